"""GPU tests of the key-value cache in 8 bits (type F8) and of attention through windows that leave first tokens in sight
(es_hip_attn_*_sinks_dev), with caches of every type, against the formula in 64 bits (tests/_attn8.py). Unused codes are NaN and
unused scales infinite, so that whatever reads past a sequence shows. What an append leaves is exact; the tolerance of the attention
is the one derived in _attn.tolerance, with the matrix products over an 8-bit cache's elements as exact as over those of 16 bits:
fp32 queries in two terms of fp16 (the 22 bits that it counts) and weights in the same or better, 16-bit queries as they are and their
weights in a prompt rounded once to the queries' type."""
import numpy as np
import pytest

import es_hip_quant as E
from _attn import Cache, from_bits, to_bits, tolerance
from _attn8 import RUN, VALUES, Cache8, attention
from test_hip_attn import Hip, queries, strided, write

pytestmark = pytest.mark.gpu
F8 = [(E.F32, E.F8), (E.F16, E.F8), (E.BF16, E.F8)]
ALL = F8 + [(E.F32, E.F16), (E.F32, E.BF16), (E.F16, E.F16), (E.BF16, E.BF16)]
NAMES = {E.F32: "f32", E.F16: "f16", E.BF16: "bf16", E.F8: "f8"}
ids = lambda p: "/".join(NAMES[t] for t in p) if isinstance(p, tuple) and p in ALL else None


def cache_of(ct, heads, dim, page, lens, rng, **more):
    return Cache8(heads, dim, page, lens, rng, **more) if ct == E.F8 else Cache(ct, heads, dim, page, lens, rng, **more)


def as_queries(cache, t):
    """weights of an 8-bit cache's rows have the queries' type where that is of 16 bits (for _attn.tolerance)"""
    if isinstance(cache, Cache8) and t != E.F32:
        cache.t = t


def run(hip, cache, starts, q, t, scale, window=0, sinks=0, seq=None, qpad=0, opad=0, lead=0, decode=False):
    """the call's output [ntok, heads, dim] in storage; everything around the rows checked to be as it was"""
    ntok, heads, dim = q.shape
    kv, keep = cache.upload(hip, seq)
    n, row, es, nseq = starts[-1], heads * dim, q.dtype.itemsize, len(starts) - 1
    dq = hip.upload(strided(q, row + qpad, lead))
    before = strided(np.zeros_like(q), row + opad, lead)
    before[...] = 7 if t == E.F32 else 0x1234
    do, ds = hip.upload(before), hip.upload(np.array(starts, np.int32))
    ws = hip.attn_decode_workspace(kv, nseq, heads) if decode else hip.attn_prompt_workspace(kv, nseq, ntok, heads, t)
    dw = hip.alloc(ws)
    hip.memset(dw, 0xFF, ws)   # (NaN)
    q_at, out_at, qs, os_ = dq.offset(lead * es), do.offset(lead * es), row + qpad if qpad else 0, row + opad if opad else 0
    if decode and sinks:
        hip.attn_decode_sinks_dev(kv, nseq, heads, t, q_at, qs, scale, window, sinks, out_at, os_, dw, ws)
    elif decode:
        hip.attn_decode_dev(kv, nseq, heads, t, q_at, qs, scale, window, out_at, os_, dw, ws)
    elif sinks:
        hip.attn_prompt_sinks_dev(kv, nseq, ds, ntok, heads, t, q_at, qs, scale, window, sinks, out_at, os_, dw, ws)
    else:
        hip.attn_prompt_dev(kv, nseq, ds, ntok, heads, t, q_at, qs, scale, window, out_at, os_, dw, ws)
    got = hip.download(do, np.zeros_like(before))
    out, mask = np.zeros_like(q), np.ones(len(got), bool)
    for i in range(ntok):
        at = lead + i * (row + opad)
        out[i] = got[at:at + row].reshape(heads, dim)
        if i < n:
            mask[at:at + row] = False
    assert np.array_equal(got[mask], before[mask])   # rows behind the last sequence and the gaps: as they were
    return out


def allowed(cache, x, t, scale, mag, low, want, decode):
    """_attn.tolerance, and what it does not count: weights below fp16's range in a prompt over 8 bits whose products are of fp16, and outputs
    below fp16's smallest normal number, whose steps are 2^-24"""
    tol = tolerance(cache, x, t, scale, mag, want)
    return tol + (low if t != E.BF16 and not decode else 0) + (2.0 ** -25 if t == E.F16 else 0)


def check(cache, starts, q, t, scale, got, window=0, sinks=0, seq=None, decode=False):
    x = from_bits(q, t)
    as_queries(cache, t)
    want, mag, low = attention(cache, starts, x, scale, window, sinks, seq)
    n = starts[-1]
    tol = allowed(cache, x, t, scale, mag, low, want, decode)
    got = from_bits(got, t)[:n]
    err = np.abs(got - want[:n])
    bad = ~(err <= tol[:n])
    if t == E.F16:   # (65520, half a step above its largest number, and what is greater are infinities in fp16)
        bad &= ~(np.isinf(got) & (np.sign(got) == np.sign(want[:n])) & (np.abs(want[:n]) + tol[:n] >= 65520))
    assert not bad.any(), (np.argwhere(bad)[:5], err[bad][:5], tol[:n][bad][:5], want[:n][bad][:5])


def both(hip, c, starts, q, t, scale, **k):
    got = run(hip, c, starts, q, t, scale, **k)
    check(c, starts, q, t, scale, got, k.get("window", 0), k.get("sinks", 0), k.get("seq"), k.get("decode", False))
    return got


# ---- append ------------------------------------------------------------------------------------------------------------------
def same_cache(hip, keep, c, at=(0, 1), scales=(4, 5)):
    """the pools as the model has them: codes equal (a NaN's sign aside), scales equal"""
    for i in range(2):
        code, scale = hip.download(keep[at[i]], np.zeros_like(c.code[i])), hip.download(keep[scales[i]], np.zeros_like(c.scale[i]))
        nan = (c.code[i] & 127) == 127
        assert np.array_equal((code & 127) == 127, nan)
        assert np.array_equal(VALUES[code[~nan]], VALUES[c.code[i][~nan]])   # (a number rounded to 0 keeps its sign or loses it)
        assert np.array_equal(scale, c.scale[i])


@pytest.mark.parametrize("dim,kvh,page", [(16, 1, 16), (64, 8, 16), (80, 3, 32), (128, 4, 64), (256, 2, 1024)])
@pytest.mark.parametrize("st", [E.F32, E.F16, E.BF16], ids=lambda t: NAMES[t])
def test_append(hip, st, dim, kvh, page):
    """prompts of 0 to 100 tokens, one that brings more than there is room for, one without pages, rows behind the last; then further
    calls into runs that are partly filled, with rows of larger and smaller size"""
    rng = np.random.default_rng(dim + kvh)
    final = [21, 120, 37, 53, 50, 64]
    c = Cache8(kvh, dim, page, final, rng)
    c.table[5, :] = -1                                # no page: nothing is written
    length = np.array([1, 100, 17, 33, 50, 64])
    for r, n in ((2, 17), (3, 17)):                   # tokens from before the first call
        c.append(r, 0, *rng.standard_normal((2, n, kvh, dim)))
    kv, keep = c.upload(hip)
    row, es = kvh * dim, 4 if st == E.F32 else 2
    for step, (new, spread) in enumerate([([1, 100, 0, 16, 60, 3], 100.0), ([1] * 6, 1e3), ([3, 2, 5, 1, 0, 0], 3e-3), ([16, 17, 14, 18, 0, 0], 1e4)]):
        if step:
            length = np.minimum(length + new, final)
        starts = [0] + np.cumsum(new).tolist()
        ntok = starts[-1] + 2
        x = rng.standard_normal((2, ntok, kvh, dim)) * spread
        if step == 0:
            x[0, 0, 0, :4] = [np.inf, 6e4, -6e4, 1e-7]
            x[1, 0, 0, :3] = [np.nan, 448.0, 2.0 ** -24]
            x[0, 5:25] = 0                            # whole runs of zeros
            x[1, 40, :, 0] = [np.nan, -np.inf][step]
        k, v = to_bits(x[0], st), to_bits(x[1], st)
        dk, dv, ds = hip.upload(strided(k, row + 5, 1)), hip.upload(strided(v, row + 16)), hip.upload(np.array(starts, np.int32))
        write(hip, keep[3], length.astype(np.int32))
        hip.kv_append_dev(kv, 6, ds, ntok, st, dk.offset(es), row + 5, dv, row + 16)
        for r, (n, f) in enumerate(zip(length, new)):
            lost = max(0, f - n)
            if f - lost:
                s = slice(starts[r] + lost, starts[r + 1])
                c.append(r, n - f + lost, from_bits(k[s], st), from_bits(v[s], st))
        same_cache(hip, keep, c)


def test_append_range(hip):
    """rows from the smallest to the largest numbers of fp32, powers of two and their neighbours, the border of every scale"""
    rng = np.random.default_rng(3)
    edges = np.array([0.875 * 2.0 ** e for e in range(-120, 128)], np.float32)   # 448 * 2^j
    x = np.concatenate([edges, np.nextafter(edges, np.float32(np.inf)), np.nextafter(edges, np.float32(0)),
                        np.array([0.0, 1e-45, 2.0 ** -126, 3.3e38, np.finfo(np.float32).max], np.float32)])
    n = len(x) * RUN
    c = Cache8(1, 16, 16, [n], rng)
    rows = np.zeros((2, n, 1, 16), np.float32)
    for i, y in enumerate(x):   # a run each: the largest, and numbers of every size below it
        rows[0, i * RUN:(i + 1) * RUN, 0] = y * np.exp2(-rng.uniform(0, 22, (RUN, 16))) * rng.choice([-1, 1], (RUN, 16))
        rows[0, i * RUN + i % RUN, 0, i % 16] = y
        rows[1, i * RUN:(i + 1) * RUN, 0] = (rng.integers(0, 449 * 16, (RUN, 16)) / 16).astype(np.float32)   # (ties among them)
    kv, keep = c.upload(hip)
    dk, dv, ds = hip.upload(rows[0]), hip.upload(rows[1]), hip.upload(np.array([0, n], np.int32))
    hip.kv_append_dev(kv, 1, ds, n, E.F32, dk, 0, dv, 0)
    c.append(0, 0, rows[0].astype(np.float64), rows[1].astype(np.float64))
    same_cache(hip, keep, c)


@pytest.mark.parametrize("nseq", [5, 64, 65, 130, 4097])
def test_append_finds_its_sequence(hip, nseq):
    """batches of more sequences than a wave probes at once, of 0 to 40 tokens each, by number; and one token each"""
    rng = np.random.default_rng(nseq)
    lens = rng.integers(1, 60, nseq).tolist()
    c = Cache8(1, 16, 16, lens, rng)
    new = [int(rng.integers(0, min(n, 40) + 1)) for n in lens]
    seq = rng.permutation(nseq).tolist()
    starts = [0] + np.cumsum([new[s] for s in seq]).tolist()
    x = rng.standard_normal((2, starts[-1], 1, 16))
    for r, n in enumerate(lens):   # what was there before the call
        if n > new[r]:
            y = rng.standard_normal((2, n - new[r], 1, 16)) * 0.1
            c.append(r, 0, y[0], y[1])
    kv, keep = c.upload(hip, seq)
    k, v = x.astype(np.float32)
    dk, dv, ds = hip.upload(k), hip.upload(v), hip.upload(np.array(starts, np.int32))
    hip.kv_append_dev(kv, nseq, ds, starts[-1], E.F32, dk, 0, dv, 0)
    for b, s in enumerate(seq):
        if new[s]:
            c.append(s, lens[s] - new[s], k[starts[b]:starts[b + 1]].astype(float), v[starts[b]:starts[b + 1]].astype(float))
    same_cache(hip, keep, c)
    x = rng.standard_normal((2, nseq + 2, 1, 16)).astype(np.float32) * 7
    seq2 = hip.upload(np.array([-1] + seq + [nseq], np.int32))   # padded with numbers of no sequence
    kv.seq = int(seq2)
    dk, dv = hip.upload(x[0]), hip.upload(x[1])
    hip.kv_append_dev(kv, nseq + 2, None, nseq + 2, E.F32, dk, 0, dv, 0)
    for b, s in enumerate(seq):
        c.append(s, lens[s] - 1, x[0, b + 1:b + 2].astype(float), x[1, b + 1:b + 2].astype(float))
    same_cache(hip, keep, c)


@pytest.mark.parametrize("kvh,dim,page,nl,n,pad", [(1, 16, 16, 1, 1, 0), (2, 64, 16, 3, 40, 32), (3, 80, 32, 2, 500, 0), (8, 256, 64, 2, 3, 1), (70, 16, 1024, 1, 2, 0)])
def test_copy_pages(hip, kvh, dim, page, nl, n, pad):
    """codes and scales of every layer, with `pad` runs of 16 tokens between the layers"""
    rng = np.random.default_rng(n)
    npages = 2 * n + 3
    pb, ps = kvh * dim * page, kvh * page // RUN
    layer, layer_s = npages * pb + pad * RUN * dim, npages * ps + pad
    x = rng.integers(0, 256, (2, nl, layer), dtype=np.uint8)
    y = rng.standard_normal((2, nl, layer_s)).astype(np.float32)
    d = [hip.upload(a) for a in (x[0], x[1], y[0], y[1])]
    kv = E.Kv8(E.F8, kvh, dim, page, npages, int(d[0]), int(d[1]), None, None, None, 0, 0, int(d[2]), int(d[3]))
    p = rng.permutation(npages)
    src, dst = p[:n].copy(), p[n:2 * n]
    if n > 2:
        src[1] = src[0]   # one page to two places
    hip.kv_copy_pages_dev(kv, nl, layer if pad else 0, src, dst)
    for a, b in zip(src, dst):
        x[:, :, b * pb:(b + 1) * pb] = x[:, :, a * pb:(a + 1) * pb]
        y[:, :, b * ps:(b + 1) * ps] = y[:, :, a * ps:(a + 1) * ps]
    for dev, want in zip(d, (x[0], x[1], y[0], y[1])):
        assert np.array_equal(hip.download(dev, np.zeros_like(want)), want)


# ---- attention over 8 bits ---------------------------------------------------------------------------------------------------
LENS = [1, 2, 15, 16, 17, 31, 33, 64, 127, 128, 129, 200, 333]


@pytest.mark.parametrize("dim", [16, 64, 80, 128, 208, 256])
@pytest.mark.parametrize("types", F8, ids=ids)
def test_decode_lengths(hip, types, dim):
    t, ct = types
    rng = np.random.default_rng(dim)
    c = cache_of(ct, 2, dim, 16, LENS, rng)
    c.fill(rng)
    both(hip, c, list(range(len(LENS) + 1)), queries(rng, len(LENS), 8, dim, t), t, dim ** -0.5, decode=True)


@pytest.mark.parametrize("heads,kvh", [(1, 1), (7, 1), (17, 1), (32, 4), (40, 1), (9, 9)])
@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("types", F8, ids=ids)
def test_heads(hip, types, decode, heads, kvh):
    t, ct = types
    rng = np.random.default_rng(heads)
    c = cache_of(ct, kvh, 64, 32, [300, 5], rng)
    c.fill(rng)
    starts = [0, 1, 2] if decode else [0, 60, 65]
    both(hip, c, starts, queries(rng, starts[-1], heads, 64, t), t, 0.125, decode=decode, qpad=24, opad=40, lead=1)


@pytest.mark.parametrize("dim,heads,kvh,page,lens", [(64, 4, 1, 16, [6000]), (128, 40, 2, 32, [1900, 130, 4000]), (208, 17, 1, 16, [2049, 700]),
                                                     (256, 6, 3, 64, [5000, 1]), (80, 8, 8, 1024, [2500])])
@pytest.mark.parametrize("types", F8, ids=ids)
def test_decode_long(hip, types, dim, heads, kvh, page, lens):
    """lengths that are split over many workgroups and joined"""
    t, ct = types
    rng = np.random.default_rng(page)
    c = cache_of(ct, kvh, dim, page, lens, rng)
    c.fill(rng, 2.0)
    starts = list(range(len(lens) + 1))
    q = queries(rng, len(lens), heads, dim, t, 2.0)
    got = both(hip, c, starts, q, t, dim ** -0.5, decode=True)
    assert np.array_equal(got, run(hip, c, starts, q, t, dim ** -0.5, decode=True))   # the same from call to call


@pytest.mark.parametrize("types", F8, ids=ids)
def test_decode_most_parts(hip, types):
    """one K/V head of 64 elements, whose one long sequence is split over more workgroups than any other call's"""
    t, ct = types
    rng = np.random.default_rng(70)
    c = cache_of(ct, 1, 64, 1024, [70000, 3], rng)
    c.fill(rng)
    both(hip, c, [0, 1, 2], queries(rng, 2, 2, 64, t), t, 0.125, decode=True)


@pytest.mark.parametrize("dim", [16, 64, 80, 128, 208, 256])
@pytest.mark.parametrize("types", F8, ids=ids)
def test_prompt_packed(hip, types, dim):
    """whole prompts and pieces of them, of one token and more, an empty one among them, rows behind the last"""
    t, ct = types
    rng = np.random.default_rng(dim)
    lens, new = [1, 20, 65, 130, 7, 40, 300], [1, 20, 65, 100, 0, 1, 3]
    c = cache_of(ct, 2, dim, 16, lens, rng)
    c.fill(rng)
    starts = [0] + np.cumsum(new).tolist()
    both(hip, c, starts, queries(rng, starts[-1] + 3, 6, dim, t), t, dim ** -0.5)


@pytest.mark.parametrize("dim,heads,kvh,page,lens,new", [(64, 4, 1, 64, [3000], [5]), (128, 32, 4, 32, [2200, 1300], [33, 64]), (208, 5, 1, 16, [2500, 30, 700], [17, 30, 1]),
                                                         (256, 6, 3, 64, [1900], [70]), (80, 8, 8, 1024, [1500], [200])])
@pytest.mark.parametrize("types", F8, ids=ids)
def test_prompt_behind_long_prefix(hip, types, dim, heads, kvh, page, lens, new):
    """few rows over many keys: split and joined"""
    t, ct = types
    rng = np.random.default_rng(lens[0])
    c = cache_of(ct, kvh, dim, page, lens, rng)
    c.fill(rng, 2.0)
    starts = [0] + np.cumsum(new).tolist()
    q = queries(rng, starts[-1], heads, dim, t, 2.0)
    got = both(hip, c, starts, q, t, dim ** -0.5)
    assert np.array_equal(got, run(hip, c, starts, q, t, dim ** -0.5))


@pytest.mark.parametrize("dim", [16, 128])
def test_prompt_whole_tiles_over_long_prefix(hip, dim):
    """enough rows that no tile is split, over more keys than a wave looks up the pages of at a time"""
    rng = np.random.default_rng(35)
    c = Cache8(16, dim, 16, [2500], rng)
    c.fill(rng)
    both(hip, c, [0, 300], queries(rng, 300, 128, dim, E.F32), E.F32, dim ** -0.5)


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("types", F8, ids=ids)
def test_scales_far_apart(hip, types, decode):
    """runs of very different size, in K and V, from one to the next: nothing of one run's scale reaches another's"""
    t, ct = types
    rng = np.random.default_rng(44)
    n = 700
    c = Cache8(1, 64, 16, [n], rng)
    x = rng.standard_normal((2, n, 1, 64))
    size = np.exp2(rng.integers(-40, 41, (2, -(-n // RUN)))).repeat(RUN, 1)[:, :n, None, None]
    x[0] *= np.minimum(size[0], 1.0)
    x[1] *= size[1]
    c.append(0, 0, x[0], x[1])
    new = 1 if decode else 90
    both(hip, c, [0, new], queries(rng, new, 4, 64, t), t, 0.125, decode=decode)


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("types", F8, ids=ids)
def test_values(hip, types, decode):
    """queries of zeros, tiny and huge, against runs of zeros (the least scale), of tiny and of huge keys; hidden keys stay hidden"""
    t, ct = types
    rng = np.random.default_rng(8)
    n = 300
    c = Cache8(1, 64, 16, [n] * 6, rng)
    for r in range(6):
        x = rng.standard_normal((2, n, 1, 64))
        x[0, 16:64], x[1, 100:140] = 0, 0
        x[0, 64:96] *= 2.0 ** -90
        x[0, 128:160] *= 16
        c.append(r, 0, x[0], x[1])
    new = 1 if decode else 70
    x = rng.standard_normal((6, new, 4, 64)).astype(np.float32)
    x[0] = 0
    x[1] *= 30
    x[2] *= 1e-6 if t != E.F16 else 1e-4
    x[3, :, :, ::2] *= 1e-4
    x[4, :, :2] *= 200
    x[5, :, 1] = 0
    x = x.reshape(6 * new, 4, 64)
    starts = list(range(0, 6 * new + 1, new))
    both(hip, c, starts, to_bits(x, t), t, 0.125, decode=decode)
    both(hip, c, starts, to_bits(x, t), t, 0.125, decode=decode, window=100, sinks=20)
    if t != E.F16:   # beyond fp16's range either way: an fp32 row is scaled before it is split
        both(hip, c, starts, to_bits(x * np.float32(1e-20), t), t, 1e19, decode=decode)
        both(hip, c, starts, to_bits(x * np.float32(1e-20), t), t, 0.125, decode=decode, window=250, sinks=3)   # (hidden keys in a run of zeros)
        both(hip, c, starts, to_bits(x * np.float32(1e20), t), t, 1e-21, decode=decode)


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("types", F8, ids=ids)
def test_batches_as_they_come(hip, types, decode):
    """by sequence numbers: padded, empty, lengths that are negative or past the table, holes and page numbers out of range"""
    t, ct = types
    rng = np.random.default_rng(5)
    c = Cache8(2, 128, 16, [40, 0, 100, 96], rng, max_pages=7)
    c.len[3] = 112
    c.table[3] = rng.permutation(c.npages)[:7]   # (whole pages, so that none of its slots is NaN)
    c.fill(rng)
    c.table[2, 2:4] = [-1, c.npages]
    seq = [2, -1, 0, 1, 4, 3, 0, 1 << 30, -(1 << 31)]
    n = [1] * len(seq) if decode else [40, 3, 20, 2, 4, 50, 1, 2, 1]
    starts = [0] + np.cumsum(n).tolist()
    q = queries(rng, starts[-1], 8, 128, t)
    got = both(hip, c, starts, q, t, 0.09, seq=seq, decode=decode)
    for b in (1, 3, 4, 7, 8):
        assert not from_bits(got[starts[b]:starts[b + 1]], t).any()
    c.len[1], c.len[3] = -5, 1 << 30   # the device's own numbers, taken within the table
    got = run(hip, c, starts, q, t, 0.09, seq=seq, decode=decode)
    c.len[1], c.len[3] = 0, 112
    check(c, starts, q, t, 0.09, got, seq=seq)


# (keys, queries): one whole tile; one whose keys are split
@pytest.mark.parametrize("n,new", [(150, 150), (2000, 60), (900, 1)])
# (16-bit caches without sinks: tests/test_hip_attn.py and test_hip_attn_split.py)
@pytest.mark.parametrize("types,window,sinks", [(p, 300, 70) for p in ALL] + [(p, w, 0) for p in F8 for w in (0, 300)], ids=ids)
@pytest.mark.parametrize("dim", [64, 128, 208])
def test_nan_reaches_who_sees_it(hip, types, dim, window, sinks, n, new):
    """in V: that element of the rows that see it, and no other; in K: the rows that see it"""
    t, ct = types
    rng = np.random.default_rng(dim + n)
    c = cache_of(ct, 1, dim, 16, [n], rng)
    c.fill(rng)
    as_queries(c, t)
    scale, decode = dim ** -0.5, new == 1
    q = queries(rng, new, 4, dim, t)
    x = from_bits(q, t)
    want, mag, low = attention(c, [0, new], x, scale, window, sinks)
    tol = allowed(c, x, t, scale, mag, low, want, decode)
    pos = np.arange(n - new, n)
    sees = lambda j: (pos >= j) & ((pos < j + window) | (j < sinks) if window else True)
    at = lambda j: (c.table[0, j // 16], slice(None), j % 16)
    codes, nan = ((c.code[0], c.code[1]), 0x7F) if ct == E.F8 else ((c.k, c.v), to_bits(np.array([np.nan], np.float32), ct)[0])
    bad = {n - 40: 3, n - 17: 8 * (dim // 16), n - 2: dim - 1, 5: 20, 69: 21, 75: 22, n // 2: 11, max(0, n - new // 2 - 300): 17}
    rest = np.ones_like(want, bool)
    for j, d in bad.items():
        codes[1][at(j)][:, d] = nan
        rest[sees(j), :, d] = False
    got = from_bits(run(hip, c, [0, new], q, t, scale, window, sinks, decode=decode), t)
    assert np.isnan(got[~rest]).all()
    assert (np.abs(got - want) <= tol)[rest].all()
    for j in (7, n - 25):
        kept = codes[0][at(j)][:, 0].copy()
        codes[0][at(j)][:, 0] = nan
        got = from_bits(run(hip, c, [0, new], q, t, scale, window, sinks, decode=decode), t)
        codes[0][at(j)][:, 0] = kept
        assert np.isnan(got[sees(j)]).all()
        assert (np.abs(got - want) <= tol)[rest & ~sees(j)[:, None, None]].all()


# ---- windows with sinks ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("window,sinks", [(1, 1), (2, 4), (16, 16), (17, 63), (100, 64), (100, 65), (128, 300), (1000, 4), (700, 1500), (5000, 4), (3, 1 << 30)])
@pytest.mark.parametrize("types", ALL, ids=ids)
def test_decode_sinks(hip, types, window, sinks):
    t, ct = types
    rng = np.random.default_rng(window + sinks)
    lens = [1, 5, 16, 99, 100, 165, 640, 2000, 0]
    c = cache_of(ct, 2, 64, 16, lens, rng)
    c.fill(rng)
    for r, n in enumerate(lens):   # pages that lie between belong to others by now
        c.table[r, min(-(-sinks // 16), c.max_pages):max(0, n - window) // 16] = [-1, c.npages, 1 << 30, -(1 << 31)][r % 4]
    both(hip, c, list(range(len(lens) + 1)), queries(rng, len(lens), 4, 64, t), t, 0.125, window=window, sinks=sinks, decode=True)


@pytest.mark.parametrize("window,sinks", [(1, 1), (31, 4), (64, 64), (65, 70), (129, 130), (500, 3)])
@pytest.mark.parametrize("types", ALL, ids=ids)
def test_prompt_sinks(hip, types, window, sinks):
    """prompts and pieces, queries that stand among the sinks and before the window's end"""
    t, ct = types
    rng = np.random.default_rng(window + sinks)
    lens, new = [400, 700, 290, 60, 3], [400, 37, 1, 20, 5]
    c = cache_of(ct, 2, 64, 16, lens, rng)
    c.fill(rng)
    for r, (n, f) in enumerate(zip(lens, new)):
        c.table[r, -(-sinks // 16):max(0, n - f - window + 1) // 16] = [-1, c.npages, 1 << 30][r % 3]
    starts = [0] + np.cumsum(new).tolist()
    both(hip, c, starts, queries(rng, starts[-1] + 2, 4, 64, t), t, 0.125, window=window, sinks=sinks)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens,new,window,sinks", [([1900], [900], 100, 4), ([3000], [70], 2000, 700), ([2500, 30, 1800, 0], [17, 30, 64, 3], 900, 200),
                                                   ([3000], [5], 1000, 900), ([1700, 1600], [200, 1], 1111, 130), ([2600], [500], 200, 1100)])
@pytest.mark.parametrize("types", ALL, ids=ids)
def test_sinks_over_chunks(hip, types, dim, lens, new, window, sinks):
    """tiles whose keys are split: chunks that end inside the sinks, that hold sinks and window, and none that the tile sees"""
    t, ct = types
    rng = np.random.default_rng(window)
    c = cache_of(ct, 1, dim, 16, lens, rng)
    c.fill(rng)
    starts = [0] + np.cumsum(new).tolist()
    both(hip, c, starts, queries(rng, starts[-1], 4, dim, t), t, dim ** -0.5, window=window, sinks=sinks)


@pytest.mark.parametrize("dim,heads,kvh", [(128, 40, 2), (208, 6, 3), (256, 5, 1)])
@pytest.mark.parametrize("types", ALL, ids=ids)
def test_sinks_wide_heads(hip, types, dim, heads, kvh):
    t, ct = types
    rng = np.random.default_rng(dim)
    lens = [1900, 130, 2700]
    c = cache_of(ct, kvh, dim, 32, lens, rng)
    c.fill(rng)
    both(hip, c, [0, 1, 2, 3], queries(rng, 3, heads, dim, t), t, dim ** -0.5, window=900, sinks=70, decode=True)
    both(hip, c, [0, 40, 50, 51], queries(rng, 51, heads, dim, t), t, dim ** -0.5, window=300, sinks=33)


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("types", ALL, ids=ids)
def test_sinks_of_none_and_of_all(hip, types, decode):
    """0 sinks: the windowed call, bit for bit; as many as there are tokens: no window, bit for bit"""
    t, ct = types
    rng = np.random.default_rng(1)
    c = cache_of(ct, 2, 64, 16, [900, 1300], rng)
    c.fill(rng)
    starts = [0, 1, 2] if decode else [0, 30, 70]
    q = queries(rng, starts[-1], 4, 64, t)
    kv, keep = c.upload(hip)
    dq, do, ds = hip.upload(q), hip.alloc(q.nbytes), hip.upload(np.array(starts, np.int32))
    ws = hip.attn_workspace_upto(kv, 2, 70, 4)
    dw = hip.alloc(ws)

    def call(f, *more):
        f = getattr(hip, "attn_%s%s_dev" % ("decode" if decode else "prompt", f))
        args = (kv, 2, 4, t, dq) if decode else (kv, 2, ds, starts[-1], 4, t, dq)
        f(*args, 0, 0.125, *more, do, 0, dw, ws)
        return hip.download(do, np.zeros_like(q))

    assert np.array_equal(call("", 200), call("_sinks", 200, 0))
    assert np.array_equal(call("", 0), call("_sinks", 200, c.max_pages * 16))
    assert np.array_equal(call("", 0), call("_sinks", 0, 7))


# ---- together ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("t", [E.F32, E.F16, E.BF16], ids=lambda t: NAMES[t])
def test_a_stream_through_a_pool(hip, t):
    """prompts into an 8-bit pool, a fork, branches decoded through a window with sinks, one cut back and gone on with, the pool
    compacted between steps: always the cache that the same calls leave in the model, and the attention over it"""
    rng = np.random.default_rng(12)
    heads, kvh, dim, page, nl, window, sinks = 8, 2, 64, 32, 2, 40, 5
    pool = E.KvPool(hip, E.F8, nl, kvh, dim, page, 40, 6, 12)
    model = {}   # sequence -> per layer a cache of one row
    most = None

    def step(seqs, new):
        nonlocal most
        pool.extend(seqs, new)
        starts = [0] + np.cumsum(new).tolist()
        ntok, one = starts[-1], all(n == 1 for n in new)
        dseq, ds = hip.upload(np.array(seqs, np.int32)), hip.upload(np.array(starts, np.int32))
        for l in range(nl):
            k, v = (to_bits(x, t) for x in rng.standard_normal((2, ntok, kvh, dim)).astype(np.float32) * np.exp2(rng.integers(-2, 3)))
            dk, dv = hip.upload(k), hip.upload(v)
            kv = pool.view(l, dseq)
            if most is None:
                most = hip.attn_workspace_upto(kv, 6, 100, heads)
            hip.kv_append_dev(kv, len(seqs), None if one else ds, ntok, t, dk, 0, dv, 0)
            q = queries(rng, ntok, heads, dim, t)
            dq, out, dw = hip.upload(q), hip.alloc(q.nbytes), hip.alloc(most)
            if one:
                hip.attn_decode_sinks_dev(kv, len(seqs), heads, t, dq, 0, 0.125, window, sinks, out, 0, dw, most)
            else:
                hip.attn_prompt_sinks_dev(kv, len(seqs), ds, ntok, heads, t, dq, 0, 0.125, window, sinks, out, 0, dw, most)
            got = hip.download(out, np.zeros_like(q))
            for i, s in enumerate(seqs):
                c, s_ = model[s][l], slice(starts[i], starts[i + 1])
                c.append(0, int(c.len[0]), from_bits(k[s_], t), from_bits(v[s_], t))
                c.len[0] += new[i]
                assert pool.len(s) == c.len[0]
                check(c, [0, new[i]], q[s_], t, 0.125, got[s_], window, sinks)

    def new_seq(like=None):
        s = pool.create() if like is None else pool.fork(like)
        model[s] = []
        for l in range(nl):
            c = Cache8(kvh, dim, page, [12 * page], rng)
            c.len[0] = 0
            if like is not None:
                o = model[like][l]
                c.table, c.len = o.table.copy(), o.len.copy()
                c.code, c.scale, c.npages = [x.copy() for x in o.code], [x.copy() for x in o.scale], o.npages
            model[s].append(c)
        return s

    a, b = new_seq(), new_seq()
    step([a, b], [37, 20])
    f = new_seq(a)
    step([a, b, f], [1, 1, 1])
    pool.truncate(f, 30)
    for c in model[f]:
        c.len[0] = 30
    step([f], [1])
    pool.free(b)
    del model[b]
    used = pool.compact()
    assert used == 40 - pool.free_pages() and max(pool.pages(a) + pool.pages(f)) < used
    step([f, a], [1, 1])
    g = new_seq(f)
    step([a, g, f], [40, 3, 18])
    for _ in range(20):
        step([a, g, f], [1, 1, 1])
    pool.close()


@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("ct", [E.F8, E.F16], ids=lambda t: NAMES[t])
def test_captured_calls_follow_the_lengths(hip, ct, prompt):
    """append and attention with sinks captured once and replayed over growing lengths and new rows, eager work between: every replay
    is the eager result (an append of the same rows twice is one); two graphs share the workspace"""
    rt, rng = Hip(), np.random.default_rng(21)
    c = cache_of(ct, 2, 64, 16, [960] * 3, rng)
    c.fill(rng)
    c.len[:] = [700, 90, 5]
    kv, keep = c.upload(hip)
    starts = [0, 2, 3, 6] if prompt else [0, 1, 2, 3]
    n = starts[-1]
    ds = hip.upload(np.array(starts, np.int32))
    new, q, out = hip.alloc(2 * n * 128 * 4), [hip.alloc(n * 512 * 4) for _ in range(2)], [hip.alloc(n * 512 * 4) for _ in range(3)]
    wb = hip.attn_prompt_workspace(kv, 3, n, 8, E.F32) if prompt else hip.attn_decode_workspace(kv, 3, 8)
    assert wb
    ws, s = hip.alloc(wb), rt.stream()

    def call(i, o):
        hip.kv_append_dev(kv, 3, ds if prompt else None, n, E.F32, new, 0, new.offset(n * 512), 0, s.value)
        if prompt:
            hip.attn_prompt_sinks_dev(kv, 3, ds, n, 8, E.F32, q[i], 0, 0.125, 300, 70, o, 0, ws, wb, s.value)
        else:
            hip.attn_decode_sinks_dev(kv, 3, 8, E.F32, q[i], 0, 0.125, 300, 70, o, 0, ws, wb, s.value)

    graphs = [rt.capture(s, lambda i=i: call(i, out[i])) for i in range(2)]
    for step in range(4):
        for x in (new, *q):
            write(hip, x, rng.standard_normal(x.nbytes // 4).astype(np.float32))
        c.len += 1 + 70 * (step == 2)
        write(hip, keep[3], c.len)
        for g in graphs:
            rt.launch(g, s)
        hip.synchronize()
        for i in range(2):
            call(i, out[2])
            hip.synchronize()
            got = [hip.download(o, np.zeros(n * 512, np.float32)) for o in (out[i], out[2])]
            assert np.isfinite(got[0]).all() and np.array_equal(*got), (step, i)
    for g in graphs:
        assert rt.L.hipGraphExecDestroy(g) == 0
    assert rt.L.hipStreamDestroy(s) == 0


@pytest.mark.parametrize("ct", [E.F8, E.F16], ids=lambda t: NAMES[t])
def test_two_streams_at_once(hip, ct):
    """decode and a prompt over one cache, sinks and none, on two streams with workspaces of their own: the bits of each call alone"""
    rt, rng = Hip(), np.random.default_rng(33)
    c = cache_of(ct, 2, 128, 16, [3000, 1700, 9], rng)
    c.fill(rng)
    kv, keep = c.upload(hip)
    starts = [0, 64, 100, 103]
    n, ds = starts[-1], hip.upload(np.array(starts, np.int32))
    q = hip.upload(queries(rng, n, 8, 128, E.F32).astype(np.float32))
    sizes = hip.attn_decode_workspace(kv, 3, 8), hip.attn_prompt_workspace(kv, 3, n, 8, E.F32)
    assert all(sizes)
    ws, rows, streams = [hip.alloc(b) for b in sizes], (3, n), [rt.stream() for _ in range(2)]

    def call(i, window, sinks, o, s):
        if i:
            hip.attn_prompt_sinks_dev(kv, 3, ds, n, 8, E.F32, q, 0, 0.1, window, sinks, o, 0, ws[1], sizes[1], s.value)
        else:
            hip.attn_decode_sinks_dev(kv, 3, 8, E.F32, q, 0, 0.1, window, sinks, o, 0, ws[0], sizes[0], s.value)

    for window, sinks in ((0, 0), (900, 70)):
        outs = [[hip.alloc(m * 1024 * 4) for _ in range(9)] for m in rows]
        for i in range(2):
            call(i, window, sinks, outs[i][8], streams[0])
            hip.synchronize()
        for k in range(8):
            for i in range(2):
                call(i, window, sinks, outs[i][k], streams[i])
        hip.synchronize()
        for i, m in enumerate(rows):
            alone = hip.download(outs[i][8], np.zeros(m * 1024, np.float32))
            assert np.isfinite(alone).all()
            for k in range(8):
                assert np.array_equal(hip.download(outs[i][k], np.zeros(m * 1024, np.float32)), alone), (i, k)
    for s in streams:
        assert rt.L.hipStreamDestroy(s) == 0


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("types", ALL, ids=ids)
def test_nothing_outside_the_buffers(hip, types, dim):
    """starts out of order, beyond the rows, negative: what they give is undefined, where it goes is not"""
    t, ct = types
    rng = np.random.default_rng(dim)
    c = cache_of(ct, 1, dim, 16, [900, 900, 900, 900], rng)
    c.fill(rng)
    c.table[3, 2:5] = [-1, c.npages, -(1 << 31)]
    q = queries(rng, 64, 4, dim, t)
    G = 1 << 16   # guard bytes before and after
    size, bufs = {}, {}
    kv, keep = c.upload(hip)
    ws = hip.attn_prompt_workspace(kv, 4, 64, 4, t)
    assert ws
    parts = [("k", c.code[0]), ("v", c.code[1]), ("ks", c.scale[0]), ("vs", c.scale[1])] if ct == E.F8 else [("k", c.k), ("v", c.v)]
    for name, data in parts + [("out", np.zeros_like(q)), ("ws", np.zeros(ws, np.uint8))]:
        raw = np.full(data.nbytes + 2 * G, 0xA5, np.uint8)
        raw[G:G + data.nbytes] = np.ascontiguousarray(data).reshape(-1).view(np.uint8)
        size[name], bufs[name] = data.nbytes, hip.upload(raw)
    kv.k, kv.v = int(bufs["k"].offset(G)), int(bufs["v"].offset(G))
    if ct == E.F8:
        kv.k_scale, kv.v_scale = int(bufs["ks"].offset(G)), int(bufs["vs"].offset(G))
    dq = hip.upload(q)
    for starts in ([0, 64, 0, 64, 0], [-5, 1 << 30, 3, -(1 << 31), 64], [64, 48, 32, 16, 0], [1 << 30] * 5, [0, 16, 32, 48, 64]):
        ds = hip.upload(np.array(starts, np.int32))
        hip.kv_append_dev(kv, 4, ds, 64, t, dq, 4 * dim, dq, 4 * dim)
        for window, sinks in ((0, 0), (700, 0), (300, 100)):
            hip.attn_prompt_sinks_dev(kv, 4, ds, 64, 4, t, dq, 0, 0.125, window, sinks, bufs["out"].offset(G), 0, bufs["ws"].offset(G), ws)
        for name, b in bufs.items():
            raw = hip.download(b, np.zeros(size[name] + 2 * G, np.uint8))
            assert (raw[:G] == 0xA5).all() and (raw[-G:] == 0xA5).all(), (name, starts)


def test_far_offsets(hip):
    """pools of more than 2^32 bytes, codes and scales in their last pages"""
    heads, dim, page, npages = 16, 256, 1024, 1050
    pool, scales = npages * heads * page * dim, npages * heads * (page // RUN) * 4
    assert pool > 1 << 32
    rng = np.random.default_rng(2)
    k, v, ks, vs = hip.alloc(pool), hip.alloc(pool), hip.alloc(scales), hip.alloc(scales)
    table, ln = hip.upload(np.array([[npages - 1, 3]], np.int32)), hip.upload(np.array([1100], np.int32))
    kv = E.Kv8(E.F8, heads, dim, page, npages, int(k), int(v), int(table), int(ln), None, 1, 2, int(ks), int(vs))
    x = rng.standard_normal((2, 1100, heads, dim)).astype(np.float32)
    dk, dv, ds = hip.upload(x[0]), hip.upload(x[1]), hip.upload(np.array([0, 1100], np.int32))
    hip.kv_append_dev(kv, 1, ds, 1100, E.F32, dk, 0, dv, 0)
    hip.kv_copy_pages_dev(kv, 1, 0, [npages - 1], [npages - 2])
    table2 = hip.upload(np.array([[npages - 2, 3]], np.int32))
    kv.table = int(table2)
    c = Cache8(heads, dim, page, [1100], rng)
    c.append(0, 0, x[0].astype(float), x[1].astype(float))
    for n in (1, 30):
        q = queries(rng, n, heads, dim, E.F32)
        dq, do, ds = hip.upload(q), hip.alloc(q.nbytes), hip.upload(np.array([0, n], np.int32))
        ws = hip.attn_workspace_upto(kv, 1, 30, heads)
        dw = hip.alloc(ws)
        if n == 1:
            hip.attn_decode_dev(kv, 1, heads, E.F32, dq, 0, 1 / 16, 0, do, 0, dw, ws)
        else:
            hip.attn_prompt_dev(kv, 1, ds, n, heads, E.F32, dq, 0, 1 / 16, 0, do, 0, dw, ws)
        check(c, [0, n], q, E.F32, 1 / 16, hip.download(do, np.zeros_like(q)))
