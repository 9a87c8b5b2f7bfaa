"""GPU tests of the paged key-value cache and its attention (es_hip_kv_append_dev, es_hip_attn_decode_dev, es_hip_attn_prompt_dev,
es_hip_kv_copy_pages_dev, es_hip_kv_pool_*) against the formula in 64 bits (tests/_attn.py). Pools are filled with NaN wherever no
token lies, so that whatever reads past a sequence shows. The tolerance is derived in _attn.tolerance."""
import ctypes as C
import glob

import numpy as np
import pytest

import es_hip_quant as E
from _attn import Cache, attention, from_bits, to_bits, tolerance

pytestmark = pytest.mark.gpu
TYPES = [(E.F32, E.F16), (E.F32, E.BF16), (E.F16, E.F16), (E.BF16, E.BF16)]
NAMES = {E.F32: "f32", E.F16: "f16", E.BF16: "bf16"}
ids = lambda p: "/".join(NAMES[t] for t in p) if isinstance(p, tuple) and len(p) == 2 and p in TYPES else None


def strided(x, stride, lead=0):
    """rows of x [n, ...] every `stride` elements after `lead`, the rest a pattern that must survive"""
    n = x.shape[0]
    flat = x.reshape(n, -1)
    stride = stride or flat.shape[1]
    buf = np.full(lead + max(n, 1) * stride, 7 if x.dtype == np.float32 else 0x1234, x.dtype)
    for i in range(n):
        buf[lead + i * stride: lead + i * stride + flat.shape[1]] = flat[i]
    return buf


def run(hip, cache, starts, q, t, scale, window=0, seq=None, qpad=0, opad=0, lead=0, decode=False, extra=0):
    """the call's output [ntok + extra, heads, dim] in storage; everything around the rows checked to be as it was"""
    ntok, heads, dim = q.shape
    kv, keep = cache.upload(hip, seq)
    n = starts[-1]
    row = heads * dim
    dq = hip.upload(strided(q, row + qpad, lead))
    before = strided(np.full_like(q, 0 if t != E.F32 else 0), row + opad, lead)
    before[...] = 7 if t == E.F32 else 0x1234
    do = hip.upload(before)
    es = q.dtype.itemsize
    nseq = len(starts) - 1
    if decode:
        ws = hip.attn_decode_workspace(kv, nseq, heads)
        dw = hip.alloc(ws)
        hip.memset(dw, 0xFF, ws)   # (NaN)
        hip.attn_decode_dev(kv, nseq, heads, t, dq.offset(lead * es), row + qpad if qpad else 0, scale, window, do.offset(lead * es),
                            row + opad if opad else 0, dw, ws)
    else:
        ds = hip.upload(np.array(starts, np.int32))
        ws = hip.attn_prompt_workspace(kv, nseq, ntok, heads, t)
        dw = hip.alloc(ws)
        hip.memset(dw, 0xFF, ws)
        hip.attn_prompt_dev(kv, nseq, ds, ntok, heads, t, dq.offset(lead * es), row + qpad if qpad else 0, scale, window,
                            do.offset(lead * es), row + opad if opad else 0, dw, ws)
    got = hip.download(do, np.zeros_like(before))
    out = np.zeros_like(q)
    mask = np.ones(len(got), bool)
    for i in range(ntok):
        at = lead + i * (row + opad)
        out[i] = got[at:at + row].reshape(heads, dim)
        if i < n:
            mask[at:at + row] = False
    assert np.array_equal(got[mask], before[mask])   # rows behind the last sequence and the gaps: as they were
    return out


def check(cache, starts, q, t, scale, got, window=0, seq=None):
    x = from_bits(q, t)
    want, mag = attention(cache, starts, x, scale, window, seq)
    n = starts[-1]
    tol = tolerance(cache, x, t, scale, mag, want)
    err = np.abs(from_bits(got, t)[:n] - want[:n])
    bad = ~(err <= tol[:n])
    assert not bad.any(), (np.argwhere(bad)[:5], err[bad][:5], tol[:n][bad][:5], want[:n][bad][:5])


def queries(rng, ntok, heads, dim, t, spread=1.0):
    return to_bits((rng.standard_normal((ntok, heads, dim)) * spread).astype(np.float32), t)


# ---- decode ------------------------------------------------------------------------------------------------------------------
LENS = [1, 2, 15, 16, 17, 31, 33, 64, 127, 128, 129, 200, 333]


@pytest.mark.parametrize("dim", [8, 64, 72, 128, 200, 256])
@pytest.mark.parametrize("types", TYPES, ids=ids)
def test_decode_lengths(hip, types, dim):
    t, ct = types
    rng = np.random.default_rng(dim)
    c = Cache(ct, 2, dim, 16, LENS, rng)
    c.fill(rng)
    q = queries(rng, len(LENS), 8, dim, t)
    starts = list(range(len(LENS) + 1))
    check(c, starts, q, t, dim ** -0.5, run(hip, c, starts, q, t, dim ** -0.5, decode=True))


@pytest.mark.parametrize("heads,kvh", [(1, 1), (7, 1), (14, 2), (16, 1), (17, 1), (32, 4), (40, 1), (9, 9), (6, 3)])
@pytest.mark.parametrize("types", TYPES, ids=ids)
def test_decode_heads(hip, types, heads, kvh):
    t, ct = types
    rng = np.random.default_rng(heads)
    c = Cache(ct, kvh, 64, 32, [300, 5], rng)
    c.fill(rng)
    q = queries(rng, 2, heads, 64, t)
    check(c, [0, 1, 2], q, t, 0.125, run(hip, c, [0, 1, 2], q, t, 0.125, decode=True, qpad=24, opad=40, lead=1))


@pytest.mark.parametrize("page", [16, 64, 1024])
@pytest.mark.parametrize("lens", [[6000], [5000, 1, 700], [2049, 4096]])
@pytest.mark.parametrize("types", TYPES, ids=ids)
def test_decode_long(hip, types, lens, page):
    """lengths that are split over many workgroups and joined"""
    t, ct = types
    rng = np.random.default_rng(page)
    c = Cache(ct, 1, 64, page, lens, rng)
    c.fill(rng, 2.0)
    starts = list(range(len(lens) + 1))
    q = queries(rng, len(lens), 4, 64, t, 2.0)
    got = run(hip, c, starts, q, t, 0.125, decode=True)
    check(c, starts, q, t, 0.125, got)
    assert np.array_equal(got, run(hip, c, starts, q, t, 0.125, decode=True))   # the same from call to call


@pytest.mark.parametrize("dim,heads,kvh,page", [(128, 40, 2, 32), (200, 17, 1, 16), (256, 6, 3, 64), (72, 8, 8, 16)])
@pytest.mark.parametrize("types", TYPES, ids=ids)
def test_decode_long_heads(hip, types, dim, heads, kvh, page):
    """split tiles of every width, more than one tile to a K/V head among them"""
    t, ct = types
    rng = np.random.default_rng(dim)
    c = Cache(ct, kvh, dim, page, [1900, 130, 4000], rng)
    c.fill(rng)
    q = queries(rng, 3, heads, dim, t)
    check(c, [0, 1, 2, 3], q, t, dim ** -0.5, run(hip, c, [0, 1, 2, 3], q, t, dim ** -0.5, decode=True))


@pytest.mark.parametrize("types", TYPES, ids=ids)
def test_decode_many_sequences(hip, types):
    """more sequences than a wave has lanes, of 0 to 1500 tokens, by number"""
    t, ct = types
    rng = np.random.default_rng(31)
    lens = [int(x) for x in np.exp(rng.uniform(0, np.log(1500), 150))]
    lens[3] = lens[70] = 0
    c = Cache(ct, 2, 64, 16, lens, rng)
    c.fill(rng)
    seq = [int(x) for x in rng.permutation(150)] + [-1, 70, 7]
    starts = list(range(len(seq) + 1))
    q = queries(rng, len(seq), 8, 64, t)
    check(c, starts, q, t, 0.125, run(hip, c, starts, q, t, 0.125, seq=seq, decode=True), seq=seq)


def test_decode_many_kv_heads(hip):
    """so many K/V heads that each has one workgroup, which goes through more than 64 blocks of a sequence"""
    rng = np.random.default_rng(32)
    c = Cache(E.F16, 512, 8, 16, [9000, 333], rng)
    x = rng.standard_normal((2,) + c.k.shape).astype(np.float32)
    c.k, c.v = to_bits(x[0], E.F16), to_bits(x[1], E.F16)
    q = queries(rng, 2, 512, 8, E.F32)
    check(c, [0, 1, 2], q, E.F32, 0.4, run(hip, c, [0, 1, 2], q, E.F32, 0.4, decode=True))


@pytest.mark.parametrize("rise", [0.01, 0.045, 0.2, -0.2])
@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("types", TYPES, ids=ids)
def test_scores_that_rise_slowly(hip, types, prompt, rise):
    """by less than what moves the reference of the weights, from one step of keys to the next, and by more"""
    t, ct = types
    rng = np.random.default_rng(37)
    n, dim = 700, 64
    c = Cache(ct, 1, dim, 16, [n], rng)
    c.fill(rng)
    k = from_bits(c.k, ct)
    for j in range(n):
        page, i = c.table[0, j // 16], j % 16
        k[page, 0, i] *= 0.05
        k[page, 0, i, 0] = rise * np.log(2) * j
    c.k = to_bits(k, ct)
    new = 130 if prompt else 1
    q = from_bits(queries(rng, new, 4, dim, t), t)
    q[..., 0] = 1.0
    q = to_bits(q, t)
    check(c, [0, new], q, t, 1.0, run(hip, c, [0, new], q, t, 1.0, decode=not prompt))


@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("types", TYPES, ids=ids)
def test_out_in_place_of_q(hip, types, prompt):
    t, ct = types
    rng = np.random.default_rng(33)
    c = Cache(ct, 2, 64, 16, [2000, 90], rng)
    c.fill(rng)
    starts = [0, 60, 150] if prompt else [0, 1, 2]
    q = queries(rng, starts[-1], 8, 64, t)
    kv, keep = c.upload(hip)
    dq, ds = hip.upload(q), hip.upload(np.array(starts, np.int32))
    ws = hip.attn_prompt_workspace(kv, 2, starts[-1], 8, t) if prompt else hip.attn_decode_workspace(kv, 2, 8)
    dw = hip.alloc(ws)
    if prompt:
        hip.attn_prompt_dev(kv, 2, ds, starts[-1], 8, t, dq, 0, 0.125, 0, dq, 0, dw, ws)
    else:
        hip.attn_decode_dev(kv, 2, 8, t, dq, 0, 0.125, 0, dq, 0, dw, ws)
    check(c, starts, q, t, 0.125, hip.download(dq, np.zeros_like(q)))


@pytest.mark.parametrize("window", [1, 2, 16, 17, 100, 128, 1000, 5000])
@pytest.mark.parametrize("types", TYPES, ids=ids)
def test_decode_window(hip, types, window):
    t, ct = types
    rng = np.random.default_rng(window)
    lens = [1, 16, 99, 100, 101, 640, 2000]
    c = Cache(ct, 2, 64, 16, lens, rng)
    c.fill(rng)
    for r, n in enumerate(lens):   # pages that the window has left behind belong to others by now
        c.table[r, :max(0, n - window) // 16] = [-1, c.npages, 1 << 30, -(1 << 31)][r % 4]
    starts = list(range(len(lens) + 1))
    q = queries(rng, len(lens), 4, 64, t)
    check(c, starts, q, t, 0.125, run(hip, c, starts, q, t, 0.125, window, decode=True), window)


@pytest.mark.parametrize("types", TYPES, ids=ids)
def test_decode_batches_as_they_come(hip, types):
    """a batch by sequence numbers: padded, one sequence twice, an empty one, a negative length, one longer than its table"""
    t, ct = types
    rng = np.random.default_rng(5)
    c = Cache(ct, 2, 128, 16, [40, 0, 77, 32], rng, max_pages=6)   # (row 3: whole pages, so that none of its slots is NaN)
    c.fill(rng)
    seq = [2, -1, 0, 2, 1, 4, 3, 0, 1 << 30, -(1 << 31)]
    starts = list(range(len(seq) + 1))
    q = queries(rng, len(seq), 8, 128, t)
    got = run(hip, c, starts, q, t, 0.09, seq=seq, decode=True)
    check(c, starts, q, t, 0.09, got, seq=seq)
    for b in (1, 4, 5, 8, 9):
        assert not from_bits(got[b], t).any()
    c.len[1], c.len[3] = -5, 1 << 30   # the device's own numbers, taken within the table
    got = run(hip, c, starts, q, t, 0.09, seq=seq, decode=True)
    c.len[1], c.len[3] = 0, 96
    check(c, starts, q, t, 0.09, got, seq=seq)


@pytest.mark.parametrize("types", TYPES, ids=ids)
def test_decode_values(hip, types):
    """scores from far apart to all equal, rows of zeros, tiny and huge queries, infinities in what is seen"""
    t, ct = types
    rng = np.random.default_rng(8)
    c = Cache(ct, 1, 64, 16, [500] * 6, rng)
    c.fill(rng)
    x = rng.standard_normal((6, 4, 64)).astype(np.float32)
    x[0] = 0
    x[1] *= 30
    x[2] *= 1e-6 if t != E.F16 else 1e-4
    x[3, :, ::2] *= 1e-4
    x[4, :2] *= 200
    x[5, 1] = 0
    q = to_bits(x, t)
    starts = list(range(7))
    check(c, starts, q, t, 0.125, run(hip, c, starts, q, t, 0.125, decode=True))
    if t == E.F32:   # beyond fp16's range either way: the row is scaled before it is split
        q = to_bits(x * np.float32(1e-20), t)
        check(c, starts, q, t, 1e19, run(hip, c, starts, q, t, 1e19, decode=True))
        q = to_bits(x * np.float32(1e20), t)
        check(c, starts, q, t, 1e-21, run(hip, c, starts, q, t, 1e-21, decode=True))
    inf = to_bits(np.array([np.inf], np.float32), ct)[0]
    c.v[c.table[0, 3], 0, 5, 7] = inf
    c.k[c.table[1, 2], 0, 1, 0] = inf
    out = from_bits(run(hip, c, starts, queries(rng, 6, 4, 64, t), t, 0.125, decode=True), t)
    assert (np.isposinf(out[0, :, 7]) | (np.isnan(out[0, :, 7]) if t == E.F32 else False)).all()   # (fp32's terms of both signs)
    assert np.isfinite(np.delete(out[0], 7, 1)).all()
    assert np.isfinite(out[2:]).all()


def test_decode_far_offsets(hip):
    """pools of more than 2^32 bytes: the last pages of them"""
    heads, dim, page, npages = 8, 256, 1024, 1100
    pool = npages * heads * page * dim * 2
    assert pool > 1 << 32
    rng = np.random.default_rng(2)
    k, v = hip.alloc(pool), hip.alloc(pool)
    table, ln = hip.upload(np.array([[npages - 1, 3]], np.int32)), hip.upload(np.array([1100], np.int32))
    kv = E.Kv(E.BF16, heads, dim, page, npages, int(k), int(v), int(table), int(ln), None, 1, 2)
    x = rng.standard_normal((2, 1100, heads, dim)).astype(np.float32)
    dk, dv, ds = hip.upload(x[0]), hip.upload(x[1]), hip.upload(np.array([0, 1100], np.int32))
    hip.kv_append_dev(kv, 1, ds, 1100, E.F32, dk, 0, dv, 0)
    hip.kv_copy_pages_dev(kv, 1, 0, [npages - 1], [npages - 2])
    table2 = hip.upload(np.array([[npages - 2, 3]], np.int32))
    kv.table = int(table2)
    c = Cache(E.BF16, heads, dim, page, [1100], rng)
    c.put(0, 0, to_bits(x[0], E.BF16), to_bits(x[1], E.BF16))
    q = queries(rng, 1, heads, dim, E.F32)
    dq, do = hip.upload(q), hip.alloc(q.nbytes)
    ws = hip.attn_decode_workspace(kv, 1, heads)
    dw = hip.alloc(ws)
    hip.attn_decode_dev(kv, 1, heads, E.F32, dq, 0, 1 / 16, 0, do, 0, dw, ws)
    check(c, [0, 1], q, E.F32, 1 / 16, hip.download(do, np.zeros_like(q)))
    q = queries(rng, 30, heads, dim, E.F32)
    dq, do, ds = hip.upload(q), hip.alloc(q.nbytes), hip.upload(np.array([0, 30], np.int32))
    ws = hip.attn_prompt_workspace(kv, 1, 30, heads, E.F32)
    dw = hip.alloc(ws)
    hip.attn_prompt_dev(kv, 1, ds, 30, heads, E.F32, dq, 0, 1 / 16, 0, do, 0, dw, ws)
    check(c, [0, 30], q, E.F32, 1 / 16, hip.download(do, np.zeros_like(q)))


# ---- prompts -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [8, 64, 72, 128, 200, 256])
@pytest.mark.parametrize("types", TYPES, ids=ids)
def test_prompt_packed(hip, types, dim):
    """whole prompts and pieces of them, of one token and more, an empty one among them, rows behind the last"""
    t, ct = types
    rng = np.random.default_rng(dim)
    lens, new = [1, 20, 65, 130, 7, 40, 100], [1, 20, 65, 100, 0, 1, 3]
    c = Cache(ct, 2, dim, 16, lens, rng)
    c.fill(rng)
    starts = [0] + np.cumsum(new).tolist()
    q = queries(rng, starts[-1] + 3, 6, dim, t)
    check(c, starts, q, t, dim ** -0.5, run(hip, c, starts, q, t, dim ** -0.5))


@pytest.mark.parametrize("heads,kvh", [(1, 1), (7, 1), (14, 2), (32, 4), (71, 1), (200, 1), (9, 9)])
@pytest.mark.parametrize("types", TYPES, ids=ids)
def test_prompt_heads(hip, types, heads, kvh):
    t, ct = types
    rng = np.random.default_rng(heads)
    c = Cache(ct, kvh, 64, 32, [70, 9], rng)
    c.fill(rng)
    q = queries(rng, 40, heads, 64, t)
    check(c, [0, 31, 40], q, t, 0.125, run(hip, c, [0, 31, 40], q, t, 0.125, qpad=24, opad=40, lead=3))


@pytest.mark.parametrize("window", [1, 2, 31, 64, 65, 129, 500])
@pytest.mark.parametrize("types", TYPES, ids=ids)
def test_prompt_window(hip, types, window):
    t, ct = types
    rng = np.random.default_rng(window)
    lens, new = [150, 400, 90], [150, 37, 1]
    c = Cache(ct, 2, 64, 16, lens, rng)
    c.fill(rng)
    for r, (n, f) in enumerate(zip(lens, new)):
        c.table[r, :max(0, n - f - window + 1) // 16] = [-1, c.npages, 1 << 30][r % 3]
    starts = [0] + np.cumsum(new).tolist()
    q = queries(rng, starts[-1], 4, 64, t)
    check(c, starts, q, t, 0.125, run(hip, c, starts, q, t, 0.125, window), window)


@pytest.mark.parametrize("window", [3000, 1 << 30, (1 << 31) - 1])
@pytest.mark.parametrize("decode", [False, True])
def test_window_wider_than_the_cache(hip, window, decode):
    """split tiles beside padding that brings more queries than it has tokens"""
    rng = np.random.default_rng(36)
    c = Cache(E.F16, 1, 64, 16, [2500, 0, 3, 700], rng)
    c.fill(rng)
    starts = [0, 1, 2, 3, 4] if decode else [0, 9, 49, 60, 63]
    q = queries(rng, starts[-1], 4, 64, E.F32)
    check(c, starts, q, E.F32, 0.125, run(hip, c, starts, q, E.F32, 0.125, window, decode=decode), window)


@pytest.mark.parametrize("lens,new", [([3000], [5]), ([2500, 30, 700], [17, 30, 1]), ([1500], [200])])
@pytest.mark.parametrize("types", TYPES, ids=ids)
def test_prompt_behind_long_prefix(hip, types, lens, new):
    """few rows over many keys: split and joined"""
    t, ct = types
    rng = np.random.default_rng(lens[0])
    c = Cache(ct, 1, 64, 64, lens, rng)
    c.fill(rng, 2.0)
    starts = [0] + np.cumsum(new).tolist()
    q = queries(rng, starts[-1], 4, 64, t, 2.0)
    got = run(hip, c, starts, q, t, 0.125)
    check(c, starts, q, t, 0.125, got)
    assert np.array_equal(got, run(hip, c, starts, q, t, 0.125))


@pytest.mark.parametrize("dim,heads,kvh,page", [(128, 32, 4, 32), (200, 5, 1, 16), (256, 6, 3, 64), (72, 8, 8, 1024)])
@pytest.mark.parametrize("types", TYPES, ids=ids)
def test_prompt_prefix_heads(hip, types, dim, heads, kvh, page):
    t, ct = types
    rng = np.random.default_rng(dim)
    lens, new = [2200, 1300], [33, 64]
    c = Cache(ct, kvh, dim, page, lens, rng)
    c.fill(rng)
    starts = [0] + np.cumsum(new).tolist()
    q = queries(rng, starts[-1], heads, dim, t)
    check(c, starts, q, t, dim ** -0.5, run(hip, c, starts, q, t, dim ** -0.5))


@pytest.mark.parametrize("types", TYPES, ids=ids)
def test_prompt_many_sequences(hip, types):
    """more sequences than a wave has lanes, split and whole tiles among them, by number"""
    t, ct = types
    rng = np.random.default_rng(34)
    lens = [int(x) for x in np.exp(rng.uniform(0, np.log(1500), 140))]
    new = [min(n, int(x)) for n, x in zip(lens, rng.integers(0, 12, 140))]
    c = Cache(ct, 1, 64, 16, lens, rng)
    c.fill(rng)
    seq = [int(x) for x in rng.permutation(140)]
    starts = [0] + np.cumsum([new[s] for s in seq]).tolist()
    q = queries(rng, starts[-1], 4, 64, t)
    check(c, starts, q, t, 0.125, run(hip, c, starts, q, t, 0.125, seq=seq), seq=seq)


def test_prompt_whole_tiles_over_long_prefix(hip):
    """enough rows that no tile is split, over more keys than a wave looks up the pages of at a time"""
    rng = np.random.default_rng(35)
    c = Cache(E.BF16, 64, 8, 16, [3000], rng)
    x = rng.standard_normal((2,) + c.k.shape).astype(np.float32)
    c.k, c.v = to_bits(x[0], E.BF16), to_bits(x[1], E.BF16)
    q = queries(rng, 300, 256, 8, E.F32)
    check(c, [0, 300], q, E.F32, 0.4, run(hip, c, [0, 300], q, E.F32, 0.4))


@pytest.mark.parametrize("types", TYPES, ids=ids)
def test_prompt_many_tiles(hip, types):
    """enough rows that no tile is split"""
    t, ct = types
    rng = np.random.default_rng(3)
    c = Cache(ct, 8, 64, 16, [700, 500], rng)
    c.fill(rng)
    q = queries(rng, 1200, 64, 64, t)
    got = run(hip, c, [0, 700, 1200], q, t, 0.125)
    x = from_bits(q, t)
    pick = np.r_[0:20, 600:720, 1180:1200]   # (the formula in Python is slow: rows around the ends)
    for b, (s, e) in enumerate([(0, 700), (700, 1200)]):
        K, V, _ = c.rows(b)
        for i in pick[(pick >= s) & (pick < e)]:
            n = i - s + 1
            for h in (0, 9, 63):
                z = 0.125 * (K[:n, h // 8] @ x[i, h])
                p = np.exp(z - z.max())
                p /= p.sum()
                want, mag = p @ V[:n, h // 8], p @ np.abs(V[:n, h // 8])
                tol = tolerance(c, x[i:i + 1, h:h + 1], t, 0.125, mag[None, None], want[None, None])[0, 0]
                assert (np.abs(from_bits(got[i, h], t) - want) <= tol).all(), (i, h)


@pytest.mark.parametrize("types", TYPES, ids=ids)
def test_prompt_rows_without_keys(hip, types):
    """more queries than tokens, no pages at all, a hole in the table, a sequence that is not there"""
    t, ct = types
    rng = np.random.default_rng(4)
    c = Cache(ct, 2, 64, 16, [10, 40, 100, 30], rng)
    c.fill(rng)
    c.table[1, :] = -1
    c.table[2, 2:4] = [-1, c.npages]
    seq = [0, 1, 2, 9]
    starts = [0, 25, 35, 135, 140]
    q = queries(rng, 140, 4, 64, t)
    got = run(hip, c, starts, q, t, 0.125, seq=seq)
    check(c, starts, q, t, 0.125, got, seq=seq)
    assert not from_bits(got[:15], t).any() and not from_bits(got[25:35], t).any() and not from_bits(got[135:], t).any()


@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("types", TYPES, ids=ids)
def test_prompt_infinities_where_unseen(hip, types, window):
    """a NaN or infinity in a token's K and V reaches the queries that see it, and no other"""
    t, ct = types
    rng = np.random.default_rng(6)
    n = 150
    c = Cache(ct, 2, 64, 16, [n], rng)
    c.fill(rng)
    q = queries(rng, n, 4, 64, t)
    clean = run(hip, c, [0, n], q, t, 0.125, window)
    check(c, [0, n], q, t, 0.125, clean, window)
    x = from_bits(clean, t)
    want, mag = attention(c, [0, n], from_bits(q, t), 0.125, window)
    tol = tolerance(c, from_bits(q, t), t, 0.125, mag, want)
    nan, inf, ninf = (to_bits(np.array([v], np.float32), ct)[0] for v in (np.nan, np.inf, -np.inf))
    at = lambda j: (c.table[0, j // 16], slice(None), j % 16)
    sees = lambda j: (np.arange(n) >= j) & ((np.arange(n) < j + window) if window else True)
    c.v[at(70)][:, 3] = inf
    c.v[at(71)][:, 3] = ninf
    c.v[at(100)][:, 9] = nan
    got = from_bits(run(hip, c, [0, n], q, t, 0.125, window), t)
    assert np.isnan(got[sees(70) & sees(71)][:, :, 3]).all()
    for rows, which in ((sees(70) & ~sees(71), np.isposinf), (sees(71) & ~sees(70), np.isneginf)):
        y = got[rows][:, :, 3]
        assert (which(y) | (np.isnan(y) if t == E.F32 else False)).all()   # (fp32's weights are terms of both signs)
    assert np.isnan(got[sees(100)][:, :, 9]).all()
    rest = np.ones_like(x, bool)
    rest[sees(70) | sees(71), :, 3] = False
    rest[sees(100), :, 9] = False
    assert (np.abs(got - x) <= 2 * tol)[rest].all()   # (both within the tolerance of the same value)
    c.k[at(120)][:, 0] = nan
    got = from_bits(run(hip, c, [0, n], q, t, 0.125, window), t)
    assert np.isnan(got[sees(120)]).all() and np.isfinite(got[rest & ~sees(120)[:, None, None]]).all()


@pytest.mark.parametrize("types", TYPES, ids=ids)
def test_prompt_starts_out_of_order(hip, types):
    """whatever the starts hold, the call ends and stays within its buffers"""
    t, ct = types
    rng = np.random.default_rng(7)
    c = Cache(ct, 1, 64, 16, [900, 900, 900, 900], rng)
    c.fill(rng)
    q = queries(rng, 64, 4, 64, t)
    kv, keep = c.upload(hip)
    dq, do = hip.upload(q), hip.alloc(q.nbytes)
    ws = hip.attn_prompt_workspace(kv, 4, 64, 4, t)
    dw = hip.alloc(ws)
    for starts in ([0, 64, 0, 64, 0], [-5, 1 << 30, 3, -(1 << 31), 64], [64, 48, 32, 16, 0], [1 << 30] * 5):
        ds = hip.upload(np.array(starts, np.int32))
        hip.attn_prompt_dev(kv, 4, ds, 64, 4, t, dq, 0, 0.125, 0, do, 0, dw, ws)
        hip.kv_append_dev(kv, 4, ds, 64, t, dq, 256, dq, 256)
        hip.synchronize()


# ---- append ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dim,kvh,page", [(8, 1, 16), (64, 8, 16), (72, 3, 32), (128, 4, 64), (256, 2, 1024)])
@pytest.mark.parametrize("types", TYPES, ids=ids)
def test_append(hip, types, dim, kvh, page):
    st, ct = types
    rng = np.random.default_rng(dim + kvh)
    lens, new = [1, 100, 17, 33, 50, 64], [1, 100, 0, 16, 60, 3]   # the fifth brings more than it has room for: its last 50
    c = Cache(ct, kvh, dim, page, lens, rng)
    c.table[5, :] = -1                                             # no page: nothing is written
    starts = [0] + np.cumsum(new).tolist()
    ntok = starts[-1] + 2
    x = rng.standard_normal((2, ntok, kvh, dim)).astype(np.float32) * 100
    x[0, 0, 0, :4] = [np.inf, 1e6, -1e6, 1e-7]
    x[1, 0, 0, :3] = [np.nan, 65519.9, 2.0 ** -24]
    k, v = to_bits(x[0], st), to_bits(x[1], st)
    kv, keep = c.upload(hip)
    row = kvh * dim
    dk, dv, ds = hip.upload(strided(k, row + 5, 1)), hip.upload(strided(v, row + 16)), hip.upload(np.array(starts, np.int32))
    es = k.dtype.itemsize
    hip.kv_append_dev(kv, 6, ds, ntok, st, dk.offset(es), row + 5, dv, row + 16)
    k, v = to_bits(from_bits(k, st), ct), to_bits(from_bits(v, st), ct)
    for r, (n, f) in enumerate(zip(lens, new)):
        if r == 5:
            continue
        lost = max(0, f - n)
        c.put(r, n - f + lost, k[starts[r] + lost:starts[r + 1]], v[starts[r] + lost:starts[r + 1]])
    for dev, want in zip(keep, (c.k, c.v)):
        got = hip.download(dev, np.zeros_like(want))
        assert np.array_equal(np.isnan(from_bits(got, ct)), np.isnan(from_bits(want, ct)))
        ok = ~np.isnan(from_bits(want, ct))
        assert np.array_equal(got[ok], want[ok])


def test_append_one_token_each(hip):
    rng = np.random.default_rng(1)
    c = Cache(E.F16, 2, 64, 16, [1, 16, 17, 200], rng)
    seq = [3, -1, 0, 1, 7]
    x = rng.standard_normal((2, 5, 2, 64)).astype(np.float32)
    kv, keep = c.upload(hip, seq)
    dk, dv = hip.upload(x[0]), hip.upload(x[1])
    hip.kv_append_dev(kv, 5, None, 5, E.F32, dk, 0, dv, 0)
    for b, r in enumerate(seq):
        if 0 <= r < 4:
            c.put(r, int(c.len[r]) - 1, to_bits(x[0, b:b + 1], E.F16), to_bits(x[1, b:b + 1], E.F16))
    for dev, want in zip(keep, (c.k, c.v)):
        assert np.array_equal(hip.download(dev, np.zeros_like(want)), want)


# ---- pages -------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kvh,dim,page,nl,n,pad", [(1, 8, 16, 1, 1, 0), (2, 64, 16, 3, 40, 32), (3, 72, 32, 2, 500, 0), (8, 256, 64, 2, 3, 256)])
def test_copy_pages(hip, kvh, dim, page, nl, n, pad):
    rng = np.random.default_rng(n)
    npages = 2 * n + 3
    pb = kvh * dim * page * 2
    layer = npages * pb + pad
    x = rng.integers(0, 256, (2, nl, layer), dtype=np.uint8)
    dk, dv = hip.upload(x[0]), hip.upload(x[1])
    kv = E.Kv(E.BF16, kvh, dim, page, npages, int(dk), int(dv), None, None, None, 0, 0)
    p = rng.permutation(npages)
    src, dst = p[:n].copy(), p[n:2 * n]
    if n > 2:
        src[1] = src[0]   # one page to two places
    hip.kv_copy_pages_dev(kv, nl, layer if pad else 0, src, dst)
    for a, b in zip(src, dst):
        x[:, :, b * pb:(b + 1) * pb] = x[:, :, a * pb:(a + 1) * pb]
    for dev, want in ((dk, x[0]), (dv, x[1])):
        assert np.array_equal(hip.download(dev, np.zeros_like(want)), want)


# ---- together ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("types", TYPES, ids=ids)
def test_prompts_forks_and_decode_through_a_pool(hip, orc, types):
    """prompts written and read, a fork, both branches decoded, one cut back, the pool compacted between steps: always the
    attention over the tokens that each sequence was given; then the output's activation blocks for the next product"""
    t, ct = types
    rng = np.random.default_rng(12)
    heads, kvh, dim, page, nl = 8, 2, 64, 16, 2
    pool = E.KvPool(hip, ct, nl, kvh, dim, page, 40, 6, 12)
    told = {}   # sequence -> per layer [K rows, V rows] in storage

    def step(seqs, new):
        pool.extend(seqs, new)
        starts = [0] + np.cumsum(new).tolist()
        ntok = starts[-1]
        dseq, ds = hip.upload(np.array(seqs, np.int32)), hip.upload(np.array(starts, np.int32))
        out = None
        for l in range(nl):
            x = rng.standard_normal((2, ntok, kvh, dim)).astype(np.float32)
            k, v = to_bits(x[0], t), to_bits(x[1], t)
            dk, dv = hip.upload(k), hip.upload(v)
            kv = pool.view(l, dseq)
            one = all(n == 1 for n in new)
            hip.kv_append_dev(kv, len(seqs), None if one else ds, ntok, t, dk, 0, dv, 0)
            k, v = to_bits(from_bits(k, t), ct), to_bits(from_bits(v, t), ct)
            for i, s in enumerate(seqs):
                told[s][l][0] = np.concatenate([told[s][l][0], k[starts[i]:starts[i + 1]]])
                told[s][l][1] = np.concatenate([told[s][l][1], v[starts[i]:starts[i + 1]]])
            c = Cache(ct, kvh, dim, page, [len(told[s][l][0]) for s in seqs], rng)
            for i, s in enumerate(seqs):
                assert pool.len(s) == c.len[i]
                c.put(i, 0, *told[s][l])
            q = queries(rng, ntok, heads, dim, t)
            dq, out = hip.upload(q), hip.alloc(q.nbytes)
            ws = hip.attn_decode_workspace(kv, len(seqs), heads) if one else hip.attn_prompt_workspace(kv, len(seqs), ntok, heads, t)
            dw = hip.alloc(ws)
            if one:
                hip.attn_decode_dev(kv, len(seqs), heads, t, dq, 0, 0.125, 0, out, 0, dw, ws)
            else:
                hip.attn_prompt_dev(kv, len(seqs), ds, ntok, heads, t, dq, 0, 0.125, 0, out, 0, dw, ws)
            got = hip.download(out, np.zeros_like(q))
            check(c, starts, q, t, 0.125, got)
        return out, got

    def new_seq(like=None):
        s = pool.create() if like is None else pool.fork(like)
        told[s] = [[np.zeros((0, kvh, dim), np.float32 if ct == E.F32 else np.uint16)] * 2 for _ in range(nl)] if like is None else \
            [list(x) for x in told[like]]
        return s

    a, b = new_seq(), new_seq()
    step([a, b], [37, 20])
    f = new_seq(a)
    assert pool.pages(f) == pool.pages(a)
    step([a, b, f], [1, 1, 1])
    assert pool.pages(f)[:2] == pool.pages(a)[:2] and pool.pages(f)[2] != pool.pages(a)[2]
    pool.truncate(f, 30)
    told[f] = [[x[0][:30], x[1][:30]] for x in told[f]]
    step([f], [1])
    pool.free(b)
    del told[b]
    used = pool.compact()
    assert used == 40 - pool.free_pages() and max(pool.pages(a) + pool.pages(f)) < used
    step([f, a], [1, 1])
    g = new_seq(f)
    out, got = step([a, g, f], [40, 3, 18])
    if t == E.F32:   # what the output projection takes next
        n, cols = 61, heads * dim
        blocks = hip.alloc(n * cols // 256 * 292)
        hip.act_prepare_dev(out, 0, n, cols, None, 0, blocks, 0)
        raw = hip.download(blocks, np.zeros(n * cols // 256 * 292, np.uint8))
        assert np.array_equal(raw, np.ascontiguousarray(orc.quantize_act(E.Q4_K, got.reshape(n, cols))).view(np.uint8).reshape(-1))
    pool.close()


class Hip:
    """the HIP runtime that the library uses: streams and graphs"""

    def __init__(self):
        self.L = C.CDLL(sorted(glob.glob("/opt/rocm/lib/libamdhip64.so*"))[0])

    def stream(self):
        s = C.c_void_p()
        assert self.L.hipStreamCreate(C.byref(s)) == 0
        return s

    def capture(self, s, call):
        g, x = C.c_void_p(), C.c_void_p()
        assert self.L.hipStreamBeginCapture(s, 2) == 0   # hipStreamCaptureModeRelaxed
        try:
            call()
        finally:
            assert self.L.hipStreamEndCapture(s, C.byref(g)) == 0
        assert self.L.hipGraphInstantiate(C.byref(x), g, None, None, C.c_size_t(0)) == 0
        assert self.L.hipGraphDestroy(g) == 0
        return x

    def launch(self, x, s):
        assert self.L.hipGraphLaunch(x, s) == 0


def write(hip, dev, arr):
    arr = np.ascontiguousarray(arr)
    hip._check(hip._L.es_hip_memcpy_h2d(int(dev), arr.ctypes.data, arr.nbytes))


@pytest.mark.parametrize("prompt", [False, True])
def test_captured_calls_follow_the_lengths(hip, prompt):
    """append and attention captured once and replayed over growing lengths and new rows, eager work between: every replay is
    the eager result; two graphs share the workspace"""
    rt, rng = Hip(), np.random.default_rng(21)
    c = Cache(E.F16, 2, 64, 16, [700, 90, 5], rng, max_pages=60, spare=200)
    c.npages = 180
    c.k, c.v = (to_bits(rng.standard_normal((180, 2, 16, 64)).astype(np.float32), E.F16) for _ in range(2))
    c.table[:] = rng.permutation(180).reshape(3, 60)
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
            hip.attn_prompt_dev(kv, 3, ds, n, 8, E.F32, q[i], 0, 0.125, 0, o, 0, ws, wb, s.value)
        else:
            hip.attn_decode_dev(kv, 3, 8, E.F32, q[i], 0, 0.125, 0, o, 0, ws, wb, s.value)

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


def test_pool_refuses_capture(hip):
    rt, s = Hip(), None
    pool = E.KvPool(hip, E.F16, 1, 2, 64, 16, 8, 4, 4)
    a = pool.create()
    pool.extend([a], [20])
    s = rt.stream()

    def calls():
        for f in (lambda: pool.create(s.value), lambda: pool.extend([a], [1], s.value), lambda: pool.fork(a, s.value),
                  lambda: pool.truncate(a, 3, s.value), lambda: pool.free(a, s.value), lambda: pool.compact(s.value)):
            with pytest.raises(E.EsHipError) as e:
                f()
            assert e.value.code == -2

    g, n = C.c_void_p(), C.c_size_t(0)
    assert rt.L.hipStreamBeginCapture(s, 2) == 0
    calls()
    assert rt.L.hipStreamEndCapture(s, C.byref(g)) == 0
    if g.value:
        assert rt.L.hipGraphGetNodes(g, None, C.byref(n)) == 0 and n.value == 0
        rt.L.hipGraphDestroy(g)
    assert pool.len(a) == 20 and pool.free_pages() == 6
    assert rt.L.hipStreamDestroy(s) == 0
    pool.close()


@pytest.mark.parametrize("types", TYPES, ids=ids)
def test_calls_on_two_streams(hip, types):
    """two callers with a workspace each, at once"""
    t, ct = types
    rt, rng = Hip(), np.random.default_rng(9)
    c = Cache(ct, 2, 64, 16, [3000, 1200], rng)
    c.fill(rng)
    kv, keep = c.upload(hip)
    wb = hip.attn_decode_workspace(kv, 2, 8)
    q = [queries(rng, 2, 8, 64, t) for _ in range(2)]
    dq, do, ws, st = [hip.upload(x) for x in q], [hip.alloc(q[0].nbytes) for _ in q], [hip.alloc(wb) for _ in q], [rt.stream() for _ in q]
    for _ in range(20):
        for i in range(2):
            hip.attn_decode_dev(kv, 2, 8, t, dq[i], 0, 0.125, 0, do[i], 0, ws[i], wb, st[i].value)
    hip.synchronize()
    for i in range(2):
        check(c, [0, 1, 2], q[i], t, 0.125, hip.download(do[i], np.zeros_like(q[i])))
        assert rt.L.hipStreamDestroy(st[i]) == 0
