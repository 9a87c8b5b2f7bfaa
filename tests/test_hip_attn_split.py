"""GPU tests of prompt attention where a call's tiles are cut into chunks of keys and joined: windows that begin inside a chunk or
leave whole chunks unseen, infinities and NaN in what some rows see, and, for heads of every width, that nothing outside a call's
buffers is written whatever the starts hold."""
import numpy as np
import pytest

from _attn import Cache, attention, from_bits, to_bits, tolerance
from test_hip_attn import TYPES, check, ids, queries, run

pytestmark = pytest.mark.gpu


# The first: 29 tiles of 32 tokens that see 131 keys each, of chunks of 128 or 256; the others: windows that reach over several
# chunks, from inside one.
@pytest.mark.parametrize("lens,new,window", [([1900], [900], 100), ([3000], [5], 1000), ([3000], [70], 2900), ([2500, 30, 1800, 0], [17, 30, 64, 3], 1300),
                                             ([1700, 1600], [200, 1], 1111)])
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("types", TYPES, ids=ids)
def test_windows_over_chunks(hip, types, dim, lens, new, window):
    t, ct = types
    rng = np.random.default_rng(window)
    c = Cache(ct, 1, dim, 16, lens, rng)
    c.fill(rng)
    for r, (n, f) in enumerate(zip(lens, new)):   # pages that the window has left behind belong to others by now
        c.table[r, :max(0, n - f - window + 1) // 16] = [-1, c.npages, 1 << 30][r % 3]
    starts = [0] + np.cumsum(new).tolist()
    q = queries(rng, starts[-1], 4, dim, t)
    check(c, starts, q, t, dim ** -0.5, run(hip, c, starts, q, t, dim ** -0.5, window), window)


# (keys, queries): one whole tile; one whose keys are split
@pytest.mark.parametrize("n,new", [(150, 150), (2000, 60)])
@pytest.mark.parametrize("window", [0, 1200])
@pytest.mark.parametrize("dim", [64, 128, 200, 256])
@pytest.mark.parametrize("types", TYPES, ids=ids)
def test_infinities_reach_who_sees_them(hip, types, dim, window, n, new):
    t, ct = types
    rng = np.random.default_rng(dim + n)
    c = Cache(ct, 1, dim, 16, [n], rng)
    c.fill(rng)
    scale = dim ** -0.5
    q = queries(rng, new, 4, dim, t)
    x = from_bits(q, t)
    want, mag = attention(c, [0, new], x, scale, window)
    tol = tolerance(c, x, t, scale, mag, want)
    pos = np.arange(n - new, n)
    sees = lambda j: (pos >= j) & ((pos < j + window) if window else True)
    at = lambda j: (c.table[0, j // 16], slice(None), j % 16)
    bad = {n - 40: (3, np.inf), n - 39: (3, -np.inf), n - 30: (dim - 1, np.nan), n - 17: (8 * (dim // 16), np.inf)}
    if n > new:   # keys that all rows see, some do, and none does
        bad.update({n // 2: (11, np.inf), n - new // 2 - 1200: (17, np.nan), 5: (20, -np.inf)})
    rest = np.ones_like(want, bool)
    for j, (d, y) in bad.items():
        c.v[at(j)][:, d] = to_bits(np.array([y], np.float32), ct)[0]
        rest[sees(j), :, d] = False
    got = from_bits(run(hip, c, [0, new], q, t, scale, window), t)
    assert not np.isfinite(got[~rest]).any()
    assert (np.abs(got - want) <= tol)[rest].all()
    c.k[at(n - 25)][:, 0] = to_bits(np.array([np.nan], np.float32), ct)[0]
    got = from_bits(run(hip, c, [0, new], q, t, scale, window), t)
    assert np.isnan(got[sees(n - 25)]).all()
    assert (np.abs(got - want) <= tol)[rest & ~sees(n - 25)[:, None, None]].all()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("types", TYPES, ids=ids)
def test_nothing_outside_the_buffers(hip, types, dim):
    """starts out of order, beyond the rows, negative: what they give is undefined, where it goes is not"""
    t, ct = types
    rng = np.random.default_rng(dim)
    c = Cache(ct, 1, dim, 16, [900, 900, 900, 900], rng)
    c.fill(rng)
    c.table[3, 2:5] = [-1, c.npages, -(1 << 31)]
    q = queries(rng, 64, 4, dim, t)
    G = 1 << 16   # guard bytes before and after
    size, bufs = {}, {}
    kv, keep = c.upload(hip)
    ws = hip.attn_prompt_workspace(kv, 4, 64, 4, t)
    assert ws
    for name, data in (("k", c.k), ("v", c.v), ("out", np.zeros_like(q)), ("ws", np.zeros(ws, np.uint8))):
        raw = np.full(data.nbytes + 2 * G, 0xA5, np.uint8)
        raw[G:G + data.nbytes] = np.ascontiguousarray(data).reshape(-1).view(np.uint8)
        size[name], bufs[name] = data.nbytes, hip.upload(raw)
    kv.k, kv.v = int(bufs["k"].offset(G)), int(bufs["v"].offset(G))
    dq = hip.upload(q)
    for starts in ([0, 64, 0, 64, 0], [-5, 1 << 30, 3, -(1 << 31), 64], [64, 48, 32, 16, 0], [1 << 30] * 5, [0, 16, 32, 48, 64]):
        ds = hip.upload(np.array(starts, np.int32))
        hip.kv_append_dev(kv, 4, ds, 64, t, dq, 4 * dim, dq, 4 * dim)
        for window in (0, 700):
            hip.attn_prompt_dev(kv, 4, ds, 64, 4, t, dq, 0, 0.125, window, bufs["out"].offset(G), 0, bufs["ws"].offset(G), ws)
        for name, b in bufs.items():
            raw = hip.download(b, np.zeros(size[name] + 2 * G, np.uint8))
            assert (raw[:G] == 0xA5).all() and (raw[-G:] == 0xA5).all(), (name, starts)
