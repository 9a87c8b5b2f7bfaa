"""CPU tests of the 8-bit key-value cache's host side and of windows with sinks: argument checks of the device calls and their
launches, with the HIP calls answered by a stub; a pool's bookkeeping; the model that the GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest

import es_hip_quant as E
from _attn8 import LEAST, VALUES, Cache8, exponent_for, nearest
from test_kv_pool import child  # noqa: F401 (a fixture)

REFUSE = r"""
out = {}
P = 1 << 20
def kv8(k_scale=4096, v_scale=4096, **k):
    a = kv(**{"type": E.F8, **k})
    return E.Kv8(*[getattr(a, n) for n, _ in E.Kv._fields_], k_scale, v_scale)
ap = lambda k, nseq=3, start=None, ntok=3, t=E.F32, kk=P, ks=0, v=P, vs=0: code(L.kv_append_dev, k, nseq, start, ntok, t, kk, ks, v, vs)
de = lambda k, nseq=3, heads=32, t=E.F32, w=0, s=0, wb=1 << 30: code(L.attn_decode_sinks_dev, k, nseq, heads, t, P, 0, 0.1, w, s, P, 0, P, wb)
pr = lambda k, nseq=3, start=P, ntok=9, heads=32, t=E.F32, w=0, s=0, wb=1 << 30: code(L.attn_prompt_sinks_dev, k, nseq, start, ntok, heads, t, P, 0, 0.1, w, s, P, 0, P, wb)
cp = lambda k, nl=2, lb=0, s=[1, 2], d=[3, 4]: code(L.kv_copy_pages_dev, k, nl, lb, s, d)
for n, b in dict(ks=dict(k_scale=None), vs=dict(v_scale=None), align=dict(v_scale=4098), dim8=dict(dim=72), dim0=dict(dim=0), big=dict(dim=272), page=dict(page=8)).items():
    k = kv8(**b)
    out.update({"append " + n: ap(k), "decode " + n: de(k), "prompt " + n: pr(k), "copy " + n: cp(k)})
    if L.attn_decode_workspace(k, 3, 32) or L.attn_prompt_workspace(k, 3, 9, 32, E.F32) or L.attn_workspace_upto(k, 3, 9, 32): out["workspace " + n] = 0
k = kv8()
out.update({"a type": ap(k, t=E.F8), "a type2": ap(k, t=2), "a many": ap(k, start=P, ntok=(1 << 31) - 1), "a manyseq": ap(kv8(seq=4096), nseq=1 << 26, ntok=1 << 26),
            "d f8": de(k, t=E.F8), "d bf16": de(kv(), t=E.BF16), "p f8": pr(k, t=E.F8), "c layer": cp(k, lb=100 * 4 * 16 * 128 + 16),
            "d sinks": de(kv(), s=-1, w=5), "p sinks": pr(kv(), s=-1, w=5), "d window": de(k, s=1, w=-1), "p start": pr(k, start=None, s=1, w=5)})
launched = counts[0]
fine = {"append": ap(k), "starts": ap(k, start=P, ntok=9), "f16": ap(k, t=E.F16), "bf16": ap(k, t=E.BF16), "none": ap(k, ntok=0, start=P),
        "decode": de(k), "prompt": pr(k), "bf16 q": de(k, t=E.BF16), "f16 q": pr(k, t=E.F16), "copy": cp(k), "sinks": de(kv(), w=9, s=2), "p sinks": pr(kv(), w=9, s=1 << 30),
        "all": de(kv(), w=(1 << 31) - 1, s=(1 << 31) - 1)}
print(json.dumps({"bad": out, "launched": launched, "fine": fine, "after": [counts[i] for i in range(5)]}))
"""


def test_refusals(child):  # noqa: F811
    got = child(REFUSE)
    assert {k: v for k, v in got["bad"].items() if v != -2} == {}
    assert got["launched"] == 0
    assert set(got["fine"].values()) == {0}
    # four appends and a copy of one launch, seven attention calls of two: nothing allocated, copied or waited for
    assert got["after"] == [5 + 2 * 7, 0, 0, 0, 0]


GRIDS = r"""
rows = []
P = 1 << 20
for nseq, heads, ntok, starts in [(1, 4, 1, 0), (48, 8, 48, 0), (1, 3, 4096, 1), (300, 2, 777, 1), (5, 1, 5, 1)]:
    k = E.Kv8(E.F8, heads, 64, 16, 100, 4096, 8192, 4096, 4096, None, nseq, 64, 4096, 4096)
    n = counts[0]
    L.kv_append_dev(k, nseq, P if starts else None, ntok, E.F32, P, 0, P, 0)
    rows.append([nseq, heads, ntok, starts, counts[0] - n, list(shapes[n % 64])])
print(json.dumps(rows))
"""


def test_every_run_has_a_wave(child):  # noqa: F811
    """whatever the starts and lengths, a wave for each run of 16 tokens that a call may touch, found by the slot that it has"""
    for nseq, heads, ntok, starts, launches, (x, y, threads, _) in child(GRIDS):
        assert launches == 1 and y == 2 and threads == 256
        if not starts:
            assert x * 4 >= nseq * heads
            continue
        rng = np.random.default_rng(nseq)
        for _ in range(200):
            start = np.concatenate([[0], np.sort(rng.integers(0, ntok + 1, nseq - 1)), [ntok]])
            n = np.diff(start)
            first = rng.integers(0, 100, nseq)   # where the call's tokens begin
            runs = np.where(n > 0, (first + n - 1) // 16 - first // 16 + 1, 0)
            slot = start // 16 + 2 * np.arange(nseq + 1)
            assert (runs <= np.diff(slot)).all() and slot[-1] <= x * 4 // heads


def test_pool_in_8_bits(hiplib):
    """bookkeeping as with any type; heads of a multiple of 16 elements"""
    p = E.KvPool(hiplib, E.F8, 0, 2, 64, 16, 8, 3, 4)
    s = p.create()
    p.extend([s], [20])
    f = p.fork(s)
    p.extend([f], [1])
    assert p.pages(s)[0] == p.pages(f)[0] and p.pages(s)[1] != p.pages(f)[1] and p.free_pages() == 5
    with pytest.raises(E.EsHipError):
        E.KvPool(hiplib, E.F8, 0, 2, 72, 16, 8, 3, 4)


def test_view_leaves_what_follows_a_16_bit_cache(child):  # noqa: F811
    """a program built when es_hip_kv ended before the scales has no room for them"""
    got = child(r"""
out = []
for t in (E.F16, E.F8):
    p = E.KvPool(L, t, 2, 2, 64, 16, 8, 3, 4)
    kv = E.Kv8(k_scale=77, v_scale=78)
    L._check(L._L.es_hip_kv_pool_view(p.h, 1, C.byref(kv)))
    a = E.Kv8()
    L._check(L._L.es_hip_kv_pool_view(p.h, 0, C.byref(a)))
    out.append([kv.k_scale, kv.v_scale, kv.k - a.k, kv.v - a.k, (kv.k_scale or 0) - (a.k_scale or 0), (kv.v_scale or 0) - a.k, kv.heads, kv.max_pages])
    p.close()
print(json.dumps(out))
""")
    page = 2 * 16 * 64
    assert got[0][:4] == [77, 78, 8 * page * 2, 2 * 8 * page * 2 + 8 * page * 2] and got[0][6:] == [2, 4]
    scales = 8 * 2   # a layer's
    assert got[1][2:6] == [8 * page, 3 * 8 * page, scales * 4, 4 * 8 * page + 3 * scales * 4]


def test_model():
    """the GPU tests' model of the format"""
    assert np.nanmax(VALUES) == 448
    assert nearest(np.array([449.0, -460.0, 2.0 ** -10, 3 * 2.0 ** -10, np.inf, np.nan])).tolist() == [0x7E, 0xFE, 0, 2, 0x7F, 0x7F]
    assert exponent_for(np.array([448.0, np.inf])) == 0 and exponent_for(np.array([-448.1])) == 1 and exponent_for(np.zeros(3)) == LEAST
    for c in range(256):
        assert np.isnan(VALUES[c]) or VALUES[nearest(VALUES[c:c + 1])[0]] == VALUES[c]


def test_tokens_one_by_one():
    """what a run holds does not hang on how its tokens came, but for what lies below 2^-14 of its largest (numbers that a smaller scale
    rounds to more bits than the last one has below 2^-6)"""
    rng = np.random.default_rng(0)
    for _ in range(20):
        x = rng.standard_normal((2, 16, 1, 16)) * np.exp2(rng.integers(-8, 9, (2, 16, 1, 1)))
        a, b = (Cache8(1, 16, 16, [16], rng) for _ in range(2))
        a.append(0, 0, x[0], x[1])
        for i in range(16):
            b.append(0, i, x[0, i:i + 1], x[1, i:i + 1])
        for i, (p, q) in enumerate(zip(a.rows(0)[:2], b.rows(0)[:2])):
            assert np.array_equal(a.scale[i][a.table[0, 0]], b.scale[i][b.table[0, 0]])
            s = a.scale[i][a.table[0, 0], 0, 0]
            normal = np.abs(p) > 2.0 ** -6 * s
            assert np.array_equal(p[normal], q[normal]) and (np.abs(p - q) <= 2.0 ** -9 * s).all()
