"""How many bits fp32 queries and the softmax weights keep on their way through attention's matrix products: 22 or more, as
es_hip_quant.h promises. Queries, keys and values are chosen so that an output element is one key's weight and that weight hangs on the
low bits; the GPU's outputs are checked, and, on the CPU, that the checks tell a model of the arithmetic from one that keeps fewer.

Every case has 32 keys (one wave's in decode: no joining between) and compares out_j / out_0, where key 0's weight is 1: what all
weights have in common, the sum above all, cancels. u = 2^-24 is half a step of fp32 relative to the value."""
import numpy as np
import pytest

import es_hip_quant as E
from _attn import Cache, from_bits, to_bits

N = 32
U = 2.0 ** -24
LN2 = np.float32(0.693147182464599609375)   # times the fp32 log2(e) it is 1 in fp32: scores are exponents of 2
TERMS = {E.F16: 2, E.BF16: 3}
TYPES = [E.F16, E.BF16]
NAMES = {E.F16: "f16", E.BF16: "bf16"}


def near(ct):
    """Exponents -j 2^-21: weights 1 - j 2^-21 ln 2. The exponents are exact, the weights' first terms are 1 and the rest has few
    bits, so that what is left is 2^x (a step, u here, for each of the two) and the outputs' last rounding (u each)."""
    return [2.0 ** -10], -np.arange(N)[:, None] * 2.0 ** -11, LN2, 4 * U


def spread(ct):
    """Exponents -j / 32, exact: weights of every mantissa. 2^x (a step: 2 u), the weights' terms (fp16: 2^-11 of 2^-11; bf16:
    2^-24, both within 2^-22 = 4 u), the scale's roundings (u), the outputs' (2 u)."""
    return [1.0], -np.arange(N)[:, None] / 32, LN2, 9 * U


def low_terms(ct):
    """q0 = q1 plus what only q0's last term carries, K = (j, -j): scores are that last term times j, from 0 to 4 in powers of two.
    The products and their sums are exact. The exponent's roundings (scale, its product with log2(e), the fused one: u each of at
    most 4), 2^x and the terms of the weights as above, the outputs': 12 ln 2 u + 2 u + 4 u + 2 u, for either key."""
    last, rest = (5 * 2.0 ** -14, 1.0) if ct == E.F16 else (5 * 2.0 ** -22, 1 + 3 * 2.0 ** -10)
    j = np.arange(N)
    return [rest + last, rest], np.stack([j, -j], 1).astype(float), np.float32(LN2 / (8 * last)), 2 * 17 * U


def many_low_terms(ct):
    """A score of 128 from the queries' first terms and, for every other key, 3 steps of fp32 at 128 (2^-16 each) from 32 elements' second
    terms, 3/8 of a step from any 8 of them: lost one by one if they are added to the 128. Exponents are 0 and -3/4; the rest as in
    low_terms (only decode has registers for a sum per term)."""
    q = np.ones(64)
    q[1::2] -= 3 * 2.0 ** -21
    k = np.zeros((N, 64))
    k[1::2, 0::2], k[1::2, 1::2] = 1, -1
    k[:, 0] += 128
    return q, k, LN2 * np.float32(2 ** 14), 2 * 17 * U


CASES = [near, spread, low_terms, many_low_terms]


def off(case, ct, out):
    """out[..., j] = weight of key j over the sum: the largest relative error of out_j / out_0, over the tolerance"""
    q, k, scale, tol = case(ct)
    s = k @ np.array(q)
    want = np.exp(float(scale) * (s - s[0]))
    out = np.asarray(out, float)
    return (np.abs(out / out[..., :1] / want - 1) / tol).max()


# ---- the checks on models of the arithmetic ------------------------------------------------------------------------------------
def split(x, ct, n):
    r, y = np.asarray(x, np.float32), []
    for _ in range(n):
        y.append(from_bits(to_bits(r, ct), ct).astype(np.float32))
        r = r - y[-1]
    return [t.astype(float) for t in y]


def scores(k, terms, apart):
    """sums rounded to fp32 after every 8 products: one for each term, then added from the smallest on, or one for all"""
    total = np.zeros(len(k))
    for q in terms[::-1] if apart else terms:
        s = np.zeros(len(k)) if apart else total
        for i in range(0, len(q), 8):
            s = (s + k[:, i:i + 8] @ q[i:i + 8]).astype(np.float32).astype(float)
        total = (total + s).astype(np.float32).astype(float) if apart else s
    return total


def model(case, ct, q_terms, w_terms, before, after, apart=True):
    """weights 2^(s - m + before) 2^after, in fp32 where the kernels are"""
    q, k, scale, _ = case(ct)
    c2 = np.float32(scale * np.float32(1.44269504088896340736))
    s = scores(k, split(q, ct, q_terms), apart)
    m = np.float32((s * c2).max())
    w = np.exp2((s * float(c2) + float(np.float32(before) - m)).astype(np.float32).astype(float)).astype(np.float32) * np.float32(2.0 ** after)
    return (sum(split(w, ct, w_terms)) * float(np.float32(1) / w.sum(dtype=np.float32))).astype(np.float32)


@pytest.mark.parametrize("ct", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("case", CASES)
def test_checks_accept_what_keeps_the_bits(case, ct):
    for after in (0, 15, 12, -8):
        assert off(case, ct, model(case, ct, TERMS[ct], TERMS[ct], 0, after if (after > 0) == (ct == E.F16) else 0)) <= 1


@pytest.mark.parametrize("ct", TYPES, ids=NAMES.get)
def test_checks_refuse_what_does_not(ct):
    n = TERMS[ct]
    for before in ((15, 12) if ct == E.F16 else (-8,)):   # added to the exponent, a constant rounds it
        assert off(near, ct, model(near, ct, n, n, before, 0)) > 1.2
    assert off(spread, ct, model(spread, ct, n, n - 1, 0, 0)) > 4
    assert off(low_terms, ct, model(low_terms, ct, n - 1, n, 0, 0)) > 100
    assert off(many_low_terms, ct, model(many_low_terms, ct, n, n, 0, 0, apart=False)) > 100


def cut(x, ct):
    """fp32 -> the type's bits, towards zero"""
    if ct == E.BF16:
        return (x.view(np.uint32) >> 16).astype(np.uint16)
    y = to_bits(x, ct)
    return y - (from_bits(y, ct) > x).astype(np.uint16)


# Decode with 16-bit queries: out_j = (w_j v_j - w_0) / l, where v_j is 2^(j / 32) in the cache's type, so that what is left has few of
# the weights' leading bits and the output's rounding is small next to theirs.
def against(ct, terms=None):
    """v, exact outputs, tolerance (and a model's outputs, of terms cut off): two terms of a weight, the last bit of the second set, are within
    2^-14 of it in bf16, 2^-20 in fp16, the exponent with its constant within 3.3e-7 and 2^x within 2 u, for w_j and for w_0; then the
    output's own rounding"""
    a = np.arange(N) / 32
    v = from_bits(to_bits(np.exp2(a), ct), ct)
    w = np.exp2(-a)
    exact = (w * v - 1) / w.sum()
    tol = 2 * ((2.0 ** -14 if ct == E.BF16 else 2.0 ** -20) + 3.3e-7 + 2 * U) / w.sum() + {E.F16: 2.0 ** -11, E.BF16: 2.0 ** -8}[ct] * np.abs(exact)
    if terms is None:
        return v, exact, tol
    w32 = w.astype(np.float32) * np.float32(2 ** 15)
    first = cut(w32, ct) if terms == 2 else to_bits(w32, ct)
    x = from_bits(first, ct)
    if terms == 2:
        x = x + from_bits(cut(w32 - x.astype(np.float32), ct) | 1, ct)
    out = (x * v - x[0]) / float(w32.sum())
    return v, exact, tol, from_bits(to_bits(out.astype(np.float32), ct), ct)


@pytest.mark.parametrize("ct", TYPES, ids=NAMES.get)
def test_checks_of_16_bit_decode(ct):
    for terms in (1, 2):
        _, exact, tol, out = against(ct, terms)
        assert (np.abs(out - exact) <= tol)[1:].all() == (terms == 2)


# ---- on the GPU ----------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("ct", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("case,prompt", [(c, p) for c in CASES for p in (False, True) if not (p and c is many_low_terms)])
def test_bits_of_queries_and_weights(hip, case, ct, prompt, dim):
    qs, ks, scale, _ = case(ct)
    c = Cache(ct, 1, dim, 16, [N], np.random.default_rng(1))
    k = np.zeros((N, 1, dim))
    k[:, 0, :len(qs)] = ks
    v = np.zeros((N, 1, dim))
    v[np.arange(N), 0, np.arange(N)] = 1
    c.put(0, 0, to_bits(k, ct), to_bits(v, ct))
    kv, keep = c.upload(hip)
    heads, new = 2, 1
    q = np.zeros((new, heads, dim), np.float32)
    q[..., :len(qs)] = qs
    dq, do, ds = hip.upload(q), hip.alloc(q.nbytes), hip.upload(np.array([0, new], np.int32))
    ws = hip.attn_prompt_workspace(kv, 1, new, heads, E.F32) if prompt else hip.attn_decode_workspace(kv, 1, heads)
    dw = hip.alloc(max(ws, 16))
    if prompt:
        hip.attn_prompt_dev(kv, 1, ds, new, heads, E.F32, dq, 0, float(scale), 0, do, 0, dw, ws)
    else:
        hip.attn_decode_dev(kv, 1, heads, E.F32, dq, 0, float(scale), 0, do, 0, dw, ws)
    got = hip.download(do, np.zeros_like(q))
    assert not got[..., N:].any()
    r = off(case, ct, got[..., :N])
    print(f"{case.__name__} {NAMES[ct]} {'prompt' if prompt else 'decode'} {dim}: {r:.3f} of the tolerance", flush=True)
    assert r <= 1


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("ct", TYPES, ids=NAMES.get)
def test_decode_of_16_bit_queries_keeps_two_terms_of_the_weights(hip, ct, dim):
    v, exact, tol = against(ct)
    c = Cache(ct, 1, dim, 16, [N], np.random.default_rng(1))
    k, vs = np.zeros((N, 1, dim)), np.zeros((N, 1, dim))
    k[:, 0, 0] = -np.arange(N) / 32
    vs[np.arange(N), 0, np.arange(N)] = v
    vs[0, 0, :N] = -1
    c.put(0, 0, to_bits(k, ct), to_bits(vs, ct))
    kv, keep = c.upload(hip)
    q = np.zeros((1, 2, dim))
    q[..., 0] = 1
    q = to_bits(q, ct)
    dq, do = hip.upload(q), hip.alloc(q.nbytes)
    ws = hip.attn_decode_workspace(kv, 1, 2)
    dw = hip.alloc(max(ws, 16))
    hip.attn_decode_dev(kv, 1, 2, ct, dq, 0, float(LN2), 0, do, 0, dw, ws)
    got = from_bits(hip.download(do, np.zeros_like(q)), ct)
    r = (np.abs(got[..., 1:N] - exact[1:]) / tol[1:]).max()
    print(f"16-bit decode {NAMES[ct]} {dim}: {r:.3f} of the tolerance", flush=True)
    assert r <= 1
