"""GPU tests of attention over the key-value cache in 8 bits where fp32's and fp16's ranges end, against the formula in 64 bits
(tests/_attn8.py) with the tolerance derived in _attn.tolerance, and of tokens that no query sees, over 8 and 16 bits, whatever they hold."""
import numpy as np
import pytest

import es_hip_quant as E
from _attn import from_bits, to_bits
from _attn8 import RUN, Cache8, attention
from test_hip_attn import queries
from test_hip_attn8 import ALL, F8, allowed, as_queries, both, cache_of, ids, run

pytestmark = pytest.mark.gpu

LN2 = np.float32(0.6931472)   # as a call's scale: scores are exponents of 2


def scored(c, scores, v):
    """row 0's tokens, whole runs of one score (a negative whole number) and one V each: q = (1, 1, 0, ...) sees the scores. K's elements are a
    multiple of 8 and the rest, which 8 bits hold exactly."""
    n = len(scores) * RUN
    k = np.zeros((n, 1, c.dim))
    k[:, 0, 0] = np.repeat([s // 8 * 8 for s in scores], RUN)
    k[:, 0, 1] = np.repeat([s % 8 for s in scores], RUN)
    c.append(0, 0, k, v)
    assert np.array_equal(c.rows(0)[0], k)


def lost(c, x, scale):
    """What keys whose p is below 2^-118 of the row's largest add to it [ntok, heads, 1..]: a prompt with bf16 queries keeps weights as 2^-8 p in
    fp32 (so that no sum passes the range of its V's), whose least normal number is 2^-126; what is below may count as none."""
    k, v, _ = c.rows(0)
    pos = np.arange(len(k) - len(x), len(k))
    out = np.zeros(x.shape)
    for h in range(x.shape[1]):
        s = np.where(np.arange(len(k)) <= pos[:, None], scale * (x[:, h] @ k[:, 0].T), -np.inf)
        p = np.exp(s - s.max(1, keepdims=True))
        out[:, h] = np.where(p < 2.0 ** -118, p, 0.0) / p.sum(1, keepdims=True) @ np.abs(v[:, 0])
    return out


@pytest.mark.parametrize("first", ["largest score first", "largest sum first"])
@pytest.mark.parametrize("dim", [64, 128, 208])
@pytest.mark.parametrize("types", F8, ids=ids)
def test_prompt_scores_and_scales_far_apart(hip, types, dim, first):
    """Keys whose score lies 80 to 125 powers of two below the row's largest, where p is a normal number of fp32 yet, with V as many above that
    of the largest's: they are most of the sum, and of ordinary size."""
    t, ct = types
    rng = np.random.default_rng(dim)
    below = [0, 80, 101, 112, 115, 118, 121, 123, 125]
    for near in (0.0, 1e-3, 1.0):   # V of the largest score
        order = below if first == "largest score first" else below[::-1]
        c = Cache8(1, dim, 16, [len(order) * RUN], rng)
        v = rng.standard_normal((len(order) * RUN, 1, dim))
        for i, b in enumerate(order):
            v[i * RUN:(i + 1) * RUN] *= 2.0 ** b if b else near
        scored(c, [-b for b in order], v)
        x = np.zeros((100, 4, dim), np.float32)
        x[:, :, :2] = 1
        x[:, 1, :2] = 0.5      # a row whose scores lie half as far apart: V's largest outweigh all
        x[::3, 2, :2] = 0.9375
        if t != E.F32:         # (fp16: outputs of up to 2^60 are infinities, which the check knows)
            x[:, 1] = x[:, 0]
        q = to_bits(x, t)
        got = from_bits(run(hip, c, [0, 100], q, t, LN2), t)
        as_queries(c, t)
        want, mag, low = attention(c, [0, 100], x.astype(float), LN2)
        tol = allowed(c, x.astype(float), t, LN2, mag, low, want, False) + (lost(c, x.astype(float), LN2) if t == E.BF16 else 0)
        good = np.abs(got - want) <= tol
        if t == E.F16:   # (what lies within the tolerance from 65520 on, on either side of 0, is an infinity of fp16)
            good |= np.isinf(got) & (np.sign(got) * want + tol >= 65520)
        assert good.all(), (np.argwhere(~good)[:5], got[~good][:5], want[~good][:5], tol[~good][:5])


def hide(c, starts, window, sinks, garbage):
    """Runs of 16 tokens that no query of the call sees, their table entries as they are, hold NaN codes and these scales in turn; how many
    of them share 64 tokens with what some query sees"""
    near = 0
    for r in range(len(c.len)):
        n, f = int(c.len[r]), starts[r + 1] - starts[r]
        since = max(0, n - f - window + 1)   # the first token that the first query's window shows
        for u in range(-(-sinks // RUN), since // RUN):
            g, o = c.table[r, u * RUN // c.page], u * RUN % c.page
            for i in range(2):
                c.code[i][g, :, o:o + RUN] = 0x7F
                c.scale[i][g, :, o // RUN] = garbage[(u + i) % len(garbage)]
            near += u // 4 == since // 64 or (sinks > 0 and u // 4 == (sinks - 1) // 4 // RUN)
    return near


@pytest.mark.parametrize("window,sinks", [(17, 0), (100, 0), (333, 0), (31, 4), (65, 70), (300, 17), (129, 130)])
@pytest.mark.parametrize("dim", [64, 128, 208])
@pytest.mark.parametrize("types", F8, ids=ids)
def test_scales_of_hidden_runs(hip, types, dim, window, sinks):
    """pages between sinks and window that are others' by now, and hold scales that nobody has written: no influence"""
    t, ct = types
    for decode in (True, False):
        rng = np.random.default_rng(window + sinks + dim)
        lens = [640, 705, 1000, 399, 260, 1800]
        new = [1] * 6 if decode else [1, 37, 70, 20, 5, 130]
        starts = [0] + np.cumsum(new).tolist()
        c = Cache8(2, dim, 32, lens, rng)
        c.fill(rng)
        q = queries(rng, starts[-1], 4, dim, t)
        before = both(hip, c, starts, q, t, dim ** -0.5, window=window, sinks=sinks, decode=decode)
        assert hide(c, starts, window, sinks, [np.inf, np.nan, -np.inf, 0.0, -3.0]) >= 4
        assert np.array_equal(before, run(hip, c, starts, q, t, dim ** -0.5, window, sinks, decode=decode))


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("types", F8, ids=ids)
def test_scores_of_0_under_large_scales(hip, types, decode):
    """queries that are 0 where keys are huge, and huge where keys are 0: every score is 0, and the output V's mean"""
    t, ct = types
    rng = np.random.default_rng(6)
    c = Cache8(1, 64, 16, [80], rng)
    x = rng.standard_normal((2, 80, 1, 64))
    x[0, :, :, 32:] = 0
    x[0, 16:48] *= 2.0 ** 100
    c.append(0, 0, x[0], x[1])
    new = 1 if decode else 40
    q = np.zeros((new, 4, 64), np.float32)
    q[:, :, 32:] = rng.standard_normal((new, 4, 32))
    for size, scale in ((2.0 ** 60, 1.0), (1.0, 2.0 ** 60), (2.0 ** 40, 2.0 ** 20)):
        if t == E.F16 and size > 1:
            continue
        y = to_bits(q * np.float32(size), t)
        got = from_bits(run(hip, c, [0, new], y, t, scale, decode=decode), t)
        as_queries(c, t)
        want, mag, low = attention(c, [0, new], from_bits(y, t), scale)
        none = np.zeros_like(want)   # (no products but with 0: the scores are exact)
        assert (np.abs(got - want) <= allowed(c, none, t, 1.0, mag, low, want, decode)).all()


@pytest.mark.parametrize("window,sinks", [(100, 0), (31, 4), (65, 70), (300, 17), (129, 130)])
@pytest.mark.parametrize("dim", [64, 128, 208])
@pytest.mark.parametrize("types", ALL[3:], ids=ids)
def test_hidden_tokens_of_16_bits(hip, types, dim, window, sinks):
    """the same over 16-bit caches: tokens that no query sees hold NaN and infinities, one by one"""
    t, ct = types
    for decode in (True, False):
        rng = np.random.default_rng(window + sinks + dim)
        lens = [640, 705, 1000, 399, 260, 1800]
        new = [1] * 6 if decode else [1, 37, 70, 20, 5, 130]
        starts = [0] + np.cumsum(new).tolist()
        c = cache_of(ct, 2, dim, 32, lens, rng)
        c.fill(rng)
        q = queries(rng, starts[-1], 4, dim, t)
        before = both(hip, c, starts, q, t, dim ** -0.5, window=window, sinks=sinks, decode=decode)
        bad = to_bits(np.array([np.nan, np.inf, -np.inf], np.float32), ct)
        for r, (n, f) in enumerate(zip(lens, new)):
            j = np.arange(sinks, max(sinks, n - f - window + 1))
            g, o = c.table[r, j // 32], j % 32
            c.k[g, :, o], c.v[g, :, o] = bad[j % 3, None, None], bad[(j + 1) % 3, None, None]
        assert np.array_equal(before, run(hip, c, starts, q, t, dim ** -0.5, window, sinks, decode=decode))
