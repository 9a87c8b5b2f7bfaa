"""GPU tests of attention where a workgroup takes many steps and many tiles: sizes at which a decode call counts the beginning of a tile as a block
(tests/_deal.py), at which a wave goes on past the 32 steps (decode), or 64 runs of 16 keys (prompts), whose pages and scales it holds, and
at which two steps of keys are on their way. Against the formula in 64 bits (tests/_attn8.py) for a few K/V heads; the others hold the
same again, and have to give the same bits."""
import copy

import numpy as np
import pytest

import es_hip_quant as E
from _deal import Deal
from test_hip_attn import queries
from test_hip_attn8 import ALL, F8, cache_of, check, ids, run

pytestmark = pytest.mark.gpu


def alike(c, kvh):
    """the cache with kvh heads that repeat c's"""
    full = copy.copy(c)
    full.heads = kvh
    again = lambda x: np.tile(x, (1, kvh // c.heads) + (1,) * (x.ndim - 2))
    if hasattr(c, "code"):
        full.code, full.scale = [again(x) for x in c.code], [again(x) for x in c.scale]
    else:
        full.k, full.v = again(c.k), again(c.v)
    return full


def go(hip, c, kvh, G, starts, rng, t, decode, window=0, sinks=0):
    dim, few = c.dim, c.heads
    q = queries(rng, starts[-1], few * G, dim, t)
    got = run(hip, alike(c, kvh), starts, np.tile(q, (1, kvh // few, 1)), t, dim ** -0.5, window, sinks, decode=decode)
    first = np.ascontiguousarray(got[:, :few * G])
    check(c, starts, q, t, dim ** -0.5, first, window, sinks, decode=decode)
    assert np.array_equal(got, np.tile(first, (1, kvh // few, 1)))


SHORT = [1, 130, 5000, 700]
MANY = [5000 if i % 35 == 3 else 1 + 37 * i % 400 for i in range(75)]
# K/V heads, query heads to each, elements, lengths, window, sinks
BEGINNINGS = [(64, 1, 16, SHORT, 0, 0), (128, 1, 80, SHORT, 0, 0), (128, 2, 64, MANY, 0, 0), (64, 40, 80, SHORT, 0, 0), (64, 17, 16, [3000, 200, 2500], 0, 0),
              (64, 1, 128, SHORT, 900, 70), (128, 1, 256, [1, 2000, 150], 0, 0), (64, 2, 64, MANY + [9] * 60, 700, 4), (64, 1, 208, [4000, 3, 3000], 0, 0)]


@pytest.mark.parametrize("kvh,G,dim,lens,window,sinks", BEGINNINGS)
@pytest.mark.parametrize("types", F8, ids=ids)
def test_beginnings_that_count(hip, types, kvh, G, dim, lens, window, sinks):
    t, ct = types
    rng = np.random.default_rng(len(lens) + dim)
    c = cache_of(ct, 2, dim, 16, lens, rng)
    d = Deal(True, dim, 16, c.max_pages, kvh, kvh * G, lens, window, sinks)
    assert d.extra == 1 and d.joined()
    c.fill(rng)
    go(hip, c, kvh, G, list(range(len(lens) + 1)), rng, t, True, window, sinks)


# a window with sinks hides the tokens between: as many steps, with keys renumbered
@pytest.mark.parametrize("dim,kvh,lens,window,sinks", [(64, 128, [10000], 0, 0), (80, 128, [10000], 0, 0), (128, 128, [10100], 0, 0), (208, 128, [10000], 0, 0),
                                                       (64, 256, [9000, 4700], 0, 0), (128, 256, [4500, 4800], 0, 0), (64, 128, [12000], 9500, 70), (128, 128, [12000], 9500, 130),
                                                       (208, 256, [5100, 5300], 4600, 70)])
@pytest.mark.parametrize("types", ALL, ids=ids)
def test_decode_of_many_steps(hip, types, dim, kvh, lens, window, sinks):
    t, ct = types
    rng = np.random.default_rng(dim + window)
    c = cache_of(ct, 2, dim, 16, lens, rng)
    d = Deal(ct == E.F8, dim, 16, c.max_pages, kvh, kvh, lens, window, sinks)
    assert d.steps() > 33
    c.fill(rng)
    go(hip, c, kvh, 1, list(range(len(lens) + 1)), rng, t, True, window, sinks)


@pytest.mark.parametrize("window,sinks", [(0, 0), (1300, 70)])
@pytest.mark.parametrize("dim", [64, 128, 208, 256])
@pytest.mark.parametrize("types", ALL, ids=ids)
def test_prompt_of_many_steps(hip, types, dim, window, sinks):
    """tiles that are one part each (there are as many as parts are aimed for) of more keys than 64 runs"""
    t, ct = types
    rng = np.random.default_rng(dim + window)
    new = 520
    assert new * 8 // 128 + 1 >= 512 // 16   # tiles; parts aimed for, a K/V head, with two workgroups to a CU
    c = cache_of(ct, 2, dim, 16, [2500], rng)
    c.fill(rng)
    go(hip, c, 16, 8, [0, new], rng, t, False, window, sinks)
