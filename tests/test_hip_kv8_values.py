"""GPU test of what an append into an 8-bit cache does with infinities and NaN, of either sign, in K and in V, in new runs and in partly
filled ones: they become NaN, count for no scale, and stay NaN when their run is rounded to a larger one. Exact, against tests/_attn8.py."""
import numpy as np
import pytest

import es_hip_quant as E
from _attn import from_bits, to_bits
from _attn8 import Cache8
from test_hip_attn import write
from test_hip_attn8 import NAMES, same_cache

pytestmark = pytest.mark.gpu
BAD = [np.inf, -np.inf, np.nan]


@pytest.mark.parametrize("dim,kvh,page", [(16, 1, 16), (80, 3, 32), (256, 2, 64)])
@pytest.mark.parametrize("st", [E.F32, E.F16, E.BF16], ids=lambda t: NAMES[t])
def test_append_what_is_not_finite(hip, st, dim, kvh, page):
    rng = np.random.default_rng(dim)
    total = 60
    c = Cache8(kvh, dim, page, [total], rng)
    kv, keep = c.upload(hip)
    pos = 0
    # tokens of the call, their size, and the tokens all of whose elements are bad
    for n, size, whole in ((20, 1.0, ()), (3, 300.0, ()), (1, 1e-3, ()), (9, 5e3, ()), (5, 1.0, range(5)), (2, 20.0, ()), (14, 1.0, (2,)), (6, 1e-2, ())):
        x = rng.standard_normal((2, n, kvh, dim)) * size
        for i in range(2):   # in K, and at other places in V
            for j, bad in enumerate(BAD):
                x[i, (j + i) % n, j % kvh, (5 * j + 3 + i) % dim] = bad
        for j in whole:
            x[:, j] = rng.choice(BAD, x[:, j].shape)
        k, v = to_bits(x[0], st), to_bits(x[1], st)
        write(hip, keep[3], np.array([pos + n], np.int32))
        hip.kv_append_dev(kv, 1, hip.upload(np.array([0, n], np.int32)), n, st, hip.upload(k), 0, hip.upload(v), 0)
        c.append(0, pos, from_bits(k, st), from_bits(v, st))
        same_cache(hip, keep, c)
        pos += n
    assert pos == total
    assert all(((code & 127) == 127)[c.table[0]].sum() > 2 * kvh for code in c.code)
