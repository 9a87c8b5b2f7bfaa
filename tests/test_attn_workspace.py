"""CPU tests of es_hip_attn_workspace_upto: one workspace of that size serves every attention call up to the given one (the HIP calls
answered by the stub of test_kv_pool.py)."""
import pytest

from test_kv_pool import child   # noqa: F401  (a fixture)

CALLS = r"""
import random
P, out = 1 << 20, []
for shape, heads, most_seq, most_tok in CASES:
    k = kv(**shape)
    b = L.attn_workspace_upto(k, most_seq, most_tok, heads)
    rng, refused, need = random.Random(1), [], 0
    sizes = [(s, n) for s in {1, 2, 3, most_seq // 2, most_seq - 1, most_seq} for n in {1, 2, 64, 512, most_tok // 2, most_tok - 1, most_tok}]
    sizes += [(int(most_seq ** rng.random()), int(most_tok ** rng.random())) for _ in range(300)]
    for s, n in sizes:
        if not 0 < s <= most_seq or not 0 < n <= most_tok: continue
        for t in (E.F32, k.type):
            need = max(need, L.attn_prompt_workspace(k, s, n, heads, t), L.attn_decode_workspace(k, s, heads))
            if code(L.attn_prompt_dev, k, s, P, n, heads, t, P, 0, 0.1, 0, P, 0, P if b else None, b): refused.append(["prompt", s, n, t])
            if code(L.attn_decode_dev, k, s, heads, t, P, 0, 0.1, 0, P, 0, P if b else None, b): refused.append(["decode", s, t])
    out.append([b, need, refused])
print(json.dumps(out))
"""
# (cache, query heads, most sequences, most tokens): a pool of 256 pages of 32 as an integration has, wide and narrow heads, one K/V
# head and as many as there are workgroups, tables too short for parts
CASES = [
    (dict(heads=8, dim=64, page=32, max_pages=256, rows=64, type=1), 32, 64, 2048),
    (dict(heads=8, dim=64, page=32, max_pages=256, rows=64, type=30), 32, 64, 16384),
    (dict(heads=4, dim=128, page=16, max_pages=512, rows=1, type=1), 32, 1, 16384),
    (dict(heads=4, dim=128, page=16, max_pages=512, rows=300, type=30), 32, 300, 5000),
    (dict(heads=1, dim=256, page=64, max_pages=100, rows=9, type=30), 71, 9, 3000),
    (dict(heads=2, dim=72, page=16, max_pages=41, rows=40, type=1), 14, 40, 100),
    (dict(heads=512, dim=8, page=16, max_pages=100, rows=5, type=1), 512, 5, 300),
    (dict(heads=256, dim=64, page=16, max_pages=100, rows=5, type=1), 256, 5, 300),
    (dict(heads=8, dim=64, page=16, max_pages=32, rows=20, type=1), 32, 20, 5000),
]


@pytest.mark.parametrize("i", range(len(CASES)))
def test_one_workspace_for_every_smaller_call(child, i):   # noqa: F811
    (bound, need, refused), = child(f"CASES = {[CASES[i]]!r}\n" + CALLS)
    assert refused == []
    assert need <= bound <= 2 * need


def test_no_bytes_where_calls_are_refused(child):   # noqa: F811
    got = child(r"""
good = kv()
print(json.dumps([L.attn_workspace_upto(k, s, n, h) for k, s, n, h in
                  [(kv(dim=100), 3, 9, 32), (good, 3, 9, 30), (good, -1, 9, 32), (good, 3, -1, 32), (good, 0, 9, 32), (good, 3, 1 << 28, 32)]]
                 + [L.attn_workspace_upto(good, 3, 0, 32) - L.attn_decode_workspace(good, 3, 32)]))
""")
    assert got == [0] * 7


def test_no_bytes_for_a_type_that_the_call_refuses(child):   # noqa: F811
    got = child(r"""
P, out = 1 << 20, []
for cache in (E.F16, E.BF16):
    k = kv(type=cache)
    for t in (E.F32, E.F16, E.BF16, 2, 99):
        fine = code(L.attn_prompt_dev, k, 3, P, 9, 32, t, P, 0, 0.1, 0, P, 0, P, 1 << 30) == 0
        out.append([fine, L.attn_prompt_workspace(k, 3, 9, 32, t) > 0, "type" in L.last_error() or "F32" in L.last_error()])
print(json.dumps(out))
""")
    assert all(fine == some for fine, some, _ in got) and sum(fine for fine, _, _ in got) == 4
    assert all(named for fine, _, named in got if not fine)
