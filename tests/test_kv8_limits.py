"""CPU test of how much an append into an 8-bit cache takes: exactly what the header says, in launches that the runtime takes (fewer than
2^32 threads along a dimension), with the HIP calls answered by a stub."""
from test_kv_pool import child  # noqa: F401 (a fixture)

LIMITS = r"""
P = 1 << 20
def call(heads, nseq, ntok, starts):
    k = E.Kv8(E.F8, heads, 64, 16, 100, 4096, 8192, 4096, 4096, 4096, 8, 64, 4096, 4096)
    n = counts[0]
    rc = code(L.kv_append_dev, k, nseq, P if starts else None, ntok, E.F32, P, 0, P, 0)
    return [rc, counts[0] - n, shapes[n % 64][0] * shapes[n % 64][2] if counts[0] > n else 0]
most = (1 << 26) - 4
rows = []
for heads in (1, 3, 8, 4096):
    n = most // heads
    rows.append([call(heads, n, n, False), call(heads, n + 1, n + 1, False)])
    t = min((n - 3) * 16 + 15, (1 << 31) - 1)   # one sequence: t / 16 + 2 + 1 of each head
    rows.append([call(heads, 1, t, True), call(heads, 1, t + 1, True)])
    b = (n - 1) // 2   # sequences that bring nothing, but for 15 tokens
    rows.append([call(heads, b, 15, True), call(heads, b + 1, 15, True)])
print(json.dumps(rows))
"""


def test_append_takes_what_the_header_says(child):  # noqa: F811
    for fits, more in child(LIMITS):
        assert fits[:2] == [0, 1] and fits[2] < 1 << 32
        assert more == [-2, 0, 0]
