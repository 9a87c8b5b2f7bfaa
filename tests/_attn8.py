"""A paged key-value cache in 8 bits in host memory, what an append leaves in it, and attention through windows with sinks from the
formula in 64 bits: what the GPU tests of es_hip_kv_append_dev and es_hip_attn_* on caches of type F8 compare with."""
import numpy as np

import es_hip_quant as E

LEAST, MOST, RUN = -100, 120, 16


def _values():
    """what the 256 codes stand for: 1 sign, 4 exponent (bias 7) and 3 mantissa bits, no infinities"""
    c = np.arange(256)
    e, m = c >> 3 & 15, c & 7
    x = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    x = np.where((c & 127) == 127, np.nan, x)
    return np.where(c & 128, -x, x)


VALUES = _values()
POSITIVE = VALUES[:127]   # ascending


def nearest(y):
    """the code of the number nearest to y (|y| <= 448), ties to the even code; NaN for what is not finite"""
    a = np.abs(np.where(np.isfinite(y), y, 0.0))
    i = np.clip(np.searchsorted(POSITIVE, a), 1, 126)
    lo, hi = POSITIVE[i - 1], POSITIVE[i]
    mid = (lo + hi) / 2
    i = np.where((a < mid) | ((a == mid) & ((i - 1) % 2 == 0)), i - 1, i)
    return np.where(np.isfinite(y), i | np.where(np.signbit(y), 128, 0), 127).astype(np.uint8)


def exponent_for(x):
    """the least e with |x| <= 448 * 2^e for all finite elements of x"""
    big = np.abs(x[np.isfinite(x)]).max(initial=0.0)
    if big == 0:
        return LEAST
    m, e = np.frexp(big)   # big = m * 2^e, 448 = 0.875 * 2^9
    return int(np.clip(e - 8 if m > 0.875 else e - 9, LEAST, MOST))


class Cache8:
    """pools filled with what must not be read (NaN codes, infinite scales), a page table, lengths"""

    t = E.BF16   # the type of a prompt's weights, that of its queries if that is of 16 bits (for _attn.tolerance)

    def __init__(self, heads, dim, page, lens, rng, spare=3, max_pages=None):
        self.heads, self.dim, self.page = heads, dim, page
        self.len = np.array(lens, np.int32)
        need = [-(-n // page) for n in lens]
        self.max_pages = max_pages or max(1, max(need))
        self.npages = sum(need) + spare
        self.code = [np.full((self.npages, heads, page, dim), 0x7F, np.uint8) for _ in range(2)]
        self.scale = [np.full((self.npages, heads, page // RUN), np.inf, np.float32) for _ in range(2)]
        self.table = np.full((len(lens), self.max_pages), -1, np.int32)
        p = rng.permutation(self.npages)
        at = 0
        for r, n in enumerate(need):
            self.table[r, :n] = p[at:at + n]
            at += n

    def append(self, r, pos, k, v):
        """one call's rows k, v [n, heads, dim] (64 bits) at positions pos.. of row r"""
        n = len(k)
        for u in range(pos // RUN, (pos + n - 1) // RUN + 1):
            g, o = self.table[r, u * RUN // self.page], u * RUN % self.page
            if not 0 <= g < self.npages:
                continue
            lo, hi = max(pos, u * RUN), min(pos + n, (u + 1) * RUN)
            for x, code, scale in ((k, self.code[0], self.scale[0]), (v, self.code[1], self.scale[1])):
                for h in range(self.heads):
                    y = x[lo - pos:hi - pos, h]
                    e = exponent_for(y)
                    if lo > u * RUN:
                        old = int(np.log2(scale[g, h, o // RUN]))
                        e = max(e, old)
                        kept = code[g, h, o:o + lo - u * RUN]
                        if e > old:
                            kept[:] = nearest(VALUES[kept] * 2.0 ** (old - e))
                    code[g, h, o + lo - u * RUN:o + hi - u * RUN] = nearest(y * 2.0 ** -e)
                    scale[g, h, o // RUN] = 2.0 ** e

    def fill(self, rng, spread=1.0):
        """every sequence's tokens, with a spread of its own in every run"""
        for r, n in enumerate(self.len):
            if n > 0:
                x = rng.standard_normal((2, n, self.heads, self.dim)) * spread
                x[1] *= np.exp2(rng.integers(-3, 4, -(-n // RUN))).repeat(RUN)[:n, None, None]
                self.append(r, 0, x[0], x[1])

    def rows(self, r):
        """row r's K and V [len, heads, dim] in 64 bits, and which of its tokens lie in a page"""
        n, tab = int(self.len[r]), self.table[r]
        j = np.arange(n)
        g = tab[j // self.page]
        ok = (g >= 0) & (g < self.npages)
        g = np.where(ok, g, 0)
        o = j % self.page
        with np.errstate(invalid="ignore"):
            k, v = (VALUES[self.code[i][g, :, o]] * self.scale[i][g, :, o // RUN][..., None].astype(np.float64) for i in range(2))
        return k, v, ok

    def v_scales(self, r):
        """the scale of each of row r's V rows [len, heads] (0 where it has no page)"""
        j = np.arange(int(self.len[r]))
        g = self.table[r][j // self.page]
        ok = (g >= 0) & (g < self.npages)
        return np.where(ok[:, None], self.scale[1][np.where(ok, g, 0), :, j % self.page // RUN], 0.0)

    def upload(self, hip, seq=None):
        """(Kv, buffers to keep: K, V, table, lengths, scales of K and of V)"""
        keep = [hip.upload(x) for x in (*self.code, self.table, self.len, *self.scale)]
        ds = None if seq is None else hip.upload(np.array(seq, np.int32))
        kv = E.Kv8(E.F8, self.heads, self.dim, self.page, self.npages, int(keep[0]), int(keep[1]), int(keep[2]), int(keep[3]),
                  None if ds is None else int(ds), len(self.len), self.max_pages, int(keep[4]), int(keep[5]))
        return kv, keep + [ds]


def attention(cache, starts, q, scale, window=0, sinks=0, seq=None):
    """q [ntok, heads, dim] in 64 bits -> out, per output the sum of |p v| (the scale of its rounding errors), and, of an 8-bit cache, what
    weights below fp16's range may change in a prompt's row.

    Those go into the products as p * (V's scale) relative to the row's largest such, which stands between 2^12 and 2^15; two terms of
    fp16 (or one) are off by at most half of its smallest step, 2^-25, which is 2^-37 of the largest. n keys of numbers up to 448 add that up."""
    out, mag, low = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape)
    G = q.shape[1] // cache.heads
    for b in range(len(starts) - 1):
        r = b if seq is None else seq[b]
        if r < 0 or r >= len(cache.len):
            continue
        K, V, ok = cache.rows(r)
        n, f = len(K), starts[b + 1] - starts[b]
        pos, j = np.arange(n - f, n)[:, None], np.arange(n)
        seen = ok & (j <= pos) & ((j > pos - window) | (j < sinks) if window else True)
        some = seen.any(1)
        if not some.any():
            continue
        any_sees = seen.any(0)[:, None, None]
        K, V = np.where(any_sees, K, 0.0), np.where(any_sees, V, 0.0)
        for h in range(q.shape[1]):
            s = np.where(seen, scale * (q[starts[b]:starts[b + 1], h] @ K[:, h // G].T), -np.inf)
            p = np.exp(s - np.where(some, s.max(1), 0.0)[:, None])
            p /= np.where(some, p.sum(1), 1.0)[:, None]
            out[starts[b]:starts[b + 1], h] = p @ V[:, h // G]
            mag[starts[b]:starts[b + 1], h] = p @ np.abs(V[:, h // G])
            if isinstance(cache, Cache8):
                largest = (p * np.where(any_sees[:, 0, 0], cache.v_scales(r)[:, h // G], 0.0)).max(1)
                low[starts[b]:starts[b + 1], h] = (n * 448 * 2.0 ** -37 * largest)[:, None]
    return out, mag, low
