"""A paged key-value cache in host memory and the attention over it from the formula, in 64 bits: what the GPU tests of
es_hip_kv_* and es_hip_attn_* compare with."""
import numpy as np

import es_hip_quant as E

EPS = {E.F32: 2.0 ** -23, E.F16: 2.0 ** -10, E.BF16: 2.0 ** -7}   # steps at 1; a rounding is off by half of one


def to_bits(x, t):
    """float array -> the type's storage (float32, or uint16 bits), rounded to nearest even"""
    x = np.asarray(x)
    if t == E.F32:
        return x.astype(np.float32)
    if t == E.F16:
        with np.errstate(over="ignore"):
            return x.astype(np.float32).astype(np.float16).view(np.uint16)
    u = x.astype(np.float32).view(np.uint32)
    r = (u + 0x7FFF + ((u >> 16) & 1)) >> 16
    return np.where(np.isnan(x), 0x7FC0, r).astype(np.uint16)


def from_bits(b, t):
    """storage -> float64"""
    if t == E.F32:
        return b.astype(np.float64)
    if t == E.F16:
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


class Cache:
    """pools of npages pages filled with what must not be read (NaN), a page table of `rows` rows, lengths"""

    def __init__(self, t, heads, dim, page, lens, rng, spare=3, max_pages=None, fill=np.nan):
        self.t, self.heads, self.dim, self.page = t, heads, dim, page
        self.len = np.array(lens, np.int32)
        need = [-(-n // page) for n in lens]
        self.max_pages = max_pages or max(1, max(need))
        self.npages = sum(need) + spare
        shape = (self.npages, heads, page, dim)
        self.k = to_bits(np.full(shape, fill, np.float32), t)
        self.v = to_bits(np.full(shape, fill, np.float32), t)
        self.table = np.full((len(lens), self.max_pages), -1, np.int32)
        p = rng.permutation(self.npages)
        at = 0
        for r, n in enumerate(need):
            self.table[r, :n] = p[at:at + n]
            at += n

    def put(self, r, pos, k, v):
        """rows k, v [n, heads, dim] (storage) at positions pos.. of row r"""
        for i in range(len(k)):
            g, o = self.table[r, (pos + i) // self.page], (pos + i) % self.page
            self.k[g, :, o], self.v[g, :, o] = k[i], v[i]

    def fill(self, rng, spread=1.0):
        for r, n in enumerate(self.len):
            x = rng.standard_normal((2, n, self.heads, self.dim)).astype(np.float32) * spread
            self.put(r, 0, to_bits(x[0], self.t), to_bits(x[1], self.t))

    def rows(self, r):
        """row r's K and V [len, heads, dim] in 64 bits, and which of its tokens lie in a page"""
        n, tab = int(self.len[r]), self.table[r]
        j = np.arange(n)
        g = tab[j // self.page]
        ok = (g >= 0) & (g < self.npages)
        g = np.where(ok, g, 0)
        return (from_bits(self.k[g, :, j % self.page], self.t), from_bits(self.v[g, :, j % self.page], self.t), ok)

    def upload(self, hip, seq=None):
        """(Kv, buffers to keep)"""
        keep = [hip.upload(x) for x in (self.k, self.v, self.table, self.len)]
        ds = None if seq is None else hip.upload(np.array(seq, np.int32))
        kv = E.Kv(self.t, self.heads, self.dim, self.page, self.npages, int(keep[0]), int(keep[1]), int(keep[2]), int(keep[3]),
                  None if ds is None else int(ds), len(self.len), self.max_pages)
        return kv, keep + [ds]


def attention(cache, starts, q, scale, window=0, seq=None):
    """q [ntok, heads, dim] in 64 bits -> out, and per output the sum of |p v| (the scale of its rounding errors)"""
    out, mag = np.zeros(q.shape), np.zeros(q.shape)
    G = q.shape[1] // cache.heads
    for b in range(len(starts) - 1):
        r = b if seq is None else seq[b]
        if r < 0 or r >= len(cache.len):
            continue
        K, V, ok = cache.rows(r)
        n, f = len(K), starts[b + 1] - starts[b]
        pos, j = np.arange(n - f, n)[:, None], np.arange(n)
        seen = ok & (j <= pos) & ((j > pos - window) if window else True)
        some = seen.any(1)
        if not some.any():
            continue
        K, V = np.where(ok[:, None, None], K, 0.0), np.where(ok[:, None, None], V, 0.0)
        for h in range(q.shape[1]):
            s = np.where(seen, scale * (q[starts[b]:starts[b + 1], h] @ K[:, h // G].T), -np.inf)
            p = np.exp(s - np.where(some, s.max(1), 0.0)[:, None])
            p /= np.where(some, p.sum(1), 1.0)[:, None]
            out[starts[b]:starts[b + 1], h] = p @ V[:, h // G]
            mag[starts[b]:starts[b + 1], h] = p @ np.abs(V[:, h // G])
    return out, mag


def tolerance(cache, q, t, scale, mag, out):
    """How far an output may be from the formula's: a row of it is sum p v with relative errors of p, and a last rounding.

    s = scale q.k is summed in fp32 from exact products of the terms of q (what q loses in its terms, 2^-22 of its row's
    largest, stays below): at most (dim + 4) half steps of 2^-24 relative to scale sum |q k|, and rounded once more when it is
    scaled to base 2 and to the maximum's reference (2 half steps of its size). An error e of s is one of e (relative) in p, and as
    p is divided by their sum, of at most 2 e in the weight. 2^x itself: 1 step. Weights kept as a 16-bit q has them are rounded once to the
    cache's type (half a step); else to 2^-22 or less. The sums over the keys are of fp32: the matrix products add 32 (or 16) at a time, so n keys
    take n / 16 additions, half a step each, relative to the sum of |p v|, the parts' joining a few more."""
    big = 0.0
    for r in range(len(cache.len)):
        K, _, ok = cache.rows(r)
        big = max(big, np.abs(K[ok]).max(initial=0.0))
    qk = scale * np.abs(q).sum(-1, keepdims=True) * big
    u = 2.0 ** -24
    e = (cache.dim + 4) * u * qk + 2.0 ** -22 * qk * 2 + 4 * u * (qk + 1)
    w = EPS[cache.t] / 2 if t != E.F32 else 2.0 ** -22
    n = int(cache.len.max(initial=1))
    rel = 2 * e + 2 * u + w + (n / 16 + 48) * u
    return rel * mag + EPS[t] / 2 * (np.abs(out) + rel * mag) + 1e-30
