"""The speed of the paged key-value cache in 8 bits and of attention that keeps a few first tokens in sight of a window, through
the library's C ABI.

A case is one call with its sizes:

  append  K and V rows of new tokens quantized into their pages (es_hip_kv_append_dev on a cache of type ES_HIP_F8)
  decode  attention of one new token per sequence over its pages (es_hip_attn_decode_dev, or with sinks es_hip_attn_decode_sinks_dev)
  prompt  causal attention of packed prompts or prompt chunks over their pages (es_hip_attn_prompt_dev, es_hip_attn_prompt_sinks_dev)

The 8-bit cache holds numbers of 8 bits (1 sign, 4 exponent, 3 mantissa bits: up to 448, no infinities) and, for every 16 tokens
of a page and K/V head, one scale for K and one for V: a power of two. With own true, run() makes the library's calls; otherwise it
computes the same in plain torch operations. listed() holds the named cases, draw() gives more of the same ranges, prepare() makes
what a program holds before the call (the cache, its page tables, the rows), exact() the same results in 64 bits.
"""
import os
import random
import sys

import numpy as np
import torch

own = False
LIB = None
F8, LOWEST, HIGHEST = 256, -100, 120     # the 8-bit cache's type number and the range of its scales' exponents
TYPES = {"f32": (torch.float32, 0), "f16": (torch.float16, 1), "bf16": (torch.bfloat16, 30), "f8": (torch.float8_e4m3fn, F8)}
RUN = 16                                 # tokens that share a scale


def _lib():
    """the binding and the loaded library"""
    global LIB
    if LIB is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "stream-_amd"))
        import es_hip_quant as E

        LIB = (E, E.Lib())
        if not LIB[1].available():
            raise RuntimeError(LIB[1].last_error())
    return LIB


# ---- the cases -------------------------------------------------------------------------------------------------------
# seqs sequences of lo..hi tokens, the last `new` of each (0: all of them) being the call's own;
# heads query heads over kv heads of dim elements; pages of `page` tokens; q and cache types; window 0: none; sinks: first tokens
# that the window leaves in sight
def listed():
    return [
        # one sequence's next token into a partly filled run: the smallest call, all latency
        dict(name="append_t1", kind="append", seqs=1, lo=700, hi=700, new=1, kv=4, dim=128, page=32, src="f32"),
        # a decode batch's tokens, each into a run of its own, from 16-bit rows
        dict(name="append_t48", kind="append", seqs=48, lo=50, hi=4000, new=1, kv=8, dim=128, page=16, src="bf16"),
        # four prompts of different lengths written at once
        dict(name="append_packed", kind="append", seqs=4, lo=333, hi=4096, new=0, kv=8, dim=64, page=16, src="f32"),
        # a chat's next token in a 1B model (2048 wide, 512 of K and V) after a short prompt
        dict(name="decode_t1", kind="decode", seqs=1, lo=500, hi=500, heads=32, kv=8, dim=64, page=32, q="f32", cache="f8", window=0, sinks=0),
        # a decode batch of 32 sequences of very different lengths (4096 of q, 512 of K and V)
        dict(name="decode_t32", kind="decode", seqs=32, lo=77, hi=8192, heads=32, kv=4, dim=128, page=16, q="f32", cache="f8", window=0, sinks=0),
        # one sequence with a book in its context
        dict(name="decode_long", kind="decode", seqs=1, lo=131072, hi=131072, heads=32, kv=4, dim=128, page=64, q="bf16", cache="f8", window=0,
             sinks=0),
        # the engine's batch of 64 tokens, deep in a long prompt
        dict(name="prompt_t64", kind="prompt", seqs=1, lo=8001, hi=8001, new=64, heads=32, kv=4, dim=128, page=32, q="f32", cache="f8", window=0,
             sinks=0),
        # eight prompts of different lengths, packed
        dict(name="prompt_packed", kind="prompt", seqs=8, lo=99, hi=3333, new=0, heads=32, kv=8, dim=128, page=16, q="bf16", cache="f8",
             window=0, sinks=0),
        # a long document in one call
        dict(name="prompt_t16384", kind="prompt", seqs=1, lo=16384, hi=16384, new=0, heads=32, kv=4, dim=128, page=64, q="bf16", cache="f8",
             window=0, sinks=0),
        # a batch on a 0.5B model (896 wide: 14 heads over 2) that streams: the last 4096 tokens and the first 4
        dict(name="decode_sinks", kind="decode", seqs=48, lo=1000, hi=12000, heads=14, kv=2, dim=64, page=32, q="bf16", cache="bf16",
             window=4096, sinks=4),
        # the same kind of stream over an 8-bit cache: wide heads, a short window, a system prompt of 100 tokens kept
        dict(name="decode_sinks_f8", kind="decode", seqs=64, lo=3000, hi=20000, heads=32, kv=8, dim=128, page=64, q="f32", cache="f8",
             window=2048, sinks=100),
        # a long document read through a window of 1024 with its first 4 tokens in sight
        dict(name="prompt_sinks", kind="prompt", seqs=1, lo=12001, hi=12001, new=0, heads=32, kv=8, dim=64, page=32, q="f16", cache="f16",
             window=1024, sinks=4),
    ]


def _log(rng, lo, hi):
    """a whole number in [lo, hi], spread evenly over its logarithm"""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["append", "append", "decode", "decode", "decode", "prompt", "prompt", "prompt"])
    kv, dim, page = rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 64, 80, 96, 128, 128, 256]), rng.choice([16, 16, 32, 64, 128])
    if kind == "append":
        src = rng.choice(["f32", "f32", "bf16", "f16"])
        if rng.random() < 0.5:
            return dict(kind=kind, seqs=_log(rng, 1, 64), lo=1, hi=_log(rng, 2, 2000), new=1, kv=kv, dim=dim, page=page, src=src)
        return dict(kind=kind, seqs=rng.randint(1, 4), lo=1, hi=_log(rng, 2, 3000), new=rng.choice([0, 0, _log(rng, 1, 128)]), kv=kv, dim=dim,
                    page=page, src=src)
    cache = rng.choice(["f8", "f8", "f16", "bf16"])
    q, heads = rng.choice(["f32", "bf16" if cache == "f8" else cache]), kv * rng.choice([1, 2, 4, 4, 5, 7, 8])
    seqs = _log(rng, 1, 64) if kind == "decode" else rng.choice([1, 1, 2, 5])
    hi = _log(rng, 16, 200000 // (seqs * kv) if kind == "decode" else 6000 // seqs)
    # 16-bit caches without sinks are no new call: those have both
    window = rng.randint(1, hi) if cache != "f8" else rng.choice([0, 0, rng.randint(1, hi)])
    sinks = (_log(rng, 1, max(1, hi // 8)) if window and (cache != "f8" or rng.random() < 0.5) else 0)
    c = dict(kind=kind, seqs=seqs, lo=max(1, hi // rng.choice([1, 2, 20] if kind == "decode" else [1, 1, 3])), hi=hi, heads=heads, kv=kv, dim=dim,
             page=page, q=q, cache=cache, window=window, sinks=sinks)
    if kind == "prompt":
        c["new"] = rng.choice([0, 0, _log(rng, 1, 128)])
    return c


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _lengths(c, seed):
    """each sequence's tokens in the cache and how many of them are the call's own: the same lengths in an order of the seed's"""
    r = random.Random(17)
    total = [c["hi"]] + [_log(r, c["lo"], c["hi"]) for _ in range(c["seqs"] - 1)]
    random.Random(seed).shuffle(total)
    fresh = [1 if c["kind"] == "decode" else min(n, c["new"] or n) for n in total]
    return total, fresh


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _rows(g, shape, dtype, outliers):
    """normal rows; K rows have a few channels of larger spread, as attention keys do"""
    x = torch.randn(shape, device="cuda", generator=g)
    if outliers:
        x[..., 3::29] *= 3.0
    return x.to(dtype)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _exponent(amax):
    """the least e in [LOWEST, HIGHEST] with amax <= 448 * 2^e"""
    m, e = torch.frexp(amax)                     # amax = m * 2^e, 448 = 0.875 * 2^9
    return torch.where(m > 0.875, e - 8, e - 9).clamp(LOWEST, HIGHEST)


def _power(e):
    """2^e in fp32"""
    return (e.int() + 127 << 23).view(torch.float32)


def _eight(x, e):
    """x * 2^-e (exact), rounded to the nearest number of 8 bits"""
    return (x * _power(-e)).to(torch.float8_e4m3fn)


def _pools(g, shape, cache):
    """K and V of [pages, heads, tokens, elements], and, of an 8-bit cache, the scales of every 16 tokens"""
    if cache != "f8":
        return _rows(g, shape, TYPES[cache][0], True), _rows(g, shape, TYPES[cache][0], False), None, None
    got = []
    for outliers in (True, False):
        x = _rows(g, shape, torch.float32, outliers).view(shape[0], shape[1], shape[2] // RUN, RUN, shape[3])
        e = _exponent(x.abs().amax((3, 4)))
        got.append((_eight(x, e[..., None, None]).view(shape), _power(e)))
    return got[0][0], got[1][0], got[0][1], got[1][1]


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = {"case": c}
    total, fresh = _lengths(c, seed)
    page = c["page"]
    most = max(-(-n // page) for n in total)
    used = sum(-(-n // page) for n in total)
    npages = used + 5
    p = np.random.RandomState(seed % (1 << 31)).permutation(npages)
    table, at = np.full((c["seqs"], most), -1, np.int32), 0
    for b, n in enumerate(total):
        k = -(-n // page)
        table[b, :k] = p[at: at + k]
        at += k
    s["k"], s["v"], s["ks"], s["vs"] = _pools(g, (npages, c["kv"], page, c["dim"]), c.get("cache", "f8"))
    s["table"], s["len"], s["start"] = _ints(table), _ints(total), _ints([0] + list(np.cumsum(fresh)))
    s["total"], s["fresh"], s["most"] = total, fresh, most
    ntok = sum(fresh)
    if c["kind"] == "append":
        src = TYPES[c["src"]][0]
        s["nk"], s["nv"] = _rows(g, (ntok, c["kv"], c["dim"]), src, True), _rows(g, (ntok, c["kv"], c["dim"]), src, False)
    else:
        s["q"] = _rows(g, (ntok, c["heads"], c["dim"]), TYPES[c["q"]][0], False)
        s["out"] = torch.zeros_like(s["q"])
    return s


# ---- one pass: plain -------------------------------------------------------------------------------------------------
def _plain_append(s):
    """The scale of a run that gets tokens: what they need, and no less than it was where the run has earlier tokens, whose numbers
    are then rounded once more to the larger scale."""
    page, dim = s["case"]["page"], s["case"]["dim"]
    start, n = s["start"].long(), s["len"].long()
    t = torch.arange(s["nk"].shape[0], device="cuda")
    b = torch.searchsorted(start, t, right=True) - 1
    pos = n[b] - (start[b + 1] - t)
    at = s["table"].long()[b, pos // page]
    run, off = pos % page // RUN, pos % RUN
    before = pos - off < n[b] - (start[b + 1] - start[b])          # the run has tokens from before the call
    old = torch.arange(RUN, device="cuda") < (n[b] - (start[b + 1] - start[b]) - (pos - off))[:, None]   # [token, token of its run]
    for pool, scales, rows in ((s["k"], s["ks"], s["nk"].float()), (s["v"], s["vs"], s["nv"].float())):
        runs = pool.view(torch.uint8).view(pool.shape[0], pool.shape[1], page // RUN, RUN, dim)
        need = _exponent(rows.abs().amax(2))                       # [token, head]
        had = torch.frexp(scales[at, :, run])[1] - 1
        place = (at * (page // RUN) + run)[:, None].expand(-1, rows.shape[1])
        e = torch.full((pool.shape[0] * (page // RUN), rows.shape[1]), LOWEST, dtype=torch.int64, device="cuda")
        e.scatter_reduce_(0, place, torch.where(before[:, None], torch.maximum(need, had), need).long(), "amax")
        e = e.gather(0, place).int()
        kept = runs[at, :, run].view(torch.float8_e4m3fn)          # [token, head, 16, dim]
        again = _eight(kept.float(), (e - had)[..., None, None]).view(torch.uint8)
        runs[at, :, run] = torch.where(old[:, None, :, None], again, kept.view(torch.uint8))
        scales[at, :, run] = _power(e)
        runs[at, :, run, off] = _eight(rows, e[..., None]).view(torch.uint8)
    return [s["k"], s["ks"], s["v"], s["vs"]]


def _plain_rows(pool, scales, at, L):
    """[sequence, head, token, element] in fp32 of the sequences' pages `at`"""
    x = pool[at].float() if scales is None else pool.view(torch.uint8)[at].view(torch.float8_e4m3fn).float()
    if scales is not None:
        x = x.view(*x.shape[:3], -1, RUN, x.shape[4]).mul_(scales[at][..., None, None]).view(x.shape)
    return x.permute(0, 2, 1, 3, 4).reshape(x.shape[0], x.shape[2], L, x.shape[4])


def _plain_attention(s):
    """gathers each sequence's pages, padded to the longest, and takes the masked softmax over them in fp32"""
    c = s["case"]
    B, kv, dim, G = c["seqs"], c["kv"], c["dim"], c["heads"] // c["kv"]
    start, n = s["start"].long(), s["len"].long()
    ntok, Q, L = s["q"].shape[0], max(s["fresh"]), s["most"] * c["page"]
    at = s["table"].long().clamp_min(0)
    k, v = _plain_rows(s["k"], s["ks"], at, L), _plain_rows(s["v"], s["vs"], at, L)
    i = torch.arange(Q, device="cuda")
    own_rows = start[1:] - start[:-1]
    row = torch.where(i < own_rows[:, None], start[:-1, None] + i, ntok)                       # [B, Q]; past the end: a row of zeros
    q = torch.cat([s["q"], s["q"].new_zeros(1, c["heads"], dim)]).float()[row]                 # [B, Q, heads, dim]
    q = q.reshape(B, Q, kv, G, dim).permute(0, 2, 3, 1, 4).reshape(B, kv, G * Q, dim)
    pos = (n - own_rows)[:, None] + i                                                          # [B, Q]
    j = torch.arange(L, device="cuda")
    hidden = j > pos[..., None]
    if c["window"]:
        hidden |= (j <= pos[..., None] - c["window"]) & (j >= c["sinks"])
    p = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(dim ** -0.5).view(B, kv, G, Q, L)
    p.masked_fill_(hidden[:, None, None], float("-inf"))
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(p.view(B, kv, G * Q, L), v) / p.sum(-1).view(B, kv, G * Q, 1)
    o = o.view(B, kv, G, Q, dim).permute(0, 3, 1, 2, 4).reshape(B * Q, c["heads"], dim).to(s["out"].dtype)
    out = s["out"].new_zeros(ntok + 1, c["heads"], dim)
    out[row.reshape(-1)] = o
    return out[:ntok]


# ---- one pass: the library's calls -----------------------------------------------------------------------------------
def _kv(s):
    """the library's view of the cache, kept with the state as a program keeps it"""
    if "kv" not in s:
        E, _ = _lib()
        c = s["case"]
        fields = (TYPES[c.get("cache", "f8")][1], c["kv"], c["dim"], c["page"], s["k"].shape[0], s["k"].data_ptr(), s["v"].data_ptr(),
                  s["table"].data_ptr(), s["len"].data_ptr(), None, c["seqs"], s["most"])
        s["kv"] = E.Kv(*fields) if s["ks"] is None else E.Kv8(*fields, s["ks"].data_ptr(), s["vs"].data_ptr())
    return s["kv"]


def _workspace(s, nbytes):
    if "ws" not in s:
        s["ws"] = torch.empty(max(nbytes(), 16), dtype=torch.uint8, device="cuda")
    return s["ws"].data_ptr(), s["ws"].numel()


def _own_run(s):
    _, L = _lib()
    c, kv = s["case"], _kv(s)
    ntok = sum(s["fresh"])
    if c["kind"] == "append":
        L.kv_append_dev(kv, c["seqs"], s["start"].data_ptr(), ntok, TYPES[c["src"]][1], s["nk"].data_ptr(), 0, s["nv"].data_ptr(), 0)
        return [s["k"], s["ks"], s["v"], s["vs"]]
    t, scale, q, out = TYPES[c["q"]][1], c["dim"] ** -0.5, s["q"].data_ptr(), s["out"].data_ptr()
    if c["kind"] == "decode":
        ws = _workspace(s, lambda: L.attn_decode_workspace(kv, c["seqs"], c["heads"]))
        if c["sinks"]:
            L.attn_decode_sinks_dev(kv, c["seqs"], c["heads"], t, q, 0, scale, c["window"], c["sinks"], out, 0, *ws)
        else:
            L.attn_decode_dev(kv, c["seqs"], c["heads"], t, q, 0, scale, c["window"], out, 0, *ws)
    else:
        ws = _workspace(s, lambda: L.attn_prompt_workspace(kv, c["seqs"], ntok, c["heads"], t))
        if c["sinks"]:
            L.attn_prompt_sinks_dev(kv, c["seqs"], s["start"].data_ptr(), ntok, c["heads"], t, q, 0, scale, c["window"], c["sinks"], out, 0, *ws)
        else:
            L.attn_prompt_dev(kv, c["seqs"], s["start"].data_ptr(), ntok, c["heads"], t, q, 0, scale, c["window"], out, 0, *ws)
    return s["out"]


def run(s):
    if own:
        return _own_run(s)
    return _plain_append(s) if s["case"]["kind"] == "append" else _plain_attention(s)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    c = case
    es = {"f32": 4, "f16": 2, "bf16": 2, "f8": 1}
    total, fresh = _lengths(c, 0)
    if c["kind"] == "append":
        runs = sum((n - 1) // RUN - (n - f) // RUN + 1 for n, f in zip(total, fresh))
        return {"bytes": 2 * sum(fresh) * c["kv"] * c["dim"] * (es[c["src"]] + 1) + 2 * runs * c["kv"] * 4, "flops": 0}
    w = c["window"] or 1 << 30
    seen = lambda p: min(p + 1, w + min(c["sinks"], max(0, p + 1 - w)))  # noqa: E731
    pairs = sum(seen(p) for n, f in zip(total, fresh) for p in range(n - f, n))
    read = sum(min(n, f + w - 1 + min(c["sinks"], max(0, n - f + 1 - w))) for n, f in zip(total, fresh))
    row = c["dim"] * es[c["cache"]] + (4 / RUN if c["cache"] == "f8" else 0)
    return {"bytes": 2 * read * c["kv"] * row + 2 * sum(fresh) * c["heads"] * c["dim"] * es[c["q"]],
            "flops": 4 * pairs * c["heads"] * c["dim"]}


# ---- in 64 bits ------------------------------------------------------------------------------------------------------
def _nearest(y):
    """y (64 bits) rounded to the nearest number of 8 bits, ties to even: steps of 2^-9 up to 2^-6, then of an eighth of the binade"""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def _exact_append(s):
    """sequence by sequence and run by run, from the definition: the least power of two whose 448-fold covers what the run is to hold"""
    c, table = s["case"], s["table"].cpu().numpy()
    k, v = s["k"].double(), s["v"].double()
    got = [k, s["ks"].double(), v, s["vs"].double()]
    t = 0
    for b, (n, f) in enumerate(zip(s["total"], s["fresh"])):
        for r in range((n - f) // RUN, (n - 1) // RUN + 1):
            lo, hi = max(n - f, r * RUN), min(n, (r + 1) * RUN)
            page, u, o = int(table[b, r * RUN // c["page"]]), r * RUN % c["page"] // RUN, r * RUN % c["page"]
            for x, pool, scales in ((s["nk"], got[0], got[1]), (s["nv"], got[2], got[3])):
                x = x[t + lo - n + f: t + hi - n + f].double().transpose(0, 1)                 # [head, token, element]
                e = torch.ceil(torch.log2(x.abs().amax((1, 2)) / 448)).clamp(LOWEST, HIGHEST)
                if lo > r * RUN:
                    e = torch.maximum(e, torch.log2(scales[page, :, u]))
                    kept = pool[page, :, o: o + lo - r * RUN]
                    pool[page, :, o: o + lo - r * RUN] = _nearest(kept * (scales[page, :, u] / torch.exp2(e))[:, None, None])
                pool[page, :, o + lo - r * RUN: o + hi - r * RUN] = _nearest(x / torch.exp2(e)[:, None, None])
                scales[page, :, u] = torch.exp2(e)
        t += f
    return got


def exact(case, seed):
    """sequence by sequence and head by head from the definition"""
    s = prepare(case, seed)
    c = case
    if c["kind"] == "append":
        return _exact_append(s)
    table, page = s["table"].cpu().numpy(), c["page"]
    t = 0
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    G = c["heads"] // c["kv"]

    def rows(pool, scales, pages, h, n):
        if scales is None:
            return pool[pages, h].reshape(-1, c["dim"])[:n].double()
        x = torch.stack([pool[p, h].double() for p in pages]).view(-1, RUN, c["dim"])
        return (x * scales[pages, h].reshape(-1, 1, 1).double()).view(-1, c["dim"])[:n]

    for b, (n, f) in enumerate(zip(s["total"], s["fresh"])):
        pages = [int(x) for x in table[b, : -(-n // page)]]
        pos = torch.arange(n - f, n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")
        seen = (key <= pos) & ((key > pos - (c["window"] or n + 1)) | (key < c["sinks"]))
        for g in range(c["kv"]):
            k, v = rows(s["k"], s["ks"], pages, g, n), rows(s["v"], s["vs"], pages, g, n)
            for h in range(g * G, (g + 1) * G):
                z = torch.where(seen, (s["q"][t: t + f, h].double() @ k.t().contiguous()) / c["dim"] ** 0.5, -torch.inf)
                out[t: t + f, h] = torch.softmax(z, dim=1) @ v
        t += f
    return out
