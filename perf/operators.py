"""The speed of the paged key-value cache and of the attention that reads it, through the library's C ABI.

A case is one call with its sizes:

  append  K and V rows of new tokens written to their pages (es_hip_kv_append_dev)
  decode  attention of one new token per sequence over its pages (es_hip_attn_decode_dev)
  prompt  causal attention of packed prompts or prompt chunks over their pages (es_hip_attn_prompt_dev)
  pages   pages copied in every layer, as forks and compaction do (es_hip_kv_copy_pages_dev)

With own true, run() makes these calls; otherwise it computes the same in plain torch operations. listed() holds the named
cases, draw() gives more of the same ranges, prepare() makes what a program holds before the call (the cache, its page tables,
the rows), exact() the same results in 64 bits.
"""
import os
import random
import sys

import numpy as np
import torch

own = False
LIB = None
TYPES = {"f32": (torch.float32, 0), "f16": (torch.float16, 1), "bf16": (torch.bfloat16, 30)}


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
# heads query heads over kv heads of dim elements; pages of `page` tokens; q and cache types; window 0: none
def listed():
    return [
        # one sequence's next token: the smallest call, all latency
        dict(name="append_t1", kind="append", seqs=1, lo=700, hi=700, new=1, kv=4, dim=128, page=32, src="f32", cache="f16"),
        # four prompts of different lengths written at once
        dict(name="append_packed", kind="append", seqs=4, lo=333, hi=4096, new=0, kv=8, dim=64, page=16, src="f32", cache="bf16"),
        # a chat's next token in a 1B model (2048 wide, 512 of K and V) after a short prompt
        dict(name="decode_t1", kind="decode", seqs=1, lo=500, hi=500, heads=32, kv=8, dim=64, page=32, q="f32", cache="f16", window=0),
        # a decode batch of 32 sequences of very different lengths (4096 of q, 512 of K and V)
        dict(name="decode_t32", kind="decode", seqs=32, lo=77, hi=8192, heads=32, kv=4, dim=128, page=16, q="f32", cache="f16", window=0),
        # one sequence with a book in its context
        dict(name="decode_long", kind="decode", seqs=1, lo=131072, hi=131072, heads=32, kv=4, dim=128, page=64, q="f16", cache="f16",
             window=0),
        # a batch on a 0.5B model (896 wide: 14 heads over 2) whose layer sees the last 4096 tokens alone
        dict(name="decode_window", kind="decode", seqs=48, lo=1000, hi=12000, heads=14, kv=2, dim=64, page=32, q="bf16", cache="bf16",
             window=4096),
        # the engine's batch of 64 tokens, deep in a long prompt
        dict(name="prompt_t64", kind="prompt", seqs=1, lo=8001, hi=8001, new=64, heads=32, kv=4, dim=128, page=32, q="f32", cache="f16",
             window=0),
        # a whole prompt of 512 tokens in a 1B model
        dict(name="prompt_t512", kind="prompt", seqs=1, lo=512, hi=512, new=0, heads=32, kv=8, dim=64, page=16, q="f32", cache="bf16",
             window=0),
        # eight prompts of different lengths, packed
        dict(name="prompt_packed", kind="prompt", seqs=8, lo=99, hi=3333, new=0, heads=32, kv=8, dim=128, page=16, q="bf16",
             cache="bf16", window=0),
        # a long document in one call
        dict(name="prompt_t16384", kind="prompt", seqs=1, lo=16384, hi=16384, new=0, heads=32, kv=4, dim=128, page=64, q="f16",
             cache="f16", window=0),
        # the last pages of 32 forked sequences, in every layer
        dict(name="pages_fork", kind="pages", pages=600, moved=32, layers=16, kv=8, dim=64, page=16, cache="f16"),
        # a fragmented cache's upper half moved down
        dict(name="pages_compact", kind="pages", pages=4001, moved=1500, layers=4, kv=4, dim=128, page=32, cache="bf16"),
    ]


def _log(rng, lo, hi):
    """a whole number in [lo, hi], spread evenly over its logarithm"""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "decode", "prompt", "prompt", "prompt", "pages"])
    kv, dim, page = rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 64, 80, 96, 128, 128, 256]), rng.choice([16, 16, 32, 64, 128])
    cache = rng.choice(["f16", "bf16"])
    if kind == "pages":
        pages = _log(rng, 64, 4000)
        return dict(kind=kind, pages=pages, moved=_log(rng, 1, pages // 3), layers=rng.randint(1, 4), kv=kv, dim=dim, page=min(page, 32),
                    cache=cache)
    if kind == "append":
        if rng.random() < 0.5:
            return dict(kind=kind, seqs=_log(rng, 1, 64), lo=1, hi=_log(rng, 2, 2000), new=1, kv=kv, dim=dim, page=page,
                        src=rng.choice(["f32", cache]), cache=cache)
        return dict(kind=kind, seqs=rng.randint(1, 4), lo=1, hi=_log(rng, 2, 3000), new=0, kv=kv, dim=dim, page=page,
                    src=rng.choice(["f32", cache]), cache=cache)
    q, heads = rng.choice(["f32", cache]), kv * rng.choice([1, 2, 4, 4, 5, 7, 8])
    if kind == "decode":
        seqs = _log(rng, 1, 64)
        hi = _log(rng, 16, 200000 // (seqs * kv))
        return dict(kind=kind, seqs=seqs, lo=max(1, hi // rng.choice([1, 2, 20])), hi=hi, heads=heads, kv=kv, dim=dim, page=page, q=q,
                    cache=cache, window=rng.choice([0, 0, 0, rng.randint(1, hi)]))
    seqs = rng.choice([1, 1, 2, 5])
    hi = _log(rng, 16, 6000 // seqs)
    return dict(kind=kind, seqs=seqs, lo=max(1, hi // rng.choice([1, 1, 3])), hi=hi, new=rng.choice([0, 0, _log(rng, 1, 128)]),
                heads=heads, kv=kv, dim=dim, page=page, q=q, cache=cache, window=rng.choice([0, 0, 0, rng.randint(1, hi)]))


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


def prepare(case, seed):
    c, g = case, _gen(seed)
    cache = TYPES[c["cache"]][0]
    s = {"case": c}
    if c["kind"] == "pages":
        shape = (c["layers"], c["pages"], c["kv"], c["page"], c["dim"])
        s["k"], s["v"] = _rows(g, shape, cache, True), _rows(g, shape, cache, False)
        p = np.random.RandomState(seed % (1 << 31)).permutation(c["pages"]).astype(np.int32)
        s["src"], s["dst"] = p[: c["moved"]].copy(), p[c["moved"]: 2 * c["moved"]].copy()
        return s
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
    shape = (npages, c["kv"], page, c["dim"])
    s["k"], s["v"] = _rows(g, shape, cache, True), _rows(g, shape, cache, False)
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
    page = s["case"]["page"]
    start, n = s["start"].long(), s["len"].long()
    t = torch.arange(s["nk"].shape[0], device="cuda")
    b = torch.searchsorted(start, t, right=True) - 1
    pos = n[b] - (start[b + 1] - t)
    at = s["table"].long()[b, pos // page]
    s["k"][at, :, pos % page] = s["nk"].to(s["k"].dtype)
    s["v"][at, :, pos % page] = s["nv"].to(s["v"].dtype)
    return [s["k"], s["v"]]


def _plain_attention(s):
    """gathers each sequence's pages, padded to the longest, and takes the masked softmax over them in fp32"""
    c = s["case"]
    B, kv, dim, G = c["seqs"], c["kv"], c["dim"], c["heads"] // c["kv"]
    start, n = s["start"].long(), s["len"].long()
    ntok, Q, L = s["q"].shape[0], max(s["fresh"]), s["most"] * c["page"]
    at = s["table"].long().clamp_min(0)
    k = s["k"][at].permute(0, 2, 1, 3, 4).reshape(B, kv, L, dim).float()
    v = s["v"][at].permute(0, 2, 1, 3, 4).reshape(B, kv, L, dim).float()
    i = torch.arange(Q, device="cuda")
    own_rows = start[1:] - start[:-1]
    row = torch.where(i < own_rows[:, None], start[:-1, None] + i, ntok)                       # [B, Q]; past the end: a row of zeros
    q = torch.cat([s["q"], s["q"].new_zeros(1, c["heads"], dim)]).float()[row]                 # [B, Q, heads, dim]
    q = q.reshape(B, Q, kv, G, dim).permute(0, 2, 3, 1, 4).reshape(B, kv, G * Q, dim)
    pos = (n - own_rows)[:, None] + i                                                          # [B, Q]
    j = torch.arange(L, device="cuda")
    hidden = j > pos[..., None]
    if c["window"]:
        hidden |= j <= pos[..., None] - c["window"]
    p = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(dim ** -0.5).view(B, kv, G, Q, L)
    p.masked_fill_(hidden[:, None, None], float("-inf"))
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(p.view(B, kv, G * Q, L), v) / p.sum(-1).view(B, kv, G * Q, 1)
    o = o.view(B, kv, G, Q, dim).permute(0, 3, 1, 2, 4).reshape(B * Q, c["heads"], dim).to(s["out"].dtype)
    out = s["out"].new_zeros(ntok + 1, c["heads"], dim)
    out[row.reshape(-1)] = o
    return out[:ntok]


def _plain_pages(s):
    src, dst = torch.tensor(s["src"], device="cuda"), torch.tensor(s["dst"], device="cuda")
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    return [s["k"], s["v"]]


# ---- one pass: the library's calls -----------------------------------------------------------------------------------
def _kv(s):
    """the library's view of the cache, kept with the state as a program keeps it"""
    if "kv" not in s:
        E, _ = _lib()
        c, paged = s["case"], "table" in s
        s["kv"] = E.Kv(TYPES[c["cache"]][1], c["kv"], c["dim"], c["page"], s["k"].shape[-4], s["k"].data_ptr(), s["v"].data_ptr(),
                       s["table"].data_ptr() if paged else None, s["len"].data_ptr() if paged else None, None,
                       c["seqs"] if paged else 0, s["most"] if paged else 0)
    return s["kv"]


def _workspace(s, nbytes):
    if "ws" not in s:
        s["ws"] = torch.empty(max(nbytes(), 16), dtype=torch.uint8, device="cuda")
    return s["ws"].data_ptr(), s["ws"].numel()


def _own_run(s):
    _, L = _lib()
    c, kv = s["case"], _kv(s)
    if c["kind"] == "pages":
        L.kv_copy_pages_dev(kv, c["layers"], 0, s["src"], s["dst"])
        return [s["k"], s["v"]]
    ntok = sum(s["fresh"])
    if c["kind"] == "append":
        L.kv_append_dev(kv, c["seqs"], s["start"].data_ptr(), ntok, TYPES[c["src"]][1], s["nk"].data_ptr(), 0, s["nv"].data_ptr(), 0)
        return [s["k"], s["v"]]
    t, scale = TYPES[c["q"]][1], c["dim"] ** -0.5
    if c["kind"] == "decode":
        ws = _workspace(s, lambda: L.attn_decode_workspace(kv, c["seqs"], c["heads"]))
        L.attn_decode_dev(kv, c["seqs"], c["heads"], t, s["q"].data_ptr(), 0, scale, c["window"], s["out"].data_ptr(), 0, *ws)
    else:
        ws = _workspace(s, lambda: L.attn_prompt_workspace(kv, c["seqs"], ntok, c["heads"], t))
        L.attn_prompt_dev(kv, c["seqs"], s["start"].data_ptr(), ntok, c["heads"], t, s["q"].data_ptr(), 0, scale, c["window"],
                          s["out"].data_ptr(), 0, *ws)
    return s["out"]


def run(s):
    if own:
        return _own_run(s)
    return {"append": _plain_append, "decode": _plain_attention, "prompt": _plain_attention, "pages": _plain_pages}[s["case"]["kind"]](s)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    c = case
    es = {"f32": 4, "f16": 2, "bf16": 2}
    if c["kind"] == "pages":
        return {"bytes": 2 * 2 * c["moved"] * c["layers"] * c["kv"] * c["page"] * c["dim"] * 2, "flops": 0}
    total, fresh = _lengths(c, 0)
    if c["kind"] == "append":
        return {"bytes": 2 * sum(fresh) * c["kv"] * c["dim"] * (es[c["src"]] + 2), "flops": 0}
    w = c["window"] or 1 << 30
    pairs = sum(min(p + 1, w) for n, f in zip(total, fresh) for p in range(n - f, n))
    read = sum(min(n, f + w - 1) for n, f in zip(total, fresh))
    return {"bytes": 2 * read * c["kv"] * c["dim"] * 2 + 2 * sum(fresh) * c["heads"] * c["dim"] * es[c["q"]],
            "flops": 4 * pairs * c["heads"] * c["dim"]}


# ---- in 64 bits ------------------------------------------------------------------------------------------------------
def exact(case, seed):
    """sequence by sequence and head by head from the definition"""
    s = prepare(case, seed)
    c = case
    if c["kind"] == "pages":
        got = []
        for x in (s["k"], s["v"]):
            y = x.double()
            for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
                y[:, b] = x[:, a].double()
            got.append(y)
        return got
    table, page = s["table"].cpu().numpy(), c["page"]
    t = 0
    if c["kind"] == "append":
        got = [s["k"].double(), s["v"].double()]
        for b, (n, f) in enumerate(zip(s["total"], s["fresh"])):
            for j in range((n - f) // page, -(-n // page)):
                lo, hi = max(n - f, j * page), min(n, (j + 1) * page)
                for y, x in zip(got, (s["nk"], s["nv"])):
                    y[int(table[b, j]), :, lo - j * page: hi - j * page] = x[t + lo - n + f: t + hi - n + f].double().transpose(0, 1)
            t += f
        return got
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    G = c["heads"] // c["kv"]
    for b, (n, f) in enumerate(zip(s["total"], s["fresh"])):
        pages = [int(x) for x in table[b, : -(-n // page)]]
        pos = torch.arange(n - f, n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")
        seen = (key <= pos) & (key > pos - (c["window"] or n + 1))
        for h in range(c["heads"]):
            k = s["k"][pages, h // G].reshape(-1, c["dim"])[:n].double()
            v = s["v"][pages, h // G].reshape(-1, c["dim"])[:n].double()
            z = torch.where(seen, (s["q"][t: t + f, h].double() @ k.t().contiguous()) / c["dim"] ** 0.5, -torch.inf)
            out[t: t + f, h] = torch.softmax(z, dim=1) @ v
        t += f
    return out
