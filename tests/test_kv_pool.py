"""CPU tests of the key-value cache's host side: a pool's bookkeeping (es_hip_kv_pool_* and es_hip_kv_seq_*, nlayers = 0) against
a plain model of sequences, shared pages and copies before writing, its refusals, and the argument checks of the device
calls, with the HIP calls answered by a stub."""
import json
import os
import subprocess
import sys

import numpy as np
import pytest

import es_hip_quant as E

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Model:
    """what a pool must do: every token is a name; a page holds names; sequences list pages"""

    def __init__(self, page, npages, max_seqs, max_pages):
        self.page, self.npages, self.max_seqs, self.max_pages = page, npages, max_seqs, max_pages
        self.seqs = {}     # number -> [length, pages]

    def refs(self):
        c = {}
        for _, pages in self.seqs.values():
            for g in pages:
                c[g] = c.get(g, 0) + 1
        return c

    def free(self):
        used = self.refs()
        return [g for g in range(self.npages) if g not in used]

    def create(self):
        s = next((i for i in range(self.max_seqs) if i not in self.seqs), None)
        if s is not None:
            self.seqs[s] = [0, []]
        return s

    def extend(self, seqs, n):
        """the copies made, or None: too few pages; ValueError: refused"""
        if len(set(seqs)) < len(seqs) or any(s not in self.seqs for s in seqs):
            raise ValueError
        if any(k < 0 or self.seqs[s][0] + k > self.max_pages * self.page for s, k in zip(seqs, n)):
            raise ValueError
        before = {s: [v[0], list(v[1])] for s, v in self.seqs.items()}
        copies = []
        for s, k in zip(seqs, n):
            q = self.seqs[s]
            for i in range(k):
                if (q[0] + i) % self.page == 0 or i == 0 and self.refs()[q[1][-1]] > 1:
                    if not self.free():
                        self.seqs = before
                        return None
                    g = self.free()[0]
                    if (q[0] + i) % self.page:
                        copies.append((q[1][-1], g))
                        q[1][-1] = g
                    else:
                        q[1].append(g)
            q[0] += k
        return copies

    def fork(self, s):
        f = next((i for i in range(self.max_seqs) if i not in self.seqs), None)
        if f is not None:
            self.seqs[f] = [self.seqs[s][0], list(self.seqs[s][1])]
        return f

    def truncate(self, s, n):
        self.seqs[s] = [n, self.seqs[s][1][:-(-n // self.page)]]


def same(pool, model):
    for s in range(model.max_seqs):
        if s in model.seqs:
            assert pool.len(s) == model.seqs[s][0]
            assert pool.pages(s) == model.seqs[s][1]
        else:
            with pytest.raises(E.EsHipError):
                pool.len(s)
    assert pool.free_pages() == len(model.free())


@pytest.mark.parametrize("seed", range(8))
def test_pool_follows_the_model(hiplib, seed):
    rng = np.random.default_rng(seed)
    page, npages, max_seqs, max_pages = [(16, 20, 6, 7), (32, 9, 4, 20), (16, 200, 12, 40), (64, 5, 3, 2)][seed % 4]
    pool, m = E.KvPool(hiplib, E.F16, 0, 2, 64, page, npages, max_seqs, max_pages), Model(page, npages, max_seqs, max_pages)
    refused = busy = shared = 0
    for _ in range(400):
        live = sorted(m.seqs)
        op = rng.integers(0, 12)
        if op == 0 or not live:
            want = m.create()
            if want is None:
                with pytest.raises(E.EsHipError) as e:
                    pool.create()
                assert e.value.code == E.EBUSY
            else:
                assert pool.create() == want
        elif op < 6:
            seqs = [int(x) for x in rng.choice(live, size=rng.integers(1, len(live) + 1), replace=False)]
            n = [int(x) for x in rng.integers(0, 2 * page, size=len(seqs))]
            if rng.random() < 0.05:
                seqs[-1] = max_seqs
            try:
                want = m.extend(seqs, n)
            except ValueError:
                refused += 1
                with pytest.raises(E.EsHipError) as e:
                    pool.extend(seqs, n)
                assert e.value.code == -2
            else:
                if want is None:
                    busy += 1
                    with pytest.raises(E.EsHipError) as e:
                        pool.extend(seqs, n)
                    assert e.value.code == E.EBUSY
                else:
                    shared += len(want)
                    pool.extend(seqs, n)
        elif op < 8:
            s = int(rng.choice(live))
            want = m.fork(s)
            if want is None:
                with pytest.raises(E.EsHipError) as e:
                    pool.fork(s)
                assert e.value.code == E.EBUSY
            else:
                assert pool.fork(s) == want
        elif op == 8:
            s = int(rng.choice(live))
            n = int(rng.integers(0, m.seqs[s][0] + 1))
            m.truncate(s, n)
            pool.truncate(s, n)
        elif op == 9:
            s = int(rng.choice(live))
            del m.seqs[s]
            pool.free(s)
        else:
            used = m.npages - len(m.free())
            assert pool.compact() == used
            assert sorted({g for s in m.seqs for g in pool.pages(s)}) == list(range(used))
            to = {}
            for s in m.seqs:   # pages are renamed one to one, and those below `used` stay
                new = pool.pages(s)
                assert len(new) == len(m.seqs[s][1])
                for a, b in zip(m.seqs[s][1], new):
                    assert to.setdefault(a, b) == b and (a >= used or a == b)
                m.seqs[s][1] = new
            assert len(set(to.values())) == len(to)
        same(pool, m)
    assert busy or npages > 100
    assert shared
    assert refused
    pool.close()


@pytest.mark.parametrize("args", [
    (E.F32, 0, 2, 64, 16, 4, 2, 2), (7, 0, 2, 64, 16, 4, 2, 2), (E.F16, -1, 2, 64, 16, 4, 2, 2), (E.F16, 0, 0, 64, 16, 4, 2, 2),
    (E.F16, 0, 2, 60, 16, 4, 2, 2), (E.F16, 0, 2, 264, 16, 4, 2, 2), (E.F16, 0, 2, 0, 16, 4, 2, 2), (E.F16, 0, 2, 64, 8, 4, 2, 2),
    (E.F16, 0, 2, 64, 48, 4, 2, 2), (E.F16, 0, 2, 64, 2048, 4, 2, 2), (E.F16, 0, 2, 64, 16, 0, 2, 2), (E.F16, 0, 2, 64, 16, 4, 0, 2),
    (E.F16, 0, 2, 64, 16, 4, 2, 0), (E.F16, 0, 2, 64, 1024, 4, 2, 1 << 21)])
def test_pool_refuses(hiplib, args):
    with pytest.raises(E.EsHipError) as e:
        E.KvPool(hiplib, *args)
    assert e.value.code == -2


def test_pool_refuses_what_a_sequence_cannot_do(hiplib):
    p = E.KvPool(hiplib, E.BF16, 0, 2, 64, 16, 8, 3, 4)
    s = p.create()
    for bad in (lambda: p.extend([s, s], [1, 1]), lambda: p.extend([s], [-1]), lambda: p.extend([s], [65]), lambda: p.extend([1], [1]),
                lambda: p.truncate(s, 1), lambda: p.truncate(s, -1), lambda: p.fork(2), lambda: p.free(-1), lambda: p.view(0)):
        with pytest.raises(E.EsHipError) as e:
            bad()
        assert e.value.code == -2
    p.extend([s], [64])
    assert p.len(s) == 64 and p.free_pages() == 4
    p.free(s)
    assert p.free_pages() == 8
    with pytest.raises(E.EsHipError):
        p.len(s)


def test_a_device_pool_needs_a_device(hiplib):
    if hiplib.available():
        pytest.skip("a device is present")
    with pytest.raises(E.EsHipError) as e:
        E.KvPool(hiplib, E.F16, 1, 2, 64, 16, 4, 2, 2)
    assert e.value.code == -1


# ---- argument checks and launches, the HIP calls answered by the stub ---------------------------------------------------------
@pytest.fixture(scope="module")
def child(hiplib, tmp_path_factory):
    if not os.path.isdir("/opt/rocm/include/hip"):
        pytest.skip("no HIP headers")
    so = tmp_path_factory.mktemp("stub") / "stub.so"
    subprocess.run(["gcc", "-O2", "-w", "-shared", "-fPIC", "-I/opt/rocm/include", "-o", str(so), os.path.join(ROOT, "tests", "_hip_stub.c")],
                   check=True)
    common = r"""
import ctypes as C, json, os, sys
sys.path.insert(0, os.path.join(ROOT, "stream-_amd"))
import es_hip_quant as E
L, S = E.Lib(), C.CDLL(STUB)
assert L.available(), L.last_error()
counts = (C.c_long * 5).in_dll(S, "counts")
shapes = (C.c_long * 4 * 64).in_dll(S, "shapes")
def kv(**k):
    d = dict(type=E.F16, heads=4, dim=128, page=16, npages=100, k=4096, v=8192, table=4096, len=4096, seq=None, rows=8, max_pages=64)
    d.update(k)
    return E.Kv(*[d[n] for n, _ in E.Kv._fields_])
def code(f, *a):
    try: f(*a)
    except E.EsHipError as e: return e.code
    return 0
"""

    def run(code):
        r = subprocess.run([sys.executable, "-c", f"ROOT, STUB = {ROOT!r}, {str(so)!r}\n" + common + code], capture_output=True, text=True,
                           env=dict(os.environ, LD_PRELOAD=str(so)), timeout=300)
        assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
        return json.loads(r.stdout.splitlines()[-1])

    return run


REFUSE = r"""
out = {}
P = 1 << 20
bad_kv = dict(type=dict(type=2), f32=dict(type=E.F32), heads=dict(heads=0), dim=dict(dim=100), dim0=dict(dim=0), dimbig=dict(dim=264), page=dict(page=8),
              pow2=dict(page=24), npages=dict(npages=0), k=dict(k=None), align=dict(v=8200), table=dict(table=None), len=dict(len=None),
              rows=dict(rows=2), maxp=dict(max_pages=0), far=dict(max_pages=1 << 27), talign=dict(table=4098))
ap = lambda k, nseq=3, start=None, ntok=3, t=E.F32, kk=P, ks=0, v=P, vs=0: code(L.kv_append_dev, k, nseq, start, ntok, t, kk, ks, v, vs)
de = lambda k, nseq=3, heads=32, t=E.F32, q=P, qs=0, sc=0.1, w=0, o=P, os_=0, ws=P, wb=1 << 30: code(L.attn_decode_dev, k, nseq, heads, t, q, qs, sc, w, o, os_, ws, wb)
pr = lambda k, nseq=3, start=P, ntok=9, heads=32, t=E.F32, q=P, qs=0, sc=0.1, w=0, o=P, os_=0, ws=P, wb=1 << 30: code(L.attn_prompt_dev, k, nseq, start, ntok, heads, t, q, qs, sc, w, o, os_, ws, wb)
cp = lambda k, nl=2, lb=0, s=[1, 2], d=[3, 4]: code(L.kv_copy_pages_dev, k, nl, lb, s, d)
for n, b in bad_kv.items():
    out["append " + n], out["decode " + n], out["prompt " + n] = ap(kv(**b)), de(kv(**b)), pr(kv(**b))
    if n in ("type", "heads", "dim", "page", "npages", "k", "align"): out["copy " + n] = cp(kv(**b))
k = kv()
inf, nan = float("inf"), float("nan")
out.update({
 "a ntok": ap(k, ntok=-1), "a no start": ap(k, ntok=4), "a type": ap(k, t=E.BF16), "a k": ap(k, kk=None), "a v": ap(k, v=P + 2), "a stride": ap(k, ks=511),
 "a nseq": ap(k, nseq=-1, ntok=-1), "a start": ap(k, start=P + 2),
 "d heads": de(k, heads=30), "d heads0": de(k, heads=0), "d type": de(k, t=E.BF16), "d q": de(k, q=None), "d o": de(k, o=None), "d align": de(k, q=P + 2),
 "d scale0": de(k, sc=0.0), "d scale-": de(k, sc=-1.0), "d inf": de(k, sc=inf), "d nan": de(k, sc=nan), "d window": de(k, w=-1), "d stride": de(k, os_=4000),
 "d ws": de(k, ws=None), "d small": de(k, wb=16), "d wsalign": de(k, ws=P + 8), "d many": de(kv(seq=4096), nseq=1 << 20),
 "p start": pr(k, start=None), "p ntok": pr(k, ntok=-1), "p salign": pr(k, start=P + 1), "p stride": pr(k, qs=1),
 "p many": pr(k, ntok=1 << 28),
 "c range": cp(k, s=[1, 100]), "c neg": cp(k, d=[-1, 4]), "c twice": cp(k, d=[3, 3]), "c both": cp(k, s=[1, 3]), "c self": cp(k, s=[1], d=[1]),
 "c layers": cp(k, nl=-1), "c layer bytes": cp(k, lb=16), "c odd": cp(k, lb=(1 << 30) + 8),
})
launched = counts[0]
fine = {"append": ap(k), "same type": ap(k, t=E.F16), "decode": de(k), "prompt": pr(k), "copy": cp(k), "none": ap(k, ntok=0, start=P), "empty": de(k, nseq=0),
        "no copy": cp(k, s=[], d=[]), "no layers": cp(k, nl=0), "short": code(L.attn_decode_dev, kv(max_pages=32), 3, 32, E.F32, P, 0, 0.1, 0, P, 0, None, 0)}
print(json.dumps({"bad": out, "launched": launched, "fine": fine, "after": [counts[i] for i in range(5)]}))
"""


def test_refusals(child):
    got = child(REFUSE)
    assert {k: v for k, v in got["bad"].items() if v != -2} == {}
    assert got["launched"] == 0
    assert set(got["fine"].values()) == {0}
    # append, append, decode + join, prompt + join, copy, a short cache's decode alone: nothing allocated, copied or waited for
    assert got["after"] == [8, 0, 0, 0, 0]


GRIDS = r"""
P = 1 << 20
rows = []
def one(f, *a):
    n = counts[0]
    f(*a)
    return [[shapes[(n + i) % 64][j] for j in range(4)] for i in range(counts[0] - n)]
for nseq, heads, kvh, maxp, ntok in [(1, 32, 4, 8, 1), (1, 32, 4, 8192, 1), (48, 14, 2, 400, 48), (600, 32, 8, 64, 600), (2, 71, 1, 64, 2),
                                     (3, 32, 32, 33, 3)]:
    k = kv(heads=kvh, rows=nseq, max_pages=maxp)
    ws = L.attn_decode_workspace(k, nseq, heads)
    rows.append(["decode", nseq, heads, kvh, maxp * 16, ws, one(L.attn_decode_dev, k, nseq, heads, E.F32, P, 0, 0.1, 0, P, 0, P, ws)])
for nseq, heads, kvh, maxp, ntok, t in [(1, 32, 4, 500, 64, E.F16), (1, 32, 4, 1024, 16384, E.F16), (8, 32, 8, 210, 9000, E.F16), (5, 14, 2, 100, 5, E.F16),
                                        (1, 32, 4, 500, 64, E.BF16), (5, 14, 2, 100, 5, E.BF16), (40, 14, 2, 100, 70, E.BF16)]:
    k = kv(heads=kvh, rows=nseq, max_pages=maxp, type=t)   # (a CU holds one workgroup with a bf16 cache, else two)
    ws = L.attn_prompt_workspace(k, nseq, ntok, heads, E.F32)
    pairs = [t == E.F16]
    rows.append(["prompt", nseq, heads, kvh, ntok, ws, one(L.attn_prompt_dev, k, nseq, P, ntok, heads, E.F32, P, 0, 0.1, 0, P, 0, P, ws)] + pairs)
print(json.dumps(rows))
"""


def test_every_part_has_room(child):
    """for any lengths: a prompt's parts never outnumber the grid, nor their sums the workspace; a decode call's blocks are dealt
    out whole, each group begins at most one tile that others go on with, and the workspace holds two parts a group"""
    for kind, nseq, heads, kvh, tokens, ws, launches, *pairs in child(GRIDS):
        pairs = pairs == [True]
        G = heads // kvh
        grid = launches[0][0]
        assert grid % kvh == 0
        rng = np.random.default_rng(1)
        for _ in range(200):
            if kind == "decode":
                assert len(launches) == (2 if ws else 1)
                groups, tiles = grid // kvh, -(-G // 16)
                assert (ws > 0) == (tokens > 512)
                blocks = np.repeat(np.maximum(1, -(-rng.integers(0, tokens + 1, nseq) // (128 if ws else 512))), tiles)
                at = np.concatenate([[0], np.cumsum(blocks)])
                each = -(-at[-1] // groups)
                a, b = at[:-1] // each, (at[1:] - 1) // each
                assert b.max() < groups
                begun = a[b > a]
                assert len(set(begun)) == len(begun)
                if ws:
                    assert ws >= 2 * groups * kvh * 16 * (128 + 2) * 4
                else:
                    assert not len(begun)
                continue
            cut = np.sort(rng.integers(0, tokens + 1, nseq - 1))
            n, span = np.diff(np.concatenate([[0], cut, [tokens]])), rng.integers(0, 1 << 20, nseq)
            tiles = -(-n * G // 128)
            assert len(launches) == (2 if ws else 1)
            if ws:   # the chunk that the device takes: total work over the parts aimed for, longer until the last chunks have room
                target = grid // kvh - (tokens * G // 128 + nseq)
                step = 128 if pairs else 64
                rounded = lambda keys: max(128, -(-keys // step) * step)
                if nseq == 1:
                    chunk = int(span[0] / max(1, target // max(1, int(tiles[0]))) + 64) // 64 * 64
                    chunk = max(128, chunk * 2 if pairs and chunk <= 384 else chunk)
                else:
                    chunk = rounded(-(-int((tiles * span).sum()) // target))
                    for _ in range(0 if pairs else 8):
                        n = int((tiles * np.maximum(1, -(-span // chunk))).sum())
                        if n <= target:
                            break
                        chunk = max(chunk + 64, rounded(chunk * n // target))
                if (span * (tiles > 0)).max() <= chunk + 512:
                    chunk = 1 << 30
                parts = (tiles * np.maximum(1, -(-span // chunk))).sum()
                assert ws >= parts * kvh * 128 * (128 + 2) * 4
            else:
                parts = tiles.sum()
            assert parts * kvh <= grid
