"""CPU test of how decode deals out its blocks (tests/_deal.py, a model of the kernels' indexing): every block is taken once, a workgroup's two
places in the workspace are never written twice, and what is joined is what was written, in order."""
import numpy as np

from _deal import Deal


def test_every_block_is_taken_once_and_joined_once():
    rng = np.random.default_rng(0)
    reached = {0: 0, 1: 0}
    for _ in range(3000):
        nseq = int(rng.choice([1, 2, 3, 7, 40, 64, 65, 150]))
        page, kvh = int(rng.choice([16, 64])), int(rng.choice([1, 2, 8, 64, 128, 300]))
        lens = [int(n) for n in np.exp2(rng.uniform(0, rng.uniform(4, 13), nseq))]
        most = -(-max(lens) // page)
        window, sinks = (int(rng.integers(1, 3000)), int(rng.integers(0, 300))) if rng.random() < 0.4 else (0, 0)
        d = Deal(rng.random() < 0.7, int(rng.choice([16, 80, 256])), page, most, kvh, kvh * int(rng.choice([1, 4, 17, 40])), lens, window, sinks)
        reached[d.extra] += 1
        tiles, slots = {}, {}
        for group, seq, tile, block, here, slot in d.taken():
            tiles.setdefault((seq, tile), []).append((block, here, slot))
            assert slot is None or slots.setdefault(slot, (seq, tile)) == (seq, tile) and here > 0
        parts = d.joined()
        assert len(tiles) == nseq * d.tiles
        written = [p[2] for t in tiles.values() for p in t if p[2] is not None]
        assert len(written) == len(set(written))
        for key, took in tiles.items():
            ends = np.cumsum([0] + [h for _, h, _ in took])
            assert [b for b, _, _ in took] == ends[:-1].tolist() and ends[-1] == d.blocks[key[0]]
            assert [s for _, _, s in took] == parts.get(key, [None])
    assert min(reached.values()) > 300
