"""How a decode call's blocks of keys are dealt out to workgroups, and which parts its second launch joins: a model of the kernels'
indexing (Deal, attn_decode_kernel and attn_decode_join_kernel in es_hip_attn_kernels.h), by which tests choose sizes and say what those reach."""


class Deal:
    def __init__(self, eight, dim, page, max_pages, kvh, heads, lens, window=0, sinks=0):
        most, nseq = page * max_pages, len(lens)
        per_cu = 3 if eight and dim <= 64 else 2 if dim <= 128 else 1
        self.target = min(max((256 * per_cu if nseq > 1 else 256) // kvh, 1), 512)
        self.block = 512 if most <= 512 else 128
        self.tiles = -(-(heads // kvh) // 16)
        window = 0 if window >= most or sinks >= most else window
        kept = -(-sinks // 64) * 64 if window else 0
        base = [max(0, max(0, n - window) // 64 * 64 - kept) if window else 0 for n in lens]
        self.blocks = [max(1, -(-(n - b) // self.block)) for n, b in zip(lens, base)]
        total = self.tiles * sum(self.blocks)
        self.each = -(-total // self.target)
        self.extra = int(eight and nseq > 1 and 3 * min(self.blocks) <= self.each)
        if self.extra:
            total += self.tiles * nseq
            self.each = -(-total // self.target)
        self.total = total
        self.first = [0]   # of each sequence, and the end
        for b in self.blocks:
            self.first.append(self.first[-1] + self.tiles * (b + self.extra))

    def steps(self):
        """the most steps of 32 keys that one wave takes in a row"""
        return min(max(self.blocks), self.each) * self.block // 128

    def taken(self):
        """what every workgroup does: (workgroup, sequence, tile, first block, blocks, slot in the workspace or None)"""
        out = []
        for group in range(self.target):
            pos, end = group * self.each, min(self.total, (group + 1) * self.each)
            while pos < end:
                seq = next(i for i in range(len(self.blocks)) if pos < self.first[i + 1])
                tile, block = divmod(pos - self.first[seq], self.blocks[seq] + self.extra)
                block -= self.extra
                if block < 0:
                    pos += 1
                    if pos >= end:
                        break
                    block = 0
                here = min(self.blocks[seq] - block, end - pos)
                begins = group == (pos - block) // self.each
                out.append((group, seq, tile, block, here, None if here == self.blocks[seq] else group * 2 + begins))
                pos += here
        return out

    def joined(self):
        """(sequence, tile) -> the slots that are joined, in the order of their keys; nothing where a tile is one part"""
        out = {}
        for seq, n in enumerate(self.blocks):
            for tile in range(self.tiles):
                at = self.first[seq] + tile * (n + self.extra) + self.extra
                first, parts = at // self.each, (at + n - 1) // self.each - at // self.each + 1
                if parts > 1:
                    out[seq, tile] = [(first + i) * 2 + (i == 0) for i in range(parts)]
        return out
