"""The page operators of the 8-bit cache one sequence after the other in plain Python, and the packing of tokens in 64 bits (for
the tests; written from the definitions)."""
import torch

BLOCK = 64


def blocks_of(n):
    return (n + BLOCK - 1) // BLOCK


class Pages:
    """refs, table, lens as lists."""

    def __init__(self, pages, sequences, blocks):
        self.refs, self.table, self.lens, self.blocks = [0] * pages, [[-1] * blocks for _ in range(sequences)], [0] * sequences, blocks

    def fork(self, parent):
        old, lens = [list(r) for r in self.table], list(self.lens)
        for b, p in enumerate(parent):
            if p == b:
                continue
            for page in old[b]:
                if page >= 0:
                    self.refs[page] -= 1
            n = blocks_of(lens[p]) if p >= 0 else 0
            self.table[b] = (old[p][:n] if p >= 0 else []) + [-1] * (self.blocks - n)
            for page in self.table[b]:
                if page >= 0:
                    self.refs[page] += 1
            self.lens[b] = lens[p] if p >= 0 else 0

    def reserve(self, count):
        B = len(self.lens)
        free = [p for p, n in enumerate(self.refs) if n == 0]
        granted, copies, refused = [0] * B, [[-1] * B, [-1] * B], False
        for b, n in enumerate(count):
            a, z = self.lens[b] // BLOCK, blocks_of(self.lens[b] + n)
            if n <= 0 or z > self.blocks:
                continue
            row = self.table[b]
            shared = self.lens[b] % BLOCK > 0 and self.refs[row[a]] > 1
            want = [a] * shared + [j for j in range(a, z) if row[j] < 0]
            refused |= len(want) > len(free)
            if refused:
                continue
            granted[b] = n
            for j in want:
                if row[j] >= 0:
                    copies[0][b], copies[1][b] = row[j], free[0]
                    self.refs[row[j]] -= 1
                row[j] = free.pop(0)
                self.refs[row[j]] = 1
        return granted, copies

    def free(self, keep):
        for b, n in enumerate(keep):
            self.lens[b] = min(self.lens[b], max(n, 0))
            for j in range(blocks_of(self.lens[b]), self.blocks):
                if self.table[b][j] >= 0:
                    self.refs[self.table[b][j]] -= 1
                    self.table[b][j] = -1


def packed(cells, scale, row, index, transposed):
    """Blocks of the tokens index (a list) of the sequence whose pages row names: [(int8 cells (heads, 64, D) or (heads, D, 64), scale
    (heads,))]. The integers are those of FP32 with one rounding per operation, as the definition has them."""
    heads = cells.shape[1]
    out = []
    for i in range(0, len(index), BLOCK):
        part = index[i:i + BLOCK]
        pages, slots = [int(row[t // BLOCK]) for t in part], [t % BLOCK for t in part]
        s = torch.stack([scale[p] for p in pages]).float()                    # (tokens, heads)
        top = s.amax(0)
        ratio = s / torch.where(top > 0, top, torch.ones_like(top))
        new = torch.zeros(heads, BLOCK, cells.shape[3] if not transposed else cells.shape[2], device=cells.device)
        for j, (p, t) in enumerate(zip(pages, slots)):
            x = cells[p, :, :, t] if transposed else cells[p, :, t]
            new[:, j] = (x.float() * ratio[j][:, None]).round()
        out.append(((new.transpose(1, 2) if transposed else new).to(torch.int8), top))
    return out
