"""Pages of the 8-bit cache: forks, reservations, frees against a sequence-by-sequence model; copies bit for bit; packed tokens
against the definition, integer for integer."""
import random

import pytest
import torch

import pages_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def K():
    from yanlongvla_b200 import kernels
    kernels.device_error()
    return kernels


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device='cuda')


class Both:
    """The kernels and the model side by side."""

    def __init__(self, K, pages, sequences, blocks, refs=None):
        self.K, self.m = K, ref.Pages(pages, sequences, blocks)
        if refs is not None:                                                   # pages that other tables name
            self.m.refs = list(refs)
        self.base = list(self.m.refs)
        self.owner = K.KV8Pages(ints(self.m.refs))
        self.table, self.lens = self.owner.table(sequences, blocks), ints([0] * sequences)

    def check(self):
        assert self.table.tolist() == self.m.table
        assert self.lens.tolist() == self.m.lens
        assert self.owner.refs.tolist() == self.m.refs
        named = list(self.base)
        for row in self.m.table:
            for p in row:
                if p >= 0:
                    named[p] += 1
        assert named == self.m.refs                                            # the model counts what its tables say

    def fork(self, parent):
        self.K.kv8_fork(self.owner, self.table, self.lens, ints(parent))
        self.m.fork(parent)
        self.check()

    def reserve(self, count, advance=True):
        granted, copies = self.K.kv8_reserve(self.owner, self.table, self.lens, ints(count))
        g, c = self.m.reserve(count)
        assert granted.tolist() == g and copies.tolist() == c
        self.check()
        if advance:
            self.lens += granted
            self.m.lens = [a + b for a, b in zip(self.m.lens, g)]
        return g, c

    def free(self, keep):
        self.K.kv8_free(self.owner, self.table, self.lens, ints(keep))
        self.m.free(keep)
        self.check()


@pytest.mark.parametrize('sequences,blocks,pages,seed', [(1, 1, 1, 0), (1, 9, 4, 1), (3, 5, 12, 2), (7, 33, 60, 3), (40, 18, 300, 4), (33, 65, 2000, 5),
                                                         (300, 7, 900, 6), (1030, 4, 2500, 7)])
def test_random_histories(K, sequences, blocks, pages, seed):
    rng = random.Random(seed)
    s = Both(K, pages, sequences, blocks)
    refusals = 0
    for step in range(24):
        kind = rng.choice(('reserve', 'reserve', 'fork', 'free', 'reserved only'))
        if kind == 'fork':
            s.fork([rng.choice((b, b, rng.randrange(sequences), -1 if rng.random() < 0.2 else b)) for b in range(sequences)])
        elif kind == 'free':
            s.free([rng.choice((1 << 30, s.m.lens[b], rng.randrange(s.m.lens[b] + 1), 0)) for b in range(sequences)])
        else:
            count = [rng.choice((0, 1, 63, 64, 65, rng.randrange(1, 200))) for _ in range(sequences)]
            g, _ = s.reserve(count, advance=kind == 'reserve')
            refusals += g != [n if s.m.lens[b] + n <= blocks * 64 or g[b] else 0 for b, n in enumerate(count)]
    K.device_error()


def test_writers_of_one_page(K):
    s = Both(K, 20, 6, 4)
    s.reserve([70, 0, 0, 0, 0, 0])
    s.fork([0, 0, 0, 0, 4, 5])
    g, c = s.reserve([0, 1, 1, 0, 0, 0])                                       # two of four write: both get a page
    assert c[1][1:3] == [2, 3] and g == [0, 1, 1, 0, 0, 0]
    s.fork([0, 0, 0, 0, 0, 0])
    _, c = s.reserve([5] * 6)                                                  # all write: the last keeps the page
    assert c[0][:5] == [1] * 5 and c[0][5] == -1
    s.fork([-1] * 6)
    assert s.m.refs == [0] * 20
    assert K.device_error() == 0


def test_permutation_of_sequences(K):
    s = Both(K, 64, 5, 6)
    s.reserve([10, 100, 200, 300, 0])
    s.fork([3, 0, 4, 1, 2])
    assert s.m.lens == [300, 10, 0, 100, 200]
    s.fork([4, 3, 2, 1, 0])
    assert K.device_error() == 0


def test_shared_page_with_a_refused_writer(K):
    """Of three writers that are all who name a page, the free pages serve one: the page stays with the other two."""
    s = Both(K, 3, 3, 2)
    s.reserve([70, 0, 0])
    s.fork([0, 0, 0])
    g, c = s.reserve([1, 1, 1])
    assert g == [1, 0, 0] and c == [[1, -1, -1], [2, -1, -1]] and s.m.refs == [3, 2, 1]
    assert K.device_error() == 2 and K.device_error() == 0


@pytest.mark.parametrize('pages,offset', [(16384, 0), (16385, 0), (40007, 0), (50000, 3)])
def test_large_pools(K, pages, offset):
    """Free pages far apart, more than one look at 16384 of them, and an address that is no multiple of 16."""
    rng = random.Random(pages)
    refs = [1 if rng.random() < 0.98 else 0 for _ in range(pages)]
    s = Both(K, pages, 50, 40, refs)
    if offset:
        wide = torch.zeros(pages + offset, dtype=torch.int32, device='cuda')
        wide[offset:] = s.owner.refs
        s.owner = K.KV8Pages(wide[offset:])
    for _ in range(3):
        s.reserve([rng.randrange(0, 800) for _ in range(50)])
        s.fork([rng.choice((b, rng.randrange(50))) for b in range(50)])
    K.device_error()


def test_many_sequences(K):
    n = 4096
    s = Both(K, 3 * n, n, 3)
    s.reserve([b % 130 for b in range(n)])
    s.fork([b ^ 1 if b % 3 else b for b in range(n)])
    s.reserve([b % 7 for b in range(n)])
    s.free([b % 90 for b in range(n)])
    K.device_error()


def test_indices_out_of_range(K):
    s = Both(K, 8, 3, 2)
    s.reserve([64, 64, 70])
    K.device_error()
    before = s.table.clone(), s.lens.clone(), s.owner.refs.clone()

    def same():
        return all(torch.equal(a, b) for a, b in zip(before, (s.table, s.lens, s.owner.refs)))
    K.kv8_fork(s.owner, s.table, s.lens, ints([0, 3, 1 << 30]))               # a parent past the sequences: unchanged
    assert K.device_error() == 2 and same()
    g, c = K.kv8_reserve(s.owner, s.table, s.lens, ints([-1, 65, 1 << 30]))   # counts below zero, past the table
    assert K.device_error() == 2 and same() and g.tolist() == [0, 0, 0] and c.tolist() == [[-1] * 3] * 2
    bad = s.lens.clone()
    bad[0], bad[1] = -5, 1 << 30
    K.kv8_reserve(s.owner, s.table, bad, ints([0, 1, 0]))
    assert K.device_error() == 2 and same()
    s.free([-3, 64, 70])
    assert K.device_error() == 2


# ------------------------------------------------------------------------------------------------ copies
def filled(K, pages, heads, D, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    c = K.KV8Cache.empty(pages, heads, D)
    for t in (c.k, c.v):
        t.copy_(torch.randint(-127, 128, t.shape, device='cuda', generator=g))
    for t in (c.k_scale, c.v_scale):
        t.copy_(torch.rand(t.shape, device='cuda', generator=g) + 0.01)
    return c


def parts(c):
    return c.k, c.v, c.k_scale, c.v_scale


@pytest.mark.parametrize('heads,D,layers', [(1, 32, 1), (8, 64, 3), (3, 48, 2), (5, 80, 2), (16, 128, 2), (2, 96, 130)])
def test_copy(K, heads, D, layers):
    caches = [filled(K, 12, heads, D, i) for i in range(layers)]
    want = [[t.clone() for t in parts(c)] for c in caches]
    pairs = [(0, 3), (0, 5), (7, 11), (-1, 2), (4, -1), (9, 9), (-1, -1)]
    for w in want:
        for t in w:
            for a, b in pairs:
                if a >= 0 and b >= 0:
                    t[b] = t[a]
    K.kv8_copy(caches if layers > 1 else caches[0], ints(pairs).t().contiguous())
    for c, w in zip(caches, want):
        for t, u in zip(parts(c), w):
            assert torch.equal(t, u)
    K.kv8_copy(caches, ints([[12, 0], [0, 1 << 30]]))
    assert K.device_error() == 2
    for c, w in zip(caches, want):
        assert all(torch.equal(t, u) for t, u in zip(parts(c), w))


# ------------------------------------------------------------------------------------------------ compact
def check_compact(K, caches, table, lens, index, new_table, kept):
    """Every page of every layer is what the definition says, those that no new block names what they were."""
    want = [[t.clone() for t in parts(c)] for c in caches]
    B, M = index.shape
    for b in range(B):
        m = M if kept is None else int(kept[b])
        idx = index[b, :m].tolist()
        for w in want:
            for cells, scale, transposed in ((w[0], w[2], False), (w[1], w[3], True)):
                made = ref.packed(cells, scale, table[b].tolist(), idx, transposed)
                for j, (x, s) in enumerate(made):
                    cells[int(new_table[b, j])] = x
                    scale[int(new_table[b, j])] = s
    K.kv8_compact(caches if len(caches) > 1 else caches[0], table, lens, index, new_table, kept=kept)
    for c, w in zip(caches, want):
        for t, u in zip(parts(c), w):
            assert torch.equal(t, u)


@pytest.mark.parametrize('D', [32, 48, 64, 80, 96, 128])
@pytest.mark.parametrize('heads,layers,lens,kept', [(1, 1, [1], [1]), (2, 2, [130, 64, 300], [64, 0, 170]), (3, 1, [70, 200], None)])
def test_compact(K, D, heads, layers, lens, kept):
    rng = random.Random(D)
    held = [ref.blocks_of(n) for n in lens]
    M = max(kept) if kept else 65
    new = [ref.blocks_of(n) for n in (kept or [M] * len(lens))]
    pages = sum(held) + sum(new) + 2
    order = rng.sample(range(pages), pages)
    table, new_table = ([[order.pop() for _ in range(n)] + [-1] * (max(v) - n) for n in v] for v in (held, new))
    caches = [filled(K, pages, heads, D, 10 * i + D) for i in range(layers)]
    caches[0].k_scale[table[-1][0]] = 0.0                                      # a block of zeros
    caches[0].k[table[-1][0]] = 0
    index = [(sorted(rng.sample(range(n), M)) if n >= M and b % 2 == 0 else [rng.randrange(n) for _ in range(M)]) for b, n in enumerate(lens)]
    check_compact(K, caches, ints(table), ints(lens), ints(index), ints(new_table), None if kept is None else ints(kept))
    assert K.device_error() == 0


@pytest.mark.parametrize('index', [list(range(64)), list(range(32, 96)), list(range(63, -1, -1)), [5] * 64, list(range(0, 640, 10)),
                                   list(range(640)), list(range(1, 640, 64)) + [639]])
def test_compact_runs(K, index):
    """Whole blocks, blocks across two and many pages, backwards, one token many times."""
    caches = [filled(K, 30, 2, 64, 3)]
    n = ref.blocks_of(len(index))
    check_compact(K, caches, ints([list(range(10, 20))]), ints([640]), ints([index]), ints([list(range(20, 20 + n))]), None)


def test_whole_blocks_keep_their_integers(K):
    c = filled(K, 4, 2, 64, 5)
    K.kv8_compact(c, ints([[0, 1]]), ints([128]), ints([list(range(128))]), ints([[3, 2]]))
    for t in parts(c):
        assert torch.equal(t[3], t[0]) and torch.equal(t[2], t[1])


def test_compact_numbers_out_of_range(K):
    c = filled(K, 6, 2, 64, 6)
    before = [t.clone() for t in parts(c)]
    K.kv8_compact(c, ints([[0, 7], [1, 2]]), ints([100, 70]), ints([[3, 64, -1], [69, 70, 1 << 30]]), ints([[3], [4]]))
    assert K.device_error() == 2
    assert torch.equal(c.k[3, :, 0], before[0][0, :, 3]) and not c.k[3, :, 1:].any() and not c.v[4, :, :, 1:].any()
    assert torch.equal(c.v[4, :, :, 0], before[1][2, :, :, 5])
    K.kv8_compact(c, ints([[0]]), ints([64]), ints([[1] * 65]), ints([[6]]))       # a page past the cache, a block past the table
    assert K.device_error() == 2
    K.kv8_compact(c, ints([[0]]), ints([64]), ints([[1, 2]]), ints([[5]]), kept=ints([3]))
    assert K.device_error() == 2
    for i in (0, 1, 2):
        assert all(torch.equal(t[i], u[i]) for t, u in zip(parts(c), before))


# ------------------------------------------------------------------------------------------------ together
def test_branches_of_a_memory(K):
    """Fork, reserve, copy, append, read: each branch holds its parent's tokens and its own, the parent stays as it was; the whole of it
    in a CUDA graph, replayed, does the same again."""
    pages, heads, D, blocks = 40, 2, 64, 6
    owner, caches = K.KV8Pages.empty(pages), [K.KV8Cache.empty(pages, heads, D) for _ in range(2)]
    table, lens = owner.table(4, blocks), ints([0] * 4)
    g = torch.Generator(device='cuda').manual_seed(0)
    x = torch.randn(2, 2, 4, 100, heads * D, device='cuda', generator=g, dtype=torch.bfloat16)

    def add(count, new):
        granted, copies = K.kv8_reserve(owner, table, lens, count)
        K.kv8_copy(caches, copies)
        for c, (k, v) in zip(caches, new):
            K.kv8_append(c, k, v, table, lens, count=granted)
        lens.add_(granted)

    def read():
        return [t.clone() for c in caches for t in K.kv8_read(c, table, ints([0] * 4), lens, 200)]

    first, second, parent = ints([100, 0, 0, 0]), ints([0, 30, 100, 0]), ints([0, 0, 0, 3])
    add(first, [(x[0, 0], x[0, 1]), (x[1, 0], x[1, 1])])
    alone = read()
    K.kv8_fork(owner, table, lens, parent)
    for t in read():
        assert torch.equal(t[0], t[1]) and torch.equal(t[0], t[2])
    new = [(x[1, 1], x[0, 0]), (x[0, 1], x[1, 0])]
    add(second, new)
    got = read()
    assert lens.tolist() == [100, 130, 200, 0]
    for t, a, n in zip(got, alone, [t for p in new for t in p]):
        assert torch.equal(t[0], a[0])                                         # the parent
        step = n.float().abs().amax() / 127                                    # a value is off by at most a step and a half: its own
        for b, m in ((1, 30), (2, 100)):                                       # rounding, one more when its block's scale grew; and BF16's
            assert (t[b, 100:100 + m].float() - n[b, :m].float()).abs().max() <= 1.5 * step + 2.0 ** -8 * n.float().abs().amax()
            assert (t[b, :100].float() - a[0, :100].float()).abs().max() <= step + 2.0 ** -7 * a.float().abs().amax()
    # the same in a graph, from the same begin
    state = [t.clone() for t in (owner.refs, table, lens)] + [t.clone() for c in caches for t in parts(c)]
    keep = ints([100, 0, 0, 0])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            K.kv8_free(owner, table, lens, keep)
            K.kv8_fork(owner, table, lens, parent)
            add(second, new)
        for _ in range(3):
            graph.replay()
    torch.cuda.current_stream().wait_stream(stream)
    for a, b in zip(state[:3], (owner.refs, table, lens)):
        assert torch.equal(a, b)
    for a, b in zip(got, read()):
        assert torch.equal(a, b)
    assert K.device_error() == 0


def test_compact_with_pages_of_the_pool(K):
    """The oldest tokens are dropped: new pages from the pool, the old ones back to it, a branch that shares them unharmed."""
    pages, heads, D = 24, 2, 64
    owner, c = K.KV8Pages.empty(pages), K.KV8Cache.empty(pages, heads, D)
    table, lens = owner.table(2, 8), ints([0, 0])
    g = torch.Generator(device='cuda').manual_seed(1)
    k, v = (torch.randn(2, 300, heads * D, device='cuda', generator=g, dtype=torch.bfloat16) for _ in range(2))
    granted, _ = K.kv8_reserve(owner, table, lens, ints([300, 0]))
    K.kv8_append(c, k, v, table, lens, count=granted)
    lens += granted
    K.kv8_fork(owner, table, lens, ints([0, 0]))
    whole = [t.clone() for t in K.kv8_read(c, table, ints([0, 0]), lens, 300)]
    index, kept = ints([[*range(32), *range(192, 300)], [0] * 140]), ints([140, 0])
    new = owner.table(2, 8)
    granted, _ = K.kv8_reserve(owner, new, ints([0, 0]), kept)
    K.kv8_compact(c, table, lens, index, new, kept=granted)
    K.kv8_free(owner, table, lens, ints([0, 1 << 30]))                        # the first row's old pages; the branch holds them
    table[0], lens[0] = new[0], granted[0]
    got = K.kv8_read(c, table, ints([0, 0]), lens, 300)
    for t, w in zip(got, whole):
        assert torch.equal(t[1], w[1])
        step = w.float().abs().amax() / 127
        assert (t[0, :140].float() - w[0, index[0].long()].float()).abs().max() <= 0.5 * step + 2.0 ** -7 * w.float().abs().amax()
    named = torch.bincount(table[table >= 0].long(), minlength=pages).int()
    assert torch.equal(named, owner.refs)
    assert K.device_error() == 0


def test_refusals(K):
    owner, c, other = K.KV8Pages.empty(8), K.KV8Cache.empty(8, 2, 64), K.KV8Cache.empty(8, 2, 32)
    table, lens, more = owner.table(2, 3), ints([0, 0]), ints([0, 0])
    for call in (K.kv8_fork, K.kv8_reserve, K.kv8_free):
        for bad in ((table.long(), lens, more), (table.t(), lens, more), (table[0], lens, more), (table, ints([0]), more), (table, lens, ints([0] * 3)),
                    (table, lens.cpu(), more), (table, lens.float(), more), (table[:0], lens[:0], more[:0])):
            with pytest.raises(K.TcqError):
                call(owner, *bad)
    for bad in (ints([0, 1]), ints([[0, 1]]), ints([[0, 1]] * 3), torch.zeros(2, 2, device='cuda'), ints([[], []])):
        with pytest.raises(K.TcqError):
            K.kv8_copy(c, bad)
    with pytest.raises(K.TcqError, match='one shape'):
        K.kv8_copy([c, other], ints([[0], [1]]))
    for bad in ((table, lens, ints([0]), table), (table, lens, ints([[0]]), table), (table, lens, ints([[0], [0]]), table[:1]),
                (table, ints([0]), ints([[0], [0]]), table)):
        with pytest.raises(K.TcqError):
            K.kv8_compact(c, *bad)
    with pytest.raises(K.TcqError):
        K.kv8_compact(c, table, lens, ints([[0], [0]]), table, kept=ints([1]))
    assert K.device_error() == 0


def test_compact_bad_numbers_next_to_good_ones(K):
    """A token of zeros where the number is past the sequence, the tokens next to it as they are."""
    c = filled(K, 6, 9, 64, 8)                                                 # nine heads: more than a CTA takes at once
    k0, v0 = c.k[0].clone(), c.v[0].clone()
    K.kv8_compact(c, ints([[0]]), ints([60]), ints([[64, 1, 2, 3, 4, 5, 6, 60, 8, 9, 10, 11, -1, 13]]), ints([[3]]))
    assert K.device_error() == 2
    for j in (1, 2, 3, 4, 5, 6, 8, 9, 10, 11, 13):
        assert torch.equal(c.k[3, :, j], k0[:, j]) and torch.equal(c.v[3, :, :, j], v0[:, :, j])
    for j in (0, 7, 12, *range(14, 64)):
        assert not c.k[3, :, j].any() and not c.v[3, :, :, j].any()


def test_compact_rounds_the_product_first(K):
    """rint(fl(q r)), not rint(q r): of some 10^8 products a few tens lie so near a half that the two differ."""
    P, g = 3000, torch.Generator(device='cuda').manual_seed(1)
    c = K.KV8Cache.empty(3 * P, 8, 64)
    for cells, scale in ((c.k, c.k_scale), (c.v, c.v_scale)):
        cells.copy_(torch.randint(-127, 128, cells.shape, device='cuda', generator=g))
        scale.copy_(torch.rand(scale.shape, device='cuda', generator=g) + 0.02)
    at = torch.arange(64, device='cuda')
    index = (2 * torch.arange(P, device='cuda')[:, None] + at // 32) * 64 + at % 32 + 8         # half of each of two pages
    pages = torch.arange(3 * P, device='cuda', dtype=torch.int32)[None]
    K.kv8_compact(c, pages[:, :2 * P].contiguous(), ints([2 * P * 64]), index.view(1, -1).int(), pages[:, 2 * P:].contiguous())
    differ = 0
    for cells, scale, transposed in ((c.k, c.k_scale, False), (c.v, c.v_scale, True)):
        old = scale[:2 * P].view(P, 2, 8)
        ratio = (old / old.amax(1, keepdim=True))[..., None, None]
        q = (cells[:2 * P, :, :, 8:40] if transposed else cells[:2 * P, :, 8:40].transpose(2, 3)).reshape(P, 2, 8, 64, 32)
        got = cells[2 * P:] if transposed else cells[2 * P:].transpose(2, 3)
        got = got.reshape(P, 8, 64, 2, 32).permute(0, 3, 1, 2, 4)
        want = (q.float() * ratio).round()
        assert torch.equal(got.float(), want)
        differ += (want != (q.double() * ratio.double()).round()).sum().item()
    assert differ > 0
