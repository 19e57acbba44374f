"""Operators of a policy whose memory branches and forgets and whose action head reads states of ragged lengths, with their
plain forms and the cases they are timed on.

  cross     attention of the action head's tokens to an encoder's states of another length: several candidates may share an
            observation's states, states end early (lens) or are left out one by one (mask)
  branch    sequences of a paged 8-bit cache continued several ways: fork (share the pages), reserve (pages for new tokens; a
            shared page that is written to is replaced by a page of its own), copy those pages in every layer, read the begun
            blocks back, free the branches again
  compact   tokens of a paged 8-bit cache kept by their numbers and packed into new pages in every layer, then read back

The cache is that of `operators.py`: K (pages, kv_heads, 64, D) int8, V (pages, kv_heads, D, 64) int8, scales (pages, kv_heads)
FP32, table (B, blocks) int32, -1 where a sequence has no page. refs (pages,) int32 counts the table entries that name a page;
0 is a free page, and free pages are given out from the lowest number on, by sequence and block.

Compact: a block's scale is the largest of the scales its tokens come with, q' = rint(q * (s_old / s)).
"""
import math

import torch

own = False

BLOCK = 64
DTYPES = {'bf16': torch.bfloat16, 'f16': torch.float16}


# --------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # the policy's own call: 17 action tokens of one robot, 32 heads of 48, over the 160 states of its prefix
        dict(name='cross_chunk', op='cross', B=1, S=1, T=17, N=160, heads=32, kv_heads=32, D=48, ragged=False, mask=False, dtype='bf16'),
        # the same of 32 robots whose instructions differ in length
        dict(name='cross_chunks', op='cross', B=32, S=1, T=17, N=160, heads=32, kv_heads=32, D=48, ragged=True, mask=False, dtype='bf16'),
        # 16 candidate chunks for each of eight robots, the states shared by a robot's candidates
        dict(name='cross_candidates', op='cross', B=8, S=16, T=17, N=160, heads=32, kv_heads=32, D=48, ragged=True, mask=False, dtype='bf16'),
        # one token of each of four robots over the states of a long episode, grouped heads of 64
        dict(name='cross_token', op='cross', B=4, S=1, T=1, N=16411, heads=32, kv_heads=8, D=64, ragged=True, mask=False, dtype='bf16'),
        # 256 query tokens over the patches of ten images, 16 heads of 72, images and patches left out
        dict(name='cross_images', op='cross', B=2, S=1, T=256, N=2560, heads=16, kv_heads=16, D=72, ragged=False, mask=True, dtype='bf16'),
        # two prompts of 4096 tokens over 4200 states, heads of 128, FP16
        dict(name='cross_prompt', op='cross', B=2, S=1, T=4096, N=4200, heads=32, kv_heads=8, D=128, ragged=True, mask=False, dtype='f16'),
        # one robot's memory (six frames, in the middle of a block) continued three ways by a frame of 160 tokens, 24 layers
        dict(name='branch_robot', op='branch', B=1, S=3, length=1003, new=160, kv_heads=8, D=64, layers=24),
        # 32 robots, eight ways each, memories of very different lengths
        dict(name='branch_fleet', op='branch', B=32, S=8, length=16411, new=160, kv_heads=8, D=64, layers=4),
        # one robot forgets the oldest frames and keeps its instruction: 24 layers
        dict(name='compact_frames', op='compact', B=1, length=1603, keep=0.9, pattern='recent', kv_heads=8, D=64, layers=24),
        # four robots keep about half of their tokens, chosen one by one
        dict(name='compact_chosen', op='compact', B=4, length=16411, keep=0.5, pattern='chosen', kv_heads=8, D=64, layers=8),
        # two long episodes lose their oldest quarter, heads of 128
        dict(name='compact_episode', op='compact', B=2, length=65531, keep=0.75, pattern='recent', kv_heads=8, D=128, layers=4),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(('cross', 'cross', 'branch', 'compact'))
    if op == 'cross':
        D = rng.choice((32, 40, 48, 64, 72, 80, 96, 128))
        kv_heads = rng.choice((1, 2, 8, 16, 32))
        heads = kv_heads * rng.choice((1, 2, 4, 7)) if kv_heads < 32 else 32
        T = 1 if rng.random() < 0.25 else _log(rng, 2, 4096)
        S = rng.choice((1, 1, 3, 16)) if T <= 64 else 1
        B = _log(rng, 1, 32)
        # no more products than the listed prompts, no more rows than theirs, no more states than twice theirs
        most = min(16411, 2 * 32 * 128 * 4096 * 4200 // (B * S * heads * D * T), 4 * 4200 * 8 * 128 // (B * kv_heads * D))
        T = min(T, max(1, 2 * 4096 * 32 * 128 // (B * S * heads * D)))
        return dict(op=op, B=B, S=S, T=T, N=_log(rng, 1, max(1, most)), heads=heads, kv_heads=kv_heads, D=D,
                    ragged=rng.random() < 0.5, mask=rng.random() < 0.4, dtype=rng.choice(('bf16', 'f16')))
    D, kv_heads, layers = rng.choice((32, 48, 64, 80, 96, 128)), rng.choice((1, 2, 8, 16)), rng.choice((1, 3, 8, 24))
    B = _log(rng, 1, 32)
    if op == 'branch':
        S = rng.choice((1, 2, 3, 8))
        most = min(16411, 32 * 16411 * 8 * 64 * 4 // (B * kv_heads * D * layers))
        return dict(op=op, B=B, S=S, length=_log(rng, 1, max(1, most)), new=_log(rng, 1, 640), kv_heads=kv_heads, D=D, layers=layers)
    most = min(65531, 2 * 65531 * 8 * 128 * 4 // (B * kv_heads * D * layers))
    return dict(op=op, B=B, length=_log(rng, 2, max(2, most)), keep=rng.uniform(0.05, 1.0), pattern=rng.choice(('recent', 'chosen')),
                kv_heads=kv_heads, D=D, layers=layers)


def _lens(c):
    """Lengths of a case's sequences: `length` (N), spread down to about an eighth over the batch."""
    B, L = c['B'], c['N'] if c['op'] == 'cross' else c['length']
    if c['op'] == 'cross' and not c['ragged']:
        return [L] * B
    return [max(1, L // 8 + (L - L // 8) * (b * 5 % B + 1) // B) for b in range(B)]


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _kept(c):
    """Tokens that each sequence keeps."""
    return [max(1, int(n * c['keep'])) for n in _lens(c)]


def _visible(c):
    """States of all sequences that are seen (the mask leaves out about two thirds)."""
    return sum(_lens(c)) // (3 if c['mask'] else 1)


def work(case):
    c = case
    D = c['D']
    row = c['kv_heads'] * D
    if c['op'] == 'cross':
        q = c['B'] * c['S'] * c['T'] * c['heads'] * D
        seen = _visible(c)
        return dict(bytes=4 * seen * row + 4 * q + (c['B'] * c['N'] if c['mask'] else 0), flops=4 * seen * c['S'] * c['T'] * c['heads'] * D)
    if c['op'] == 'branch':
        lens, S = _lens(c), c['S']
        copied = S * sum(n % BLOCK > 0 for n in lens)                       # begun blocks: read, written, read back as BF16
        held = sum(_blocks(n) for n in lens)
        pages = 2 * BLOCK * row + 8 * c['kv_heads']
        return dict(bytes=c['layers'] * copied * (3 * pages + 4 * BLOCK * row) + 8 * held * (1 + S) + 8 * _pool(c), flops=2 * c['layers'] * copied * BLOCK * row)
    kept = sum(_kept(c))
    return dict(bytes=c['layers'] * kept * row * 2 * (3 + 2) + 4 * kept, flops=4 * c['layers'] * kept * row)


def _pool(c):
    """Pages of a branch case's pool: its sequences, room for their branches, and an eighth more."""
    held = sum(_blocks(n) for n in _lens(c))
    more = c['S'] * sum(_blocks(n + c['new']) - n // BLOCK for n in _lens(c))
    return held + more + (held + more) // 8 + 1


# ---------------------------------------------------------------------------------------------------------- the inputs
class State:
    pass


def _int(v):
    return torch.tensor(v, dtype=torch.int32, device='cuda')


def _fill_cache(s, c, g, pages):
    """Every layer's pages in one allocation, filled with what quantized normal keys and values look like."""
    L, H, D = c['layers'], c['kv_heads'], c['D']
    s.pages = pages
    chan = 28 * (1 + 0.5 * (torch.rand(D, device='cuda', generator=g) < 0.1))
    s.k = torch.empty(L * pages, H, BLOCK, D, device='cuda', dtype=torch.int8)
    s.v = torch.empty(L * pages, H, D, BLOCK, device='cuda', dtype=torch.int8)
    step = max(1, (1 << 26) // (H * BLOCK * D))
    for i in range(0, L * pages, step):
        s.k[i:i + step] = (torch.randn(s.k[i:i + step].shape, device='cuda', generator=g) * chan).round_().clamp_(-127, 127)
        s.v[i:i + step] = (torch.randn(s.v[i:i + step].shape, device='cuda', generator=g) * 31).round_().clamp_(-127, 127)
    s.k_scale = 0.02 + 0.03 * torch.rand(L * pages, H, device='cuda', generator=g)
    s.v_scale = 0.01 + 0.04 * torch.rand(L * pages, H, device='cuda', generator=g)
    s.layer_at = (torch.arange(L, device='cuda', dtype=torch.int32) * pages)[:, None, None]


def prepare(case, seed):
    c = case
    g = torch.Generator(device='cuda').manual_seed(seed)
    s = State()
    s.case = c
    B, D, lens = c['B'], c['D'], _lens(c)
    if c['op'] == 'cross':
        dt, N, row = DTYPES[c['dtype']], c['N'], c['kv_heads'] * D
        s.q = (torch.randn(B * c['S'], c['T'], c['heads'] * D, device='cuda', generator=g) * 1.5).to(dt)
        s.kv = torch.randn(B, N, 2 * row, device='cuda', generator=g).to(dt)         # one projection's output, keys and values side by side
        s.lens = _int(lens) if c['ragged'] else None
        s.mask = None
        if c['mask']:                                                                # every other run of 64 states, and a third of the rest
            run = torch.arange(N, device='cuda') // 64 % 2 == 0
            s.mask = run & (torch.rand(B, N, device='cuda', generator=g) < 2 / 3)
        # what lies in padding is left from another use: not always finite
        seen = _seen(s, N)
        s.kv[~seen & (torch.rand(B, N, device='cuda', generator=g) < 0.5)] = math.nan
        s.out = torch.empty_like(s.q)
        s.k, s.v = s.kv[..., :row], s.kv[..., row:]
    elif c['op'] == 'branch':
        S, pages = c['S'], _pool(c)
        _fill_cache(s, c, g, pages)
        rows, blocks = B * (1 + S), max(_blocks(n + c['new']) for n in lens)
        held = [_blocks(n) for n in lens]
        order = torch.randperm(pages, device='cuda', generator=g).to(torch.int32)
        s.table = torch.full((rows, blocks), -1, dtype=torch.int32, device='cuda')
        at = 0
        for b, n in enumerate(held):
            s.table[b, :n] = order[at:at + n]
            at += n
        s.refs = torch.zeros(pages, dtype=torch.int32, device='cuda')
        s.refs[order[:at].long()] = 1
        s.lens = _int(lens + [0] * (B * S))
        s.parent = _int(list(range(B)) + [b for b in range(B) for _ in range(S)])    # the sequences stay, their branches follow
        s.count = _int([0] * B + [c['new']] * (B * S))
        s.keep = _int([1 << 30] * B + [0] * (B * S))
        s.block = torch.arange(blocks, device='cuda', dtype=torch.int32)
    else:
        kept = _kept(c)
        held, want = sum(_blocks(n) for n in lens), sum(_blocks(n) for n in kept)
        _fill_cache(s, c, g, held + want)
        order = torch.randperm(held + want, device='cuda', generator=g).to(torch.int32)
        s.table = torch.full((B, max(_blocks(n) for n in lens)), -1, dtype=torch.int32, device='cuda')
        s.new_table = torch.full((B, max(_blocks(n) for n in kept)), -1, dtype=torch.int32, device='cuda')
        s.index = torch.zeros(B, max(kept), dtype=torch.int32, device='cuda')
        at = 0
        for b, (n, m) in enumerate(zip(lens, kept)):
            s.table[b, :_blocks(n)] = order[at:at + _blocks(n)]
            at += _blocks(n)
            s.new_table[b, :_blocks(m)] = order[at:at + _blocks(m)]
            at += _blocks(m)
            if c['pattern'] == 'recent':                                             # an instruction of up to 32 tokens, and the newest
                first = min(32, m)
                s.index[b, :first] = torch.arange(first, device='cuda')
                s.index[b, first:m] = torch.arange(n - (m - first), n, device='cuda')
            else:
                s.index[b, :m] = torch.randperm(n, device='cuda', generator=g)[:m].sort().values.to(torch.int32)
        s.lens, s.kept = _int(lens), _int(kept)
        s.begin = torch.zeros(c['layers'] * B, dtype=torch.int32, device='cuda')
        s.end = s.kept.repeat(c['layers'])
        s.read_table = (s.new_table + s.layer_at).reshape(c['layers'] * B, -1)
        row = c['kv_heads'] * D
        s.out = tuple(torch.empty(c['layers'] * B, max(kept), row, device='cuda', dtype=torch.bfloat16) for _ in range(2))
    # what a user's program keeps between calls: the framework's handles of the same tensors
    if own:
        from yanlongvla_b200 import kernels as K
        s.K = K
        if c['op'] != 'cross':
            s.whole = K.KV8Cache(s.k, s.v, s.k_scale, s.v_scale)
            P = s.pages
            s.caches = [K.KV8Cache(s.k[i * P:(i + 1) * P], s.v[i * P:(i + 1) * P], s.k_scale[i * P:(i + 1) * P], s.v_scale[i * P:(i + 1) * P])
                        for i in range(c['layers'])]
        if c['op'] == 'branch':
            s.owner = K.KV8Pages(s.refs)
    return s


def _seen(s, N):
    """(B, N) truth values: the states that are there."""
    seen = torch.ones(s.kv.shape[0], N, dtype=torch.bool, device='cuda')
    if s.lens is not None:
        seen &= torch.arange(N, device='cuda') < s.lens[:, None]
    if s.mask is not None:
        seen &= s.mask
    return seen


# ---------------------------------------------------------------------------------------------------- the plain forms
def _plain_cross(s):
    c = s.case
    B, S, T, N, D, H = c['B'], c['S'], c['T'], c['N'], c['D'], c['kv_heads']
    G = c['heads'] // H
    seen = _seen(s, N)
    q = s.q.float().view(B, S, T, H, G, D).permute(0, 3, 1, 2, 4, 5).reshape(B, H, S * T * G, D)
    k = s.k.float().view(B, N, H, D).transpose(1, 2)
    v = s.v.float().masked_fill(~seen[..., None], 0.0).view(B, N, H, D).transpose(1, 2)
    score = (q @ k.transpose(2, 3)).mul_(D ** -0.5)
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    e = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = e.sum(-1, keepdim=True)
    o = (e @ v) / torch.where(total == 0, 1.0, total)
    return o.view(B, H, S, T, G, D).permute(0, 2, 3, 1, 4, 5).reshape(B * S, T, -1).to(s.q.dtype)


def _refer(refs, table, by):
    """refs[p] += by for each entry p of table."""
    flat = table.reshape(-1).long()
    refs.scatter_add_(0, flat.clamp(min=0), (flat >= 0).to(torch.int32) * by)


def _plain_branch(s):
    c = s.case
    # fork: sequence b becomes what parent[b] was, with the pages that hold its tokens
    old, lens = s.table.clone(), s.lens.clone()
    take = s.parent.clamp(min=0).long()
    new_lens = torch.where(s.parent >= 0, lens[take], 0)
    stays = (s.parent == torch.arange(len(take), device='cuda'))[:, None]
    s.table.copy_(torch.where(stays, old, torch.where(s.block < (new_lens[:, None] + BLOCK - 1) // BLOCK, old[take], -1)))
    s.lens.copy_(new_lens)
    _refer(s.refs, old, -1)
    _refer(s.refs, s.table, 1)
    # reserve: pages for the new tokens, and for a begun block that others share
    rows, blocks = s.table.shape
    first, last = s.lens // BLOCK, (s.lens + s.count + BLOCK - 1) // BLOCK            # blocks that the new tokens touch
    begun = (s.lens % BLOCK > 0) & (s.count > 0)
    at = torch.gather(s.table, 1, first.clamp(max=blocks - 1).long()[:, None])[:, 0]
    at = torch.where(begun, at, -1)
    same = (at[:, None] == at) & begun[:, None] & begun                               # writers of one begun page
    writers, is_last = same.sum(1), ~(same & (torch.arange(rows, device='cuda') > torch.arange(rows, device='cuda')[:, None])).any(1)
    held = s.refs[at.clamp(min=0).long()]
    own_page = begun & (held == writers) & is_last                                    # the last of them keeps a page no one else names
    copied = begun & ~own_page
    need = ((s.block >= first[:, None]) & (s.block < last[:, None]) & (s.table < 0) & (s.count > 0)[:, None]) \
        | ((s.block == first[:, None]) & copied[:, None])
    each = need.sum(1)
    upto = each.cumsum(0)
    free = (s.refs == 0).cumsum(0)
    fits = upto <= free[-1]                                                          # behind a sequence that does not fit, none does
    granted = torch.where(fits, s.count, 0).to(torch.int32)
    need &= fits[:, None]
    copied &= fits
    number = (need.reshape(-1).cumsum(0)).view(rows, blocks)                          # the how-manieth free page, from 1
    page = torch.searchsorted(free, number).to(torch.int32)
    fresh = torch.where(need, page, s.table)
    copies = torch.stack((torch.where(copied, at, -1),
                          torch.where(copied, torch.gather(fresh, 1, first.clamp(max=blocks - 1).long()[:, None])[:, 0], -1)))
    _refer(s.refs, copies[0], -1)
    s.table.copy_(fresh)
    _refer(s.refs, torch.where(need, page, -1), 1)
    # copy the pages in every layer; a pair that names none moves the first sequence's first page, which no pair writes, onto itself
    go = copies[0] >= 0
    src, dst = torch.where(go, copies[0], s.table[0, 0]), torch.where(go, copies[1], s.table[0, 0])
    src, dst = (s.layer_at[:, 0] + src).reshape(-1).long(), (s.layer_at[:, 0] + dst).reshape(-1).long()
    for x in (s.k, s.v, s.k_scale, s.v_scale):
        x[dst] = x[src]
    # read the begun blocks back
    tables = s.table + s.layer_at
    page = torch.gather(tables, 2, first.clamp(max=blocks - 1).long()[None, :, None].expand(c['layers'], -1, -1))[..., 0].reshape(-1).clamp(min=0).long()
    slot = torch.arange(BLOCK, device='cuda') < (s.lens - first * BLOCK)[:, None]
    slot = slot.repeat(c['layers'], 1)[..., None, None]
    k = (s.k[page].float() * s.k_scale[page][..., None, None]).transpose(1, 2)
    v = (s.v[page].float() * s.v_scale[page][..., None, None]).permute(0, 3, 1, 2)
    shape = (c['layers'] * rows, BLOCK, -1)
    k, v = (torch.where(slot, x, 0.0).reshape(shape).to(torch.bfloat16) for x in (k, v))
    # free what the branches hold
    gone = s.block >= ((torch.minimum(s.keep, s.lens + granted) + BLOCK - 1) // BLOCK)[:, None]
    gone &= s.table >= 0
    _refer(s.refs, torch.where(gone, s.table, -1), -1)
    s.table.masked_fill_(gone, -1)
    s.lens.copy_(torch.minimum(s.keep, s.lens + granted))
    return granted, copies, tables, k, v, s.refs, s.table, s.lens


def _plain_compact(s):
    c = s.case
    L, B, H, D = c['layers'], c['B'], c['kv_heads'], c['D']
    M, blocks = s.index.shape[1], s.new_table.shape[1]
    slot = torch.arange(blocks * BLOCK, device='cuda')
    live = slot < s.kept[:, None]
    idx = torch.gather(s.index, 1, slot.clamp(max=M - 1)[None].expand(B, -1))
    idx = torch.where(live, idx, 0)
    page, off = torch.gather(s.table, 1, (idx // BLOCK).long()), (idx % BLOCK).long()
    pick = torch.where(live.view(B, blocks, BLOCK).any(2), torch.arange(blocks, device='cuda'), 0)   # an absent block repeats the first
    each = torch.arange(B, device='cuda')[:, None]
    ks, vs = [], []
    for i in range(L):
        src = (page + i * s.pages).long()
        to = torch.gather(s.new_table, 1, pick).long() + i * s.pages
        for cells, scale, out, values in ((s.k, s.k_scale, ks, False), (s.v, s.v_scale, vs, True)):
            x = (cells[src, :, :, off] if values else cells[src, :, off]).float()     # (B, slots, H, D)
            sc = scale[src] * live[..., None]
            top = sc.view(B, blocks, BLOCK, H).amax(2)
            ratio = sc.view(B, blocks, BLOCK, H) / torch.where(top > 0, top, 1.0)[:, :, None]
            q = (x.view(B, blocks, BLOCK, H, D) * ratio[..., None]).round()
            q = torch.where(live.view(B, blocks, BLOCK, 1, 1), q, 0.0)
            cells[to] = (q.permute(0, 1, 3, 4, 2) if values else q.transpose(2, 3)).to(torch.int8)[each, pick]
            scale[to] = top[each, pick]
            out.append((q * top[:, :, None, :, None]).reshape(B, blocks * BLOCK, H * D)[:, :M].to(torch.bfloat16))
    return torch.cat(ks), torch.cat(vs)


def run(state):
    s = state
    c = s.case
    if not own:
        return {'cross': _plain_cross, 'branch': _plain_branch, 'compact': _plain_compact}[c['op']](s)
    K = s.K
    if c['op'] == 'cross':
        return K.cross_attention(s.q, s.k, s.v, c['heads'], c['kv_heads'], lens=s.lens, mask=s.mask, out=s.out)
    if c['op'] == 'branch':
        K.kv8_fork(s.owner, s.table, s.lens, s.parent)
        granted, copies = K.kv8_reserve(s.owner, s.table, s.lens, s.count)
        K.kv8_copy(s.caches, copies)
        tables = s.table + s.layer_at
        begin = (s.lens - s.lens % BLOCK).repeat(c['layers'])
        k, v = K.kv8_read(s.whole, tables.view(-1, tables.shape[2]), begin, s.lens.repeat(c['layers']), BLOCK)
        s.lens += granted
        K.kv8_free(s.owner, s.table, s.lens, s.keep)
        return granted, copies, tables, k, v, s.refs, s.table, s.lens
    K.kv8_compact(s.caches, s.table, s.lens, s.index, s.new_table, kept=s.kept)
    return K.kv8_read(s.whole, s.read_table, s.begin, s.end, s.index.shape[1], out=s.out)


# --------------------------------------------------------------------------------------------------- in 64 bits
def _exact_cross(c, s):
    B, S, T, N, D, H = c['B'], c['S'], c['T'], c['N'], c['D'], c['kv_heads']
    G = c['heads'] // H
    out = torch.zeros(B, S, T, H, G, D, dtype=torch.float64, device='cuda')
    for b, n in enumerate(_lens(c)):
        there = torch.arange(n, device='cuda')
        if s.mask is not None:
            there = there[s.mask[b, :n]]
        if not len(there):
            continue
        for h in range(H):
            k, v = (x[b, there, h * D:(h + 1) * D].double() for x in (s.k, s.v))
            q = s.q.view(B, S * T, H, G * D)[b, :, h].double().reshape(-1, D)
            rows = torch.empty_like(q)
            step = max(1, (1 << 26) // len(there))
            for i in range(0, len(q), step):
                rows[i:i + step] = torch.softmax(q[i:i + step] @ k.T / math.sqrt(D), -1) @ v
            out[b, :, :, h] = rows.view(S, T, G, D)
    return out.view(B * S, T, -1)


def _exact_branch(c, s):
    """The book-keeping sequence by sequence on the host, the values read where the parents hold them."""
    B, S, H, D, L = c['B'], c['S'], c['kv_heads'], c['D'], c['layers']
    table, lens, refs = s.table.tolist(), s.lens.tolist(), s.refs.tolist()
    rows, blocks = len(table), len(table[0])
    origin = [list(r) for r in table]
    end_table, end_refs, end_lens = [list(r) for r in table], list(refs), list(lens)
    for b in range(B, rows):
        table[b], lens[b] = list(table[(b - B) // S]), lens[(b - B) // S]
        for p in table[b]:
            if p >= 0:
                refs[p] += 1
    free = [p for p, n in enumerate(refs) if n == 0]
    granted, copies = [0] * rows, [[-1] * rows, [-1] * rows]
    for b in range(B, rows):
        granted[b] = c['new']
        for j in range(lens[b] // BLOCK, _blocks(lens[b] + c['new'])):
            old = table[b][j]
            if old >= 0:                                             # the begun block: its parent still names it
                copies[0][b], copies[1][b] = old, free[0]
            table[b][j] = free.pop(0)
    tables = torch.tensor(table, device='cuda', dtype=torch.int32)[None] + s.layer_at
    values = []
    for cells, scale, axis in ((s.k, s.k_scale, 2), (s.v, s.v_scale, 3)):
        out = torch.zeros(L, rows, BLOCK, H, D, dtype=torch.float64, device='cuda')
        for b in range(rows):
            a, n = (b if b < B else (b - B) // S), lens[b] % BLOCK
            if n:
                at = torch.arange(L, device='cuda') * s.pages + origin[a][lens[b] // BLOCK]
                x = cells[at].double().movedim(axis, 1)[:, :n]       # (L, n, H, D)
                out[:, b, :n] = x * scale[at].double()[:, None, :, None]
        values.append(out.view(L * rows, BLOCK, H * D))
    dev = [torch.tensor(x, device='cuda', dtype=torch.int32) for x in (granted, copies, end_refs, end_table, end_lens)]
    assert blocks == tables.shape[2]
    return dev[0], dev[1], tables, values[0], values[1], dev[2], dev[3], dev[4]


def _exact_compact(c, s):
    L, B, H, D, M = c['layers'], c['B'], c['kv_heads'], c['D'], s.index.shape[1]
    outs = []
    for cells, scale, values in ((s.k, s.k_scale, False), (s.v, s.v_scale, True)):
        out = torch.zeros(L, B, M, H, D, dtype=torch.float64, device='cuda')
        for b, m in enumerate(_kept(c)):
            idx = s.index[b, :m].long()
            pages, off = s.table[b].long()[idx // BLOCK], idx % BLOCK
            group = torch.arange(m, device='cuda') // BLOCK
            for i in range(L):
                src = pages + i * s.pages
                for h in range(H):
                    x = (cells[:, h][src, :, off] if values else cells[:, h][src, off]).double()
                    sc = scale[src, h].double()
                    top = torch.zeros(_blocks(m), dtype=torch.float64, device='cuda').scatter_reduce(0, group, sc, 'amax')[group]
                    out[i, b, :m, h] = (x * (sc / top)[:, None]).round() * top[:, None]
        outs.append(out.view(L * B, M, H * D))
    return tuple(outs)


def exact(case, seed):
    s = prepare(case, seed)
    return {'cross': _exact_cross, 'branch': _exact_branch, 'compact': _exact_compact}[case['op']](case, s)
