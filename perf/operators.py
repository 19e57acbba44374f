"""Operators of a streaming policy's memory, with their plain forms and the cases they are timed on.

A policy that acts from a stream of camera frames keeps the keys and values of past frames. Three operators serve it:

  rotary   rotary positions with one to four axes (time, height, width, camera) on the heads of a projection's output
  append   new keys (rotated on the way) and values written into a paged cache held in 8 bits, with one scale for each
           block of 64 tokens and head; the pass also reads the touched tokens back as the values they stand for
  attend   attention of new queries over that cache, for single tokens, for a frame's tokens and for whole prompts

The cache. K is (pages, kv_heads, 64, D) int8, V is (pages, kv_heads, D, 64) int8, their scales (pages, kv_heads) FP32. A
page is one block of 64 tokens; table (B, blocks) int32 names the page of each block of each sequence.

Append, for the tokens of one call in one block and head: s = max(s_old, max|x| / 127), s_old = 0 for a block that begins in
this call; q = clamp(rint(x * (1 / s)), -127, 127); older tokens of the block, when s > s_old, q' = rint(q * (s_old * (1 / s))).
A block whose s would be below 2^-120 is held as zeros with s = 0.
"""
import math

import torch

own = False

BLOCK = 64
DTYPES = {'bf16': torch.bfloat16, 'f16': torch.float16, 'f32': torch.float32}
BYTES = {'bf16': 2, 'f16': 2, 'f32': 4}
POSITIONS = 20000          # rows of the cosine / sine tables
AXES = {1: (1,), 2: (1, 1), 3: (2, 3, 3), 4: (1, 1, 1, 1)}       # shares of the frequencies by axis


# --------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one new token of one robot's language model (32 query heads of 64): latency only
        dict(name='rotary_token', op='rotary', B=1, T=1, heads=32, D=64, axes=3, pairs=False, dtype='bf16'),
        # two camera frames and an instruction (160 tokens) of eight robots, queries and keys in one tensor
        dict(name='rotary_frames', op='rotary', B=8, T=160, heads=40, D=64, axes=3, pairs=False, dtype='bf16'),
        # a recorded episode of odd length, heads of 128, the adjacent-pair layout, FP16
        dict(name='rotary_episode', op='rotary', B=2, T=8191, heads=32, D=128, axes=3, pairs=True, dtype='f16'),
        # one generated token of each of eight robots, in the middle of a block
        dict(name='append_token', op='append', B=8, T=1, kv_heads=8, D=64, axes=3, ragged=False, start=1003, dtype='bf16'),
        # a frame's tokens of eight robots, ragged, starting inside a block
        dict(name='append_frames', op='append', B=8, T=160, kv_heads=8, D=64, axes=3, ragged=True, start=437, dtype='bf16'),
        # whole episodes ingested at once, heads of 128
        dict(name='append_episode', op='append', B=4, T=8192, kv_heads=8, D=128, axes=3, ragged=False, start=0, dtype='f16'),
        # one token over a short prefix (the policy's own 160 tokens and a few generated ones)
        dict(name='attend_token', op='attend', B=1, T=1, heads=32, kv_heads=8, D=64, length=203, ragged=False, causal=True, dtype='bf16'),
        # one token of each of 32 robots with memories of very different lengths
        dict(name='attend_tokens', op='attend', B=32, T=1, heads=32, kv_heads=8, D=64, length=8191, ragged=True, causal=True, dtype='bf16'),
        # one token of four robots over a long episode (about 130,000 tokens each)
        dict(name='attend_long', op='attend', B=4, T=1, heads=32, kv_heads=8, D=64, length=131037, ragged=False, causal=True, dtype='bf16'),
        # the action head: 17 tokens of 32 heads of 48 over the 160 features of each of 32 robots, not causal
        dict(name='attend_actions', op='attend', B=32, T=17, heads=32, kv_heads=32, D=48, length=160, ragged=False, causal=False, dtype='bf16'),
        # one robot's new frame (160 tokens) over its memory of about a hundred frames
        dict(name='attend_frame', op='attend', B=1, T=160, heads=32, kv_heads=8, D=64, length=16411, ragged=False, causal=True, dtype='bf16'),
        # two prompts of 4096 new tokens after a short memory, heads of 128
        dict(name='attend_prompt', op='attend', B=2, T=4096, heads=32, kv_heads=8, D=128, length=4200, ragged=False, causal=True, dtype='f16'),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(('rotary', 'append', 'attend', 'attend'))
    D = rng.choice((32, 48, 64, 80, 96, 128))
    axes = rng.choice((1, 2, 3, 4))
    if op == 'rotary':
        heads = rng.choice((1, 8, 16, 24, 32, 40))
        most = 2 * 8191 * 32 * 128 // (heads * D)
        B = _log(rng, 1, min(32, most))
        return dict(op=op, B=B, T=_log(rng, 1, min(8191, max(1, most // B))), heads=heads, D=D, axes=axes, pairs=rng.random() < 0.5,
                    dtype=rng.choice(('bf16', 'f16', 'f32') if most > 40000 else ('bf16', 'f16')))
    if op == 'append':
        kv_heads = rng.choice((1, 2, 8, 16, 32))
        most = 4 * 8192 * 8 * 128 // (kv_heads * D)
        B = _log(rng, 1, 32)
        return dict(op=op, B=B, T=_log(rng, 1, min(8192, max(1, most // B - BLOCK))), kv_heads=kv_heads, D=D, axes=rng.choice((0, axes)),
                    ragged=rng.random() < 0.5, start=_log(rng, 1, 4000) - 1, dtype=rng.choice(('bf16', 'f16')))
    kv_heads = rng.choice((1, 4, 8, 16))
    group = rng.choice((1, 2, 4, 7, 8))
    heads = kv_heads * group
    causal, ragged, dtype = rng.random() < 0.7, rng.random() < 0.5, rng.choice(('bf16', 'f16'))
    T = 1 if rng.random() < 0.4 else _log(rng, 2, 2048)
    B = _log(rng, 1, 32)
    # no more keys than the longest listed memory, no more bytes than its, no more products than the listed prompts'
    most = min(131037, 4 * 131037 * 8 * 64 // (B * kv_heads * D), 2 * 32 * 128 * 4096 * 2048 // (B * heads * D * T))
    if most < T:
        T = max(1, int(math.sqrt(most)))
    return dict(op=op, B=B, T=T, heads=heads, kv_heads=kv_heads, D=D, length=_log(rng, max(1, T), max(1, T, most)), ragged=ragged,
                causal=causal, dtype=dtype)


def _counts(c):
    """New tokens of each sequence: T, or spread over (T / 2, T] where ragged."""
    B, T = c['B'], c['T']
    return [T - (b * 37 % max(1, T // 2)) if c['ragged'] else T for b in range(B)]


def _lens(c):
    """Tokens in the cache for each sequence, the new ones among them: `length`, or spread down to about a sixteenth."""
    B, T, L = c['B'], c['T'], c['length']
    return [max(T, L // 16 + (L - L // 16) * (b * 7 % B + 1) // B) if c['ragged'] else L for b in range(B)]


def _starts(c):
    return [c['start'] + 29 * b if c['ragged'] else c['start'] for b in range(c['B'])]


def _sections(axes, D):
    share = AXES[axes]
    part = [D // 2 * s // sum(share) for s in share]
    part[-1] += D // 2 - sum(part)
    return tuple(part)


def work(case):
    c = case
    B, T, D = c['B'], c['T'], c['D']
    if c['op'] == 'rotary':
        n = B * T * c['heads'] * D
        return dict(bytes=2 * n * BYTES[c['dtype']] + 4 * c['axes'] * B * T + min(POSITIONS, B * T) * D * 4, flops=3 * n)
    if c['op'] == 'append':
        starts, counts = _starts(c), _counts(c)
        row = c['kv_heads'] * D
        new = sum(counts)
        back = sum(s + n - s // BLOCK * BLOCK for s, n in zip(starts, counts))
        table = min(POSITIONS, new) * D * 4 + 4 * c['axes'] * B * T if c['axes'] else 0
        blocks = sum((s + n + BLOCK - 1) // BLOCK - s // BLOCK for s, n in zip(starts, counts))
        return dict(bytes=new * row * 2 * (BYTES[c['dtype']] + 1) + back * row * 2 + B * _back(c) * row * 2 * BYTES[c['dtype']]
                    + 16 * blocks * c['kv_heads'] + table, flops=8 * new * row)
    lens = _lens(c)
    row = c['kv_heads'] * D
    keys = sum(lens)
    q = B * T * c['heads'] * D
    seen = sum(n * T - (T * (T - 1) // 2 if c['causal'] else 0) for n in lens)
    blocks = sum((n + BLOCK - 1) // BLOCK for n in lens)
    return dict(bytes=2 * keys * row + 8 * blocks * c['kv_heads'] + 4 * blocks + 2 * q * BYTES[c['dtype']], flops=4 * seen * c['heads'] * D)


def _back(c):
    """Tokens read back for each sequence: whole blocks from the first touched one, as many as the widest needs."""
    return BLOCK * max((s + n + BLOCK - 1) // BLOCK - s // BLOCK for s, n in zip(_starts(c), _counts(c)))


# ---------------------------------------------------------------------------------------------------------- the inputs
class State:
    pass


def _positions(c, g):
    """(axes, B, T) int32: frames of 8 x 8 tokens (time, row, column, camera), each sequence from an origin of its own."""
    B, T, A = c['B'], c['T'], c['axes']
    i = torch.arange(T, device='cuda', dtype=torch.int32)
    t = i if A == 1 else i // 64
    kinds = torch.stack((t, i % 64 // 8, i % 8, i // 32 % 2))
    if A == 2:
        kinds = kinds[1:]
    first = torch.randint(0, POSITIONS - T, (A, B, 1), device='cuda', generator=g, dtype=torch.int32)
    return (kinds[:A, None, :] + first).contiguous()


def _tables(D):
    inv = 10000.0 ** (-torch.arange(0, D, 2, device='cuda', dtype=torch.float64) / D)
    ang = torch.arange(POSITIONS, device='cuda', dtype=torch.float64)[:, None] * inv
    return ang.cos().float(), ang.sin().float()


def _rope_inputs(s, c, g):
    s.sections = _sections(c['axes'], c['D'])
    s.cos, s.sin = _tables(c['D'])
    s.pos = _positions(c, g)
    s.axis = torch.repeat_interleave(torch.arange(c['axes'], device='cuda'), torch.tensor(s.sections, device='cuda'))
    s.freq = torch.arange(c['D'] // 2, device='cuda')


def _cache(s, c, g, blocks, B, kv_heads, D):
    """A cache whose blocks lie in shuffled pages, filled with what quantized normal keys and values look like (a few channels
    larger than the rest); one more page that no table names."""
    pages = B * blocks + 1
    s.table = torch.randperm(B * blocks, device='cuda', generator=g).to(torch.int32).view(B, blocks).contiguous()
    chan = 28 * (1 + 0.5 * (torch.rand(D, device='cuda', generator=g) < 0.1))
    s.k = torch.empty(pages, kv_heads, BLOCK, D, device='cuda', dtype=torch.int8)
    s.v = torch.empty(pages, kv_heads, D, BLOCK, device='cuda', dtype=torch.int8)
    s.k.copy_((torch.randn(s.k.shape, device='cuda', generator=g) * chan).round_().clamp_(-127, 127))
    s.v.copy_((torch.randn(s.v.shape, device='cuda', generator=g) * 31).round_().clamp_(-127, 127))
    s.k_scale = 0.02 + 0.03 * torch.rand(pages, kv_heads, device='cuda', generator=g)
    s.v_scale = 0.01 + 0.04 * torch.rand(pages, kv_heads, device='cuda', generator=g)


def _int(v):
    return torch.tensor(v, dtype=torch.int32, device='cuda')


def prepare(case, seed):
    c = case
    g = torch.Generator(device='cuda').manual_seed(seed)
    s = State()
    s.case = c
    B, T, D, dt = c['B'], c['T'], c['D'], DTYPES[c['dtype']]
    if c['op'] == 'rotary':
        s.x = (torch.randn(B, T, c['heads'] * D, device='cuda', generator=g) * 1.5).to(dt)
        s.out = torch.empty_like(s.x)
        _rope_inputs(s, c, g)
    elif c['op'] == 'append':
        counts, starts, row = _counts(c), _starts(c), c['kv_heads'] * D
        s.new_k = (torch.randn(B, T, row, device='cuda', generator=g) * 1.2).to(dt)
        s.new_v = (torch.randn(B, T, row, device='cuda', generator=g) * 0.9).to(dt)
        _cache(s, c, g, max((a + n + BLOCK - 1) // BLOCK for a, n in zip(starts, counts)), B, c['kv_heads'], D)
        s.start, s.count = _int(starts), _int(counts)
        s.begin, s.end = _int([a // BLOCK * BLOCK for a in starts]), _int([a + n for a, n in zip(starts, counts)])
        s.back = _back(c)
        s.pos = None
        if c['axes']:
            _rope_inputs(s, c, g)
        s.out = tuple(torch.empty(B, s.back, row, device='cuda', dtype=dt) for _ in range(2))
    else:
        lens = _lens(c)
        s.q = (torch.randn(B, T, c['heads'] * D, device='cuda', generator=g) * 1.5).to(dt)
        _cache(s, c, g, (max(lens) + BLOCK - 1) // BLOCK, B, c['kv_heads'], D)
        s.lens = _int(lens)
        s.out = torch.empty_like(s.q)
    # what a user's program keeps between calls: the framework's handles of the same tensors
    if own:
        from yanlongvla_b200 import kernels as K
        if hasattr(s, 'cos'):
            s.rope = K.RopeAxes(s.cos, s.sin, s.sections, pairs=c.get('pairs', False))
        else:
            s.rope = None
        if hasattr(s, 'k'):
            s.cache = K.KV8Cache(s.k, s.v, s.k_scale, s.v_scale)
        s.K = K
    return s


# ---------------------------------------------------------------------------------------------------- the plain forms
def _rotated(x, s, pairs):
    """x (B, T, heads, D) FP32 with the positions s.pos."""
    p = s.pos[s.axis].permute(1, 2, 0).long()                       # (B, T, D / 2): the position on each frequency's axis
    cos, sin = s.cos[p, s.freq][:, :, None], s.sin[p, s.freq][:, :, None]
    if pairs:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)


def _append(s, c, x, cells, scale, transposed):
    """The append of x (B, T, heads, D) FP32 into the cells of one cache tensor; returns the touched blocks' values."""
    B, T, H, D = x.shape
    blocks = s.back // BLOCK
    first, off = s.start // BLOCK, s.start % BLOCK
    slot = torch.arange(blocks * BLOCK, device='cuda')
    t = slot - off[:, None]                                          # (B, slots): the call's token that falls into the slot
    fresh = (t >= 0) & (t < s.count[:, None])
    new = torch.gather(x.reshape(B, T, H * D), 1, t.clamp(0, T - 1).long()[:, :, None].expand(-1, -1, H * D))
    new = (new * fresh[:, :, None]).view(B, blocks, BLOCK, H, D)
    block = first[:, None] + torch.arange(blocks, device='cuda')
    touched = fresh.view(B, blocks, BLOCK).any(2)
    page = torch.gather(s.table, 1, block.clamp(max=s.table.shape[1] - 1).long()).long()
    page = torch.where(touched, page, cells.shape[0] - 1)            # untouched: the page that no table names
    older = (torch.arange(blocks, device='cuda') == 0) & (off > 0)[:, None]
    s_old = torch.where(older[:, :, None], scale[page], 0.0)
    s_new = torch.maximum(s_old, new.abs().amax((2, 4)) / 127)
    s_new = torch.where(s_new < 2.0 ** -120, 0.0, s_new)
    inv = torch.where(s_new > 0, 1 / s_new, 0.0)
    q = (new * inv[:, :, None, :, None]).round().clamp(-127, 127)
    held = cells[page].permute(0, 1, 4, 2, 3) if transposed else cells[page].transpose(2, 3)
    held = held.float()                                              # (B, blocks, 64, H, D)
    moved = (held * (s_old * inv)[:, :, None, :, None]).round()
    held = torch.where((s_new > s_old)[:, :, None, :, None], moved, held)
    q = torch.where(fresh.view(B, blocks, BLOCK, 1, 1), q, held)
    cells[page] = (q.permute(0, 1, 3, 4, 2) if transposed else q.transpose(2, 3)).to(torch.int8)
    scale[page] = s_new
    upto = (s.begin[:, None] + slot < s.end[:, None]).view(B, blocks, BLOCK, 1, 1)
    return torch.where(upto, q * s_new[:, :, None, :, None], 0.0).reshape(B, blocks * BLOCK, H * D)


def _plain(s):
    c = s.case
    B, T, D, dt = c['B'], c['T'], c['D'], DTYPES[c['dtype']]
    if c['op'] == 'rotary':
        return _rotated(s.x.float().view(B, T, c['heads'], D), s, c['pairs']).reshape(s.x.shape).to(dt)
    if c['op'] == 'append':
        k, v = (x.float().view(B, T, c['kv_heads'], D) for x in (s.new_k, s.new_v))
        if c['axes']:
            k = _rotated(k, s, False)
        return _append(s, c, k, s.k, s.k_scale, False).to(dt), _append(s, c, v, s.v, s.v_scale, True).to(dt)
    H, G = c['kv_heads'], c['heads'] // c['kv_heads']
    table = s.table.long()
    L = table.shape[1] * BLOCK
    k = (s.k[table].float() * s.k_scale[table][..., None, None]).transpose(1, 2).reshape(B, H, L, D)
    v = (s.v[table].float() * s.v_scale[table][..., None, None]).permute(0, 2, 1, 4, 3).reshape(B, H, L, D)
    q = s.q.float().view(B, T, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * T, D)
    score = (q @ k.transpose(2, 3)).mul_(D ** -0.5).view(B, H, G, T, L)
    key = torch.arange(L, device='cuda')
    last = s.lens[:, None] - (T - 1 - torch.arange(T, device='cuda') if c['causal'] else torch.zeros(T, dtype=torch.int64, device='cuda'))
    score.masked_fill_((key >= last[..., None])[:, None, None], -math.inf)       # (B, T, L): keys past the query's own position
    top = score.amax(-1, keepdim=True)
    e = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = e.sum(-1, keepdim=True)
    o = (e.view(B, H, G * T, L) @ v).view(B, H, G, T, D) / torch.where(total == 0, 1.0, total)
    return o.permute(0, 3, 1, 2, 4).reshape(B, T, -1).to(dt)


def run(state):
    s = state
    if not own:
        return _plain(s)
    c = s.case
    if c['op'] == 'rotary':
        return s.K.rope_axes(s.x, s.pos, s.rope, out=s.out)
    if c['op'] == 'append':
        s.K.kv8_append(s.cache, s.new_k, s.new_v, s.table, s.start, count=s.count, rope=s.rope, pos=s.pos)
        return s.K.kv8_read(s.cache, s.table, s.begin, s.end, s.back, out=s.out)
    return s.K.kv8_attention(s.q, s.cache, s.table, s.lens, causal=c['causal'], out=s.out)


# --------------------------------------------------------------------------------------------------- in 64 bits
def _exact_rotated(x, c, s, pairs):
    """x (B, T, heads, D) FP64, frequency by frequency."""
    y = torch.empty_like(x)
    half = c['D'] // 2
    axis = [a for a, n in enumerate(_sections(c['axes'], c['D'])) for _ in range(n)]
    for j in range(half):
        at = s.pos[axis[j]].long()
        cos, sin = s.cos[:, j].double()[at][..., None], s.sin[:, j].double()[at][..., None]
        i0, i1 = (2 * j, 2 * j + 1) if pairs else (j, j + half)
        y[..., i0] = x[..., i0] * cos - x[..., i1] * sin
        y[..., i1] = x[..., i1] * cos + x[..., i0] * sin
    return y


def _exact_append(c, s, x, cells, scale, transposed):
    B, T, H, D = x.shape
    out = torch.zeros(B, _back(c), H, D, dtype=torch.float64, device='cuda')
    for b, (start, count) in enumerate(zip(_starts(c), _counts(c))):
        base = start // BLOCK * BLOCK
        for lo in range(base, start + count, BLOCK):
            a, z = max(lo, start), min(lo + BLOCK, start + count)    # this call's tokens in the block
            new = x[b, a - start:z - start]
            page = int(s.table[b, lo // BLOCK])
            top = new.abs().amax((0, 2)) / 127                      # (H,)
            if a > lo:
                old = scale[page].double()
                top = torch.maximum(top, old)
                held = cells[page].double()
                held = (held.permute(2, 0, 1) if transposed else held.transpose(0, 1))[:a - lo]
                grown = (top > old)[:, None]
                step = torch.where(grown, (held * (old / top)[:, None]).round(), held)
                out[b, lo - base:a - base] = step * top[:, None]
            out[b, a - base:z - base] = (new / top[:, None]).round() * top[:, None]
    return out.view(B, -1, H * D)


def _exact_attention(c, s):
    B, T, H, D, G = c['B'], c['T'], c['kv_heads'], c['D'], c['heads'] // c['kv_heads']
    out = torch.empty(B, T, H, G, D, dtype=torch.float64, device='cuda')
    for b, n in enumerate(_lens(c)):
        pages = s.table[b, :(n + BLOCK - 1) // BLOCK].long()
        for h in range(H):
            k = (s.k[pages, h].double() * s.k_scale[pages, h].double()[:, None, None]).reshape(-1, D)[:n]
            v = (s.v[pages, h].double() * s.v_scale[pages, h].double()[:, None, None]).transpose(1, 2).reshape(-1, D)[:n]
            q = s.q[b].double().view(T, H, G, D)[:, h]
            step = max(1, 1 << 26 >> max(0, (G * n).bit_length() - 1))
            for t in range(0, T, step):
                score = torch.einsum('tgd,kd->tgk', q[t:t + step], k) / math.sqrt(D)
                if c['causal']:
                    at = torch.arange(n, device='cuda')[None] > n - T + torch.arange(t, min(T, t + step), device='cuda')[:, None]
                    score = score.masked_fill(at[:, None], -math.inf)
                out[b, t:t + step, h] = torch.einsum('tgk,kd->tgd', torch.softmax(score, -1), v)
    return out.view(B, T, -1)


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    B, T, D = c['B'], c['T'], c['D']
    if c['op'] == 'rotary':
        return _exact_rotated(s.x.double().view(B, T, c['heads'], D), c, s, c['pairs']).view(s.x.shape)
    if c['op'] == 'append':
        k, v = (x.double().view(B, T, c['kv_heads'], D) for x in (s.new_k, s.new_v))
        if c['axes']:
            k = _exact_rotated(k, c, s, False)
        return _exact_append(c, s, k, s.k, s.k_scale, False), _exact_append(c, s, v, s.v, s.v_scale, True)
    return _exact_attention(c, s)
