"""Streaming-memory operators (rope_axes, kv8_append, kv8_read, kv8_attention) against their definitions in 64 bits.

Tolerances, from the arithmetic:
- rope_axes: FP32 with one rounding per operation, so bit-equal to the same three PyTorch operations; against FP64 the
  error is one rounding to the type plus 3 FP32 roundings of terms no larger than |a| + |b|.
- kv8_append: s = max(s_old, amax / 127) is one FP32 division of an exact maximum (or a rotated one, 3 roundings); the integers
  are rint of a value with at most 3 FP32 roundings, so they lie within 1/2 + 127 * 2^-22 of x / s.
- kv8_read: q * s with one FP32 rounding and one to the type: bit-equal to PyTorch.
- kv8_attention: the softmax weights reach the second product in FP16 (2^-11 relative), their FP32 exponent adds less than
  2^-13; so |o - o64| <= 2^-10 sum_j p_j |v_j| + half an ulp of the output type (2^-8 |o| BF16, 2^-11 |o| F16), a factor of
  almost 2 in hand on the first term.
"""
import pytest
import torch

import memory_ref as ref

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (BF16, F16, F32)}        # 2^-8, 2^-11, 2^-24: rounding to nearest


@pytest.fixture(scope='module')
def K():
    if not torch.cuda.is_available():
        pytest.skip('no CUDA device')
    from yanlongvla_b200 import kernels
    kernels.device_error(reset=True)
    yield kernels
    assert kernels.device_error(reset=True) == 0


def gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device='cuda')


# ------------------------------------------------------------------------------------------------ rope_axes
def rope_case(K, D, axes, T, B, g, pairs, positions=5000):
    half = D // 2
    cut = sorted(torch.randint(0, half + 1, (axes - 1,), generator=torch.Generator().manual_seed(D + axes)).tolist())
    sections = [b - a for a, b in zip([0] + cut, cut + [half])]
    cos, sin = K.RopeAxes.tables(positions, D)
    pos = torch.randint(0, positions, (axes, B, T), device='cuda', generator=g, dtype=torch.int32)
    return K.RopeAxes(cos, sin, sections, pairs=pairs), pos, sections


@pytest.mark.parametrize('pairs', [False, True])
@pytest.mark.parametrize('dtype', [BF16, F16, F32])
@pytest.mark.parametrize('B,T,heads,D,axes', [(1, 1, 32, 64, 3), (2, 161, 5, 64, 2), (3, 33, 1, 72, 2), (1, 7, 3, 6, 1), (2, 5, 2, 20, 4),
                                              (1, 129, 16, 48, 3), (1, 64, 40, 128, 4), (1, 3, 2, 256, 3), (1, 1, 600, 32, 1)])
def test_rope_axes(K, B, T, heads, D, axes, dtype, pairs):
    g = gen(B * 1000 + T + D)
    rope, pos, sections = rope_case(K, D, axes, T, B, g, pairs)
    x = torch.randn(B, T, heads * D, device='cuda', generator=g).to(dtype)
    y = K.rope_axes(x, pos, rope)
    x4 = x.view(B, T, heads, D)
    # the same operations in PyTorch FP32
    axis = torch.repeat_interleave(torch.arange(axes, device='cuda'), torch.tensor(sections, device='cuda'))
    p = pos[axis].permute(1, 2, 0).long()
    j = torch.arange(D // 2, device='cuda')
    c, s = rope.cos[p, j][:, :, None], rope.sin[p, j][:, :, None]
    i0, i1 = (slice(0, None, 2), slice(1, None, 2)) if pairs else (slice(0, D // 2), slice(D // 2, None))
    a, b = x4[..., i0].float(), x4[..., i1].float()
    want = torch.empty_like(x4)
    want[..., i0], want[..., i1] = (a * c - b * s).to(dtype), (a * s + b * c).to(dtype)
    assert torch.equal(y.view_as(x4), want)
    full = ref.rotary(x4.double(), pos, rope.cos, rope.sin, sections, pairs)
    size = torch.empty_like(full)
    size[..., i0] = size[..., i1] = a.double().abs() + b.double().abs()
    assert ((y.view_as(x4).double() - full).abs() <= HALF_ULP[dtype] * full.abs() + 3 * 2.0 ** -24 * size + 2.0 ** -25).all()
    # in place, and the inverse turn
    z = x.clone()
    assert K.rope_axes(z, pos, rope, out=z) is z and torch.equal(z, y)
    back = K.rope_axes(y, pos, rope, inverse=True)
    want = ref.rotary(y.view_as(x4).double(), pos, rope.cos, rope.sin, sections, pairs, inverse=True)
    assert ((back.view_as(x4).double() - want).abs() <= HALF_ULP[dtype] * want.abs() + 4 * 2.0 ** -24 * size + 2.0 ** -25).all()


@pytest.mark.parametrize('pairs', [False, True])
def test_rope_axes_gradient(K, pairs):
    """The inverse turn is the gradient: against autograd of the formula in FP64 and against differences."""
    g = gen(5)
    B, T, heads, D = 2, 9, 3, 32
    rope, pos, sections = rope_case(K, D, 3, T, B, g, pairs)
    x = torch.randn(B, T, heads * D, device='cuda', generator=g)
    w = torch.randn(B, T, heads * D, device='cuda', generator=g)
    grad = K.rope_axes(w, pos, rope, inverse=True)
    xd = x.double().requires_grad_()
    y = ref.rotary(xd.view(B, T, heads, D), pos, rope.cos, rope.sin, sections, pairs)
    want, = torch.autograd.grad((y.reshape(w.shape) * w.double()).sum(), xd)
    assert (grad.double() - want).abs().max() <= 4 * 2.0 ** -24 * w.abs().max() * 2
    for i in (0, 17, 100):
        e = torch.zeros_like(x).view(-1)
        e[i] = 0.5                                                    # the map is linear: a difference of any step is exact
        up, down = (K.rope_axes(x + d * e.view_as(x), pos, rope) for d in (1, -1))
        slope = ((up.double() - down.double()) * w.double()).sum()
        assert abs(slope - grad.view(-1)[i].double()) <= 64 * 2.0 ** -24 * w.abs().max() * 8


def test_rope_axes_strided_and_misaligned(K):
    """Views into a wider projection output, and rows that allow only narrow vectors."""
    g = gen(11)
    B, T, heads, D = 2, 19, 4, 64
    rope, pos, _ = rope_case(K, D, 3, T, B, g, False)
    for width, first in ((1024, 256), (1030, 6), (777, 1)):
        big = torch.randn(B, T, width, device='cuda', generator=g).bfloat16()
        x = big[..., first:first + heads * D]
        want = K.rope_axes(x.contiguous(), pos, rope)
        assert torch.equal(K.rope_axes(x, pos, rope), want)
        keep = big.clone()
        K.rope_axes(x, pos, rope, out=x)
        assert torch.equal(x, want)
        big[..., first:first + heads * D] = keep[..., first:first + heads * D]
        assert torch.equal(big, keep)                                # nothing outside the view was written
    t = torch.randn(T, B, heads * D, device='cuda', generator=g).bfloat16().transpose(0, 1)      # token-major
    assert torch.equal(K.rope_axes(t, pos, rope), K.rope_axes(t.contiguous(), pos, rope))


def test_positions_out_of_range_are_reported(K):
    rope, pos, _ = rope_case(K, 64, 2, 8, 1, gen(1), False)
    x = torch.randn(1, 8, 64, device='cuda').bfloat16()
    bad, near = pos.clone(), pos.clone()
    bad[0, 0, 3], near[0, 0, 3] = 5000, 4999
    bad[1, 0, 5], near[1, 0, 5] = -1, 0
    y = K.rope_axes(x, bad, rope)
    assert K.device_error(reset=True) == 2
    assert torch.equal(y, K.rope_axes(x, near, rope)) and K.device_error(reset=True) == 0


# ------------------------------------------------------------------------------------------------ the cache
def make_cache(K, pages, heads, D, g, zero_scales=False):
    c = K.KV8Cache.empty(pages, heads, D)
    c.k.copy_(torch.randint(-127, 128, c.k.shape, device='cuda', generator=g, dtype=torch.int8))
    c.v.copy_(torch.randint(-127, 128, c.v.shape, device='cuda', generator=g, dtype=torch.int8))
    c.k_scale.copy_(0.005 + 0.02 * torch.rand(pages, heads, device='cuda', generator=g))
    c.v_scale.copy_(0.002 + 0.03 * torch.rand(pages, heads, device='cuda', generator=g))
    if zero_scales:
        c.k_scale[torch.rand(pages, heads, device='cuda', generator=g) < 0.3] = 0
        c.v_scale[torch.rand(pages, heads, device='cuda', generator=g) < 0.3] = 0
    return c


def make_table(pages, B, blocks, g):
    return torch.randperm(pages, device='cuda', generator=g)[:B * blocks].to(torch.int32).view(B, blocks).contiguous()


def check_append(cache, old_k, old_v, old_ks, old_vs, table, starts, counts, k, v, k_roundings=1):
    """The cache after an append of k, v (B, T, heads, D) FP64 against the definition; returns the set of written pages."""
    slack = 0.5 + 127 * 2.0 ** -22
    written = set()
    for b, (st, n) in enumerate(zip(starts, counts)):
        for lo in range(st // 64 * 64, st + n, 64):
            a, z = max(lo, st), min(lo + 64, st + n)
            page = int(table[b, lo // 64])
            written.add(page)
            for x, cells, scale, was, was_s, tr in ((k, cache.k, cache.k_scale, old_k, old_ks, False),
                                                    (v, cache.v, cache.v_scale, old_v, old_vs, True)):
                new = x[b, a - st:z - st].transpose(0, 1)                       # (heads, tokens, D)
                s = new.abs().amax((1, 2)) / 127
                s0 = was_s[page].double() if a > lo else torch.zeros_like(s)
                s = torch.maximum(s, s0)
                got = scale[page].double()
                assert ((got - s).abs() <= 4 * 2.0 ** -24 * s).all()
                assert (torch.where(s0 >= s * (1 + 2.0 ** -20), got == s0, got >= s0)).all()
                now = cells[page].double()
                before = was[page].double()
                if tr:
                    now, before = now.transpose(1, 2), before.transpose(1, 2)
                safe = torch.where(s > 0, s, 1.0)[:, None, None]
                assert ((now[:, a - lo:z - lo] - new / safe).abs() <= slack).all()
                keep = (got == s0)[:, None, None]
                moved = before[:, :a - lo] * (s0[:, None, None] / safe)
                off = (now[:, :a - lo] - moved).abs()
                assert torch.where(keep, now[:, :a - lo] == before[:, :a - lo], off <= slack).all()
                assert torch.equal(now[:, z - lo:], before[:, z - lo:])        # slots behind the new tokens are left alone
    return written


@pytest.mark.parametrize('D', [32, 48, 64, 80, 96, 128])
@pytest.mark.parametrize('heads,starts,counts,T,dtype', [
    (8, [0], [1], 1, BF16), (1, [63, 64, 65], [1, 1, 1], 1, F16), (3, [5, 127, 0, 64], [64, 1, 0, 65], 65, BF16),
    (2, [60, 0, 33], [200, 129, 130], 200, F16), (8, [1003, 7], [160, 96], 160, BF16)])
def test_append(K, D, heads, starts, counts, T, dtype):
    g = gen(D + T)
    B, blocks = len(starts), max((s + T + 63) // 64 for s in starts) + 1
    cache = make_cache(K, B * blocks + 3, heads, D, g)
    table = make_table(cache.pages, B, blocks, g)
    k = (torch.randn(B, T, heads * D, device='cuda', generator=g) * 0.8).to(dtype)
    v = (torch.randn(B, T, heads * D, device='cuda', generator=g) * 0.5).to(dtype)
    was = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    K.kv8_append(cache, k, v, table, i32(starts), count=i32(counts))
    written = check_append(cache, *was, table, starts, counts, k.double().view(B, T, heads, D), v.double().view(B, T, heads, D))
    rest = [p for p in range(cache.pages) if p not in written]
    for t, o in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), was):
        assert torch.equal(t[rest], o[rest])
    # once more at the same place: nothing is lost, the result is the same
    again = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    K.kv8_append(cache, k, v, table, i32(starts), count=i32(counts))
    for t, o in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), again):
        assert torch.equal(t, o)


@pytest.mark.parametrize('D,axes', [(64, 3), (48, 2), (128, 4), (80, 1)])
def test_append_turns_keys(K, D, axes):
    g = gen(D)
    B, T, heads, starts = 2, 90, 4, [37, 64]
    rope, pos, sections = rope_case(K, D, axes, T, B, g, False)
    cache = make_cache(K, 9, heads, D, g)
    table = make_table(9, B, 4, g)
    qkv = torch.randn(B, T, 3 * heads * D, device='cuda', generator=g).bfloat16()      # views into one projection
    k, v = qkv[..., heads * D:2 * heads * D], qkv[..., 2 * heads * D:]
    was = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    K.kv8_append(cache, k, v, table, i32(starts), rope=rope, pos=pos)
    kt = ref.rotary(k.double().reshape(B, T, heads, D), pos, rope.cos, rope.sin, sections, False)
    check_append(cache, *was, table, starts, [T] * B, kt, v.double().reshape(B, T, heads, D))


def test_append_token_by_token_grows_the_scale(K):
    """Tokens of growing size, one at a time: every held value stays within one step of its block's final scale per growth."""
    g = gen(3)
    cache = make_cache(K, 3, 2, 64, g)
    table = i32([[2, 0]])
    xs = torch.randn(70, 2 * 64, device='cuda', generator=g) * torch.linspace(0.2, 4, 70, device='cuda')[:, None]
    xs = xs.bfloat16()
    grown = 0
    for t in range(70):
        page, s0 = (2, 0)[t // 64], cache.k_scale[(2, 0)[t // 64], 0].clone()
        K.kv8_append(cache, xs[None, None, t], -xs[None, None, t], table, i32([t]))
        grown += int(t < 64 and cache.k_scale[page, 0] > s0)
    k, v = K.kv8_read(cache, table, i32([0]), i32([70]), 70, dtype=F32)
    assert torch.equal(k, -v)
    step = cache.k_scale[table[0].long()].repeat_interleave(64, 0)[:70]          # (tokens, heads)
    err = (k[0] - xs.float()).abs().view(70, 2, 64).amax(-1)
    assert (err <= (0.5 * (grown + 1) + 1e-3) * step).all() and grown > 3


def test_append_zeros_infinities_and_nan(K):
    cache = make_cache(K, 4, 2, 32, gen(4))
    table = i32([[3, 1]])
    x = torch.zeros(1, 66, 64, device='cuda', dtype=BF16)
    x[0, 3, 5], x[0, 4, 6], x[0, 5, 7], x[0, 6, 8] = float('nan'), float('inf'), -float('inf'), 2.0
    K.kv8_append(cache, x, x, table, i32([0]))
    k, v = K.kv8_read(cache, table, i32([0]), i32([66]), 66, dtype=F32)
    assert torch.equal(k, v) and torch.isfinite(k).all()
    assert k[0, 3, 5] == 0 and abs(k[0, 6, 8] - 2) < 1e-6 and abs(k[0, 4, 6] - 2) < 1e-6 and abs(k[0, 5, 7] + 2) < 1e-6
    assert cache.k_scale[3, 1] == 0 and (cache.k[3, 1] == 0).all()             # the second head held nothing but zeros
    assert (cache.v_scale[1] == 0).all() and (cache.v[1, :, :, :2] == 0).all()
    K.kv8_append(cache, x[:, 6:7], x[:, 6:7], table, i32([66]))                # a block of zeros takes on a scale
    k, _ = K.kv8_read(cache, table, i32([64]), i32([67]), 3, dtype=F32)
    assert (k[0, :2] == 0).all() and abs(k[0, 2, 8] - 2) < 1e-6
    tiny = torch.full((1, 1, 64), 1e-37, device='cuda', dtype=BF16)
    K.kv8_append(cache, tiny, tiny, table, i32([0]))
    assert (cache.k_scale[3] == 0).all() and (cache.k[3, :, 0] == 0).all()


def test_append_out_of_range(K):
    """Tokens behind the table's last block and tokens of a page that does not exist are dropped and reported."""
    g = gen(6)
    cache = make_cache(K, 4, 2, 64, g)
    was = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    x = torch.randn(1, 64, 128, device='cuda', generator=g).bfloat16()
    K.kv8_append(cache, x, x, i32([[1]]), i32([64]))
    assert K.device_error(reset=True) == 2
    K.kv8_append(cache, x, x, i32([[4, -1]]), i32([0]))
    assert K.device_error(reset=True) == 2
    for t, o in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), was):
        assert torch.equal(t, o)


@pytest.mark.parametrize('dtype', [BF16, F16, F32])
@pytest.mark.parametrize('D,heads,begin,lens,T', [(64, 8, [0, 64], [130, 70], 150), (48, 3, [7, 100, 0], [200, 101, 0], 77),
                                                  (128, 2, [63], [64], 1), (80, 1, [5, 500], [64, 3], 64)])
def test_read(K, D, heads, begin, lens, T, dtype):
    g = gen(D)
    B = len(begin)
    cache = make_cache(K, 4 * B + 1, heads, D, g)
    table = make_table(cache.pages, B, 4, g)
    k, v = K.kv8_read(cache, table, i32(begin), i32(lens), T, dtype=dtype)
    for b in range(B):
        n = max(0, min(T, lens[b] - begin[b]))
        for got, cells, scale, tr in ((k, cache.k, cache.k_scale, False), (v, cache.v, cache.v_scale, True)):
            x = cells[table[b].long()].float() * scale[table[b].long()][..., None, None]
            x = (x.permute(0, 3, 1, 2) if tr else x.transpose(1, 2)).reshape(-1, heads * D)
            assert torch.equal(got[b, :n], x[begin[b]:begin[b] + n].to(dtype))
            assert (got[b, n:] == 0).all()


# ------------------------------------------------------------------------------------------------ attention
def check_attention(K, q, cache, table, lens, **kw):
    o = K.kv8_attention(q, cache, table, i32(lens), **{k: (i32(v) if k == 'count' and v is not None else v) for k, v in kw.items()})
    want, a = ref.attention(q, cache, table, lens, **kw)
    tol = HALF_ULP[q.dtype] * want.abs() * (1 + 2.0 ** -10) + 2.0 ** -10 * a + 2.0 ** -25
    err = (o.double() - want).abs()
    assert o.dtype == q.dtype and o.shape == q.shape
    assert bool((err <= tol).all()), f'{int((~(err <= tol)).sum())} of {err.numel()} outputs off, worst {float((err / tol).nan_to_num(1e9).max()):.3g} times the bound'
    return o


def attention_case(K, B, T, heads, kv_heads, D, lens, dtype=BF16, seed=0, extra=1, zero_scales=False, loud=1.0):
    g = gen(seed + 17 * T + D)
    blocks = (max(max(lens), 1) + 63) // 64 + extra
    cache = make_cache(K, B * blocks + 2, kv_heads, D, g, zero_scales)
    table = make_table(cache.pages, B, blocks, g)
    q = (torch.randn(B, T, heads * D, device='cuda', generator=g) * loud).to(dtype)
    return q, cache, table


@pytest.mark.parametrize('D', [32, 48, 64, 80, 96, 128])
@pytest.mark.parametrize('heads,kv_heads', [(8, 8), (8, 2), (7, 1), (16, 2)])
@pytest.mark.parametrize('lens', [[1, 2, 63, 64, 65, 0, 127, 129], [1000, 191, 4096]])
def test_attention_one_token(K, D, heads, kv_heads, lens):
    q, cache, table = attention_case(K, len(lens), 1, heads, kv_heads, D, lens)
    check_attention(K, q, cache, table, lens)


@pytest.mark.parametrize('D', [32, 48, 64, 80, 96, 128])
@pytest.mark.parametrize('T,heads,kv_heads,lens', [
    (2, 8, 2, [2, 70, 700]), (5, 6, 2, [5, 64, 900]), (17, 4, 4, [160, 17, 128]), (17, 16, 2, [300, 17]), (33, 3, 3, [33, 500]),
    (64, 4, 1, [64, 777]), (65, 7, 1, [65, 129, 66]), (130, 8, 2, [130, 1111]), (257, 2, 2, [257, 300, 1024])])
@pytest.mark.parametrize('causal', [True, False])
def test_attention_many_tokens(K, D, T, heads, kv_heads, lens, causal):
    q, cache, table = attention_case(K, len(lens), T, heads, kv_heads, D, lens, dtype=F16 if T % 2 else BF16)
    check_attention(K, q, cache, table, lens, causal=causal)


@pytest.mark.parametrize('T,heads,kv_heads,D', [(1, 8, 2, 64), (9, 8, 8, 48), (40, 8, 2, 64), (200, 8, 2, 128), (300, 4, 4, 64)])
@pytest.mark.parametrize('causal', [True, False])
def test_attention_ragged_and_empty_rows(K, T, heads, kv_heads, D, causal):
    """Fewer queries than T, sequences shorter than their queries (rows that see no token), empty sequences, no queries at all."""
    count = [T, max(1, T // 2), 0, T, T, min(T, 3)]
    lens = [T + 100, 333, 90, max(1, T // 3), 0, 2]
    q, cache, table = attention_case(K, 6, T, heads, kv_heads, D, lens)
    o = check_attention(K, q, cache, table, lens, count=count, causal=causal)
    for b in range(6):
        assert (o[b, count[b]:] == 0).all()
        if lens[b] == 0:
            assert (o[b] == 0).all()
        elif causal:
            assert (o[b, :max(0, count[b] - lens[b])] == 0).all()


@pytest.mark.parametrize('T,D', [(1, 64), (1, 128), (24, 64), (160, 64), (160, 128)])
def test_attention_long(K, T, D):
    lens = [20011, 5000]
    q, cache, table = attention_case(K, 2, T, 8, 2, D, lens)
    check_attention(K, q, cache, table, lens)


@pytest.mark.parametrize('most', [300, 1500])
@pytest.mark.parametrize('T,heads,kv_heads,D', [(1, 8, 8, 64), (1, 16, 8, 128), (9, 8, 8, 48), (17, 8, 8, 48), (25, 8, 8, 32), (3, 40, 8, 80),
                                                (20, 16, 8, 64)])
def test_attention_many_units(K, T, heads, kv_heads, D, most):
    """More heads of more sequences than the device has SMs, short (whole units to a warp) and longer ones, some empty."""
    lens = [0 if b % 13 == 5 else max(T if b % 7 else 1, (b * 37 + 11) % most) for b in range(41)]
    q, cache, table = attention_case(K, 41, T, heads, kv_heads, D, lens)
    check_attention(K, q, cache, table, lens)
    count = [(b * 5) % (T + 1) for b in range(41)]
    check_attention(K, q, cache, table, lens, count=count, causal=False)


@pytest.mark.parametrize('lens', [[3000], [9000, 64]])
def test_attention_few_units(K, lens):
    """One key head: every part of a sequence in another warp, on one CTA and over the device."""
    for T, D in ((1, 64), (2, 128), (6, 48)):
        q, cache, table = attention_case(K, len(lens), T, 4, 1, D, lens)
        want = check_attention(K, q, cache, table, lens)
        for _ in range(3):
            assert torch.equal(K.kv8_attention(q, cache, table, i32(lens)), want)


@pytest.mark.parametrize('T', [1, 20, 300])
def test_attention_negative_scale(K, T):
    lens = [260]
    q, cache, table = attention_case(K, 1, T, 4, 2, 64, lens)
    check_attention(K, q, cache, table, lens, scale=-0.2)


@pytest.mark.parametrize('T', [1, 20, 300])
def test_attention_loud_and_quiet_scores(K, T):
    """Scores of several hundred (one key takes all the weight), none at all, and blocks of very different scales."""
    lens = [700, 300]
    for loud in (80.0, 0.0):
        q, cache, table = attention_case(K, 2, T, 8, 2, 64, lens, loud=loud, dtype=BF16)
        check_attention(K, q, cache, table, lens)
    q, cache, table = attention_case(K, 2, T, 8, 2, 64, lens)
    cache.v_scale.mul_(10.0 ** torch.randint(-12, 12, cache.v_scale.shape, device='cuda', generator=gen(1)))
    check_attention(K, q, cache, table, lens)
    q, cache, table = attention_case(K, 2, T, 8, 2, 64, lens, zero_scales=True)
    check_attention(K, q, cache, table, lens)
    cache.v_scale.zero_()
    assert (K.kv8_attention(q, cache, table, i32(lens)) == 0).all()


@pytest.mark.parametrize('T', [1, 20, 300])
def test_attention_large_and_small_queries(K, T):
    """Query rows far outside FP16's range, in BF16 (the cache's scales bring the scores back)."""
    lens = [500]
    q, cache, table = attention_case(K, 1, T, 4, 2, 64, lens)
    cache.k_scale.mul_(2.0 ** -40)
    check_attention(K, q * 2.0 ** 40, cache, table, lens)
    cache.k_scale.mul_(2.0 ** 80)
    check_attention(K, q * 2.0 ** -40, cache, table, lens)
    g = gen(9)
    wide = q * 10.0 ** torch.randint(-3, 4, q.shape, device='cuda', generator=g).bfloat16()      # six decades inside a row
    cache.k_scale.mul_(2.0 ** -50)
    check_attention(K, wide, cache, table, lens)


@pytest.mark.parametrize('T', [1, 20, 300])
def test_attention_scale_strides_and_stream(K, T):
    lens = [400, 333]
    q, cache, table = attention_case(K, 2, T, 8, 2, 64, lens)
    check_attention(K, q, cache, table, lens, scale=0.3)
    check_attention(K, q, cache, table, lens, scale=0.0)
    want = K.kv8_attention(q, cache, table, i32(lens))
    qkv = torch.zeros(2, T, 1024, device='cuda', dtype=q.dtype)
    qkv[..., 256:768] = q
    assert torch.equal(K.kv8_attention(qkv[..., 256:768], cache, table, i32(lens)), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = K.kv8_attention(q, cache, table, i32(lens))
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(other, want)
    for _ in range(3):                                               # the same bits every time
        assert torch.equal(K.kv8_attention(q, cache, table, i32(lens)), want)


@pytest.mark.parametrize('T', [1, 20, 300])
def test_attention_ignores_what_is_masked(K, T):
    """Infinite and NaN scales in pages that no token lies in, and changes behind the last token, leave the output as it is."""
    lens = [330, 65]
    q, cache, table = attention_case(K, 2, T, 8, 2, 64, lens, extra=3)
    want = K.kv8_attention(q, cache, table, i32(lens))
    for b, n in enumerate(lens):
        for blk in range((n + 63) // 64, table.shape[1]):
            cache.k_scale[int(table[b, blk])] = float('nan')
            cache.v_scale[int(table[b, blk])] = float('inf')
        last = int(table[b, n // 64])
        cache.k[last, :, n % 64:] = 127
        cache.v[last, :, :, n % 64:] = -127
    assert torch.equal(K.kv8_attention(q, cache, table, i32(lens)), want)


@pytest.mark.parametrize('T', [1, 20, 300])
def test_attention_out_of_range(K, T):
    lens = [200]
    q, cache, table = attention_case(K, 1, T, 4, 2, 64, lens, extra=0)
    near = table.clone()
    table[0, 1], near[0, 1] = cache.pages + 5, cache.pages - 1
    table[0, 2], near[0, 2] = -7, 0
    o = K.kv8_attention(q, cache, table, i32(lens))
    assert K.device_error(reset=True) == 2
    assert torch.equal(o, K.kv8_attention(q, cache, near, i32(lens)))
    o = K.kv8_attention(q, cache, near, i32([100000]))
    assert K.device_error(reset=True) == 2
    assert torch.equal(o, K.kv8_attention(q, cache, near, i32([256])))
    assert K.device_error(reset=True) == 0


@pytest.mark.parametrize('T', [1, 20, 300])
def test_attention_far_pages(K, T):
    """A cache of more than 2^31 elements: pages at its end, written, read back and attended to."""
    D, heads, pages = 128, 2, 140000
    cache = K.KV8Cache.empty(pages, heads, D)
    assert cache.k.numel() > 2 ** 31
    g = gen(2)
    n = 300 + T
    table = torch.randperm(40, device='cuda', generator=g)[:(n + 63) // 64].to(torch.int32)[None] + (pages - 40)
    k = torch.randn(1, n, heads * D, device='cuda', generator=g).bfloat16()
    v = torch.randn(1, n, heads * D, device='cuda', generator=g).bfloat16()
    K.kv8_append(cache, k, v, table, i32([0]))
    kr, vr = K.kv8_read(cache, table, i32([0]), i32([n]), n)
    assert (kr - k).abs().max() < 0.05 and (vr - v).abs().max() < 0.05
    q = torch.randn(1, T, 4 * D, device='cuda', generator=g).bfloat16()
    check_attention(K, q, cache, table, [n])


@pytest.mark.parametrize('T', [1, 20, 300])
def test_attention_in_a_graph(K, T):
    """Append and attention captured in a CUDA graph; the lengths advance on the device between replays."""
    B, heads, D = 2, 4, 64
    cache = K.KV8Cache.empty(32, 2, D)
    table = make_table(32, B, 16, gen(7))
    start, lens = i32([100, 3]), i32([0, 0])
    g = gen(8)
    past = torch.randn(B, 100, 2 * D, device='cuda', generator=g).bfloat16()
    K.kv8_append(cache, past, past, table, i32([0, 0]), count=start)
    k, v = (torch.randn(B, T, 2 * D, device='cuda', generator=g).bfloat16() for _ in range(2))
    q = torch.randn(B, T, heads * D, device='cuda', generator=g).bfloat16()
    out = torch.empty_like(q)

    def step():
        K.kv8_append(cache, k, v, table, start)
        torch.add(start, T, out=lens)
        K.kv8_attention(q, cache, table, lens, out=out)
        start.copy_(lens)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    n = [100 + 3 * T, 3 + 3 * T]
    assert lens.tolist() == n
    want, a = ref.attention(q, cache, table, n)
    assert ((out.double() - want).abs() <= HALF_ULP[BF16] * want.abs() * 1.001 + 2.0 ** -10 * a + 2.0 ** -25).all()
