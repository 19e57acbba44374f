"""Cross attention against 64 bits, at the sizes, strides and masks where it can go wrong."""
import math

import pytest
import torch

import cross_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def K():
    from yanlongvla_b200 import kernels
    kernels.device_error()
    return kernels


def rand(*shape, dtype=torch.bfloat16, seed=0, std=1.0):
    g = torch.Generator(device='cuda').manual_seed(seed + sum(shape))
    return (torch.randn(*shape, device='cuda', generator=g) * std).to(dtype)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device='cuda')


def check(K, q, k, v, heads, kv_heads=None, lens=None, mask=None, scale=None, out=None):
    o = K.cross_attention(q, k, v, heads, kv_heads, lens=lens, mask=mask, scale=scale, out=out)
    want, tol = ref.attention(q, k, v, heads, kv_heads, lens, mask, scale)
    assert o.shape == q.shape and o.dtype == q.dtype
    err = (o.double() - want).abs()
    assert (err <= tol).all(), f'off by {(err / tol.clamp(min=1e-30)).max().item():.2f} of the bound'
    again = K.cross_attention(q, k, v, heads, kv_heads, lens=lens, mask=mask, scale=scale)
    assert torch.equal(o.view(torch.int16), again.view(torch.int16))
    assert K.device_error() == 0
    return o


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('D', range(8, 129, 8))
def test_head_widths(K, D, dtype):
    for T, N in ((3, 70), (150, 300)):
        q, k, v = rand(2, T, 4 * D, dtype=dtype), rand(2, N, 2 * D, dtype=dtype, seed=1), rand(2, N, 2 * D, dtype=dtype, seed=2)
        check(K, q, k, v, 4, 2)


# rows that share a key head: S * T * heads / kv_heads
SHAPES = [(1, 1, 1, 1, 1, 1), (1, 1, 1, 2, 1, 1), (3, 1, 1, 31, 2, 2), (1, 1, 1, 32, 8, 2), (2, 1, 1, 33, 8, 1), (2, 1, 15, 64, 2, 2), (1, 1, 16, 65, 2, 2),
          (2, 1, 17, 160, 4, 4), (2, 3, 17, 160, 2, 2), (1, 16, 17, 97, 2, 2), (1, 1, 32, 127, 2, 1), (1, 1, 33, 128, 1, 1), (2, 1, 64, 129, 3, 3),
          (1, 1, 65, 255, 2, 2), (1, 1, 127, 256, 2, 2), (1, 1, 128, 257, 1, 1), (1, 1, 129, 500, 2, 2), (1, 5, 51, 383, 6, 2), (1, 1, 255, 384, 2, 2),
          (1, 1, 256, 385, 1, 1), (1, 1, 257, 640, 2, 1), (2, 1, 300, 1000, 7, 1), (1, 1, 1, 5000, 4, 4), (1, 1, 2, 16411, 2, 1), (40, 1, 1, 90, 8, 8),
          (5, 2, 9, 700, 4, 2), (1, 1, 700, 40, 2, 2), (1, 1, 1000, 1, 2, 2), (1, 1, 513, 2050, 2, 2), (1, 1, 2, 3000, 64, 1)]


@pytest.mark.parametrize('B,S,T,N,heads,kv_heads', SHAPES)
@pytest.mark.parametrize('D', [48, 64, 128])
def test_sizes(K, B, S, T, N, heads, kv_heads, D):
    for dtype in (torch.bfloat16, torch.float16):
        q, k, v = rand(B * S, T, heads * D, dtype=dtype, std=1.5), rand(B, N, kv_heads * D, dtype=dtype, seed=1), rand(B, N, kv_heads * D, dtype=dtype, seed=2)
        check(K, q, k, v, heads, kv_heads)


@pytest.mark.parametrize('T,heads,kv_heads,N', [(1, 4, 4, 5000), (1, 8, 2, 700), (17, 4, 4, 160), (40, 4, 4, 200), (150, 2, 2, 300), (300, 4, 2, 900), (130, 2, 2, 3000)])
@pytest.mark.parametrize('D', [48, 72, 128])
def test_lengths(K, T, heads, kv_heads, N, D):
    """Sequences of no state, of one, of all; what lies behind the last one is NaN or infinite."""
    lens = ints([0, 1, N, N - 1, N // 2, 31, 32, 33, 127, 128, 129])
    B = len(lens)
    q, k, v = rand(B, T, heads * D), rand(B, N, kv_heads * D, seed=1), rand(B, N, kv_heads * D, seed=2)
    behind = torch.arange(N, device='cuda') >= lens[:, None]
    k[behind], v[behind] = math.nan, math.inf
    o = check(K, q, k, v, heads, kv_heads, lens=lens)
    assert not o[0].any()
    assert torch.equal(o[1].view(T, heads, D), v[1, 0].view(kv_heads, 1, D).expand(-1, heads // kv_heads, -1).reshape(1, heads, D).expand(T, -1, -1))


@pytest.mark.parametrize('T,heads,kv_heads,N', [(1, 4, 4, 5000), (17, 4, 4, 160), (40, 4, 4, 200), (150, 2, 2, 300), (300, 4, 2, 900), (130, 2, 2, 3000)])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_masks(K, T, heads, kv_heads, N, dtype):
    """Whole runs left out, single states, all but the first or last, all; garbage where none is; a mask with wider rows."""
    D, B = 64, 9
    q, k, v = rand(B, T, heads * D, dtype=dtype), rand(B, N, kv_heads * D, dtype=dtype, seed=1), rand(B, N, kv_heads * D, dtype=dtype, seed=2)
    i = torch.arange(N, device='cuda')
    wide = torch.ones(B, N + 5, dtype=torch.bool, device='cuda')
    mask = wide[:, 3:N + 3]
    mask[0] = False
    mask[1] = i == 0
    mask[2] = i == N - 1
    mask[3] = i // 64 % 2 == 1
    mask[4] = torch.rand(N, device='cuda') < 0.5
    mask[5] = i // 128 == N // 256
    mask[6] = i % 7 == 0
    mask[7] = i >= N // 2
    k[~mask], v[~mask] = math.inf, math.nan
    lens = ints([N, N, N, N, N, N, N, N // 2, N // 3])
    o = check(K, q, k, v, heads, kv_heads, mask=mask)
    assert not o[0].any()
    o = check(K, q, k, v, heads, kv_heads, mask=mask, lens=lens)
    assert not o[0].any() and not o[7].any()


@pytest.mark.parametrize('B,T,heads,N', [(1, 1, 2, 9000), (40, 1, 16, 700), (40, 17, 16, 700), (3, 40, 2, 230)])
@pytest.mark.parametrize('D', [64, 96])
def test_masks_of_few_states(K, B, T, heads, N, D):
    """Single states far apart, at the ends of what is read of a mask at a time (128 or 256 states), none at all."""
    q, k, v = rand(B, T, heads * D), rand(B, N, heads * D, seed=1), rand(B, N, heads * D, seed=2)
    mask = torch.zeros(B, N, dtype=torch.bool, device='cuda')
    for b in range(B):
        mask[b, [[127], [128], [0, N - 1], [255, 256], [N - 1], [15, 16, 144], [31, 32, 160], []][b % 8]] = True
    if B == 1:
        mask[0, [127, 2175, N - 1]] = True
    check(K, q, k, v, heads, mask=mask)
    check(K, q, k, v, heads, mask=mask, lens=torch.arange(B, dtype=torch.int32, device='cuda') * 37 % N)


@pytest.mark.parametrize('T', [1, 17, 150, 300])
def test_strides(K, T):
    """Keys and values as columns of one projection's output, queries of a wider one, tokens of every second row, batches shared."""
    B, N, heads, D = 3, 333, 4, 64
    row = heads * D
    kv = rand(B, N, 2 * row + 8)
    q = rand(B, 2 * T, 3 * row)[:, ::2, row:2 * row]
    check(K, q, kv[..., :row], kv[..., row + 8:], heads)
    kv = rand(B, 2 * N, row, seed=3)
    check(K, q, kv[:, ::2], kv[:, 1::2], heads)
    k, v = rand(1, N, row, seed=4).expand(B, -1, -1), rand(B, N, row, seed=5)
    check(K, q, k, v, heads)
    check(K, q, v, k, heads, lens=ints([333, 0, 100]))
    by_token = rand(N, B, row, seed=6).transpose(0, 1)
    check(K, q.contiguous(), by_token, by_token, heads, out=torch.empty(B, T, row, dtype=torch.bfloat16, device='cuda'))
    k1 = rand(B, 1, row, seed=7)
    check(K, q, k1, k1, heads)


def test_strides_of_single_dimensions(K):
    """A dimension of size one may state any stride."""
    D = 48
    q, k, v = rand(1, 1, D), rand(1, 5, D, seed=1), rand(1, 1, D, seed=2)
    odd = lambda x, s: torch.as_strided(x, x.shape, s)
    check(K, odd(q, (7, 3, 1)), odd(k, (1, D, 1)), rand(1, 5, D, seed=3), 1)
    check(K, q, odd(v, (5, 3, 1)), odd(v, (1, 1, 1)), 1)


@pytest.mark.parametrize('T,N', [(1, 4000), (17, 160), (200, 1200)])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_large_scores(K, T, N, dtype):
    """Scores of some hundreds, growing along the states, so that the reference moves often; negative and zero scales."""
    heads, D = 2, 64
    q, k, v = rand(2, T, heads * D, dtype=dtype, std=4), rand(2, N, heads * D, dtype=dtype, seed=1, std=4), rand(2, N, heads * D, dtype=dtype, seed=2)
    k *= torch.linspace(0.01, 1, N, device='cuda', dtype=dtype)[None, :, None]
    for scale in (None, -0.125, 0.0, 1e-30):
        check(K, q, k, v, heads, scale=scale)
        check(K, q, k, v, heads, scale=scale, lens=ints([N - 3, 5]))


@pytest.mark.parametrize('T,N', [(1, 4000), (17, 160), (200, 1200)])
def test_nan_query_rows_stay_their_own(K, T, N):
    heads, D = 2, 64
    q, k, v = rand(2, T, heads * D), rand(2, N, heads * D, seed=1), rand(2, N, heads * D, seed=2)
    q[1, T // 2, 3] = math.nan
    o = K.cross_attention(q, k, v, heads)
    assert o[1, T // 2, :D].isnan().all()
    o[1, T // 2, :D] = 0
    assert not o.isnan().any()
    o = K.cross_attention(q, k, v, heads, lens=ints([N, 0]))
    assert not o[1].any()


def test_lengths_out_of_range(K):
    q, k = rand(2, 3, 64), rand(2, 50, 64, seed=1)
    o = K.cross_attention(q, k, k, 1, lens=ints([-1, 51]))
    assert K.device_error() == 2
    assert not o[0].any() and torch.equal(o[1], K.cross_attention(q, k, k, 1)[1])


def test_no_states(K):
    q, k = rand(2, 3, 64), rand(2, 1, 64, seed=1)[:, :0]
    o = K.cross_attention(q, k, k, 1, out=rand(2, 3, 64, seed=2))
    assert not o.any()
    o = K.cross_attention(rand(4, 1000, 64), k, k, 1, lens=ints([0, 0]))
    assert o.shape == (4, 1000, 64) and not o.any()


def test_rows_behind_are_left(K):
    wide = rand(5, 20, 64, seed=9)
    before = wide.clone()
    q, k = rand(2, 20, 64), rand(2, 77, 64, seed=1)
    out = wide[1:3]
    K.cross_attention(q, k, k, 2, out=out)
    assert torch.equal(wide[0], before[0]) and torch.equal(wide[3:], before[3:]) and not torch.equal(wide[1:3], before[1:3])


@pytest.mark.parametrize('T,N', [(1, 9000), (17, 160), (300, 700)])
def test_graphs_and_streams(K, T, N):
    """Captured, replayed on new inputs in the same buffers, next to calls on other streams."""
    heads, D = 4, 64
    q, k, v, lens = rand(2, T, heads * D), rand(2, N, heads * D, seed=1), rand(2, N, heads * D, seed=2), ints([N, N // 2])
    out = torch.empty_like(q)
    K.cross_attention(q, k, v, heads, lens=lens, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.cross_attention(q, k, v, heads, lens=lens, out=out)
    streams = [torch.cuda.Stream() for _ in range(3)]
    others = [(rand(2, T, heads * D, seed=i), rand(2, N, heads * D, seed=i + 5)) for i in range(3)]
    wants = [K.cross_attention(a, b, b, heads) for a, b in others]
    for i in range(3):
        q.copy_(rand(2, T, heads * D, seed=10 + i))
        lens.copy_(ints([N - i, i]))
        torch.cuda.synchronize()
        graph.replay()
        got = []
        for s, (a, b) in zip(streams, others):
            with torch.cuda.stream(s):
                got.append(K.cross_attention(a, b, b, heads))
        torch.cuda.synchronize()
        assert torch.equal(out, K.cross_attention(q, k, v, heads, lens=lens))
        for a, b in zip(got, wants):
            assert torch.equal(a, b)
    assert K.device_error() == 0


@pytest.mark.parametrize('T,heads,kv_heads,N', [(1, 8, 2, 9000), (1, 4, 4, 5), (17, 4, 4, 160), (150, 2, 2, 300), (130, 2, 2, 3000), (300, 4, 2, 700)])
def test_output_in_place_of_the_queries(K, T, heads, kv_heads, N):
    for D in (48, 128):
        q, k, v = rand(3, T, heads * D), rand(3, N, kv_heads * D, seed=1), rand(3, N, kv_heads * D, seed=2)
        for lens in (None, ints([N, 0, N // 2])):
            want, own = K.cross_attention(q, k, v, heads, kv_heads, lens=lens), q.clone()
            assert K.cross_attention(own, k, v, heads, kv_heads, lens=lens, out=own) is own
            assert torch.equal(own, want)
        wide = rand(6, T, heads * D)
        with pytest.raises(K.TcqError):
            K.cross_attention(wide[:3], k, v, heads, kv_heads, out=wide[1:4])
    assert K.device_error() == 0


def test_refusals(K):
    q, k = rand(2, 3, 128), rand(2, 50, 64, seed=1)
    ok = dict(q=q, k=k, v=k, heads=2, kv_heads=1)

    def refused(error=K.TcqError, **kw):
        a = {**ok, **kw}
        with pytest.raises(error):
            K.cross_attention(a.pop('q'), a.pop('k'), a.pop('v'), a.pop('heads'), a.pop('kv_heads'), **a)
    refused(q=q.float())
    refused(k=k.half(), v=k.half())
    refused(v=k.half())
    refused(v=k[:, :-1])
    refused(q=q[0])
    refused(q=q.cpu())
    refused(k=k.cpu(), v=k.cpu())
    refused(q=rand(3, 3, 128))
    refused(q=q[:0])
    refused(q=q[:, :0])
    refused(k=k[:0], v=k[:0])
    refused(heads=3)
    refused(heads=0)
    refused(kv_heads=2)
    refused(kv_heads=0)
    refused(heads=4)
    refused(q=rand(2, 3, 24), k=rand(2, 5, 12), v=rand(2, 5, 12))
    refused(q=rand(2, 3, 272), k=rand(2, 5, 136), v=rand(2, 5, 136))
    refused(q=rand(2, 3, 256)[..., ::2])
    refused(q=rand(2, 3, 132)[..., 4:])
    refused(k=rand(2, 50, 68)[..., 4:], v=rand(2, 50, 68)[..., 4:])
    refused(k=rand(2, 50, 66)[..., :64], v=rand(2, 50, 66)[..., :64])
    refused(k=k[:, :1].expand(-1, 50, -1), v=k)
    for lens in (ints([1]), ints([1, 2]).long(), torch.tensor([1, 2], dtype=torch.int32), ints([[1, 2]])):
        refused(lens=lens)
    refused(mask=torch.ones(2, 50, device='cuda'))
    refused(mask=torch.ones(2, 49, dtype=torch.bool, device='cuda'))
    refused(mask=torch.ones(2, 100, dtype=torch.bool, device='cuda')[:, ::2])
    refused(mask=torch.ones(2, 50, dtype=torch.bool))
    refused(out=torch.empty(2, 3, 128, device='cuda'))
    refused(out=torch.empty(2, 6, 128, device='cuda', dtype=torch.bfloat16)[:, ::2])
    refused(TypeError, q=None)
    refused(TypeError, heads='2')
    refused(TypeError, scale='a')
    refused(TypeError, lens=[1, 2])
    refused(q=q.clone().requires_grad_())
    refused(v=k.clone().requires_grad_())
    with torch.no_grad():
        K.cross_attention(q.clone().requires_grad_(), k, k, 2, 1)
    K.cross_attention(q, k, k, 2, 1)
    assert K.device_error() == 0


def test_first_call_in_a_capture():
    """What the first call asks the device works in a capture too, and with two threads at once."""
    import subprocess
    import sys
    from pathlib import Path
    code = '''
import threading, torch
from yanlongvla_b200 import kernels as K
x = {n: torch.randn(2, n, 256, device='cuda').bfloat16() for n in (1, 300, 700, 9000)}
def calls():
    return [K.cross_attention(x[t], x[n], x[n], 4) for t, n in ((1, 9000), (1, 300), (300, 300), (300, 700), (700, 9000))]
owner = K.KV8Pages.empty(300)
table, lens = owner.table(2, 100), torch.zeros(2, dtype=torch.int32, device='cuda')
ints = lambda v: torch.tensor(v, dtype=torch.int32, device='cuda')
n, p = ints([70, 0]), ints([0, 0])
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    a = calls()
    granted, copies = K.kv8_reserve(owner, table, lens, n)
    lens += granted
    K.kv8_fork(owner, table, lens, p)
g.replay()
torch.cuda.synchronize()
assert lens.tolist() == [70, 70] and owner.refs[:3].tolist() == [2, 2, 0]
got = [None] * 4
def work(i):
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        for _ in range(20):
            got[i] = calls()
    s.synchronize()
t = [threading.Thread(target=work, args=(i,)) for i in range(4)]
[y.start() for y in t]; [y.join() for y in t]
for b in got:
    assert all(torch.equal(u, v) for u, v in zip(a, b))
assert K.device_error() == 0
'''
    r = subprocess.run([sys.executable, '-c', code], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize('T,heads', [(300, 2), (100, 2), (17, 4)])
@pytest.mark.parametrize('D', [64, 72, 128])
def test_blocks_left_out(K, T, heads, D):
    """Blocks of 64 states of which the mask leaves all, some or none: neighbours, far ones, an odd number of them, the ragged last one."""
    N = 64 * 19 + 37
    keep = [[0, 1, 2, 3], [0, 2, 4, 6, 8], [18, 19], [19], [1], [3, 4, 9, 17], list(range(20)), [0, 19], [5, 6, 7]]
    block = torch.arange(N, device='cuda') // 64
    mask = torch.stack([torch.isin(block, torch.tensor(b, device='cuda')) for b in keep])
    mask[3:, ::5] = False
    B = len(keep)
    q, k, v = rand(B, T, heads * D), rand(B, N, heads * D, seed=1), rand(B, N, heads * D, seed=2)
    k[~mask], v[~mask] = math.nan, math.inf
    check(K, q, k, v, heads, mask=mask)
    check(K, q, k, v, heads, mask=mask, lens=ints([N, N, N - 30, N, 64, 64 * 17 + 1, 64 * 11, N - 1, 64 * 6 + 3]))
