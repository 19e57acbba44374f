"""Cross attention where its output lies in a gap of its inputs, and of large scores."""
import math

import pytest
import torch

from test_cross_gpu import check, ints, rand
from test_cross_gpu import K  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('T,N', [(1, 9000), (17, 160), (150, 300), (300, 700)])
def test_output_in_a_gap_of_the_inputs(K, T, N):
    """Memory between the sequences of a strided input, or between its rows, is apart from it."""
    heads, D = 2, 64
    W = heads * D
    for lens in (None, ints([N, N // 2])):
        q, k, v = rand(2, T, W), rand(2, N, W, seed=1), rand(2, N, W, seed=2)
        buf = rand(4, T, W, seed=3)
        before = buf.clone()
        want = check(K, buf[::3], k, v, heads, lens=lens)
        check(K, buf[::3], k, v, heads, lens=lens, out=buf[1:3])
        assert torch.equal(buf[1:3], want) and torch.equal(buf[::3], before[::3])
        buf = torch.empty(2 * N * W + 2 * T * W, dtype=torch.bfloat16, device='cuda')
        kk = buf.as_strided((2, N, W), (N * W + 2 * T * W, W, 1)).copy_(k)
        out = buf[N * W:N * W + 2 * T * W].view(2, T, W)
        assert check(K, q, kk, v, heads, lens=lens, out=out) is not None
        assert torch.equal(kk, k)
        with pytest.raises(K.TcqError):
            K.cross_attention(q, kk, v, heads, lens=lens, out=buf[N * W - 8:N * W - 8 + 2 * T * W].view(2, T, W))
    assert K.device_error() == 0


def whole(q, k, v, heads, scale, lens=None):
    """(output in 64 bits, sum p |v|) of scores that are exact: q and k are small integers."""
    B, T, W = q.shape
    N, D = k.shape[1], W // heads
    qq, kk, vv = (x.double().view(B, -1, heads, D).transpose(1, 2) for x in (q, k, v))
    s = qq @ kk.transpose(2, 3) * (1 if scale > 0 else -1)
    if lens is not None:
        s.masked_fill_((torch.arange(N, device='cuda') >= lens[:, None])[:, None, None], -float('inf'))
    p = torch.softmax((s - s.amax(-1, keepdim=True)) * abs(scale), -1)
    return ((p @ x).transpose(1, 2).reshape(B, T, W) for x in (vv, vv.abs()))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('D', [48, 64, 128])
@pytest.mark.parametrize('T,N', [(1, 9000), (17, 160), (40, 97), (130, 600), (300, 700)])
def test_large_scores_and_larger_ones(K, T, N, D, dtype):
    """Integers times a power of two, so that FP32 holds q k whole: differing scores are a power of two apart, the largest take it all, and
    share it where they are equal. Equal scores have equal weights, about 2^5: the sum takes them as they are, the product rounded to
    the type once (u each, of which the sum knows nothing: u sum p |v|); N / 32 + 64 roundings of FP32; the output's own. Scores reach some 2^7 times the scale: up to 2^23 that is what comes out, past it is reported."""
    heads = 2
    u = torch.finfo(dtype).eps / 2
    g = torch.Generator(device='cuda').manual_seed(T + N + D)
    q, k = (torch.randint(-3, 4, (2, n, heads * D), device='cuda', generator=g).to(dtype) for n in (T, N))
    v = rand(2, N, heads * D, dtype=dtype, seed=2)
    k[:, ::3] = k[:, 1:2]                                                      # equal ones
    top = (q.double().view(2, T, heads, D).transpose(1, 2) @ k.double().view(2, N, heads, D).permute(0, 2, 3, 1)).amax(-1).abs().max().item()
    for lens in (None, ints([N, N // 2 + 1])):
        for power in (10, 13, 23 - math.ceil(math.log2(top))):
            for scale in (2.0 ** power, -2.0 ** power):
                o = K.cross_attention(q, k, v, heads, lens=lens, scale=scale)
                want, a = whole(q, k, v, heads, scale, lens)
                tol = u * want.abs() + (u + (N / 32 + 64) * 2.0 ** -23) * a + (2.0 ** -25 if dtype == torch.float16 else 0)
                assert ((o.double() - want).abs() <= tol).all(), (lens, scale)
        assert K.device_error() == 0
        for scale in (2.0 ** 30, -2.0 ** 90):
            K.cross_attention(q, k, v, heads, lens=lens, scale=scale)
            assert K.device_error() == 2 and K.device_error() == 0
    k.view(2, N, heads, D)[0, 0, 0] = math.inf                                 # infinite scores are what they are: NaN, and not reported
    K.cross_attention(q, k, v, heads)
    assert K.device_error() == 0


@pytest.mark.parametrize('T,heads,kv_heads,N', [(1, 4, 4, 5000), (17, 4, 4, 160), (40, 4, 4, 200), (150, 2, 2, 300), (300, 4, 2, 900), (130, 2, 2, 3000)])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_random_masks(K, T, heads, kv_heads, N, dtype):
    """States left out one by one at random, from few to nearly all; the masks are made from a seed."""
    D, shares = 64, (0.0, 0.01, 0.5, 0.9, 0.99, 0.999)
    B = len(shares)
    g = torch.Generator(device='cuda').manual_seed(T + N)
    q, k, v = rand(B, T, heads * D, dtype=dtype), rand(B, N, kv_heads * D, dtype=dtype, seed=1), rand(B, N, kv_heads * D, dtype=dtype, seed=2)
    mask = torch.rand(B, N, device='cuda', generator=g) >= torch.tensor(shares, device='cuda')[:, None]
    k[~mask], v[~mask] = math.inf, math.nan
    check(K, q, k, v, heads, kv_heads, mask=mask)
    check(K, q, k, v, heads, kv_heads, mask=mask, lens=ints([N, N - 1, N // 2, N, N, N // 3]))
