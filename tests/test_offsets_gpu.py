"""Cross attention and the page operators at offsets past 2^31 elements, which 32-bit arithmetic would wrap."""
import pytest
import torch

import cross_ref
import pages_ref

pytestmark = pytest.mark.gpu
FAR = (1 << 31) + 64


@pytest.fixture(scope='module')
def K():
    from yanlongvla_b200 import kernels
    kernels.device_error()
    return kernels


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device='cuda')


@pytest.mark.parametrize('T,N,D', [(1, 3000, 64), (17, 160, 48), (150, 400, 128), (300, 700, 64)])
def test_sequences_far_apart(K, T, N, D):
    """The second sequence's queries, keys, values and mask lie 2^31 elements behind the first one's."""
    heads = 2
    W = heads * D
    g = torch.Generator(device='cuda').manual_seed(T)
    buf = torch.empty(FAR + 3 * N * W, dtype=torch.bfloat16, device='cuda')
    q, k, v = (buf.as_strided((2, n, W), (FAR, W, 1), at) for n, at in ((T, 0), (N, N * W), (N, 2 * N * W)))
    for x in (q, k, v):
        x.copy_(torch.randn(x.shape, device='cuda', generator=g))
    o = K.cross_attention(q, k, v, heads, lens=ints([N, N // 2]))
    want, tol = cross_ref.attention(q, k, v, heads, lens=ints([N, N // 2]))
    assert ((o.double() - want).abs() <= tol).all()
    mask = torch.empty(FAR + N, dtype=torch.bool, device='cuda').as_strided((2, N), (FAR, 1))
    mask.copy_(torch.rand(2, N, device='cuda', generator=g) < 0.3)
    o = K.cross_attention(q, k, v, heads, mask=mask)
    want, tol = cross_ref.attention(q, k, v, heads, mask=mask)
    assert ((o.double() - want).abs() <= tol).all()
    assert K.device_error() == 0


@pytest.mark.parametrize('N', [5, 300])
def test_an_output_of_more_elements(K, N):
    """2^20 + 40 tokens of 2048 elements over few states, in place: the last rows as alone."""
    heads, W, T = 16, 2048, (1 << 20) + 40
    q = torch.empty(1, T, W, dtype=torch.bfloat16, device='cuda')
    g = torch.Generator(device='cuda').manual_seed(N)
    for i in range(0, T, 1 << 16):
        q[:, i:i + (1 << 16)].normal_(generator=g)
    k, v = (torch.randn(1, N, W, device='cuda', generator=g).bfloat16() for _ in range(2))
    some = [0, 1, T // 2, *range(T - 50, T)]
    own = q[:, some].clone()
    K.cross_attention(q, k, v, heads, out=q)
    want, tol = cross_ref.attention(own, k, v, heads)
    assert ((q[:, some].double() - want).abs() <= tol).all()
    assert K.device_error() == 0


def test_pages_far_behind(K):
    """Pages of 64 KB past the first 2 GB of a cache: copied, and packed from and to."""
    heads, D, pages = 8, 128, 33000
    c = K.KV8Cache.empty(pages, heads, D)
    g = torch.Generator(device='cuda').manual_seed(0)
    old, new = [5, 32900, 32990], [32950, 32770]
    for p in old:
        for cells, scale in ((c.k, c.k_scale), (c.v, c.v_scale)):
            cells[p] = torch.randint(-127, 128, cells[p].shape, device='cuda', generator=g).to(torch.int8)
            scale[p] = torch.rand(heads, device='cuda', generator=g) + 0.01
    index = [*range(40, 64), *range(64, 170, 2), 180, 190]
    K.kv8_compact(c, ints([old]), ints([192]), ints([index]), ints([new]))
    for cells, scale, transposed in ((c.k, c.k_scale, False), (c.v, c.v_scale, True)):
        for p, (x, s) in zip(new, pages_ref.packed(cells, scale, old, index, transposed)):
            assert torch.equal(cells[p], x) and torch.equal(scale[p], s)
    pairs = [(5, 32999), (32990, 7)]
    K.kv8_copy(c, ints(pairs).t().contiguous())
    for a, b in pairs:
        for t in (c.k, c.v, c.k_scale, c.v_scale):
            assert torch.equal(t[a], t[b])
    assert K.device_error() == 0
