"""Cross attention where its output lies in a gap of its inputs."""
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
