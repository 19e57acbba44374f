"""Cross attention without a GPU: what the C ABI and the binding refuse before any CUDA call, and the definition the GPU tests compare
with, pinned to hand-made cases."""
import math

import pytest
import torch

import cross_ref as ref

A, B, C, D_, E, F_ = (i << 20 for i in range(1, 7))            # fake, aligned "device" addresses


@pytest.fixture(scope='module')
def L():
    from yanlongvla_b200 import _lib
    return _lib


def test_refuses(L):
    def cross(q=A, q_sb=512, q_st=512, k=B, k_sb=4096, k_st=128, v=C, v_sb=4096, v_st=128, dtype=L.DT_BF16, out=D_, lens=None, mask=None, mask_sb=0,
              scale=0.125, n=2, s=1, t=3, states=32, heads=8, kv_heads=2, d=64):
        return L.lib.tcq_cross_attention(q, q_sb, q_st, k, k_sb, k_st, v, v_sb, v_st, dtype, out, lens, mask, mask_sb, scale, n, s, t, states, heads,
                                         kv_heads, d, None)
    for name in ('q', 'k', 'v', 'out'):
        assert cross(**{name: None}) == 4
    assert cross(dtype=L.DT_F32) == 3 and cross(dtype=9) == 3
    for name in ('n', 's', 't', 'heads', 'kv_heads'):
        assert cross(**{name: 0}) == 1
    assert cross(states=-1) == 1 and cross(heads=7) == 1
    for d in (0, 4, 12, 60, 136, 256):
        assert cross(d=d) == 1
    assert cross(s=1 << 14, t=1 << 16) == 1 and cross(states=(1 << 30) + 1) == 1                 # more than 2^30 rows of a head, states
    for name in ('q', 'k', 'v', 'out'):
        assert cross(**{name: A + 8}) == 2
    for name in ('q_sb', 'q_st', 'k_sb', 'k_st', 'v_sb', 'v_st'):
        assert cross(**{name: 4100}) == 2
    for at in (A + 64, B, B + 64, C + 4096, D_):                                                # out in the queries, keys or values
        assert cross(out=at, **({'q': D_ + 64} if at == D_ else {})) == 4
    assert cross(q=D_, q_sb=8192, out=D_) == 4                                                   # q with gaps: its rows would move
    assert cross(k_st=0) == 4 and cross(v_st=0) == 4 and cross(k_sb=-4096) == 4                  # states on one another, backwards


def test_the_binding_refuses():
    from yanlongvla_b200 import kernels as K
    q = torch.zeros(2, 3, 64, dtype=torch.bfloat16)
    with pytest.raises(K.TcqError, match='CUDA'):
        K.cross_attention(q, q, q, 1)
    with pytest.raises(TypeError):
        K.cross_attention(q, None, q, 1)
    with pytest.raises(TypeError):
        K.cross_attention(q, q, q, 'one')


def test_definition():
    k = torch.tensor([[[0.0], [1.0], [2.0], [9.0]]]).repeat(1, 1, 1)
    v = torch.tensor([[[1.0], [2.0], [4.0], [float('nan')]]])
    q = torch.tensor([[[0.0], [math.log(2.0)]], [[-math.log(2.0)], [100.0]]])
    o, tol = ref.attention(q, k, v, 1, lens=torch.tensor([3]), scale=1.0)
    want = [[7 / 3, (1 + 4 + 16) / 7], [(4 + 4 + 4) / 7, 4.0]]
    assert torch.allclose(o[..., 0], torch.tensor(want, dtype=torch.float64)) and (tol > 0).all()
    o, _ = ref.attention(q, k, v, 1, mask=torch.tensor([[True, False, True, False]]), scale=1.0)
    assert torch.allclose(o[0, :, 0], torch.tensor([2.5, (1 + 16) / 5], dtype=torch.float64))
    o, tol = ref.attention(q, k, v, 1, lens=torch.tensor([0]))
    assert not o.any() and not tol.any()
    # two query heads on one key head, two batches of queries on one of states
    from yanlongvla_b200 import definition
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(*s, generator=g) for s in ((4, 3, 16), (2, 5, 8), (2, 5, 8)))
    o, _ = ref.attention(q, k, v, 2, 1)
    both = [torch.cat((x, x), -1) for x in (k, v)]
    assert torch.allclose(o, definition.cross_attention(q, *both, 2).double(), atol=1e-5)
