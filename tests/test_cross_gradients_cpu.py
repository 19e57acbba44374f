"""Cross attention forms no derivative: tensors that ask for one are refused, in either mode, before anything else is looked at."""
import pytest
import torch
import torch.autograd.forward_ad as fwd


def test_tangents_and_gradients_are_refused():
    from yanlongvla_b200 import kernels as K
    x = torch.zeros(2, 3, 64, dtype=torch.bfloat16)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for grad in (torch.enable_grad, torch.no_grad):                        # no_grad leaves forward mode on
            with grad():
                for a in ((dual, x, x), (x, dual, x), (x, x, dual), (x, x, x, dual)):
                    with pytest.raises(K.TcqError, match='tangent'):
                        K.cross_attention(*a[:3], 1, out=a[3] if len(a) > 3 else None)
        with pytest.raises(K.TcqError, match='CUDA'):
            K.cross_attention(*(fwd.unpack_dual(dual).primal,) * 3, 1)
    with pytest.raises(K.TcqError, match='CUDA'):                              # outside the level there is none
        K.cross_attention(dual, dual, dual, 1)
    leaf = x.clone().requires_grad_()
    for a in ((leaf, x, x), (x, leaf, x), (x, x, leaf), (x, x, x, leaf)):
        with pytest.raises(K.TcqError, match='gradient'):
            K.cross_attention(*a[:3], 1, out=a[3] if len(a) > 3 else None)
    with torch.no_grad(), pytest.raises(K.TcqError, match='CUDA'):
        K.cross_attention(leaf, leaf, leaf, 1)
    with torch.inference_mode(), pytest.raises(K.TcqError, match='CUDA'):
        y = torch.zeros(2, 3, 64, dtype=torch.bfloat16)
        K.cross_attention(y, x, leaf, 1, out=y)
