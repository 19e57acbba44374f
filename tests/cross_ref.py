"""Cross attention in 64 bits, written from its definition (for the tests; runs on any device)."""
import math

import torch


def attention(q, k, v, heads, kv_heads=None, lens=None, mask=None, scale=None):
    """q (B * S, T, heads * D), k, v (B, N, kv_heads * D). Returns the output FP64 and a bound on what an implementation may be off that
    forms scores and sums in FP32, rounds the weights to the type once and the output once:

      weights   a half step of the type each, u sum_j p_j |v_j|
      scores    D products in FP32: an error of D 2^-23 sum |q k| scale in the exponent, and 2^-21 of the exponential; a weight is off by
                that share, and so is the sum of all
      sums      N / 32 + 64 additions in FP32
      FP16      weights below 2^-14 of the smallest reference (2^5) lose steps of 2^-24: 2^-29 sum |v|
      output    u |o|
    """
    BS, T, W = q.shape
    B, N, Wk = k.shape
    kv_heads = kv_heads or heads
    D, S, G = W // heads, BS // B, heads // kv_heads
    scale = D ** -0.5 if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    seen = torch.ones(B, N, dtype=torch.bool, device=q.device)
    if lens is not None:
        seen &= torch.arange(N, device=q.device) < lens[:, None]
    if mask is not None:
        seen &= mask
    o = torch.zeros(B, kv_heads, S * T * G, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(o)
    qq = q.double().view(B, S * T, kv_heads, G, D).transpose(1, 2).reshape(B, kv_heads, S * T * G, D)
    for b in range(B):
        at = seen[b].nonzero()[:, 0]
        if not len(at):
            continue
        kk, vv = (x[b, at].double().view(-1, kv_heads, D).transpose(0, 1) for x in (k, v))
        s = qq[b] @ kk.transpose(1, 2) * scale
        p = torch.softmax(s, -1)
        o[b] = p @ vv
        a = p @ vv.abs()
        size = (qq[b].abs() @ kk.abs().transpose(1, 2)).amax(-1, keepdim=True) * abs(scale)
        share = u + 2 * (D * 2.0 ** -23 * size + 2.0 ** -21) + (len(at) / 32 + 64) * 2.0 ** -23
        tol[b] = share * a + u * o[b].abs()
        if q.dtype == torch.float16:
            tol[b] += 2.0 ** -29 * vv.abs().sum(1, keepdim=True) + 2.0 ** -25          # and outputs below FP16's normal range
    back = lambda x: x.view(B, kv_heads, S * T, G, D).transpose(1, 2).reshape(BS, T, W)
    return back(o), back(tol)
