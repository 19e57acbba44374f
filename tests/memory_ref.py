"""The streaming-memory operators in 64 bits, written from their definitions (for the tests; runs on any device)."""
import math

import torch

BLOCK = 64


def rotary(x, pos, cos, sin, sections, pairs, inverse=False):
    """x (B, T, heads, D) FP64 -> the turned heads."""
    half = x.shape[-1] // 2
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    c = torch.stack([cos[:, j].double()[pos[axis[j]].long()] for j in range(half)], -1)[:, :, None]
    s = torch.stack([sin[:, j].double()[pos[axis[j]].long()] for j in range(half)], -1)[:, :, None]
    s = -s if inverse else s
    y = torch.empty_like(x)
    i0, i1 = (slice(0, None, 2), slice(1, None, 2)) if pairs else (slice(0, half), slice(half, None))
    y[..., i0] = x[..., i0] * c - x[..., i1] * s
    y[..., i1] = x[..., i0] * s + x[..., i1] * c
    return y


def values(cells, scale, table_row, n, transposed):
    """The first n tokens (n, heads, D) FP64 that one sequence's table row stands for."""
    pages = table_row[:(n + BLOCK - 1) // BLOCK].long()
    x = cells[pages].double() * scale[pages].double()[..., None, None]
    x = x.permute(0, 3, 1, 2) if transposed else x.transpose(1, 2)
    return x.reshape(-1, cells.shape[1], x.shape[-1])[:n]


def attention(q, cache, table, lens, count=None, causal=True, scale=None):
    """q (B, T, heads * D). Returns the output (B, T, heads * D) FP64 and, for each output, sum_j p_j |v_j| (the scale that errors
    of the weights act on)."""
    B, T, W = q.shape
    Hk, D = cache.kv_heads, cache.head_dim
    G = W // D // Hk
    scale = D ** -0.5 if scale is None else scale
    o = torch.zeros(B, T, Hk, G, D, dtype=torch.float64, device=q.device)
    a = torch.zeros_like(o)
    for b in range(B):
        n = int(lens[b])
        cnt = T if count is None else int(count[b])
        if n == 0 or cnt == 0:
            continue
        k = values(cache.k, cache.k_scale, table[b], n, False)
        v = values(cache.v, cache.v_scale, table[b], n, True)
        qq = q[b, :cnt].double().view(cnt, Hk, G, D)
        s = torch.einsum('thgd,khd->thgk', qq, k) * scale
        if causal:
            hide = torch.arange(n, device=q.device)[None] > n - cnt + torch.arange(cnt, device=q.device)[:, None]
            s = s.masked_fill(hide[:, None, None], -math.inf)
        top = s.amax(-1, keepdim=True)
        e = (s - torch.where(top == -math.inf, 0.0, top)).exp()
        total = e.sum(-1, keepdim=True)
        p = e / torch.where(total == 0, 1.0, total)
        o[b, :cnt] = torch.einsum('thgk,khd->thgd', p, v)
        a[b, :cnt] = torch.einsum('thgk,khd->thgd', p, v.abs())
    return o.view(B, T, W), a.view(B, T, W)
