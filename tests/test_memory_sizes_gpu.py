"""Streaming-memory operators at sizes that take the kernels' other shapes: rotary launches with four heads to a thread, prompts of
many tiles with one CTA to a unit, tables much wider than their sequences. Checks and tolerances are those of test_memory_gpu.py."""
import pytest
import torch

from test_memory_gpu import (BF16, F16, F32, K, attention_case, check_attention, gen, rope_case,  # noqa: F401
                             test_rope_axes as check_rope_axes)

check_rope_axes.__test__ = False
pytestmark = pytest.mark.gpu


# rows * units of a head * heads above 2048 to an SM (303,104 on 148): four heads to a thread, heads that do not divide by four
@pytest.mark.parametrize('pairs', [False, True])
@pytest.mark.parametrize('B,T,heads,D,axes,dtype', [
    (2, 8001, 5, 64, 3, BF16), (1, 8001, 11, 64, 2, F16), (1, 2001, 40, 64, 3, BF16), (2, 4001, 5, 128, 4, F16), (1, 4001, 7, 128, 1, F32),
    (3, 3001, 13, 72, 2, BF16), (1, 4001, 6, 256, 3, BF16), (2, 9001, 33, 6, 1, F32), (1, 1201, 40, 128, 2, F16)])
def test_rope_axes_many_tokens(K, B, T, heads, D, axes, dtype, pairs):
    check_rope_axes(K, B, T, heads, D, axes, dtype, pairs)


@pytest.mark.parametrize('pairs', [False, True])
@pytest.mark.parametrize('width,first', [(1024, 256), (1030, 6), (777, 1)])
def test_rope_axes_many_tokens_strided(K, width, first, pairs):
    g = gen(12)
    B, T, heads, D = 2, 8001, 7, 64
    rope, pos, _ = rope_case(K, D, 3, T, B, g, pairs)
    big = torch.randn(B, T, width, device='cuda', generator=g).bfloat16()
    x = big[..., first:first + heads * D]
    want = K.rope_axes(x.contiguous(), pos, rope)
    assert torch.equal(K.rope_axes(x, pos, rope), want)
    keep = big.clone()
    K.rope_axes(x, pos, rope, out=x)
    assert torch.equal(x, want)
    big[..., first:first + heads * D] = keep[..., first:first + heads * D]
    assert torch.equal(big, keep)


@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('B,T,heads,kv_heads,D', [(8, 700, 16, 8, 64), (8, 700, 16, 8, 128), (5, 333, 40, 8, 80), (24, 40, 16, 8, 64), (24, 40, 16, 8, 128),
                                                  (7, 64, 48, 24, 96)])
def test_prompts_of_many_tiles(K, B, T, heads, kv_heads, D, causal):
    """At least as many units as SMs: one CTA walks all tiles of its rows; two groups of rows, and one."""
    lens = [T + 411 + 97 * (b % 5) for b in range(B)]
    q, cache, table = attention_case(K, B, T, heads, kv_heads, D, lens, dtype=F16 if D == 128 else BF16)
    check_attention(K, q, cache, table, lens, causal=causal)
    count = [(b * 131 + 17) % (T + 1) for b in range(B)]
    ragged = [0 if b == 3 else 1 + (b * 389) % (T + 800) for b in range(B)]
    check_attention(K, q, cache, table, ragged, count=count, causal=causal)


@pytest.mark.parametrize('T', [1, 17, 40, 160, 700])
@pytest.mark.parametrize('heads,kv_heads,D', [(8, 8, 48), (8, 2, 128)])
def test_tables_wider_than_their_sequences(K, T, heads, kv_heads, D):
    lens = [T, T + 70, 1, 203]
    q, cache, table = attention_case(K, 4, T, heads, kv_heads, D, lens, extra=100)
    o = check_attention(K, q, cache, table, lens)
    narrow = table[:, :(max(lens) + 63) // 64].contiguous()
    check_attention(K, q, cache, narrow, lens)
    assert torch.isfinite(o).all()
