"""Streaming-memory operators at the edges of what a caller may pass: NaN queries, odd strides of dimensions of size one, flags
without a truth value."""
import pytest
import torch

from test_memory_gpu import K, attention_case, check_attention, gen, i32, make_cache, rope_case  # noqa: F401  (K is the module's fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('T,heads,kv_heads,D,n', [
    (1, 8, 2, 64, 203), (1, 4, 1, 64, 9000), (8, 8, 2, 128, 900),             # few rows: one CTA, parts of a unit, in the workspace
    (160, 8, 2, 64, 2000), (40, 8, 2, 128, 3000), (100, 2, 2, 48, 900),       # a cluster's CTAs divide a unit's tiles
    (64, 8, 8, 96, 64)])                                                      # one CTA to a unit
@pytest.mark.parametrize('causal', [True, False])
def test_attention_nan_query_stays_in_its_row(K, T, heads, kv_heads, D, n, causal):
    """A query row with a NaN has a NaN output, every other row its own bits."""
    q, cache, table = attention_case(K, 1, T, heads, kv_heads, D, [n])
    want = K.kv8_attention(q, cache, table, i32([n]), causal=causal)
    for t, h in ((T // 2, heads - 1), (T - 1, 0)):
        bad = q.clone()
        bad[0, t, h * D + 5] = float('nan')
        o = K.kv8_attention(bad, cache, table, i32([n]), causal=causal)
        row = o[0, t, h * D:(h + 1) * D]
        assert row.isnan().all()
        row.copy_(want[0, t, h * D:(h + 1) * D])
        assert torch.equal(o, want)


@pytest.mark.parametrize('D', [48, 64, 128])
def test_attention_scores_are_read_before_weights_replace_them(K, D):
    """The weights of one page of a tile take the place of scores of both pages. With many tiles, most of which move no reference,
    every run gives the same bits and the definition's values, also next to other work on the device."""
    lens = [1500, 1411]
    q, cache, table = attention_case(K, 2, 700, 32, 8, D, lens)
    want = check_attention(K, q, cache, table, lens)
    other, a = torch.cuda.Stream(), torch.randn(2048, 2048, device='cuda')
    for i in range(20):
        with torch.cuda.stream(other):
            for _ in range(i % 4):
                a @ a
        assert torch.equal(K.kv8_attention(q, cache, table, i32(lens)), want)
    torch.cuda.synchronize()
