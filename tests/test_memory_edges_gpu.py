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


def odd_rows(x):
    """x (1, 1, W) as a view whose strides of the two dimensions of size one are odd."""
    W = x.shape[2]
    flat = torch.zeros(W + 17, device='cuda', dtype=x.dtype)
    flat[8:8 + W] = x[0, 0]
    y = flat[None, None, 8:8 + W]
    assert y.stride() == (W + 17, W + 17, 1) and (W + 17) % 2 == 1
    return y


def test_strides_of_dimensions_of_size_one_do_not_count(K):
    """One token of one sequence, cut from a buffer of odd length: the strides that nothing steps by are no reason to refuse it."""
    g = gen(21)
    heads, D = 2, 64
    rope, pos, _ = rope_case(K, D, 3, 1, 1, g, False)
    k, v = (torch.randn(1, 1, heads * D, device='cuda', generator=g).bfloat16() for _ in range(2))
    q = torch.randn(1, 1, 4 * heads * D, device='cuda', generator=g).bfloat16()
    table = i32([[2, 0]])
    caches = [make_cache(K, 3, heads, D, gen(22)) for _ in range(2)]
    K.kv8_append(caches[0], k, v, table, i32([70]), rope=rope, pos=pos)
    K.kv8_append(caches[1], odd_rows(k), odd_rows(v), table, i32([70]), rope=rope, pos=pos)
    for name in ('k', 'v', 'k_scale', 'v_scale'):
        assert torch.equal(getattr(caches[0], name), getattr(caches[1], name))
    assert torch.equal(K.rope_axes(odd_rows(q), pos, rope), K.rope_axes(q, pos, rope))
    assert torch.equal(K.kv8_attention(odd_rows(q), caches[0], table, i32([71])), K.kv8_attention(q, caches[0], table, i32([71])))


def test_flags_without_a_truth_value_are_refused(K):
    """causal and inverse are asked for their truth; an object that has none raises its own error and nothing is launched."""
    q, cache, table = attention_case(K, 1, 3, 4, 2, 64, [70])
    rope, pos, _ = rope_case(K, 64, 2, 3, 1, gen(1), False)
    launches = dict(K.LAUNCHES)
    with pytest.raises(RuntimeError, match='ambiguous'):
        K.kv8_attention(q, cache, table, i32([70]), causal=torch.ones(2))
    with pytest.raises(RuntimeError, match='ambiguous'):
        K.rope_axes(q, pos, rope, inverse=torch.ones(2))
    assert K.LAUNCHES == launches
    assert torch.equal(K.kv8_attention(q, cache, table, i32([70]), causal=1), K.kv8_attention(q, cache, table, i32([70])))
