"""Where the output of the cross attention may lie: every byte of it apart from the rows that are read, gaps between them included.
Addresses are made up, so calls that are not refused are made only where there is no device to run them."""
import random

import pytest
import torch

AT = 1 << 24                                                                   # elements


def rows(base, batches, sb, n, st, width):
    return {base + i * sb + j * st + e for i in range(batches) for j in range(n) for e in range(0, width, 8)}


def test_against_all_addresses():
    if torch.cuda.is_available():
        pytest.skip('made-up addresses')
    from yanlongvla_b200 import _lib as L
    rng = random.Random(0)
    outcomes = {True: 0, False: 0}
    for _ in range(4000):
        B, S, T, N, heads, kv_heads, D = (rng.choice(v) for v in ((1, 2, 3), (1, 2), (1, 2, 5), (1, 2, 3, 7), (2, 4), (1, 2), (8, 16)))
        W, row = heads * D, kv_heads * D
        size = B * S * T * W
        st = lambda w: rng.choice((w, w + 8, 2 * w + 8, w + size, w + size + 8))
        q_st, k_st, v_st = st(W), st(row), st(row)
        sb = lambda n, s, w: rng.choice((n * s, n * s + size, w, 0, 8))                # sequences next to, among and on one another
        q_sb, k_sb, v_sb = sb(T, q_st, W), sb(N, k_st, row), sb(N, v_st, row)
        q, k, v = AT, 2 * AT, 3 * AT
        base, span = rng.choice(((q, (B * S - 1) * q_sb + (T - 1) * q_st + W), (k, (B - 1) * k_sb + (N - 1) * k_st + row),
                                 (v, (B - 1) * v_sb + (N - 1) * v_st + row)))
        out = base + 8 * rng.randint(-size // 8 - 1, span // 8 + 1)
        read = rows(q, B * S, q_sb, T, q_st, W) | rows(k, B, k_sb, N, k_st, row) | rows(v, B, v_sb, N, v_st, row)
        own = q == out and (T == 1 or q_st == W) and (B * S == 1 or q_sb == T * W)
        apart = own or not (read & set(range(out, out + size, 8)))
        status = L.lib.tcq_cross_attention(2 * q, q_sb, q_st, 2 * k, k_sb, k_st, 2 * v, v_sb, v_st, L.DT_BF16, 2 * out, None, None, 0, 1.0, B, S, T, N,
                                           heads, kv_heads, D, None)
        assert (status != 4) == apart, (B, S, T, N, W, row, q_sb, q_st, k_sb, k_st, v_sb, v_st, q, k, v, out)
        outcomes[apart] += 1
    assert min(outcomes.values()) > 300


def test_lengths_and_masks():
    """The output shares no byte with the lengths and the mask's rows either."""
    if torch.cuda.is_available():
        pytest.skip('made-up addresses')
    from yanlongvla_b200 import _lib as L
    B, T, N, W = 3, 2, 20, 16
    out, far, size = 1 << 24, 1 << 28, 2 * B * T * W                           # bytes

    def cross(lens=None, mask=None, mask_sb=0, states=N):
        return L.lib.tcq_cross_attention(far, T * W, W, 2 * far, N * W, W, 3 * far, N * W, W, L.DT_BF16, out, lens, mask, mask_sb, 1.0, B, 1, T, states, 2, 2, 8, None)
    for at, apart in ((out - 4 * B, True), (out - 4 * B + 4, False), (out, False), (out + size - 4, False), (out + size, True)):
        assert (cross(lens=at) != 4) == apart
        assert (cross(lens=at, states=0) != 4)                                 # without states nothing is read
    for sb in (N, N + 1, 0, size + N):
        span = (B - 1) * sb + N
        for at in range(out - span - 2, out + size + 3):
            apart = not any(at + i * sb < out + size and at + i * sb + N > out for i in range(B))
            assert (cross(mask=at, mask_sb=sb) != 4) == apart, (sb, at - out)
