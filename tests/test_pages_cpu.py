"""The page operators without a GPU: what the C ABI and the handle refuse before any CUDA call, and the model the GPU tests compare
with, pinned to hand-made cases."""
import ctypes

import pytest
import torch

import pages_ref as ref

A, B, C, D_, E, F_ = (i << 20 for i in range(1, 7))            # fake, aligned "device" addresses


@pytest.fixture(scope='module')
def L():
    from yanlongvla_b200 import _lib
    return _lib


def caches(L, n=2, **kw):
    made = (L.Kv8Cache * max(n, 1))()
    for i in range(n):
        f = dict(k=A, v=B, k_scale=C, v_scale=D_, pages=8, kv_heads=2, head_dim=64)
        f.update(kw if i == n - 1 else {})
        made[i] = L.Kv8Cache(*(f[x] for x in ('k', 'v', 'k_scale', 'v_scale', 'pages', 'kv_heads', 'head_dim')))
    return made


def test_bookkeeping_refuses(L):
    def fork(refs=A, pages=8, table=B, blocks=4, lens=C, more=D_, n=2):
        return L.lib.tcq_kv8_fork(refs, pages, table, blocks, lens, more, n, None)

    def free(refs=A, pages=8, table=B, blocks=4, lens=C, more=D_, n=2):
        return L.lib.tcq_kv8_free(refs, pages, table, blocks, lens, more, n, None)

    def reserve(refs=A, pages=8, table=B, blocks=4, lens=C, more=D_, n=2, granted=E, copies=F_):
        return L.lib.tcq_kv8_reserve(refs, pages, table, blocks, lens, more, granted, copies, n, None)
    for call in (fork, free, reserve):
        for name in ('refs', 'table', 'lens', 'more'):
            assert call(**{name: None}) == 4
        assert call(pages=0) == 1 and call(pages=1 << 30) == 1 and call(blocks=0) == 1 and call(n=0) == 1 and call(n=4097) == 1
    assert reserve(granted=None) == 4 and reserve(copies=None) == 4


def test_copy_refuses(L):
    def copy(c, layers=2, copies=E, n=1):
        return L.lib.tcq_kv8_copy(c, layers, copies, n, None)
    assert copy(None) == 4 and copy(caches(L), layers=0) == 4 and copy(caches(L), copies=None) == 4 and copy(caches(L), n=0) == 1
    assert copy(caches(L, pages=9)) == 1 and copy(caches(L, kv_heads=1)) == 1 and copy(caches(L, head_dim=32)) == 1     # of two shapes
    assert copy(caches(L, v=B + 8)) == 2 and copy(caches(L, k=None)) == 4 and copy(caches(L, head_dim=72)) == 1


def test_compact_refuses(L):
    def compact(c, layers=2, table=A, blocks=4, lens=B, index=C, tokens=70, kept=None, new=E, new_blocks=2, n=1):
        return L.lib.tcq_kv8_compact(c, layers, table, blocks, lens, index, tokens, kept, new, new_blocks, n, None)
    c = caches(L)
    for name in ('table', 'lens', 'index', 'new'):
        assert compact(c, **{name: None}) == 4
    assert compact(None) == 4 and compact(c, layers=0) == 4
    for name in ('blocks', 'tokens', 'new_blocks', 'n'):
        assert compact(c, **{name: 0}) == 1
    assert compact(caches(L, pages=9)) == 1 and compact(caches(L, k=A + 4)) == 2


def test_the_handle_refuses():
    from yanlongvla_b200 import kernels as K
    from test_memory_host_cpu import OnDevice
    with pytest.raises(K.TcqError):
        K.KV8Pages.empty(4, device='cpu')
    for shape, dtype in (((4,), torch.int64), ((2, 2), torch.int32), ((0,), torch.int32), ((1 << 30,), torch.int32)):
        with pytest.raises(K.TcqError, match='refs must be'):
            K.KV8Pages(OnDevice(shape, dtype, 0))
    assert K.KV8Pages(OnDevice((7,), torch.int32, 1)).pages == 7


def test_operators_refuse_what_is_not_theirs():
    from yanlongvla_b200 import kernels as K
    x = torch.zeros(2, 2, dtype=torch.int32)
    for call in (K.kv8_fork, K.kv8_reserve, K.kv8_free):
        with pytest.raises(TypeError):
            call(None, x, x[0], x[0])
        with pytest.raises(TypeError):
            call(x, None, x[0], x[0])
    for c in (None, [None], [x]):
        with pytest.raises(TypeError):
            K.kv8_copy(c, x)
        with pytest.raises(TypeError):
            K.kv8_compact(c, x, x[0], x, x)
    with pytest.raises(K.TcqError, match='no cache'):
        K.kv8_copy([], x)


def test_model_of_the_pages():
    m = ref.Pages(6, 3, 4)
    assert m.reserve([70, 0, 1]) == ([70, 0, 1], [[-1] * 3, [-1] * 3]) and m.table == [[0, 1, -1, -1], [-1] * 4, [2, -1, -1, -1]]
    m.lens = [70, 0, 1]
    m.fork([0, 0, -1])
    assert m.refs == [2, 2, 0, 0, 0, 0] and m.lens == [70, 70, 0] and m.table[1] == [0, 1, -1, -1]
    assert m.reserve([1, 60, 0]) == ([1, 60, 0], [[1, -1, -1], [2, -1, -1]]) and m.table[:2] == [[0, 2, -1, -1], [0, 1, 3, -1]]
    m.lens = [71, 130, 0]
    assert m.reserve([200, 1, 1]) == ([0, 1, 1], [[-1] * 3, [-1] * 3])         # 200 more do not fit the table
    m.lens[1:] = [131, 1]
    assert m.table[2] == [4, -1, -1, -1]
    assert m.reserve([0, 100, 64])[0] == [0, 100, 0]                           # pages 5 and none
    m.free([70, 0, 5])
    assert m.refs == [1, 0, 1, 0, 1, 0] and m.lens == [70, 0, 1]


def test_packing():
    k = torch.zeros(3, 1, 64, 2, dtype=torch.int8)
    k[0, 0, 3], k[1, 0, 0] = torch.tensor([100, -7]), torch.tensor([50, 127])
    scale = torch.tensor([[0.5], [2.0], [0.0]])
    (x, s), = ref.packed(k, scale, [0, 1, 2], [64, 3, 130], False)
    assert s.tolist() == [2.0] and x[0, :3].tolist() == [[50, 127], [25, -2], [0, 0]] and not x[0, 3:].any()   # -1.75 rounds to -2
    (y, _), = ref.packed(k.transpose(2, 3).contiguous(), scale, [0, 1, 2], [64, 3, 130], True)
    assert torch.equal(y, x.transpose(1, 2))
