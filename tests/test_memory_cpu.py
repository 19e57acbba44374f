"""Streaming-memory operators without a GPU: what the C ABI and the Python layer refuse (all before any CUDA call), and the
64-bit definitions the GPU tests use, pinned to hand-made cases."""
import ctypes

import pytest
import torch

import memory_ref as ref

A, B, C, D_, E = (i << 20 for i in range(1, 6))            # fake, aligned "device" addresses


@pytest.fixture(scope='module')
def L():
    from yanlongvla_b200 import _lib
    return _lib


def cache(L, **kw):
    f = dict(k=A, v=B, k_scale=C, v_scale=D_, pages=8, kv_heads=2, head_dim=64)
    f.update(kw)
    return L.Kv8Cache(*(f[n] for n in ('k', 'v', 'k_scale', 'v_scale', 'pages', 'kv_heads', 'head_dim')))


def plan(L, sections=(8, 12, 12), **kw):
    f = dict(cos=A, sin=B, positions=100, head_dim=64, axes=len(sections), pairs=0)
    f.update(kw)
    return L.RopePlan(f['cos'], f['sin'], f['positions'], f['head_dim'], f['axes'], f['pairs'], (ctypes.c_int * 4)(*sections))


def rope(L, p, x=A, dtype=None, st=64, out=B, pos=C, B_=1, T=1, heads=1):
    return L.lib.tcq_rope_axes(x, L.DT_BF16 if dtype is None else dtype, st, st, out, st, st, pos, None if p is None else ctypes.addressof(p),
                               B_, T, heads, 0, None)


def test_rope_axes_refuses(L):
    assert rope(L, None) == 4 and rope(L, plan(L), x=None) == 4 and rope(L, plan(L), pos=None) == 4 and rope(L, plan(L, cos=None)) == 4
    assert rope(L, plan(L), dtype=L.DT_I32) == 3 and rope(L, plan(L), dtype=9) == 3
    assert rope(L, plan(L, sections=(8, 12, 11))) == 1                       # do not add up to D / 2
    assert rope(L, plan(L, sections=(40, -4, -4))) == 1
    assert rope(L, plan(L, sections=(8, 8, 8, 8), axes=5)) == 1 and rope(L, plan(L, axes=0)) == 1
    assert rope(L, plan(L, sections=(16, 16), head_dim=65)) == 1 and rope(L, plan(L, sections=(150,), head_dim=300)) == 1
    assert rope(L, plan(L, positions=0)) == 1 and rope(L, plan(L), heads=0) == 1 and rope(L, plan(L), T=0) == 1
    assert rope(L, plan(L, cos=A + 4)) == 2 and rope(L, plan(L), x=A + 1) == 2


def append(L, c, k=A, v=B, st=128, dtype=None, table=C, blocks=4, start=D_, pos=None, p=None, B_=1, T=1):
    return L.lib.tcq_kv8_append(ctypes.addressof(c) if c is not None else None, k, st, st, v, st, st, L.DT_BF16 if dtype is None else dtype,
                                table, blocks, start, None, pos, None if p is None else ctypes.addressof(p), B_, T, None)


def test_append_refuses(L):
    c = cache(L)
    assert append(L, None) == 4 and append(L, c, k=None) == 4 and append(L, c, table=None) == 4 and append(L, c, start=None) == 4
    assert append(L, c, p=plan(L)) == 4                                       # a plan without positions
    assert append(L, cache(L, k_scale=None)) == 4
    assert append(L, c, dtype=L.DT_F32) == 3
    for d in (0, 16, 40, 72, 112, 144, 256):
        assert append(L, cache(L, head_dim=d)) == 1
    assert append(L, cache(L, pages=0)) == 1 and append(L, cache(L, kv_heads=0)) == 1
    assert append(L, c, T=0) == 1 and append(L, c, B_=0) == 1 and append(L, c, blocks=0) == 1
    assert append(L, c, p=plan(L, sections=(16,), head_dim=32), pos=E) == 1    # another head width
    assert append(L, c, p=plan(L, pairs=1), pos=E) == 1                       # the pair layout
    assert append(L, c, k=A + 2) == 2 and append(L, c, st=129) == 2 and append(L, cache(L, v=B + 8)) == 2


def test_read_refuses(L):
    def read(c, k=A, v=B, dtype=L.DT_BF16, table=C, blocks=4, begin=D_, lens=E, B_=1, T=1):
        return L.lib.tcq_kv8_read(ctypes.addressof(c), k, v, dtype, table, blocks, begin, lens, B_, T, None)
    c = cache(L)
    assert read(c, k=None) == 4 and read(c, begin=None) == 4 and read(c, lens=None) == 4
    assert read(c, dtype=L.DT_I32) == 3 and read(c, T=0) == 1 and read(c, blocks=0) == 1 and read(c, v=B + 4) == 2
    assert read(cache(L, head_dim=72)) == 1


def test_attention_refuses(L):
    def attend(c, q=A, dtype=L.DT_BF16, st=512, out=B, table=C, blocks=4, lens=D_, B_=1, T=1, heads=8, ws=E, ws_bytes=1 << 30):
        return L.lib.tcq_kv8_attention(ctypes.addressof(c), q, dtype, st, st, out, table, blocks, lens, None, 1, 0.125, B_, T, heads, ws,
                                       ws_bytes, None)
    c = cache(L)
    assert attend(c, q=None) == 4 and attend(c, out=None) == 4 and attend(c, lens=None) == 4
    assert attend(c, dtype=L.DT_F32) == 3
    assert attend(c, heads=7) == 1 and attend(c, heads=0) == 1 and attend(c, T=0) == 1 and attend(c, blocks=0) == 1
    assert attend(c, blocks=1 << 26) == 1                                     # more tokens than 31 bits count
    assert attend(c, q=A + 2) == 2 and attend(c, st=513) == 2 and attend(c, out=B + 2) == 2
    assert attend(c, ws=None) == 7 and attend(c, ws_bytes=0) == 7
    assert attend(cache(L, head_dim=72)) == 1
    assert L.lib.tcq_kv8_attention_workspace(0, 1, 8, 2, 64, 4) == 0 and L.lib.tcq_kv8_attention_workspace(1, 1, 8, 2, 64, 4) > 0


def test_python_layer_refuses_cpu_tensors():
    from yanlongvla_b200 import kernels as K
    with pytest.raises(K.TcqError):
        K.RopeAxes(torch.zeros(4, 8), torch.zeros(4, 8), (8,))
    with pytest.raises(K.TcqError):
        K.KV8Cache.empty(2, 2, 64, device='cpu')


def test_reference_rotary():
    cos, sin = torch.tensor([[1.0, 1.0], [0.0, 0.6]]), torch.tensor([[0.0, 0.0], [1.0, 0.8]])
    x = torch.tensor([1.0, 2.0, 3.0, 4.0], dtype=torch.float64).view(1, 1, 1, 4)
    pos = torch.tensor([[[1]], [[0]]])
    assert ref.rotary(x, pos, cos, sin, (1, 1), False).view(-1).tolist() == [-3.0, 2.0, 1.0, 4.0]
    assert ref.rotary(x, pos, cos, sin, (1, 1), True).view(-1).tolist() == [-2.0, 1.0, 3.0, 4.0]
    back = ref.rotary(ref.rotary(x, pos, cos, sin, (1, 1), True), pos, cos, sin, (1, 1), True, inverse=True)
    assert torch.allclose(back, x)


def test_reference_attention():
    class Cache:
        kv_heads, head_dim = 1, 2
        k = torch.zeros(2, 1, 64, 2, dtype=torch.int8)
        v = torch.zeros(2, 1, 2, 64, dtype=torch.int8)
        k_scale = v_scale = torch.ones(2, 1)
    Cache.k[1, 0, :3, 0] = torch.tensor([0, 1, 0], dtype=torch.int8)
    Cache.v[1, 0, 0, :3] = torch.tensor([3, 6, 9], dtype=torch.int8)
    q = torch.tensor([[[0.0, 0.0], [0.0, 5.0], [2.0 ** 0.5 * 50, 0.0]]])
    table = torch.tensor([[1, 0]])
    o, a = ref.attention(q, Cache, table, [3])
    assert torch.allclose(o[0, :, 0], torch.tensor([3.0, 4.5, 6.0], dtype=torch.float64)) and torch.equal(o, a)
    o, _ = ref.attention(q, Cache, table, [1])                        # the first two queries lie before the first token
    assert o[0, :, 0].tolist() == [0.0, 0.0, 3.0]
    o, _ = ref.attention(q, Cache, table, [3], causal=False, count=[2])
    assert torch.allclose(o[0, :, 0], torch.tensor([6.0, 6.0, 0.0], dtype=torch.float64))
