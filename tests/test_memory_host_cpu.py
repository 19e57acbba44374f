"""The streaming-memory operators' host side without a GPU: what the handles refuse."""
import pytest
import torch


class OnDevice:
    """What the handles ask of a tensor, for a device that this machine need not have."""
    is_cuda = True

    def __init__(self, shape, dtype, index):
        self.shape, self.dtype, self.device = torch.Size(shape), dtype, torch.device('cuda', index)

    def is_contiguous(self):
        return True

    def dim(self):
        return len(self.shape)

    def get_device(self):
        return self.device.index

    def data_ptr(self):
        return 1 << 20


def cache_parts(devices, pages=3, heads=2, D=64):
    shapes = ((pages, heads, 64, D), (pages, heads, D, 64), (pages, heads), (pages, heads))
    kinds = (torch.int8, torch.int8, torch.float32, torch.float32)
    return [OnDevice(s, t, i) for s, t, i in zip(shapes, kinds, devices)]


def test_a_cache_is_on_one_device():
    from yanlongvla_b200 import kernels as K
    for devices in ((0, 1, 0, 0), (1, 0, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1)):
        with pytest.raises(K.TcqError, match='several devices'):
            K.KV8Cache(*cache_parts(devices))
    assert K.KV8Cache(*cache_parts((1, 1, 1, 1)))._handle.device == 1


def test_tables_are_on_one_device():
    from yanlongvla_b200 import kernels as K
    with pytest.raises(K.TcqError, match='several devices'):
        K.RopeAxes(OnDevice((9, 32), torch.float32, 0), OnDevice((9, 32), torch.float32, 1), (32,))
    assert K.RopeAxes(*(OnDevice((9, 32), torch.float32, 1) for _ in range(2)), (16, 16))._handle.device == 1


def test_a_cache_of_another_rank_is_refused():
    from yanlongvla_b200 import kernels as K
    k, v, ks, vs = cache_parts((0, 0, 0, 0))
    for shape in ((3, 64, 64), (3, 2, 1, 64, 64)):
        with pytest.raises(K.TcqError, match='must be'):
            K.KV8Cache(OnDevice(shape, torch.int8, 0), v, ks, vs)
