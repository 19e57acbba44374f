"""The streaming-memory operators' host side without a GPU: what the handles refuse."""
import subprocess
import sys
from pathlib import Path

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


def without_binding(prepare):
    """Run `prepare` and then the import of the operators in a fresh interpreter: the C library answers, the streaming-memory
    operators raise ImportError with what to do about it. Returns the message."""
    code = prepare + '''
from yanlongvla_b200 import kernels as K
assert K.lib.tcq_abi_version() == 1 and K.quantize and K.gemm_tcq and K.TcqError
for call, n in ((K.rope_axes, 3), (K.kv8_append, 5), (K.kv8_read, 5), (K.kv8_attention, 4)):
    try:
        call(*[None] * n)
    except ImportError as e:
        message = str(e)
    else:
        raise SystemExit('no ImportError')
print(message)
'''
    r = subprocess.run([sys.executable, '-c', code], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    assert 'python -m yanlongvla_b200.build' in r.stdout
    return r.stdout


def test_the_package_imports_without_its_binding():
    without_binding("import sys; sys.modules['yanlongvla_b200._bind'] = None\n")


def test_a_binding_of_another_pytorch_is_not_used():
    assert 'this is 0.0.1' in without_binding("import torch; torch.__version__ = '0.0.1'\n")


def test_the_binding_is_for_this_pytorch():
    from yanlongvla_b200 import _bind
    assert _bind.torch_version == torch.__version__
