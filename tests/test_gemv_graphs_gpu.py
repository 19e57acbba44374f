"""CUDA graphs with the fused decode-GEMV: each graph has a zero-filled workspace of its own (partial sums and arrival counters), so
graphs may be replayed in any order, on any streams, between calls of any size."""
import pytest
import torch

from test_memory_graphs_gpu import nodes

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def K():
    if not torch.cuda.is_available():
        pytest.skip('no CUDA device')
    from yanlongvla_b200 import kernels
    return kernels


class Step:
    """One product of random weights on buffers of its own, its output outside a graph, and a graph of it."""

    def __init__(self, K, M, N, Kd, tc=False, seed=0):
        g = torch.Generator(device='cuda').manual_seed(seed)
        ri = lambda lo, hi, dt, *shape: torch.randint(lo, hi, shape, device='cuda', generator=g, dtype=dt)
        bits, t8 = ri(-32768, 32768, torch.int16, N // 16 * Kd // 16, 32), ri(-127, 128, torch.int8, 512, 2)
        q = ri(-128, 128, torch.int8, M, Kd) if tc else ri(-2 ** 31, 2 ** 31 - 1, torch.int32, Kd // 4, M)
        s, rs = 0.01 + torch.rand(M, device='cuda', generator=g), 0.01 + torch.rand(N, device='cuda', generator=g)
        self.z = torch.empty(M, N, device='cuda')
        self.call = lambda: (K.gemm_tcq_tc if tc else K.gemm_tcq)(bits, t8, q, s, rs, self.z, Kd)
        self.call()
        self.want = self.z.clone()
        self.z.fill_(float('nan'))

    def run(self):
        torch.full((48 << 20,), 255, dtype=torch.uint8, device='cuda')        # so that new memory is not zero by chance
        self.call()

    def capture(self, **kw):
        torch.cuda.synchronize()
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph, **kw):
            self.run()
        return self

    def check(self):
        torch.cuda.synchronize()
        assert torch.equal(self.z, self.want)
        self.z.fill_(float('nan'))


def test_a_second_graph_clears_its_own_workspace(K):
    step = Step(K, 1, 1536, 4096)
    for calls in (1, 1, 3):
        g = torch.cuda.CUDAGraph(keep_graph=True)
        with torch.cuda.graph(g):
            for _ in range(calls):
                step.call()
        assert nodes(g) == calls + 1


def test_graphs_in_any_order_and_on_two_streams(K):
    a, b, c = Step(K, 1, 1536, 4096, seed=1).capture(), Step(K, 8, 4096, 2048, seed=2).capture(), Step(K, 17, 1536, 4096, tc=True, seed=3).capture()
    for step in (c, b, a, a, c, b):
        step.graph.replay()
        step.check()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(10):
        for step, s in zip((a, b, c), streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                for _ in range(4):
                    step.graph.replay()
        for step in (a, b, c):
            step.check()


def test_a_larger_call_between_replays(K):
    """The stream's workspace is replaced by a larger call: a graph captured there before gives its output still, and leaves the
    tensors that took the old workspace's place alone."""
    small, large = Step(K, 1, 1536, 4096, seed=1), Step(K, 16, 32768, 256, seed=2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        small.run()
        small.check()
    small.capture(stream=s)
    with torch.cuda.stream(s):
        small.graph.replay()
        small.check()
        large.run()
        large.check()
        kept = [torch.full((n << 18,), 90, dtype=torch.uint8, device='cuda') for n in (1, 1, 1, 2, 4, 8, 16, 32)]
        for _ in range(3):
            small.graph.replay()
            small.check()
            large.run()
            large.check()
    assert all(bool((t == 90).all()) for t in kept)
