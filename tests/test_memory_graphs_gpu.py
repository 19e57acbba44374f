"""CUDA graphs with attention over the cache: each graph has a workspace of its own, cleared by its own replay, so graphs may be
replayed in any order, on any streams, between calls of any size, and a graph's memory is nobody else's.

The cases divide a sequence over many warps, whose arrival counters and parts are what the workspace holds. Before the
attention each captured step fills memory with ones and lets it go, so that a workspace in the graph's pool is not zero by chance."""
import ctypes

import pytest
import torch

from test_memory_gpu import K, attention_case, i32  # noqa: F401  (K is the module's fixture)

pytestmark = pytest.mark.gpu


class Step:
    """One attention call on buffers of its own, its expected output, and a graph of it."""

    def __init__(self, K, T, D=64, n=9000, seed=0):
        self.K = K
        self.q, self.cache, self.table = attention_case(K, 1, T, 4, 1, D, [n], seed=seed)
        self.lens = i32([n])
        self.want = K.kv8_attention(self.q, self.cache, self.table, self.lens)
        self.out = torch.empty_like(self.want)
        self.reset()

    def reset(self):
        self.out.fill_(float('nan'))

    def run(self):
        torch.full((48 << 20,), 255, dtype=torch.uint8, device='cuda')
        self.K.kv8_attention(self.q, self.cache, self.table, self.lens, out=self.out)

    def capture(self, **kw):
        torch.cuda.synchronize()
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph, **kw):
            self.run()
        return self

    def check(self):
        torch.cuda.synchronize()
        assert torch.equal(self.out, self.want)
        self.reset()


def nodes(graph):
    """How many nodes a torch.cuda.CUDAGraph(keep_graph=True) has."""
    rt = ctypes.CDLL('libcudart.so.12')                       # the one PyTorch has loaded
    n = ctypes.c_size_t(0)
    assert rt.cudaGraphGetNodes(ctypes.c_void_p(graph.raw_cuda_graph()), None, ctypes.byref(n)) == 0
    return n.value


def test_a_second_graph_clears_its_own_workspace(K):
    """Two graphs captured on one stream: the second, too, holds a node that clears the counters (looked at, not replayed); more
    calls in a graph share one."""
    step = Step(K, 1)
    for calls in (1, 1, 3):
        g = torch.cuda.CUDAGraph(keep_graph=True)
        with torch.cuda.graph(g):
            for _ in range(calls):
                K.kv8_attention(step.q, step.cache, step.table, step.lens, out=step.out)
        assert nodes(g) == calls + 1


@pytest.mark.parametrize('Ta,Tb', [(1, 1), (1, 8), (8, 2)])
def test_graphs_in_any_order(K, Ta, Tb):
    a, b = Step(K, Ta, seed=1).capture(), Step(K, Tb, seed=2).capture()
    for step in (b, a, a, b, b, a):
        step.graph.replay()
        step.check()


def test_graphs_on_two_streams(K):
    a, b = Step(K, 1, seed=1).capture(), Step(K, 4, n=40000, seed=2).capture()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for step, s in zip((a, b), streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                for _ in range(4):
                    step.graph.replay()
        a.check()
        b.check()


def test_a_larger_call_between_replays(K):
    """A step captured on a stream that has been warmed up; then a call there that needs more workspace, and tensors that take
    whatever memory was let go: the replays still give the step's output and leave those tensors alone."""
    small, large = Step(K, 1, seed=1), Step(K, 8, seed=2)
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
        kept = [torch.full((n << 20,), 90, dtype=torch.uint8, device='cuda') for n in (1, 2, 4, 8, 16, 32, 1, 2, 4, 8, 16, 32)]
        for _ in range(3):
            small.graph.replay()
            small.check()
            large.run()
            large.check()
    assert all(bool((t == 90).all()) for t in kept)


def test_calls_of_growing_size_in_one_graph(K):
    steps = [Step(K, 1, seed=1), Step(K, 8, seed=2), Step(K, 2, D=128, seed=3), Step(K, 40, seed=4), Step(K, 1, seed=5)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for step in steps:
            step.run()
    for _ in range(3):
        graph.replay()
        for step in steps:
            step.check()


def test_graphs_that_share_a_pool_and_one_that_is_gone(K):
    """Graphs of one memory pool, replayed in the order of their captures; the next is captured after one was destroyed."""
    pool = torch.cuda.graph_pool_handle()
    steps = [Step(K, T, seed=T).capture(pool=pool) for T in (1, 4, 2)]
    for _ in range(2):
        for step in steps:
            step.graph.replay()
            step.check()
    del steps[1].graph
    last = Step(K, 8, seed=9).capture()
    for step in (steps[0], steps[2], last, steps[0]):
        step.graph.replay()
        step.check()
    last.run()                                        # and a call outside any graph
    last.check()


def test_capture_numbers(K):
    """tcq_capture_id: none outside a capture, one number throughout a capture, another in the next."""
    from yanlongvla_b200._lib import lib
    n = ctypes.c_uint64(7)

    def number():
        assert lib.tcq_capture_id(torch.cuda.current_stream().cuda_stream, ctypes.byref(n)) == 0
        return n.value

    x, seen = torch.zeros(4, device='cuda'), []
    assert number() == 0 and lib.tcq_capture_id(None, None) == 4
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            first = number()
            x.add_(1)
            assert number() == first != 0
        seen.append(first)
        assert number() == 0
    assert seen[0] != seen[1]
