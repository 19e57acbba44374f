"""A pooled memory's counts on the host, on the device that they follow: captured windows, robots that the pool does not serve, windows that
some robots do not fill."""
import pytest
import torch

from test_stream_gpu import P, frames, setup  # noqa: F401  (P and setup are the module's fixtures)
from test_stream_frames_gpu import layer_inputs
from test_stream_pool_gpu import K, Memory, ints, named  # noqa: F401  (K and Memory are fixtures)

pytestmark = pytest.mark.gpu


def test_a_captured_window_goes_on(P, K, Memory):
    """The window of test_a_window_in_a_graph with reserve() before each replay, over more frames than fit without forgetting."""
    c = P.PolicyConfig(vit_layers=1, llm_layers=2, dit_layers=1)
    n, B, keep = c.prefix_tokens, 2, 200
    eager, graphed = (Memory(c, B, 400, pages=20) for _ in range(2))
    held = layer_inputs(c, B, n, 0)

    def step(memory, inputs):
        memory.keep_recent(keep)
        memory.begin_frame(inputs[0][0])
        return [memory.attend(i, q.clone(), k, v) for i, (q, k, v) in enumerate(inputs)]

    graph = torch.cuda.CUDAGraph()
    step(eager, held)
    step(graphed, held)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        outs = step(graphed, held)
    assert (graphed.tokens, graphed.frames) == (n, 1)
    for f in range(1, 9):
        inputs = layer_inputs(c, B, n, f)
        want = step(eager, inputs)
        for to, x in zip(held, inputs):
            for a, b in zip(to, x):
                a.copy_(b)
        graphed.reserve(kept=keep)
        graph.replay()
        torch.cuda.synchronize()
        assert eager.lens.tolist() == graphed.lens.tolist() == [min(f * n, keep) + n] * B
        assert (graphed.tokens, graphed.frames) == (eager.tokens, eager.frames) == (min(f * n, keep) + n, f + 1)
        assert graphed.served.all()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)
        named(graphed)
    with pytest.raises(K.TcqError, match='does not fit'):
        graphed.reserve()
    assert K.device_error() == 0


@pytest.mark.parametrize('captured', [False, True])
def test_robots_without_pages_get_no_actions(P, setup, K, Memory, captured):
    """The second robot's pages run out in the second frame: served says so, its actions are zeros, the other's what they are in a pool
    that serves both; after the first robot has forgotten it is served again."""
    c, model = setup
    n, S = c.prefix_tokens, 2
    obs = [(*o[:3], torch.randn(2 * S, *o[3].shape[1:], device='cuda', generator=torch.Generator(device='cuda').manual_seed(i)))
           for i, o in enumerate(frames(P, c, 2, 3))]
    small, large = Memory(c, 2, 3 * n, pages=8), Memory(c, 2, 3 * n, pages=16)
    held = [t.clone() for t in obs[0]]
    with torch.no_grad():
        if captured:
            model(*obs[0], memory=Memory(c, 2, n, pages=6))                    # what the first call sets up, outside the capture
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = model(*held, memory=small)

        def act(f):
            if not captured:
                return model(*obs[f], memory=small)
            for a, b in zip(held, obs[f]):
                a.copy_(b)
            small.reserve()
            graph.replay()
            return out.clone()
        for f, served in ((0, [True, True]), (1, [True, False])):
            want, got = model(*obs[f], memory=large), act(f)
            assert small.served.tolist() == served and large.served.all()
            assert torch.equal(got[:S], want[:S]) and want.ne(0).any(-1).any(-1).all()
            assert torch.equal(got[S:], want[S:] if served[1] else torch.zeros_like(want[S:]))
        assert K.device_error() == 2
        assert small.lens.tolist() == [2 * n, n]
        small.fork(ints([-1, 1]))
        assert act(2)[S:].ne(0).any() and small.served.all() and small.lens.tolist() == [n, 2 * n]
    named(small)
    assert K.device_error() == 0


def test_the_count_is_not_below_what_is_there(P, setup, K, Memory):
    """As test_a_pool_without_pages_left: a keep that the pool does not serve lowers no count."""
    c, model = setup
    n = c.prefix_tokens
    memory = Memory(c, 2, 2 * n, pages=8)
    with torch.no_grad():
        for obs in frames(P, c, 2, 2):
            model(*obs, memory=memory)
        memory.keep_recent(100)
        assert K.device_error() == 2 and memory.lens.tolist() == [2 * n, n] and memory.tokens == 2 * n
        with pytest.raises(K.TcqError, match='does not fit'):
            memory.begin_frame()
    named(memory)


def test_robots_within_the_window_stay_where_they_are(P, setup, K, Memory):
    c, model = setup
    n = c.prefix_tokens
    memory = Memory(c, 3, 2 * n, pages=5 + 3 + 5 + 4 + 4)                    # room for what the two long ones keep, next to all
    begin = ints([0] * 3)
    with torch.no_grad():
        for f, obs in enumerate(frames(P, c, 3, 2)):
            memory.begin_frame(count=ints([n, 100 - 60 * f, n - 7 * f]))
            for i, (q, k, v) in enumerate(layer_inputs(c, 3, n, f)):
                memory.attend(i, q, k, v)
    before = memory.table.clone(), [K.kv8_read(cache, memory.table, begin, memory.lens, 2 * n, dtype=torch.float32) for cache in memory.caches]
    memory.keep_recent(2 * n - 90)
    assert K.device_error() == 0 and memory.lens.tolist() == [2 * n - 90, 140, 2 * n - 90] and memory.tokens == 2 * n - 90
    assert torch.equal(memory.table[1], before[0][1])
    named(memory)
    for cache, was in zip(memory.caches, before[1]):
        got = K.kv8_read(cache, memory.table, begin, memory.lens, 2 * n, dtype=torch.float32)
        for x, y, scale in zip(got, was, (cache.k_scale, cache.v_scale)):
            assert torch.equal(x[1], y[1])
            # half a step of the largest scale, as in test_keep_recent
            assert (x[0, :2 * n - 90] - y[0, 90:]).abs().max() <= scale.max() * (0.5 + 127 * 2.0 ** -22)
    assert K.device_error() == 0
