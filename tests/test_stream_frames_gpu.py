"""The streaming policy's memory as its caller sees it: frames that do not belong to it, steps captured in CUDA graphs."""
import pytest
import torch

from test_stream_gpu import P, frames, setup  # noqa: F401  (P and setup are the module's fixtures)

pytestmark = pytest.mark.gpu


def test_a_refused_frame_leaves_the_memory_as_it_was(P, setup):
    """A frame of another batch, or of another length, is refused before anything of the memory has moved."""
    from yanlongvla_b200 import kernels as K
    from yanlongvla_b200.stream import StreamMemory
    c, model = setup
    first, second = frames(P, c, 2, 2)
    memory = StreamMemory(c, 2, 3 * c.prefix_tokens)
    with torch.no_grad():
        model(*first, memory=memory)
        state = [t.clone() for t in (memory.pos, memory.start, memory.lens)]
        with pytest.raises(K.TcqError, match='frame'):
            model(*(t[:1] for t in second), memory=memory)
        with pytest.raises(K.TcqError, match='frame'):
            model.backbone(model.embed(*second[:2])[:, 1:], memory)
        assert (memory.tokens, memory.frames) == (c.prefix_tokens, 1)
        assert all(torch.equal(a, b) for a, b in zip(state, (memory.pos, memory.start, memory.lens)))
        got = model(*second, memory=memory)
        memory.forget()
        model(*first, memory=memory)
        assert torch.equal(model(*second, memory=memory), got)


def layer_inputs(c, B, n, seed):
    """q, k, v of every layer for one frame of n tokens."""
    g = torch.Generator(device='cuda').manual_seed(seed)
    D = c.llm_hidden // c.llm_heads
    return [[torch.randn(B, n, h * D, device='cuda', generator=g).bfloat16() for h in (c.llm_heads, c.llm_kv_heads, c.llm_kv_heads)]
            for _ in range(c.llm_layers)]


@pytest.mark.parametrize('captured_at', [0, 2])
@pytest.mark.parametrize('B', [1, 2])
def test_a_captured_step_moves_the_memory_on(P, B, captured_at):
    """A frame's step captured in a graph, as the first frame or later, gives what the step gives outside one at every replay: outputs,
    positions, lengths and caches; reserve() counts and refuses; forget() starts again."""
    from yanlongvla_b200 import kernels as K
    from yanlongvla_b200.stream import StreamMemory
    c = P.PolicyConfig(vit_layers=1, llm_layers=2, dit_layers=1)
    n, most = c.prefix_tokens, 5
    eager, graphed = (StreamMemory(c, B, most * n + 7) for _ in range(2))
    inputs = [layer_inputs(c, B, n, 100 + f) for f in range(most)]
    held = layer_inputs(c, B, n, 0)
    outs = [torch.empty_like(q) for q, _, _ in held]

    def step():
        graphed.begin_frame(held[0][0])
        for i, (q, k, v) in enumerate(held):
            outs[i].copy_(graphed.attend(i, q.clone(), k, v))

    def load(f):
        for to, x in zip(held, inputs[f]):
            for a, b in zip(to, x):
                a.copy_(b)

    graph = torch.cuda.CUDAGraph()
    for _ in range(2):
        for f in range(most):
            eager.begin_frame()
            want = [eager.attend(i, q.clone(), k, v) for i, (q, k, v) in enumerate(inputs[f])]
            load(f)
            if f == captured_at and _ == 0:
                torch.cuda.synchronize()
                with torch.cuda.graph(graph):
                    step()
                assert (graphed.tokens, graphed.frames) == (n * f, f)             # a capture runs nothing
            if f < captured_at and _ == 0:
                step()
            else:
                graphed.reserve()
                graph.replay()
            torch.cuda.synchronize()
            assert (graphed.tokens, graphed.frames) == (eager.tokens, eager.frames) == (n * (f + 1), f + 1)
            assert graphed.pos[0].unique().tolist() == [f]
            for name in ('pos', 'start', 'lens'):
                assert torch.equal(getattr(graphed, name), getattr(eager, name))
            for a, b in zip(outs, want):
                assert torch.equal(a, b)
            for a, b in zip(graphed.caches, eager.caches):
                for name in ('k', 'v', 'k_scale', 'v_scale'):
                    assert torch.equal(getattr(a, name), getattr(b, name))
        for refused in (graphed.reserve, graphed.begin_frame):
            with pytest.raises(K.TcqError, match='does not fit'):
                refused()
        assert (graphed.tokens, graphed.frames) == (most * n, most) and graphed.lens.tolist() == [most * n] * B
        eager.forget()
        graphed.forget()
    assert K.device_error() == 0


def test_the_whole_policy_in_a_graph(P, setup):
    """A chunk with a memory, captured as the first frame: every replay gives the actions of the run outside a graph."""
    from yanlongvla_b200.stream import StreamMemory
    c, model = setup
    eager, graphed = (StreamMemory(c, 1, 4 * c.prefix_tokens) for _ in range(2))
    held = [t.clone() for t in frames(P, c, 1, 1)[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad():
        wants = [model(*obs, memory=eager).clone() for obs in frames(P, c, 1, 4)]
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            actions = model(*held, memory=graphed)
        for obs, want in zip(frames(P, c, 1, 4), wants):
            for to, x in zip(held, obs):
                to.copy_(x)
            graphed.reserve()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(actions, want)
    assert torch.equal(graphed.lens, eager.lens) and graphed.tokens == eager.tokens
