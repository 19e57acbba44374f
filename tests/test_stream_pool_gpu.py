"""A streaming memory with a pool of pages: the same as one without, forked, thinned out, with frames of differing length, in graphs,
and when the pool is empty."""
import pytest
import torch

from test_stream_gpu import P, frames, setup  # noqa: F401  (P and setup are the module's fixtures)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def K():
    from yanlongvla_b200 import kernels
    kernels.device_error()
    return kernels


@pytest.fixture(scope='module')
def Memory():
    from yanlongvla_b200.stream import StreamMemory
    return StreamMemory


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device='cuda')


def named(memory):
    """The pool counts what the table says."""
    t = memory.table
    assert torch.equal(torch.bincount(t[t >= 0].long(), minlength=memory.pages.pages).int(), memory.pages.refs)


def test_a_pool_is_the_same_memory(P, setup, K, Memory):
    c, model = setup
    plain, pooled = Memory(c, 2, 3 * c.prefix_tokens), Memory(c, 2, 3 * c.prefix_tokens, pages=16)
    with torch.no_grad():
        for _ in range(2):
            for obs in frames(P, c, 2, 3):
                assert torch.equal(model(*obs, memory=plain), model(*obs, memory=pooled))
            assert torch.equal(plain.lens, pooled.lens)
            named(pooled)
            plain.forget()
            pooled.forget()
            assert not pooled.pages.refs.any() and (pooled.table == -1).all()
    assert K.device_error() == 0


def test_forked_robots_go_on_alone(P, setup, K, Memory):
    """Three robots of which two start from the first one's past act as three that have seen the same."""
    c, model = setup
    forked, told = (Memory(c, 3, 3 * c.prefix_tokens, pages=24) for _ in range(2))
    first, second, third = frames(P, c, 3, 3)
    same = [t[:1].expand(3, *t.shape[1:]).contiguous() for t in first]
    with torch.no_grad():
        model(*first, memory=forked)
        model(*same, memory=told)
        forked.fork(ints([0, 0, 0]))
        assert (forked.pages.refs.max().item(), int((forked.pages.refs > 0).sum())) == (3, 3)
        for obs in (second, third):
            assert torch.equal(model(*obs, memory=forked), model(*obs, memory=told))
            named(forked)
        with pytest.raises(K.TcqError, match='pool'):
            Memory(c, 1, 64).fork(ints([0]))
    assert K.device_error() == 0


def test_keep_recent(P, setup, K, Memory):
    """What is kept is what was there, but for the steps of blocks that now share a scale; new frames follow it."""
    c, model = setup
    n = c.prefix_tokens
    memory = Memory(c, 2, 3 * n, pages=2 * 8 + 2 * 6)
    obs = frames(P, c, 2, 6)
    begin = ints([0, 0])
    with torch.no_grad():
        for o in obs[:3]:
            model(*o, memory=memory)
        before = [K.kv8_read(cache, memory.table, begin, memory.lens, 3 * n, dtype=torch.float32) for cache in memory.caches]
        memory.keep_recent(2 * n - 7)
        named(memory)
        assert memory.lens.tolist() == [2 * n - 7] * 2 and memory.tokens == 2 * n - 7
        for cache, was in zip(memory.caches, before):
            got = K.kv8_read(cache, memory.table, begin, memory.lens, 2 * n - 7, dtype=torch.float32)
            for x, y in zip(got, was):
                # half a step of the largest scale s; in FP32 the quotient and its product with an integer up to 127 are off by 2^-24
                # each, 127 2^-23 of a step, and so are the two values, 127 s at most, together: 127 2^-22 s
                step = (cache.k_scale if y is was[0] else cache.v_scale).max()
                assert (x - y[:, n + 7:]).abs().max() <= step * (0.5 + 127 * 2.0 ** -22)
        with pytest.raises(K.TcqError, match='does not fit'):
            for o in obs[3:]:
                model(*o, memory=memory)
                named(memory)
        assert memory.lens.tolist() == [3 * n - 7] * 2
        memory.keep_recent(0)
        assert memory.tokens == 0 and not memory.pages.refs.any()
        with pytest.raises(K.TcqError, match='do not fit'):
            memory.keep(ints([[0] * (3 * n + 64)] * 2))
    assert K.device_error() == 0


def test_frames_of_differing_length(P, setup, K, Memory):
    """Padding of the instruction has no effect, on the memory neither, with and without a pool."""
    c, model = setup
    first, second = frames(P, c, 2, 2)
    lens = ints([5, c.lang_tokens])
    outs = []
    with torch.no_grad():
        for pages in (None, 16):
            for seed in (0, 1):
                memory = Memory(c, 2, 2 * c.prefix_tokens, pages=pages)
                for images, lang, state, noise in (first, second):
                    lang = lang.clone()
                    lang[0, 5:] = torch.randint(0, c.vocab, (c.lang_tokens - 5,), generator=torch.Generator().manual_seed(seed)).cuda()
                    outs.append(model(images, lang, state, noise, memory=memory, lang_lens=lens))
                image = c.cameras * c.image_tokens
                assert memory.lens.tolist() == [2 * (image + 5), 2 * (image + c.lang_tokens)]
    for f in (0, 1):
        for other in outs[f + 2::2]:
            assert torch.equal(outs[f], other)
    assert K.device_error() == 0


def test_counts_of_a_frame(P, setup, K, Memory):
    """A count that is none of the frame's is refused before anything moves; one past the frame is the whole frame."""
    c, _ = setup
    n = c.prefix_tokens
    for pages in (None, 8):
        memory = Memory(c, 2, n, pages=pages)
        for bad in (ints([n, n]).long(), ints([n]), torch.tensor([n, n], dtype=torch.int32)):
            with pytest.raises(K.TcqError, match='count'):
                memory.begin_frame(count=bad)
        assert memory.tokens == memory.frames == 0 and memory.pos[0].eq(-1).all() and not memory.lens.any()
        memory.begin_frame(count=ints([n + 1, -1]))
        assert memory.lens.tolist() == [n, 0]


def test_a_pool_without_pages_left(P, setup, K, Memory):
    """The robot that is not served remembers nothing of the frame, the other all of it."""
    c, model = setup
    first, second = frames(P, c, 2, 2)
    memory = Memory(c, 2, 2 * c.prefix_tokens, pages=8)                         # three pages a frame and robot, five for two
    with torch.no_grad():
        model(*first, memory=memory)
        assert K.device_error() == 0
        assert torch.isfinite(model(*second, memory=memory)).all()
        assert K.device_error() == 2 and memory.lens.tolist() == [2 * c.prefix_tokens, c.prefix_tokens]
        named(memory)
        memory.keep_recent(100)                                                # four pages: one is left, none after one robot's
        assert K.device_error() == 2 and memory.lens.tolist() == [2 * c.prefix_tokens, c.prefix_tokens]
        named(memory)


def test_what_keep_refuses_and_cuts(P, setup, K, Memory):
    """An index or a number of tokens that keep refuses costs no page of the pool; more tokens than a robot remembers are cut, on the
    host's count too."""
    c, model = setup
    n = c.prefix_tokens
    memory = Memory(c, 2, 2 * n, pages=16)
    with torch.no_grad():
        model(*frames(P, c, 2, 1)[0], memory=memory)
    refs, index = memory.pages.refs.clone(), ints([[0] * 8] * 2)
    for bad in (index.long(), index[:1], index[0], index[:, :0], index.cpu()):
        with pytest.raises(K.TcqError, match='index'):
            memory.keep(bad)
    for bad in (ints([8, 8]).long(), ints([8]), torch.tensor([8, 8], dtype=torch.int32)):
        with pytest.raises(K.TcqError, match='kept'):
            memory.keep(index, bad)
    assert torch.equal(memory.pages.refs, refs) and memory.lens.tolist() == [n, n] and memory.tokens == n
    named(memory)
    memory.keep(index[:, ::2], ints([9, -1]))                                   # the same token four times; a view of every other number
    assert memory.lens.tolist() == [4, 0] and memory.tokens == 4
    named(memory)
    memory.keep(ints([[3, 2, 1, 0, 0, 0, 0]] * 2))
    assert memory.lens.tolist() == [4, 0] and memory.tokens == 4
    named(memory)
    assert K.device_error() == 0


def test_a_window_in_a_graph(P, K, Memory):
    """A frame with what goes before it forgotten, captured once: replays give what the steps outside a graph give."""
    c = P.PolicyConfig(vit_layers=1, llm_layers=2, dit_layers=1)
    from test_stream_frames_gpu import layer_inputs
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
    for f in range(1, 6):
        inputs = layer_inputs(c, B, n, f)
        want = step(eager, inputs)
        for to, x in zip(held, inputs):
            for a, b in zip(to, x):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert eager.lens.tolist() == graphed.lens.tolist() == [min(f * n, keep) + n] * B
        for a, b in zip(outs, want):
            assert torch.equal(a, b)
        named(graphed)
    assert K.device_error() == 0


def test_the_command(capsys):
    from yanlongvla_b200 import stream
    actions = stream.main(['--robots', '2', '--frames', '4', '--window', '2', '--candidates', '3', '--vit-layers', '1', '--llm-layers', '2', '--dit-layers', '2'])
    assert actions.shape == (6, 16, 32) and torch.isfinite(actions).all()
    out = capsys.readouterr().out
    assert 'frame 3: 320 tokens remembered' in out
    from yanlongvla_b200 import kernels
    assert kernels.device_error() == 0
