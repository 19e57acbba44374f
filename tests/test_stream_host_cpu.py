"""What a StreamMemory counts on the host, over page operators in plain Python."""
import pytest
import torch

from stream_fake import memory, named

N = 160                                                                        # tokens of a frame


def ints(v):
    return torch.tensor(v, dtype=torch.int32)


def test_a_captured_window_goes_on(monkeypatch):
    """A captured step that keeps the newest tokens before its frame: reserve(kept=) before each replay counts what it keeps."""
    m, K = memory(monkeypatch, 2, 400, pages=20)

    def step():
        m.keep_recent(200)
        m.begin_frame()
    step()
    for f in range(1, 12):
        m.reserve(kept=200)
        m.replay(step)
        assert m.lens.tolist() == [min(f * N, 200) + N] * 2 and m.tokens == min(f * N, 200) + N and m.frames == f + 1
        named(m)
    assert K.flag == 0
    with pytest.raises(K.TcqError, match='does not fit'):                      # nothing kept: the count of before
        m.reserve()
    for kept in (-1, 1.5, '3'):
        with pytest.raises((K.TcqError, TypeError)):
            m.reserve(kept=kept)
    assert m.tokens == 360 and m.frames == 12


def test_a_captured_forget_leaves_the_counts(monkeypatch):
    """A capture runs nothing: what it records does not empty the memory on the host while the device still holds it."""
    m, K = memory(monkeypatch, 1, 2 * N + 8)
    m.begin_frame()
    m.replay(lambda: (m.forget(), m.begin_frame()))                            # the capture of a step; on this machine it has run
    assert (m.tokens, m.frames) == (N, 1)
    m.begin_frame()
    with pytest.raises(K.TcqError, match='does not fit'):
        m.begin_frame()
    m.forget()
    assert (m.tokens, m.frames) == (0, 0) and not m.lens.any()


@pytest.mark.parametrize('way', ['keep', 'keep_recent'])
def test_the_count_is_not_below_what_is_there(monkeypatch, way):
    """Robots whose tokens the pool does not hold next to the old ones keep their memory, and the host's count with it."""
    m, K = memory(monkeypatch, 2, 2 * N, pages=10)                              # five pages a robot for two frames: none is left
    m.begin_frame()
    m.begin_frame()

    def keep(n):
        if way == 'keep':
            m.keep(ints([list(range(n))] * 2))
        else:
            m.keep_recent(n)
    keep(100)
    assert K.flag == 2 and m.lens.tolist() == [2 * N] * 2 and m.tokens == 2 * N
    with pytest.raises(K.TcqError, match='does not fit'):
        m.begin_frame()
    named(m)
    m.forget()
    m.begin_frame(count=ints([N, 10]))                                          # four pages; two more for robot 0, one for robot 1
    keep(100)
    assert m.lens.tolist() == [100, 10] and m.tokens == 100
    named(m)


def test_no_look_at_the_device_where_the_pool_is_large(monkeypatch):
    """A window as the command sizes it is kept without reading a length back; where the pool might be too small, one is read."""
    for pages, reads in ((2 * (6 + 4), 0), (2 * (6 + 4) - 1, 3)):
        m, K = memory(monkeypatch, 2, 360, pages=pages)
        seen = []
        monkeypatch.setattr(m, '_longest', lambda own=m._longest: (seen.append(1), own())[1])
        for _ in range(6):
            m.keep_recent(200)
            m.begin_frame(count=ints([N, 10]))
            assert m.tokens == int(m.lens.max())
            named(m)
        assert len(seen) == reads


def test_what_a_replay_keeps_in_a_small_pool(monkeypatch):
    """Whether a pool that may be too small serves the keep of a replay is not known before it: the count stays."""
    m, K = memory(monkeypatch, 2, 360, pages=2 * (5 + 4) - 1)

    def step():
        m.keep_recent(200)
        m.begin_frame()
    m.begin_frame()
    m.begin_frame()
    with pytest.raises(K.TcqError, match='does not fit'):
        m.reserve(kept=200)
    assert (m.tokens, m.frames) == (2 * N, 2)
    m.forget()
    m.begin_frame()
    m.reserve(kept=200)                                                        # four pages a robot at most before it, three kept
    m.replay(step)
    assert m.lens.tolist() == [2 * N] * 2 and m.tokens == 2 * N
    m, K = memory(monkeypatch, 1, N)                                            # without a pool nothing is kept, all may be forgotten
    m.begin_frame()
    with pytest.raises(K.TcqError, match='pool'):
        m.reserve(kept=10)
    m.reserve(kept=0)
    assert (m.tokens, m.frames) == (N, 2)


@pytest.mark.parametrize('pages', [None, 16])
def test_short_frames_count_what_they_hold(monkeypatch, pages):
    """Frames of which padding is not remembered count in full until that is too much; then what is there counts."""
    m, K = memory(monkeypatch, 2, 2 * N, pages=pages)
    seen = []
    monkeypatch.setattr(m, '_longest', lambda own=m._longest: (seen.append(1), own())[1])
    for f in range(1, 9):
        m.begin_frame(count=ints([20, 3]))
        assert m.lens.tolist() == [20 * f, 3 * f] and m.tokens >= 20 * f and m.frames == f
    assert m.tokens == 140 + N and len(seen) == 6
    with pytest.raises(K.TcqError, match='does not fit behind 160'):
        m.max_tokens = 2 * N - 1
        m.begin_frame()
    assert m.lens.tolist() == [160, 24] and m.frames == 8 and m.pos[0].eq(7).all()


def test_frames_that_were_counted_and_not_run_count(monkeypatch):
    """What is read from the device lacks the frames that have been counted in for replays to come."""
    m, K = memory(monkeypatch, 1, 4 * N)
    m.begin_frame(count=ints([20]))
    m.reserve()
    m.reserve()
    m.reserve()                                                                # 20 on the device, three frames to come
    assert m.tokens == 4 * N
    with pytest.raises(K.TcqError, match=f'does not fit behind {20 + 3 * N} '):
        m.reserve()
    m.replay(m.begin_frame)
    m.replay(m.begin_frame)
    with pytest.raises(K.TcqError, match=f'does not fit behind {20 + 3 * N} '):
        m.reserve()
    m.replay(m.begin_frame)
    assert m.lens.tolist() == [20 + 3 * N] == [m.tokens] and m.frames == 4


def test_robots_that_are_not_served_are_told(monkeypatch):
    """served says of each robot whether the memory took what it was given of the last frame, in a replay too."""
    m, K = memory(monkeypatch, 3, 3 * N, pages=10)
    assert m.served.tolist() == [True] * 3
    served = m.served
    for counts, want in ((None, [True] * 3), (ints([0, 32, N]), [True, True, False]), (ints([0, 0, 0]), [True] * 3), (ints([N + 9, -1, 0]), [False, True, True]),
                         (ints([0, 0, 1]), [True] * 3)):
        before = m.lens.tolist()
        m.replay(lambda: m.begin_frame(count=counts))
        assert m.served is served
        assert served.tolist() == want, counts
        for b in range(3):
            took = m.lens[b].item() - before[b]
            assert took == (min(max(counts[b].item(), 0), N) if counts is not None else N) * want[b]
        named(m)
    m.forget()
    assert served.tolist() == [True] * 3
    plain, _ = memory(monkeypatch, 2, N)
    plain.begin_frame(count=ints([3, 0]))
    assert plain.served.tolist() == [True] * 2


def test_a_robot_that_is_not_served_gets_no_actions(monkeypatch):
    """Its features have seen nothing; the actions of all its candidates are zeros, those of the others what they were."""
    from yanlongvla_b200 import policy
    m, K = memory(monkeypatch, 3, N, pages=9)
    m.served.copy_(torch.tensor([True, False, True]))
    actions = torch.arange(1.0, 3 * 2 * 4 * 5 + 1).view(6, 4, 5)
    p = policy.GrootStylePolicy.__new__(policy.GrootStylePolicy)
    torch.nn.Module.__init__(p)
    p.c = policy.PolicyConfig()
    monkeypatch.setattr(policy.GrootStylePolicy, 'embed', lambda *a: torch.zeros(3, 1))
    monkeypatch.setattr(policy.GrootStylePolicy, 'backbone', lambda *a: torch.zeros(3, 1))
    monkeypatch.setattr(policy.GrootStylePolicy, 'action_head', lambda *a: actions)
    noise = torch.zeros(6, 4, 5)
    state = torch.zeros(3, 64)
    for memory_, want in ((None, actions), (m, actions * torch.tensor([1, 1, 0, 0, 1, 1.0])[:, None, None])):
        assert torch.equal(p(None, None, state, noise, memory=memory_), want)
    actions[2] = float('nan')                                                  # whatever the head made of it
    assert not p(None, None, state, noise, memory=m)[2:4].any()


def test_inputs_that_do_not_fit_leave_the_memory(monkeypatch):
    """Noise or states of another batch are refused before the memory has moved."""
    from yanlongvla_b200 import policy
    m, K = memory(monkeypatch, 2, N, pages=9)
    p = policy.GrootStylePolicy.__new__(policy.GrootStylePolicy)
    torch.nn.Module.__init__(p)
    p.c = policy.PolicyConfig()
    monkeypatch.setattr(policy.GrootStylePolicy, 'embed', lambda *a: torch.zeros(2, N, 8))
    monkeypatch.setattr(policy.GrootStylePolicy, 'backbone', lambda self, prefix, memory, lens: memory.begin_frame(prefix))
    monkeypatch.setattr(policy.GrootStylePolicy, 'action_head', lambda self, feats, state, noise, lens: noise)
    state = torch.zeros(2, 64)
    for noise in (torch.zeros(3, 4, 5), torch.zeros(1, 4, 5), torch.zeros(0, 4, 5)):
        with pytest.raises(ValueError, match='noise'):
            p(None, None, state, noise, memory=m)
    with pytest.raises(ValueError, match='state'):
        p(None, None, state[:1], torch.zeros(4, 4, 5), memory=m)
    assert m.frames == m.tokens == 0 and not m.lens.any()
    p(None, None, state, torch.zeros(4, 4, 5), memory=m)
    assert m.frames == 1


def test_robots_within_the_window_stay_where_they_are(monkeypatch):
    """keep_recent packs what is longer than the window: the others' tokens keep their pages, need no second ones and refuse no one."""
    m, K = memory(monkeypatch, 4, 400, pages=3 + 3 + 5 + 2 + 4)                 # room next to the old ones for the long robot's tokens alone
    m.begin_frame(count=ints([N, 130, N, 100]))
    m.begin_frame(count=ints([0, 0, N, 0]))
    before = m.table.clone()
    m.keep_recent(200)
    assert K.flag == 0 and m.lens.tolist() == [N, 130, 200, 100] and m.tokens == 200
    for b in (0, 1, 3):
        assert torch.equal(m.table[b], before[b])
    named(m)
    m.fork(ints([0, 1, 2, 2]))
    refs = m.pages.refs.clone()
    m.keep_recent(200)                                                         # nothing to forget: nothing moves
    assert torch.equal(m.pages.refs, refs) and m.lens.tolist() == [N, 130, 200, 200]
    m.keep_recent(130)                                                         # three pages each for three robots, seven free
    assert K.flag == 2 and m.lens.tolist() == [130, 130, 130, 200]
    named(m)


def test_a_window_longer_than_the_memory(monkeypatch):
    m, K = memory(monkeypatch, 2, 2 * N, pages=10)
    m.begin_frame()
    before = m.table.clone()
    for tokens in (N, 2 * N, 10 ** 6, 1 << 40):
        m.keep_recent(tokens)
        assert m.lens.tolist() == [N, N] and m.tokens == N and torch.equal(m.table, before)
    assert K.flag == 0


@pytest.mark.parametrize('window', ['0', '3'])
def test_the_command_has_positions_for_all_its_frames(monkeypatch, window):
    from yanlongvla_b200 import policy, stream
    made = []

    def memory(c, robots, max_tokens, max_frames=4096, pages=None):
        made.append(max_frames)
        raise KeyboardInterrupt
    monkeypatch.setattr(policy, 'build_policy', lambda runtime, c: (None, None, None))
    monkeypatch.setattr(stream, 'StreamMemory', memory)
    for frames in ('5000', '8'):
        with pytest.raises(KeyboardInterrupt):
            stream.main(['--frames', frames, '--window', window])
    assert made == [5000, 4096]


@pytest.mark.parametrize('seed', range(12))
def test_random_histories(monkeypatch, seed):
    """Frames, forks and keeps in pools of any size: the count is never below what is there, a frame is refused only where the longest memory
    leaves no room, pages are counted, and the flag is raised where a robot was not served."""
    import random
    rng = random.Random(seed)
    robots, most = rng.choice((1, 2, 5)), rng.choice((N, 3 * N + 5, 700))
    m, K = memory(monkeypatch, robots, most, pages=rng.choice((4, 9, 20, 60)))
    refused = 0
    for _ in range(60):
        K.flag = 0
        before, n = m.lens.tolist(), rng.choice((0, 1, 64, 100, 200, 500))
        kind = rng.choice(('frame', 'frame', 'frame', 'fork', 'keep', 'recent', 'replay', 'forget'))
        if kind == 'frame':
            count = ints([rng.randint(0, N) for _ in range(robots)]) if rng.random() < 0.5 else None
            try:
                m.begin_frame(count=count)
            except K.TcqError:
                refused += 1
                assert max(before) + N > most and m.lens.tolist() == before
                continue
            want = [N] * robots if count is None else count.tolist()
            assert m.served.tolist() == [a - b == w for a, b, w in zip(m.lens.tolist(), before, want)]
            assert m.served.all() == (K.flag == 0)
        elif kind == 'fork':
            m.fork(ints([rng.randrange(-1, robots) for _ in range(robots)]))
        elif kind == 'keep' and n:
            n = min(n, m.table.shape[1] * 64)
            m.keep(torch.randint(0, 50, (robots, n), dtype=torch.int32), ints([rng.randint(-1, n) for _ in range(robots)]))
        elif kind == 'recent':
            m.keep_recent(n)
            if K.flag == 0:
                assert m.lens.tolist() == [min(n, b) for b in before]
        elif kind == 'replay':
            try:
                m.reserve(kept=n)
            except K.TcqError:
                continue
            m.replay(lambda: (m.keep_recent(n), m.begin_frame()))
        elif kind == 'forget':
            m.forget()
        named(m)
        assert m.lens.max() <= m.tokens <= most
        assert all(blocks == -(-length // 64) for blocks, length in zip((m.table >= 0).sum(1).tolist(), m.lens.tolist()))
    assert refused or most > N
