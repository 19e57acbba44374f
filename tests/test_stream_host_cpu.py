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
