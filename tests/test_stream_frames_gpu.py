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
