"""A StreamMemory on the CPU: the page operators sequence by sequence in plain Python (pages_ref), caches without contents. For the host's
side of a memory: its counts, and what it hands to the operators."""
import contextlib
import types

import torch

import pages_ref as ref


class Kernels:
    """In place of `stream.K`. flag: what device_error would report; calls: the operators in the order they came in."""
    KV8_BLOCK = ref.BLOCK

    def __init__(self):
        from yanlongvla_b200.kernels import TcqError
        self.TcqError, self.flag, self.calls = TcqError, 0, []
        self.KV8Cache = types.SimpleNamespace(empty=lambda pages, heads, D, device: types.SimpleNamespace(pages=pages))
        self.KV8Pages = types.SimpleNamespace(empty=self._pages)
        self.RopeAxes = type('RopeAxes', (), {'__init__': lambda *a: None, 'tables': staticmethod(lambda *a: (None, None))})

    @staticmethod
    def _pages(pages, device):
        return types.SimpleNamespace(pages=pages, refs=torch.zeros(pages, dtype=torch.int32),
                                     table=lambda n, blocks: torch.full((n, blocks), -1, dtype=torch.int32))

    @contextlib.contextmanager
    def _model(self, name, pages, table, lens):
        self.calls.append(name)
        m = ref.Pages(0, len(lens), table.shape[1])
        m.refs, m.table, m.lens = pages.refs.tolist(), table.tolist(), lens.tolist()
        yield m
        pages.refs.copy_(torch.tensor(m.refs))
        table.copy_(torch.tensor(m.table))
        lens.copy_(torch.tensor(m.lens))

    def kv8_fork(self, pages, table, lens, parent):
        with self._model('fork', pages, table, lens) as m:
            m.fork(parent.tolist())

    def kv8_free(self, pages, table, lens, keep):
        with self._model('free', pages, table, lens) as m:
            m.free(keep.tolist())

    def kv8_reserve(self, pages, table, lens, count):
        with self._model('reserve', pages, table, lens) as m:
            granted, copies = m.reserve(count.tolist())
        if granted != count.tolist():
            self.flag = 2
        return tuple(torch.tensor(x, dtype=torch.int32) for x in (granted, copies))

    def kv8_copy(self, caches, copies):
        self.calls.append('copy')

    def kv8_compact(self, caches, table, lens, index, new_table, kept=None):
        self.calls.append('compact')


def config(tokens=160):
    """A policy whose frames have that many tokens (a square image of each of two cameras, the rest an instruction)."""
    return types.SimpleNamespace(llm_hidden=128, llm_heads=2, llm_kv_heads=1, llm_layers=2, cameras=2, image_tokens=64, lang_tokens=tokens - 128)


def memory(monkeypatch, robots, max_tokens, pages=None, **kw):
    """(the memory, its kernels); its `replay(step)` runs what a captured step's replay does: the device's part, none of the host's."""
    from yanlongvla_b200 import stream
    K = Kernels()
    monkeypatch.setattr(stream, 'K', K)
    capturing = [False]
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: capturing[0])
    m = stream.StreamMemory(config(), robots, max_tokens, device='cpu', pages=pages, **kw)

    def replay(step):
        capturing[0] = True
        step()
        capturing[0] = False
    m.replay = replay
    return m, K


def named(m):
    """The pool counts what the table says."""
    assert torch.bincount(m.table[m.table >= 0].long(), minlength=m.pages.pages).tolist() == m.pages.refs.tolist()
