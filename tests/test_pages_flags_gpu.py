"""What the page operators refuse, and device_error, agree: after each reservation of random histories, in pools that refuse often."""
import random

import pytest
import torch

from test_pages_gpu import Both, ints
from test_pages_gpu import K  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


def reserve(s, count, advance=True):
    """Whether a sequence was refused: by the pool, or by its table. The flag says the same."""
    asked = [n > 0 for n in count]
    g, _ = s.reserve(count, advance)
    refused = any(a and not n for a, n in zip(asked, g))
    assert s.K.device_error() == (2 if refused else 0)
    return refused


@pytest.mark.parametrize('sequences,blocks,pages,seed', [(1, 9, 3, 1), (3, 5, 8, 2), (7, 33, 14, 3), (40, 18, 90, 4), (33, 65, 80, 5), (300, 7, 700, 6),
                                                         (1030, 4, 2200, 7), (5, 2, 40, 8)])
def test_a_refusal_is_reported(K, sequences, blocks, pages, seed):
    rng = random.Random(seed)
    s = Both(K, pages, sequences, blocks)
    assert K.device_error() == 0
    refusals = served = 0
    for step in range(32):
        kind = rng.choice(('reserve', 'reserve', 'fork', 'free', 'reserved only'))
        if kind == 'fork':
            s.fork([rng.choice((b, b, rng.randrange(sequences), -1 if rng.random() < 0.2 else b)) for b in range(sequences)])
        elif kind == 'free':
            s.free([rng.choice((1 << 30, s.m.lens[b], rng.randrange(s.m.lens[b] + 1), 0)) for b in range(sequences)])
        else:
            few = rng.random() < 0.4                                           # some that any pool serves
            refused = reserve(s, [rng.choice((0, 1)) if few else rng.choice((0, 1, 63, 64, 65, rng.randrange(1, 200))) for _ in range(sequences)],
                              advance=kind == 'reserve')
            refusals += refused
            served += not refused
            continue
        assert K.device_error() == 0                                           # forks and frees within the sequences refuse nothing
    assert refusals > 0 and served > 0


@pytest.mark.parametrize('pages,share', [(16385, 0.98), (40007, 0.999)])
def test_a_large_pool_runs_empty(K, pages, share):
    rng = random.Random(pages)
    s = Both(K, pages, 50, 40, [1 if rng.random() < share else 0 for _ in range(pages)])
    refusals = [reserve(s, [rng.randrange(0, 300) for _ in range(50)]) for _ in range(6)]
    assert not refusals[0] or pages > 40000
    assert refusals[-1]


def test_many_sequences_are_served_or_reported(K):
    n = 4096
    s = Both(K, 2 * n, n, 3)
    assert not reserve(s, [b % 130 for b in range(n)])
    s.fork([b ^ 1 if b % 3 else b for b in range(n)])
    assert K.device_error() == 0
    assert not reserve(s, [b % 7 and 1 for b in range(n)], advance=False)
    assert reserve(s, [192] * n, advance=False)
    s.free([b % 90 for b in range(n)])
    assert K.device_error() == 0
