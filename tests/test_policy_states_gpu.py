"""The policy with instructions of differing length and with several candidates: every cross-attention of the action head against its
definition in 64 bits, padding without effect, candidates that do not see one another, and the path without either as it was."""
import pytest
import torch

import cross_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def small():
    if not torch.cuda.is_available():
        pytest.skip('no CUDA device')
    from yanlongvla_b200 import policy as P
    c = P.PolicyConfig(vit_layers=1, llm_layers=2, dit_layers=4)
    model, layers, _ = P.build_policy('cuda', 'resident', c)
    return P, c, model, layers


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device='cuda')


def candidates(c, B, S, seed=0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return torch.randn(B * S, c.chunk, c.action_dim, device='cuda', generator=g)


@pytest.mark.parametrize('B,S,lens', [(3, 1, [1, 17, 32]), (2, 5, None), (2, 16, [32, 3])])
def test_every_cross_attention_against_its_definition(small, monkeypatch, B, S, lens):
    from yanlongvla_b200 import kernels as K
    P, c, model, _ = small
    images, lang, state, _ = P.synthetic_observations(B, c, seed=5)
    calls = []
    cross = K.cross_attention

    def spy(q, k, v, heads, lens=None, **kw):
        o = cross(q, k, v, heads, lens=lens, **kw)
        want, tol = ref.attention(q, k, v, heads, lens=lens)
        assert ((o.double() - want).abs() <= tol).all()
        calls.append((tuple(q.shape), tuple(k.shape)))
        return o

    monkeypatch.setattr(K, 'cross_attention', spy)
    with torch.no_grad():
        a = model(images, lang, state, candidates(c, B, S), lang_lens=None if lens is None else ints(lens))
    assert a.shape == (B * S, c.chunk, c.action_dim) and torch.isfinite(a).all()
    assert calls == [((B * S, c.chunk + 1, c.dit_hidden), (B, c.prefix_tokens, c.dit_hidden))] * (2 * c.flow_steps)
    assert K.device_error() == 0


def test_padding_has_no_effect(small):
    P, c, model, _ = small
    images, lang, state, noise = P.synthetic_observations(3, c, seed=6)
    lens = ints([4, 31, 0])
    other = lang.clone()
    for b, n in enumerate(lens.tolist()):
        other[b, n:] = (other[b, n:] + 1 + b) % c.vocab
    with torch.no_grad():
        a, b = (model(images, x, state, noise, lang_lens=lens) for x in (lang, other))
        assert torch.equal(a, b)
        assert not torch.equal(model(images, other, state, noise), model(images, lang, state, noise))


def test_candidates_do_not_see_one_another(small):
    P, c, model, _ = small
    images, lang, state, _ = P.synthetic_observations(2, c, seed=7)
    noise = candidates(c, 2, 6)
    order = torch.tensor([3, 0, 5, 1, 4, 2], device='cuda')
    changed = noise.clone().view(2, 6, c.chunk, c.action_dim)
    changed[1, 2] += 1
    with torch.no_grad():
        a = model(images, lang, state, noise).view(2, 6, c.chunk, c.action_dim)
        p = model(images, lang, state, noise.view(2, 6, c.chunk, c.action_dim)[:, order].reshape(noise.shape)).view_as(a)
        d = model(images, lang, state, changed.view_as(noise)).view_as(a)
        with pytest.raises(ValueError, match='noise'):
            model(images, lang, state, noise[:5])
    assert torch.equal(p, a[:, order])
    same = torch.ones(2, 6, dtype=torch.bool)
    same[1, 2] = False
    assert torch.equal(d[same], a[same]) and not torch.equal(d[1, 2], a[1, 2])


def test_the_reference_runtime_has_them_too(small):
    """The runtime of PyTorch operations: one candidate each and whole instructions are the path without either; the quantizers after
    the attention turn its last bits into steps, so the rest is held to the policy's tolerance on the first attention alone."""
    from yanlongvla_b200 import definition
    P, c, _, layers = small
    model, _, _ = P.build_policy('cuda', 'reference', c, layers=layers)
    images, lang, state, noise = P.synthetic_observations(2, c, seed=8)
    with torch.no_grad():
        a = model(images, lang, state, candidates(c, 2, 3), lang_lens=ints([0, 9]))
    assert a.shape == (6, c.chunk, c.action_dim) and torch.isfinite(a).all()
    q, k, v = (torch.randn(n, t, 96, device='cuda').bfloat16() for n, t in ((4, 7), (2, 30), (2, 30)))
    v[1, 20:] = float('nan')
    o = definition.cross_attention(q, k, v, 2, lens=ints([0, 20]))
    want, tol = ref.attention(q, k, v, 2, lens=ints([0, 20]))
    assert not o[:2].any() and ((o.double() - want).abs() <= tol).all()
