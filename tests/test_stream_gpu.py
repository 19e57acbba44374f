"""The streaming policy (stream.StreamMemory): a reduced-depth policy over several frames, every attention of every layer compared
with its definition in 64 bits on the same cache, the caches with what was appended, and the stateless path left as it was.

Tolerance of the attention: as in test_memory_gpu.py (2^-10 sum p |v| + half an ulp). Cached values: a block's tokens arrive in
at most three frames, so a value is off by at most half a step when written and half a step each time the block's scale grows
afterwards (at most twice)."""
import pytest
import torch

import memory_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def P():
    if not torch.cuda.is_available():
        pytest.skip('no CUDA device')
    from yanlongvla_b200 import policy
    return policy


@pytest.fixture(scope='module')
def setup(P):
    c = P.PolicyConfig(vit_layers=1, llm_layers=2, dit_layers=2)
    model, _, _ = P.build_policy(runtime='resident', c=c)
    return c, model


def frames(P, c, B, n):
    return [P.synthetic_observations(B, c, seed=10 + f) for f in range(n)]


def test_every_attention_against_its_definition(P, setup, monkeypatch):
    from yanlongvla_b200 import kernels as K
    from yanlongvla_b200.stream import StreamMemory
    c, model = setup
    memory = StreamMemory(c, 2, 3 * c.prefix_tokens)
    seen = []
    attention, append = K.kv8_attention, K.kv8_append

    def spy(q, cache, table, lens, **kw):
        o = attention(q, cache, table, lens, **kw)
        want, a = ref.attention(q, cache, table, lens.tolist())
        err = (o.double() - want).abs()
        assert (err <= 2.0 ** -8 * want.abs() * (1 + 2.0 ** -10) + 2.0 ** -10 * a + 2.0 ** -25).all()
        seen.append(lens.tolist())
        return o

    kept = {}

    def spy_append(cache, k, v, *args, **kw):
        kept.setdefault(id(cache), []).append((ref.rotary(k.double().view(2, -1, c.llm_kv_heads, 64), kw['pos'], kw['rope'].cos, kw['rope'].sin,
                                                          kw['rope'].sections, False), v.double().view(2, -1, c.llm_kv_heads, 64)))
        return append(cache, k, v, *args, **kw)

    monkeypatch.setattr(K, 'kv8_attention', spy)
    monkeypatch.setattr(K, 'kv8_append', spy_append)
    with torch.no_grad():
        for obs in frames(P, c, 2, 3):
            assert torch.isfinite(model(*obs, memory=memory)).all()
    assert seen == [[160 * (f + 1)] * 2 for f in range(3) for _ in range(2)]
    n = 3 * c.prefix_tokens
    for cache in memory.caches:
        for b in range(2):
            for i, (cells, scale, tr) in enumerate(((cache.k, cache.k_scale, False), (cache.v, cache.v_scale, True))):
                held = ref.values(cells, scale, memory.table[b], n, tr)
                want = torch.cat([x[i][b] for x in kept[id(cache)]])
                step = scale[memory.table[b].long()].double().repeat_interleave(64, 0)[:n, :, None]
                assert ((held - want).abs() <= (1.5 + 1e-3) * step).all()


def test_memory_matters_and_forgets(P, setup):
    from yanlongvla_b200.stream import StreamMemory
    c, model = setup
    first, second = frames(P, c, 1, 2)
    memory = StreamMemory(c, 1, 2 * c.prefix_tokens)
    with torch.no_grad():
        a1, a2 = model(*first, memory=memory), model(*second, memory=memory)
        with pytest.raises(Exception, match='does not fit'):
            model(*second, memory=memory)
        memory.forget()
        assert torch.equal(model(*first, memory=memory), a1) and torch.equal(model(*second, memory=memory), a2)
        memory.forget()
        assert not torch.equal(model(*second, memory=memory), a2)            # without the first frame the second looks different


def test_stateless_path_is_unchanged(P, setup):
    c, model = setup
    obs = frames(P, c, 1, 1)[0]
    with torch.no_grad():
        prefix = model.embed(*obs[:2])
        want = model.backbone(prefix)
        assert torch.equal(model.backbone(prefix, None), want)
        assert torch.equal(model(*obs), model.action_head(want, *obs[2:]))
