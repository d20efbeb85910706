"""The verify step from end to end (nebula_b200/speculate.py) on a B200: drafted trees decode the same text as one token at
a time, in fewer steps, and the cache afterwards holds what plain decoding leaves in it."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def S(gpu_lib):
    from nebula_b200 import speculate
    return speculate


def cached(model, layer):
    """Keys of the committed positions of a layer, in order."""
    n, page = int(model.lengths.get()[0]), model.cache.page_tokens
    pool = model.k.get().view(np.float16).reshape(model.layers, -1, model.kv_heads, model.head_dim)[layer]
    p = np.arange(n)
    return pool[model.table.get()[p // page] * page + p % page].astype(np.float64)


@pytest.mark.parametrize("heads", [(24, 2, 256), (8, 2, 64)])
def test_drafted_trees_decode_the_same_text(S, heads):
    rng = np.random.default_rng(7)
    size = dict(layers=2, q_heads=heads[0], kv_heads=heads[1], head_dim=heads[2], rotary=64, page=16)
    prompt = [int(t) for t in rng.integers(0, 1024, 21)]
    one = S.Speculator(**size)
    plain = S.greedy(one, prompt, 16)

    def drafter(chosen):
        """Right and wrong candidates at three depths; every fourth step all wrong."""
        drafts, parents, at = [], [], 0
        for i in range(3):
            known = len(chosen) + i < len(plain) and len(chosen) % 4 != 3
            drafts += [int(rng.integers(1024)), plain[len(chosen) + i] if known else int(rng.integers(1024))]
            parents += [at, at]
            at = len(drafts)
        return drafts, parents

    many = S.Speculator(**size)
    text, steps = S.speculative(many, prompt, 16, drafter)
    assert text == plain
    assert steps < 12
    n = min(int(m.lengths.get()[0]) for m in (one, many))
    assert n >= 20 + 15
    for layer in range(2):
        a, b = cached(one, layer)[:n], cached(many, layer)[:n]
        # half-precision keys of activations that agree to about 1e-5: a unit in the last place here and there
        np.testing.assert_allclose(b, a, rtol=2.0 ** -9, atol=2.0 ** -9)


def test_sampled_steps_keep_the_targets_choice(S):
    """With uniforms of 0 the first draft that has any mass is accepted; with uniforms near 1 none but a certain one."""
    model = S.Speculator(layers=1, nodes=4)
    model.prefill([5, 6, 7])
    path, _ = model.step([8, 1, 2, 3], [-1, 0, 1, 2], uniforms=np.zeros(4), temperature=1.0)
    assert path == [0, 1, 2, 3]
    path, nxt = model.step([9, 1, 2, 3], [-1, 0, 0, 0], uniforms=np.full(4, 1 - 2.0 ** -24), temperature=5.0)
    assert path == [0] and 0 <= nxt < model.vocab
    assert int(model.lengths.get()[0]) == 3 + 4 + 1
