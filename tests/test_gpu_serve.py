"""A batch of users from end to end (nebula_b200/serve.py) on a B200: pages, the preparation of queries and keys, attention
with a shared prompt, the MoE layer, sampling and the commit, one after the other."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

SIZE = dict(layers=2, page=16, capacity=96)


@pytest.fixture(scope="module")
def V(gpu_lib):
    from nebula_b200 import serve
    return serve


def alone(V, prompt, question, seed, settings, count, **size):
    batch = V.Batch(1, **size)
    user = V.User(batch.read_prompt(prompt) + question, V.uniforms(seed), settings)
    batch.join(user)
    while len(user.text) < count:
        batch.step()
    return user.text[:count]


SETTINGS = [(0.0, 0, 1.0, 0.0), (0.8, 40, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (0.7, 0, 1.0, 0.05), (1.0, 0, 1.0, 0.0)]


@pytest.mark.parametrize("heads", [(24, 2, 256), (8, 2, 64)])
@pytest.mark.parametrize("length", [5, 40])
def test_users_that_come_and_go(V, heads, length):
    """Users join and leave at different steps; every text is the one that the user alone gets, and no page is lost."""
    size = dict(SIZE, q_heads=heads[0], kv_heads=heads[1], head_dim=heads[2])
    rng = np.random.default_rng(length)
    prompt = [int(t) for t in rng.integers(0, 1024, length)]
    questions = [[int(t) for t in rng.integers(0, 1024, 1 + n)] for n in range(5)]
    batch = V.Batch(3, **size)
    rest = batch.read_prompt(prompt)
    assert batch.pages_in_use() == length // 16
    users = [V.User(rest + q, V.uniforms(n), SETTINGS[n]) for n, q in enumerate(questions)]
    counts, come = [9, 20, 4, 12, 7], 0
    done = set()
    for _ in range(200):
        while come < 5 and None in batch.places:
            batch.join(users[come])
            come += 1
        batch.step()
        for at, user in enumerate(batch.places):
            if user is not None and len(user.text) == counts[users.index(user)]:
                done.add(users.index(batch.leave(at)))
        if len(done) == 5:
            break
    assert len(done) == 5
    assert batch.pages_in_use() == length // 16
    for n, user in enumerate(users):
        assert user.text == alone(V, prompt, questions[n], n, SETTINGS[n], counts[n], **size), n


def test_a_pool_that_runs_dry(V):
    batch = V.Batch(2, **dict(SIZE, pages=3))
    batch.read_prompt(list(range(20)))
    users = [V.User([7], V.uniforms(n)) for n in range(2)]
    for user in users:
        batch.join(user)
    for _ in range(16):
        batch.step()
    with pytest.raises(RuntimeError):
        batch.step()
    batch.leave(1)
    batch.step()  # one has room again
    assert len(users[0].text) == 17


def test_refusals(V):
    batch = V.Batch(1, **SIZE)
    with pytest.raises(ValueError):
        batch.read_prompt(list(range(97)))
    with pytest.raises(ValueError):
        batch.read_prompt([1024])
    with pytest.raises(ValueError):
        batch.join(V.User([], V.uniforms(0)))
    with pytest.raises(ValueError):
        batch.join(V.User([-1], V.uniforms(0)))
    batch.join(V.User([1], V.uniforms(0)))
    with pytest.raises(ValueError):
        batch.join(V.User([1], V.uniforms(0)))
    with pytest.raises(ValueError):
        batch.read_prompt([1])


def test_a_verify_step_with_a_truncated_target(V):
    """Drafts are accepted, and the next token drawn, among the top_k of the target: with one token left it is the greedy one."""
    from nebula_b200 import speculate
    prompt = [5, 6, 7]
    greedy = speculate.greedy(speculate.Speculator(layers=1, nodes=4), [*prompt, 8], 6)
    model = speculate.Speculator(layers=1, nodes=4)
    model.prefill(prompt)
    drafts = [8, greedy[0], greedy[1], (greedy[2] + 1) % model.vocab]
    path, after = model.step(drafts, [-1, 0, 1, 2], uniforms=np.full(4, 0.9), temperature=1.5, top_k=1)
    assert path == [0, 1, 2] and after == greedy[2]
    path, after = model.step([after], [-1], uniforms=[0.7], temperature=0.9, top_p=0.0)
    assert path == [0] and after == greedy[3]
    path, after = model.step([after], [-1], uniforms=[0.3], temperature=2.0, min_p=1.0)
    assert path == [0] and after == greedy[4]
