"""Operators for a batch of users on a B200, at the edges of what their header allows and next to each other."""
import numpy as np
import pytest

from test_gpu_sample import L, check  # noqa: F401  (L is a fixture)

pytestmark = pytest.mark.gpu


# ---- sampling --------------------------------------------------------------


@pytest.mark.parametrize("least", [np.nextafter(np.float32(1), np.float32(2)), 1.5, np.inf])
def test_min_p_above_one_leaves_the_first_of_equals(L, least):  # noqa: F811
    """No probability is more than the largest, so nothing stays but the token that is always kept."""
    rng = np.random.default_rng(21)
    x = np.round(rng.normal(size=(8, 5003)) * 4) / 4
    for r, n in enumerate((1, 2, 40, 300, 1500, 5003, 7, 600)):
        x[r, rng.choice(5003, n, replace=False)] = 9.0
    u = np.array([0.0, 0.9, 0.99, 0.3, 0.7, 0.999, 0.5, 0.6])
    for k, p in ((0, 1.0), (50, 1.0), (400, 1.0), (2000, 1.0), (5002, 0.9), (0, 0.9), (0, 0.0), (1, 1.0)):
        check(L, x, u, [1.0] * 8, [k] * 8, [p] * 8, [least] * 8)


# ---- users ---------------------------------------------------------------------


@pytest.fixture(scope="module")
def V(gpu_lib):
    from nebula_b200 import serve
    return serve


SIZE = dict(layers=1, page=16, capacity=64)


def alone(V, question, seed, settings, count):
    batch = V.Batch(1, **SIZE)
    user = V.User(batch.read_prompt([3, 4, 5]) + question, V.uniforms(seed), settings)
    batch.join(user)
    while len(user.text) < count:
        batch.step()
    return user.text[:count]


@pytest.mark.parametrize("place", [0, 1, 2])
def test_a_user_without_a_distribution_stops_no_other(V, place):
    """A refused row raises before anything is kept of the step; without that user the others get the texts they get alone."""
    from nebula_b200 import lib
    settings = [(0.8, 40, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (0.7, 0, 1.0, 0.05)]
    texts = [alone(V, [7 + n], n, settings[n], 8) for n in range(3)]
    batch = V.Batch(3, **SIZE)
    rest = batch.read_prompt([3, 4, 5])
    nothing = np.full(batch.hidden, np.nan, np.float32)  # a token whose embedding is not a number
    lib.call("write", batch.embed.p + 4 * 1000 * batch.hidden, nothing.ctypes.data, nothing.nbytes)
    users = [V.User(rest + [7 + n], V.uniforms(n), settings[n]) for n in range(3)]
    users[place].waiting.append(1000)
    for user in users:
        batch.join(user)
    others = [n for n in range(3) if n != place]
    for _ in range(20):
        try:
            batch.step()
        except RuntimeError as e:
            assert str(place) in str(e)
            with pytest.raises(RuntimeError):
                batch.step()  # it stays so
            assert batch.leave(place) is users[place]
            break
    else:
        pytest.fail("the row was not refused")
    while min(len(users[n].text) for n in others) < 8:
        batch.step()
    for n in others:
        assert users[n].text[:8] == texts[n], n
    assert users[place].text == []


@pytest.mark.parametrize("numbers", [[0.5, 0.25], [0.5, 0.25, float("nan")]])
def test_a_user_without_uniforms_stops_no_other(V, numbers):
    """Numbers that end, or are none, take no number from the other users."""
    settings = (1.0, 0, 1.0, 0.0)
    texts = [alone(V, [7 + n], n, settings, 8) for n in range(3)]
    batch = V.Batch(3, **SIZE)
    rest = batch.read_prompt([3, 4, 5])
    users = [V.User(rest + [7 + n], V.uniforms(n), settings) for n in range(3)]
    users[1].uniforms = iter(numbers)
    for user in users:
        batch.join(user)
    with pytest.raises(ValueError, match="1"):
        for _ in range(20):
            batch.step()
    assert len(users[1].text) == 2
    batch.leave(1)
    while len(users[0].text) < 8:
        batch.step()
    assert [users[0].text[:8], users[2].text[:8]] == [texts[0], texts[2]]


BAD = [(-1.0, 0, 1.0, 0.0), (float("nan"), 0, 1.0, 0.0), (float("inf"), 0, 1.0, 0.0), (1e39, 0, 1.0, 0.0), (1.0, 0, float("nan"), 0.0),
       (1.0, 0, 1.0, float("nan")), (1.0, 1 << 31, 1.0, 0.0), (1.0, 0.5, 1.0, 0.0), (1.0, 0, 1.0), None]


def test_settings_that_no_row_can_have_are_refused(V):
    batch = V.Batch(2, **SIZE)
    for settings in BAD:
        with pytest.raises(ValueError):
            batch.join(V.User([1], V.uniforms(0), settings))
    assert batch.places == [None, None]
    user = V.User([1], V.uniforms(0), (0.5, -3, 1.5, -1.0))
    batch.join(user)
    batch.step()
    assert len(user.text) == 1
