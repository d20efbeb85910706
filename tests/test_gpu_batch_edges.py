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
