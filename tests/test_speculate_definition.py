"""The 64-bit definition of acceptance (oracle/speculate.py) where its own steps can go wrong (no GPU needed)."""
import numpy as np

from oracle import speculate as S


def test_siblings_drawn_from_a_distribution_follow_the_target():
    """Several candidates drawn from one q for the same place: over all uniforms the first new token has the target's
    distribution, because a refusal leaves max(p - q, 0) scaled to a distribution again."""
    rng = np.random.default_rng(6)
    logits = rng.normal(size=(4, 6))
    p, q = S.target(logits[0], 0.7), S.target(rng.normal(size=6), 1.0)
    counts, n = np.zeros(6), 20000
    for _ in range(n):
        draft = [0, *rng.choice(6, size=3, p=q)]
        path, nxt, _ = S.verify(logits, draft, [-1, 0, 0, 0], [q] * 4, rng.random(4), 0.7)
        counts[draft[path[1]] if len(path) > 1 else nxt] += 1
    # five standard deviations of a count
    assert np.all(np.abs(counts / n - p) < 5 * np.sqrt(p * (1 - p) / n))
