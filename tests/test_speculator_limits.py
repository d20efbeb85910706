"""What Speculator refuses before it calls any entry point (no GPU needed): more nodes than its buffers hold, tokens outside
the vocabulary, trees that are none, a cache that is full."""
import numpy as np
import pytest

from nebula_b200 import speculate


@pytest.fixture
def model(monkeypatch):
    """A Speculator without buffers: an entry point that is reached fails the test."""

    def reached(name, *args):
        pytest.fail(f"{name} was called")

    monkeypatch.setattr(speculate.L, "call", reached)
    m = speculate.Speculator.__new__(speculate.Speculator)
    m.nodes, m.vocab, m.capacity, m.committed, m.hidden, m.layers = 4, 100, 32, 10, 64, 1
    names = "masks offsets x embed draft parents uniforms path accepted lengths logits"
    for name in names.split():
        setattr(m, name, type("Buffer", (), {"p": 0})())
    m.weights = []
    return m


BAD = [  # tokens, parents, uniforms
    ([], [], None),
    ([1, 2, 3, 4, 5], [-1, 0, 1, 2, 3], None),
    ([1] * 64, range(-1, 63), None),
    ([1, 2], [-1], None),
    ([1, 2], [-1, 0, 1], None),
    ([1, 100], [-1, 0], None),
    ([-1, 2], [-1, 0], None),
    ([1, 2, 3], [-1, 0, 2], None),
    ([1, 2, 3], [-1, 2, 0], None),
    ([1, 2, 3], [-1, 0, -2], None),
]


@pytest.mark.parametrize("tokens,parents,uniforms", BAD)
def test_trees_are_refused(model, tokens, parents, uniforms):
    with pytest.raises(ValueError):
        model.forward(tokens, parents)
    with pytest.raises(ValueError):
        model.step(tokens, parents, uniforms)


@pytest.mark.parametrize("uniforms", [[0.5], np.zeros(3), [0.5, 1.0], [0.5, -0.1], [0.5, float("nan")]])
def test_uniforms_are_refused(model, uniforms):
    with pytest.raises(ValueError):
        model.step([1, 2], [-1, 0], uniforms, 1.0)


def test_a_full_cache_is_refused(model):
    model.committed = 30
    with pytest.raises(ValueError):
        model.step([1, 2, 3], [-1, 0, 1])
    with pytest.raises(ValueError):
        model.prefill([1, 2, 3])
    model.committed = 10
    with pytest.raises(ValueError):
        model.prefill([1] * 23)  # some of them would fit
    with pytest.raises(ValueError):
        model.prefill([1, 2, 100])
    assert model.committed == 10


def test_masks_and_depths_of_unused_nodes():
    """-1: a node that is not used sees itself alone."""
    assert [int(m) for m in speculate.tree_masks([-1, 0, -1, 1])] == [0b1, 0b11, 0b100, 0b1011]
    assert list(speculate.depths([-1, 0, -1, 1])) == [0, 1, 0, 2]
