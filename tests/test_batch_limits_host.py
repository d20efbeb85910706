"""What the entry points for a batch of users and the caches that they run on refuse at the edges (no GPU needed; the pointers are
never dereferenced)."""
import pytest

import test_batch_host as batch
import test_speculate_host as verify
from test_speculator_limits import model  # noqa: F401  (a fixture)

INVALID, P4 = batch.INVALID, batch.P4


@pytest.mark.parametrize("off", [1, 2, 3])
def test_pages_held_are_whole_numbers(off):
    assert batch.attention(batch.cache(held=P4 + off)) == INVALID
    for entry in (verify.attention, verify.prep, verify.commit):
        assert entry(verify.cache(held=P4 + off)) == INVALID


def test_pages_held_that_are_announced_are_there():
    assert batch.attention(batch.cache(page_tokens=16 | batch.L.KvCache.HELD)) == INVALID
    for entry in (verify.attention, verify.prep, verify.commit):
        assert entry(verify.cache(page_tokens=16 | batch.L.KvCache.HELD)) == INVALID


POOL = dict(page_table=P4 + (1 << 16), held=P4 + (2 << 16), free_pages=P4 + (3 << 16), free_count=P4 + (4 << 16))
FREE = dict(slots=P4 + (5 << 16), taken=P4 + (6 << 16), lengths=P4 + (7 << 16), counts=P4 + (8 << 16))


@pytest.mark.parametrize("what", ["page_table", "held", "free_pages", "free_count", "lengths", "counts", "slots", "taken"])
def test_results_of_pages_overlap_nothing(what):
    """Not in part either: a sequence's result is written while another's lengths, counts or pages are read. Three sequences, 20 entries of
    the table each, 100 pages, 5 slots a sequence."""
    size = dict(page_table=60, held=3, free_pages=100, free_count=1, lengths=3, counts=3, slots=15, taken=3)
    at = {**POOL, **FREE}[what]
    for name in ("taken", "slots"):
        if name == what:
            continue
        for p in {at, at + 4 * (size[what] - 1), at - 4 * (size[name] - 1)}:
            assert batch.reserve(batch.pool(**POOL), **{**FREE, name: p}) == INVALID, (name, p - at)
    if what in ("counts", "slots", "taken"):
        return
    for p in {at, at + 4 * (size[what] - 1), at - 8}:
        assert batch.release(batch.pool(**POOL), freed=p, lengths=FREE["lengths"]) == INVALID, p - at


@pytest.mark.parametrize("settings", [dict(top_p=float("nan")), dict(min_p=float("nan")), dict(top_k=0.5), dict(top_k=1 << 31), dict(top_k=float("nan")),
                                      dict(temperature=1e39, top_k=5), dict(temperature=float("nan"), min_p=0.1), dict(temperature=-1.0, top_p=0.9)], ids=str)
def test_steps_refuse_settings_that_no_row_can_have(model, settings):  # noqa: F811
    """NaN is neither below 1 nor above 0: the target would have been left as it is."""
    with pytest.raises(ValueError):
        model.step([1, 2], [-1, 0], [0.5, 0.5], **{"temperature": 1.0, **settings})


def test_a_batch_reads_no_single_sequence():
    """What Speculator does to one sequence of its own cache would go to the first user's pages."""
    from nebula_b200 import serve
    b = serve.Batch.__new__(serve.Batch)
    with pytest.raises(NotImplementedError):
        b.forward([1], [-1])
    with pytest.raises(NotImplementedError):
        b.prefill([1])


def test_settings_of_any_kind_of_number():
    import numpy as np
    from nebula_b200.speculate import check_settings
    for settings in ((0.8, 40, 0.95, 0.0), (0, 0, 1, 0), (np.float32(1), np.int64(4), np.float64(2.0), float("inf")), (np.array(0.8), np.array(3), 1, 0), (1, 40.0, 1, 0)):
        check_settings(*settings)
    for settings in (("a", 0, 1, 0), (None, 0, 1, 0), (1, None, 1, 0), (1, 1 << 3000, 1, 0), (1, float("inf"), 1, 0)):
        with pytest.raises(ValueError):
            check_settings(*settings)
