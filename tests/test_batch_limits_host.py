"""What the entry points for a batch of users and the caches that they run on refuse at the edges (no GPU needed; the pointers are
never dereferenced)."""
import pytest

import test_batch_host as batch
import test_speculate_host as verify

INVALID, P4 = batch.INVALID, batch.P4


@pytest.mark.parametrize("off", [1, 2, 3])
def test_pages_held_are_whole_numbers(off):
    assert batch.attention(batch.cache(held=P4 + off)) == INVALID
    for entry in (verify.attention, verify.prep, verify.commit):
        assert entry(verify.cache(held=P4 + off)) == INVALID
