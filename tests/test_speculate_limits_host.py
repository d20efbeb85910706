"""Sizes and numbers at the end of their range that the verify step's entry points refuse (no GPU needed; the pointers are
never dereferenced)."""
import pytest

from test_speculate_host import INVALID, attention, cache, commit, prep


@pytest.mark.parametrize("page,table_pages", [(16, (1 << 27) - 1), (64, (1 << 25) - 1), (16, (1 << 27) - 7)])
def test_positions_end_before_a_units_end_passes_31_bits(page, table_pages):
    """The last unit of 128 keys would end past 2^31: the count of units of such a sequence is negative in 32 bits."""
    positions = page * table_pages
    assert positions <= 0x7FFFFFFF < positions + 127
    c = dict(page_tokens=page, table_pages=table_pages, layers=1)
    assert attention(cache(**c)) == INVALID
    assert prep(cache(**c)) == INVALID
    assert commit(cache(**c)) == INVALID


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf"), 3e38, -3e38])
def test_attention_refuses_a_scale_that_is_not_finite(scale):
    """Also one that is not finite any more in units of powers of two (times log2(e))."""
    assert attention(cache(), scale=scale) == INVALID
