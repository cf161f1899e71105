"""The eviction's calls next to 2^31 positions are refused on the host: their
loops count in 32 bits, a block past the last position."""

import pytest
from test_evict_abi import move, select

from instinct_amd import _lib

LAST = (1 << 31) - 1


@pytest.mark.parametrize("past", [0, 4095, 4096, 8191])
def test_select(past):
    for overrides in (dict(capacity=LAST - past), dict(keep=LAST - past)):
        assert select(out_weights=None, **overrides) == _lib.PDA_ERR_TOO_LONG


@pytest.mark.parametrize("past", [0, 8191])
def test_move(past):
    assert move(keep=LAST - past) == _lib.PDA_ERR_TOO_LONG
