"""Results of the calls of steps with many tokens a sequence that overlap what other
workgroups still read are refused on the host, before anything touches the GPU."""

import pytest

from instinct_amd import _lib
from test_many_tokens_abi import BAD, FAKE, commit, rejected

# Buffers of their own, each 0x10000 bytes apart.
COMMIT = {name: FAKE * (i + 8) for i, name in enumerate(
    ("tables", "lengths", "starts", "parents", "drafted", "targets", "out_lengths", "accepted",
     "path", "following"))}


def message():
    return _lib.library().pda_last_error().decode()


@pytest.mark.parametrize("result, size", [("out_lengths", 8), ("accepted", 8), ("path", 512),
                                          ("following", 16)])
@pytest.mark.parametrize("other, length", [
    ("tables", 64), ("lengths", 8), ("starts", 12), ("parents", 40), ("drafted", 80),
    ("targets", 80), ("out_lengths", 8), ("accepted", 8), ("path", 512), ("following", 16)])
def test_commit_refuses_overlaps(result, size, other, length):
    if result == other:
        return
    for at in (COMMIT[other] + (length - 8) // 8 * 8, COMMIT[other] - size + 8):
        rejected(commit(**dict(COMMIT, **{result: at})), BAD)
        assert "overlaps" in message() or "out_lengths must not be lengths" in message()
        assert result in message() and other in message()
