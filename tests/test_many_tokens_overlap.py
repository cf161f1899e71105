"""Results of the calls of steps with many tokens a sequence that overlap what other
workgroups still read are refused on the host, before anything touches the GPU."""

import pytest

from instinct_amd import _lib
from test_many_tokens_abi import BAD, FAKE, commit, extend, rejected

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


# Two sequences of 10 tokens in all, tables of 4 pages, a feed of 10.
EXTEND = {name: FAKE * (i + 8) for i, name in enumerate(
    ("tables", "lengths", "counts", "pages", "feed", "drawn", "parents", "starts", "out_lengths",
     "out_pages", "out_drawn", "rows", "positions", "masks"))}
SIZES = dict(tables=32, lengths=8, counts=8, pages=8, feed=40, drawn=8, parents=40, starts=12,
             out_lengths=8, out_pages=8, out_drawn=8, rows=40, positions=40, masks=80)
IN_PLACE = dict(out_lengths="lengths", out_pages="pages", out_drawn="drawn")


@pytest.mark.parametrize("result", ["tables", "starts", "out_lengths", "out_pages", "out_drawn",
                                    "rows", "positions", "masks"])
@pytest.mark.parametrize("other", list(SIZES))
def test_extend_refuses_overlaps(result, other):
    if result == other:
        return
    last = EXTEND[other] + (SIZES[other] - 1) // 8 * 8
    before = EXTEND[other] - (SIZES[result] + 7) // 8 * 8 + 8
    for at in {last, before}:
        if IN_PLACE.get(result) == other and at == EXTEND[other]:
            at = EXTEND[other] + 4  # (itself is in place)
        rejected(extend(**dict(EXTEND, batch=2, tokens=10, table_stride=4, feed_len=10,
                               **{result: at})), BAD)
        assert "overlaps" in message() and result in message() and other in message()
