"""A PageFeed and the calls that take it: what is refused, on the CPU."""

import gc
import weakref

import pytest
import torch

from instinct_amd import paging
from instinct_amd.paged_kv import KVCache, KVGroup


def cache(**kw):
    return KVCache([KVGroup("a", (0,), 2, 64)], page_size=16, capacities={"a": 32},
                   **dict(dict(device="cpu"), **kw))


def test_a_feed_or_ids_with_their_count():
    feed = paging.PageFeed(cache(), "a", 4)
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32)  # noqa: E731
    args = (i32(1, 3), i32(1), i32(1), i32(1))
    with pytest.raises(TypeError, match="counts for itself"):
        paging.extend_tables(*args, feed, feed.drawn, page_size=16, tokens=1)
    with pytest.raises(TypeError, match="page ids"):
        paging.extend_tables(*args, feed.pages, page_size=16, tokens=1)
    with pytest.raises(ValueError, match="16 rows"):
        paging.extend_tables(*args, feed, page_size=32, tokens=1)


def test_refill_and_close_stay_in_place():
    """Steps that were captured read the feed's tensors: no page that they may still draw
    is listed twice."""
    c = cache()
    feed = paging.PageFeed(c, "a", 10)
    pages, drawn = feed.pages, feed.drawn
    drawn[0] = 4
    feed.refill(8)
    assert feed.drawn is drawn and drawn.tolist() == [0, 0]
    assert pages.tolist() == [4, 5, 6, 7, 8, 9, 10, 11, -1, -1]
    assert feed.pages.data_ptr() == pages.data_ptr()
    drawn[0] = 8
    feed.refill(10)
    assert pages.tolist() == feed.pages.tolist() == list(range(12, 22))
    # Past its room: what was captured on the old tensors finds nothing.
    drawn[0] = 1
    feed.refill(11)
    assert pages.tolist() == [-1] * 10 and feed.drawn is not drawn
    assert feed.pages.tolist() == list(range(13, 24)) and feed.drawn.tolist() == [0, 0]
    pages = feed.pages
    feed.close()
    assert pages.tolist() == [-1] * 11 and feed.pages.tolist() == []
    assert c.pools["a"].free == 32 - 13
    feed.refill(3)  # a closed feed may go on
    assert feed.pages.tolist() == [13, 14, 15]


def test_outgrown_tensors_stay():
    """A graph captured on them holds addresses alone."""
    feed = paging.PageFeed(cache(), "a", 4)
    drawn = weakref.ref(feed.drawn)
    address = feed.pages.data_ptr()
    feed.refill(9)
    gc.collect()
    assert drawn() is not None and feed._outgrown[0][0].data_ptr() == address
    assert feed._outgrown[0][0].tolist() == [-1] * 4
