"""A PageFeed and the calls that take it: what is refused, on the CPU."""

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
