"""PackedPrefillBatch, DraftBatch and PageFeed check what they are asked on the host."""

import numpy as np
import pytest
import torch

from instinct_amd import batches, paging
from instinct_amd.paged_kv import KVCache, KVGroup


def cache(window=0):
    groups = [KVGroup("a", (0,), 2, 64), KVGroup("b", (1,), 2, 64, window)]
    return KVCache(groups, page_size=16, capacities={"a": 32, "b": 32}, device="cpu")


TABLES = {"a": [np.array([1, 2]), np.array([3])], "b": [np.array([1, 2]), np.array([3])]}
TOKENS = torch.zeros(6, dtype=torch.int64)


@pytest.mark.parametrize("kw, match", [
    (dict(counts=[3, 2]), "counts"), (dict(counts=[7, -1]), "counts"),
    (dict(tables=dict(TABLES, b=[np.array([1])])), "table for each"),
    (dict(tables=dict(TABLES, b=[np.array([1]), np.array([], dtype=int)])), "no page for row")])
def test_packed_prefill_refuses(kw, match):
    base = dict(counts=[4, 2], tables=TABLES)
    with pytest.raises(ValueError, match=match):
        batches.PackedPrefillBatch(cache(), TOKENS, **dict(base, **kw))


@pytest.mark.parametrize("kw, match", [
    (dict(counts=[3, 2]), "counts"), (dict(parents=[-1, 0, 1, 3, -1, 0]), "earlier"),
    (dict(parents=[-1, 0, 1, 2, -1, -2]), "earlier"), (dict(parents=[-1, 0]), "earlier"),
    (dict(positions=[3]), "positions"), (dict(positions=[3, -1]), "positions"),
    (dict(positions=[29, 0]), "no page for row 32 of sequence 0"),
    (dict(held=[1, 2]), "name its groups"), (dict(held=dict(b=[1, 2])), "windowed")])
def test_draft_refuses(kw, match):
    base = dict(counts=[4, 2], parents=[-1, 0, 1, 0, -1, 0], positions=[5, 6], tables=TABLES)
    with pytest.raises(ValueError, match=match):
        batches.DraftBatch(cache(window=8), TOKENS, **dict(base, **kw))


def test_new_rows_on_released_pages():
    released = [np.array([-1, 2, 3]), np.array([4, -1])]
    with pytest.raises(ValueError, match="'b': no page for row 0 of sequence 0"):
        batches.PackedPrefillBatch(cache(), TOKENS, counts=[4, 2],
                                   tables=dict(TABLES, b=released))
    args = dict(counts=[4, 2], parents=[-1, 0, 1, 0, -1, 0])
    tables = dict(a=[np.array([1, 2, 3]), np.array([4, 5])], b=released)
    page = cache().page_size
    with pytest.raises(ValueError, match=f"'b': no page for row {page} of sequence 1"):
        batches.DraftBatch(cache(), TOKENS, positions=[page + 1, page - 1], tables=tables, **args)
    with pytest.raises(ValueError, match=f"'b': no page for row {page + 2} of sequence 1"):
        batches.DraftBatch(cache(), TOKENS, positions=[page + 1, page + 2], tables=tables, **args)


def test_draft_of_more_than_64_nodes():
    with pytest.raises(ValueError, match="64 nodes"):
        batches.DraftBatch(cache(), torch.zeros(65, dtype=torch.int64), counts=[65],
                           parents=np.arange(-1, 64), positions=[0],
                           tables={g: [np.arange(9)] for g in "ab"})


def test_page_feed_accounts_for_its_pages():
    c = cache()
    feed = paging.PageFeed(c, "a", 10)
    assert c.pools["a"].free == 22 and feed.pages.tolist() == list(range(10))
    feed.drawn[0] = 4
    feed.refill(8)
    assert feed.pages.tolist() == [4, 5, 6, 7, 8, 9, 10, 11] and feed.drawn.tolist() == [0, 0]
    feed.drawn[0] = 3
    feed.close()
    assert c.pools["a"].free == 32 - 7
    c.pools["a"].release(range(7))  # what the tables hold
    with pytest.raises(RuntimeError):
        paging.PageFeed(c, "a", 33)
    feed = paging.PageFeed(c, "a", 2)
    feed.drawn[0] = 3
    with pytest.raises(RuntimeError, match="no row"):
        feed.refill(4)
