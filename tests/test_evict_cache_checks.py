"""KVCache.evict finds what is wrong with a call before any layer is packed (on the
CPU: the layers' calls are replaced)."""

import numpy as np
import pytest
import torch

from instinct_amd import eviction
from instinct_amd.paged_kv import KVCache, KVGroup


def two_layers():
    """A cache of two layers and a sequence of 20 rows in it whose first page is
    shared."""
    store = KVCache([KVGroup("g", (0, 3), 2, 8)], page_size=4, capacities={"g": 16},
                    device="cpu")
    table = store.pools["g"].allocate_many(5, reserved=False)
    store.pools["g"].retain(table[:1])
    return store, table


GOOD = torch.ones((1, 2, 20))


@pytest.mark.parametrize("bad, error, match", [
    (None, ValueError, "no weights of layer 3"),
    (GOOD[:, :1].contiguous(), ValueError, "weights of layer 3"),
    (GOOD.repeat(2, 1, 1), ValueError, "weights of layer 3"),
    (GOOD[0], ValueError, "weights of layer 3"),
    (GOOD.double(), TypeError, "weights of layer 3"),
    (GOOD.repeat(1, 1, 2)[..., ::2], ValueError, "weights of layer 3"),
    (GOOD[..., :19].contiguous(), ValueError, "layer 3 must hold its longest"),
])
@pytest.mark.parametrize("shared", [True, False])
def test_cache_evict_checks_every_layer_first(monkeypatch, bad, error, match, shared):
    store, table = two_layers()
    pool = store.pools["g"]
    if not shared:
        pool.release(table[:1])
    monkeypatch.setattr(eviction, "evict_rows", lambda *a, **k: pytest.fail("a layer was packed"))
    weights = {0: GOOD} if bad is None else {0: GOOD, 3: bad}
    refs = pool._refs.copy()
    with pytest.raises(error, match=match):
        store.evict("g", [table], np.array([20]), weights, keep=8)
    assert pool.free == 11 and np.array_equal(pool._refs, refs)


def test_cache_evict_gives_fresh_pages_back(monkeypatch):
    """A layer's call that fails leaves the pool as it was."""
    def fail(*args, **kw):
        raise RuntimeError("launch")

    store, table = two_layers()
    monkeypatch.setattr(eviction, "evict_rows", fail)
    refs = store.pools["g"]._refs.copy()
    with pytest.raises(RuntimeError, match="launch"):
        store.evict("g", [table], np.array([20]), {0: GOOD, 3: GOOD}, keep=8)
    assert store.pools["g"].free == 11 and np.array_equal(store.pools["g"]._refs, refs)


def test_cache_evict_checks_pages_and_lengths_first(monkeypatch):
    store, table = two_layers()
    monkeypatch.setattr(eviction, "evict_rows", lambda *a, **k: pytest.fail("a layer was packed"))
    weights = {0: GOOD, 3: GOOD}
    with pytest.raises(RuntimeError, match="does not hold"):
        store.evict("g", [np.append(table[:4], 9)], np.array([20]), weights, keep=8)
    with pytest.raises(RuntimeError, match="does not hold"):
        store.evict("g", [np.append(table[1:], table[1])], np.array([20]), weights, keep=8)
    with pytest.raises(ValueError, match="lengths"):
        store.evict("g", [table], np.array([20, 20]), weights, keep=8)
    assert store.pools["g"].free == 11
