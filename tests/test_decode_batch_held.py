"""DecodeBatch's rows and lengths where sequences hold fewer rows than they have
positions (on the CPU: the constructor alone)."""

import numpy as np
import pytest
import torch

from instinct_amd.batches import DecodeBatch
from instinct_amd.paged_kv import KVCache, KVGroup

PAGE = 16


def cache(*groups):
    return KVCache([KVGroup(name, (i,), 1, 8, window) for i, (name, window) in enumerate(groups)],
                   page_size=PAGE, capacities={name: 16 for name, _ in groups}, device="cpu")


def batch(store, tables, positions=(37, 20), **kw):
    return DecodeBatch(store, torch.zeros(2), positions=np.array(positions), tables=tables, **kw)


def rows(b, name):
    return b._write[name].tolist(), b._lengths[name].tolist(), b._longest[name]


FULL = [np.array([5]), np.array([7, 2])]
LOCAL = [np.array([-1, 4, 9]), np.array([1, 3])]


def test_groups_hold_different_rows():
    """A full group was cut, the windowed one beside it was not."""
    store = cache(("full", 0), ("local", 16))
    b = batch(store, {"full": FULL, "local": LOCAL}, held={"full": np.array([8, 20])})
    assert rows(b, "full") == ([5 * PAGE + 8, 2 * PAGE + 4], [9, 21], 21)
    assert rows(b, "local") == ([9 * PAGE + 5, 3 * PAGE + 4], [38, 21], 38)
    assert b.offsets.tolist() == [37, 20]
    assert b.lengths.tolist() == [38, 21] and b.longest == 38


def test_one_vector_is_for_one_group():
    store = cache(("full", 0), ("local", 16))
    with pytest.raises(ValueError, match="several"):
        batch(store, {"full": FULL, "local": LOCAL}, held=np.array([8, 20]))
    one = cache(("full", 0))
    for held in (np.array([8, 20]), {"full": np.array([8, 20])}):
        b = batch(one, {"full": FULL}, held=held)
        assert rows(b, "full") == ([5 * PAGE + 8, 2 * PAGE + 4], [9, 21], 21)
        assert b.lengths.tolist() == [9, 21] and b.longest == 21
        assert b.offsets.tolist() == [37, 20]


@pytest.mark.parametrize("held, match", [({"other": np.array([8, 20])}, "no group"),
                                         (np.array([8]), "each sequence"),
                                         (np.array([8, -1]), "each sequence"),
                                         ({"full": np.array([[8, 20]])}, "each sequence")])
def test_held_is_checked(held, match):
    with pytest.raises(ValueError, match=match):
        batch(cache(("full", 0)), {"full": FULL}, held=held)


def test_nothing_held_apart():
    store = cache(("full", 0), ("local", 16))
    full = [np.array([5, 6, 8]), np.array([7, 2])]
    b = batch(store, {"full": full, "local": LOCAL})
    assert rows(b, "full") == ([8 * PAGE + 5, 2 * PAGE + 4], [38, 21], 38)
    assert rows(b, "local")[1:] == ([38, 21], 38)


@pytest.mark.parametrize("held", [None, {"full": np.array([16, 20])}])
def test_a_row_needs_its_page(held):
    """The packed tables are padded with page 0, another sequence's: a sequence
    whose new row lies past its own pages (as after an eviction down to whole
    pages) is refused."""
    positions = (16, 20) if held is None else (37, 20)
    with pytest.raises(ValueError, match="no page for row 16"):
        batch(cache(("full", 0)), {"full": FULL}, positions=positions, held=held)


def test_weights_hold_every_sequence():
    """A shorter capacity would cut a sequence's newest keys from its softmax."""
    store = cache(("full", 0), ("local", 16))
    tables = {"full": FULL, "local": LOCAL}
    held = {"full": np.array([8, 20])}
    fits = {0: torch.zeros((2, 1, 21)), 1: torch.zeros((2, 1, 38))}
    assert batch(store, tables, held=held, weights=fits).weights is fits
    for layer, capacity in ((0, 20), (1, 37)):
        with pytest.raises(ValueError, match=f"layer {layer}"):
            batch(store, tables, held=held,
                  weights={**fits, layer: torch.zeros((2, 1, capacity))})
    with pytest.raises(ValueError, match="layer 5"):
        batch(store, tables, held=held, weights={5: torch.zeros((2, 1, 64))})
