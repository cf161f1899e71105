"""A DraftBatch is committed once: a second time its rows would move from where others
lie by then."""

import numpy as np
import pytest
import torch

from instinct_amd.batches import DraftBatch
from instinct_amd.paged_kv import KVCache, KVGroup

pytestmark = pytest.mark.gpu


def test_commit_once(gpu):
    cache = KVCache([KVGroup("a", (0,), 2, 64), KVGroup("b", (1,), 2, 64)], page_size=16,
                    capacities={"a": 8, "b": 8})
    tables = {g: [cache.pools[g].allocate_many(2, reserved=False)] for g in "ab"}
    nodes = torch.arange(5, device="cuda")
    batch = DraftBatch(cache, nodes, counts=[5], parents=[-1, 0, 0, 2, 3], positions=[10],
                       tables=tables)
    k = torch.randn(5, 2, 64, device="cuda").half()
    q = torch.randn(5, 4, 64, device="cuda").half()
    for layer in (0, 1):
        batch.attend(layer, q, k, -k, scale=0.1)
    targets = torch.tensor([2, -1, 3, 4, -1], device="cuda")
    with pytest.raises(TypeError):  # (nothing has moved yet)
        batch.commit(targets.int())
    kept = batch.commit(targets)
    assert {g: x.path[0, :5].tolist() for g, x in kept.items()} == dict.fromkeys("ab", [0, 2, 3, 4, -1])

    def check():
        for layer, g in enumerate("ab"):
            rows = torch.as_tensor(cache.rows(np.asarray(tables[g][0]), 10, 14), device="cuda")
            assert torch.equal(cache._pick(cache.keys[layer], rows), k[[0, 2, 3, 4]])
            assert torch.equal(cache._pick(cache.values[layer], rows), -k[[0, 2, 3, 4]])

    check()
    with pytest.raises(RuntimeError, match="moved already"):
        batch.commit(targets)
    check()
    batch.attend(0, q, k, -k, scale=0.1)
    with pytest.raises(RuntimeError, match=r"layers \[1\]"):
        batch.commit(targets)
    # The whole step again gives what it gave.
    batch.attend(1, q, k, -k, scale=0.1)
    again = batch.commit(targets)
    for g in "ab":
        assert all(torch.equal(x, y) for x, y in zip(again[g], kept[g]))
    check()
