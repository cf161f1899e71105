"""Steps of many tokens a sequence refuse what their attention does not serve before a
layer's keys and values are written (on the CPU: the write itself would refuse the arena
with another message)."""

import numpy as np
import pytest
import torch

from instinct_amd.batches import DraftBatch, PackedPrefillBatch
from instinct_amd.paged_kv import KVCache, KVGroup


def cache(head_dim):
    return KVCache([KVGroup("a", (0,), 2, 64), KVGroup("b", (1,), 2, head_dim)], page_size=16,
                   capacities={"a": 8, "b": 8}, device="cpu")


def packed(c):
    return PackedPrefillBatch(c, torch.zeros(3, dtype=torch.int64), counts=[3],
                              tables={g: [np.array([0])] for g in "ab"})


def drafts(c):
    return DraftBatch(c, torch.zeros(3, dtype=torch.int64), counts=[3], parents=[-1, 0, 0],
                      positions=[2], tables={g: [np.array([0])] for g in "ab"})


@pytest.mark.parametrize("make", [packed, drafts])
@pytest.mark.parametrize("head_dim", [7, 100, 264, 512])
def test_head_dims(make, head_dim):
    with pytest.raises(ValueError, match=f"'b'.*not {head_dim}"):
        make(cache(head_dim))


@pytest.mark.parametrize("kind", [PackedPrefillBatch, DraftBatch])
@pytest.mark.parametrize("shape", [(2, 4, 64), (3, 3, 64), (3, 4, 32), (3, 0, 64), (3, 256)])
def test_queries(kind, shape):
    step = object.__new__(kind)  # (the constructor needs a GPU)
    step.cache, step.count = cache(64), 3
    k = torch.zeros(3, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="q must be"):
        step.attend(0, torch.zeros(shape, dtype=torch.float16), k, k, scale=0.1)
