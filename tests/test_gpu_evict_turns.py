"""A second turn's prompt after an eviction: rotated at its positions, written
behind the rows that are left, against float64 over the cache's rows."""

import numpy as np
import pytest
import torch

from instinct_amd.batches import DecodeBatch, PrefillBatch
from instinct_amd.paged_kv import KVCache, KVGroup

pytestmark = pytest.mark.gpu

PAGE, HEADS, KV, DIM, WINDOW = 16, 4, 2, 64, 24
SCALE = DIM ** -0.5


def attend(q, k, v, first, window):
    """Query i [HEADS, DIM] over rows 0 .. first + i (the last ``window`` of them)."""
    out = torch.empty((len(q), HEADS, DIM), dtype=torch.float64)
    for i in range(len(q)):
        seen = slice(max(0, first + i + 1 - window) if window else 0, first + i + 1)
        for h in range(HEADS):
            j = h * KV // HEADS
            p = torch.softmax(SCALE * k[seen, j].double() @ q[i, h].double(), dim=0)
            out[i, h] = p @ v[seen, j].double()
    return out


@pytest.mark.parametrize("layout", ["pages", "rows"])
def test_prompt_after_an_eviction(gpu, layout):
    g = torch.Generator().manual_seed(8)
    cache = KVCache([KVGroup("full", (0,), KV, DIM), KVGroup("local", (1,), KV, DIM, WINDOW)],
                    page_size=PAGE, capacities={"full": 12, "local": 12}, device=gpu, layout=layout)
    tables = {name: pool.allocate_many(8, reserved=False) for name, pool in cache.pools.items()}
    names = ("full", "local")

    def random(n, heads):
        return torch.randn((n, heads, DIM), generator=g).half().to(gpu)

    def rows(layer, n):
        at = torch.as_tensor(cache.rows(tables[names[layer]], 0, n), device=gpu)
        return (t.cpu() for t in cache.gather(layer, at))

    def turn(start, count, held):
        batch = PrefillBatch(cache, torch.zeros(count), start=start, tables=tables, held=held)
        assert batch.offsets.tolist() == list(range(start, start + count))
        for layer, first in enumerate((held["full"], start)):
            q, k, v = random(count, HEADS), random(count, KV), random(count, KV)
            got = batch.attend(layer, q, k, v, scale=SCALE).cpu()
            keys, values = rows(layer, first + count)
            assert torch.equal(keys[first:], k.cpu())
            want = attend(q.cpu(), keys, values, first, WINDOW if layer else 0)
            # fp16: weights and output rounded (2^-11 each), |v - out| of a few.
            assert (got.view(count, HEADS, DIM).double() - want).abs().max() < 2e-3

    turn(0, 60, {"full": 0})
    weights = {0: torch.rand((1, KV, 128), generator=g).to(gpu)}
    cut, held = cache.evict("full", [tables["full"]], np.array([60]), weights, keep=20, recent=4)
    tables["full"] = np.append(cut[0], cache.pools["full"].allocate_many(3, reserved=False))
    turn(60, 29, {"full": 20})
    batch = DecodeBatch(cache, torch.zeros(1), positions=np.array([89]),
                        tables={n: [t] for n, t in tables.items()}, held={"full": np.array([49])},
                        weights=weights)
    q = random(1, HEADS)
    got = batch.attend(0, q, random(1, KV), random(1, KV), scale=SCALE).cpu()
    keys, values = rows(0, 50)
    want = attend(q.cpu(), keys, values, 49, 0)
    assert (got.view(1, HEADS, DIM).double() - want).abs().max() < 2e-3


def test_held_is_checked(gpu):
    cache = KVCache([KVGroup("full", (0,), KV, DIM), KVGroup("local", (1,), KV, DIM, WINDOW)],
                    page_size=PAGE, capacities={"full": 8, "local": 8}, device=gpu)
    tables = {name: pool.allocate_many(4, reserved=False) for name, pool in cache.pools.items()}
    call = lambda **kw: PrefillBatch(cache, torch.zeros(4), start=40, tables=tables,  # noqa: E731
                                     **kw)
    with pytest.raises(ValueError, match="several"):
        call(held=8)
    with pytest.raises(ValueError, match="no group"):
        call(held={"other": 8})
    with pytest.raises(ValueError, match="each sequence"):
        call(held={"full": -1})
    with pytest.raises(ValueError, match="images"):
        call(held={"full": 8}, images=[(40, 2)])
    assert call(held={"full": 40}, images=[(40, 2)])._starts == {"full": 40, "local": 40}
