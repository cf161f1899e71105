"""A cache of a full and a windowed group of which one is cut: decode steps of
both against float64 over lists of rows."""

import numpy as np
import pytest
import torch

from instinct_amd.batches import DecodeBatch
from instinct_amd.paged_kv import KVCache, KVGroup

pytestmark = pytest.mark.gpu

PAGE, HEADS, KV, DIM, WINDOW, KEEP = 16, 4, 2, 64, 24, 20
SCALE = DIM ** -0.5


def attend(q, rows):
    """Float64 attention of one sequence's heads, and the weights each kv head gave."""
    out, credit = torch.empty((HEADS, DIM), dtype=torch.float64), []
    for j in range(KV):
        k, v = (torch.stack([r[i] for r in rows[j]]) for i in (0, 1))
        heads = slice(j * HEADS // KV, (j + 1) * HEADS // KV)
        p = torch.softmax(SCALE * q[heads].double() @ k.t(), dim=-1)
        out[heads] = p @ v
        credit.append(p.sum(0))
    return out, credit


def test_one_group_cut(gpu):
    g = torch.Generator().manual_seed(11)
    cache = KVCache([KVGroup("full", (0,), KV, DIM), KVGroup("local", (1,), KV, DIM, WINDOW)],
                    page_size=PAGE, capacities={"full": 16, "local": 16}, device=gpu)
    lengths = np.array([50, 33])
    tables = {name: [pool.allocate_many(5, reserved=False) for _ in lengths]
              for name, pool in cache.pools.items()}
    rows = [[[[] for _ in range(KV)] for _ in lengths] for _ in range(2)]  # layer, sequence, kv head
    weights = {0: torch.zeros((2, KV, 80), device=gpu)}
    credits = [[[0.0] * int(n) for _ in range(KV)] for n in lengths]
    for layer, name in enumerate(("full", "local")):
        for b, n in enumerate(lengths):
            k, v = (torch.randn((int(n), KV, DIM), generator=g).half() for _ in range(2))
            at = torch.as_tensor(cache.rows(tables[name][b], 0, int(n)), device=gpu)
            cache.write(layer, at, k.to(gpu), v.to(gpu))
            for j in range(KV):
                rows[layer][b][j] = list(zip(k[:, j].double(), v[:, j].double()))
    positions, held = lengths.copy(), lengths.copy()

    def step():
        nonlocal positions, held
        batch = DecodeBatch(cache, torch.zeros(2), positions=positions, tables=tables,
                            held={"full": held}, weights=weights)
        for layer in range(2):
            q, k, v = (torch.randn((2, h, DIM), generator=g).half() for h in (HEADS, KV, KV))
            got = batch.attend(layer, q.to(gpu), k.to(gpu), v.to(gpu), scale=SCALE).cpu()
            for b in range(2):
                for j in range(KV):
                    rows[layer][b][j].append((k[b, j].double(), v[b, j].double()))
                seen = rows[layer][b] if layer == 0 else [r[-WINDOW:] for r in rows[layer][b]]
                want, credit = attend(q[b], seen)
                # fp16: weights and output rounded (2^-11 each), |v - out| of a few.
                assert (got[b].view(HEADS, DIM).double() - want).abs().max() < 2e-3
                if layer == 0:
                    for j in range(KV):
                        old = credits[b][j] + [0.0]
                        credits[b][j] = [x + y for x, y in zip(old, credit[j].tolist())]
        positions, held = positions + 1, held + 1

    for _ in range(2):
        step()
    tables["full"], held = cache.evict("full", tables["full"], held, weights, keep=KEEP, recent=4)
    assert held.tolist() == [KEEP, KEEP]
    for b in range(2):
        for j in range(KV):
            n = len(rows[0][b][j])
            pick = sorted(sorted(range(n), key=lambda t: (t < n - 4, -credits[b][j][t], t))[:KEEP])
            rows[0][b][j] = [rows[0][b][j][t] for t in pick]
            credits[b][j] = [credits[b][j][t] for t in pick]
    for _ in range(3):
        step()


@pytest.mark.parametrize("shared", [False, True])
def test_rows_to_come_start_from_nothing(gpu, shared):
    """The credits behind a cut sequence's rows are zeros, not those of dropped
    keys; other sequences' are left."""
    cache = KVCache([KVGroup("full", (0, 1), KV, DIM)], page_size=PAGE, capacities={"full": 16},
                    device=gpu)
    pool = cache.pools["full"]
    tables = [pool.allocate_many(4, reserved=False) for _ in range(2)]
    if shared:
        pool.retain(tables[0][:1])
    g = torch.Generator().manual_seed(6)
    weights = {i: torch.rand((2, KV, 70), generator=g).to(gpu) for i in range(2)}
    before = {i: w.clone() for i, w in weights.items()}
    _, held = cache.evict("full", tables, np.array([60, 30]), weights, keep=32, recent=4)
    assert held.tolist() == [32, 30]
    for i, w in weights.items():
        assert bool((w[0, :, :32] > 0).all()) and bool((w[0, :, 32:] == 0).all())
        assert torch.equal(w[1], before[i][1])
