"""A bounded cache as an engine runs it: decode steps that credit their
attention weights, an eviction, and decode steps over what is left, against a
model in float64 that keeps every head's rows in lists."""

import numpy as np
import pytest
import torch

from instinct_amd.batches import DecodeBatch
from instinct_amd.paged_kv import KVCache, KVGroup

pytestmark = pytest.mark.gpu

PAGE, HEADS, KV, DIM, LAYERS, CAPACITY = 16, 6, 2, 64, 2, 160
SCALE = DIM ** -0.5


class Model:
    """What the cache should hold: per layer, sequence and kv head a list of
    (key, value, credit)."""

    def __init__(self, layers, batch):
        self.rows = [[[[] for _ in range(KV)] for _ in range(batch)] for _ in range(layers)]

    def write(self, layer, b, k, v):
        for j in range(KV):
            self.rows[layer][b][j].append([k[j].double(), v[j].double(), 0.0])

    def attend(self, layer, b, q):
        out = torch.empty((HEADS, DIM), dtype=torch.float64)
        for j in range(KV):
            rows = self.rows[layer][b][j]
            k, v = torch.stack([r[0] for r in rows]), torch.stack([r[1] for r in rows])
            heads = slice(j * HEADS // KV, (j + 1) * HEADS // KV)
            p = torch.softmax(SCALE * q[heads].double() @ k.t(), dim=-1)
            out[heads] = p @ v
            for r, x in zip(rows, p.sum(0).tolist()):
                r[2] += x
        return out

    def evict(self, layer, b, keep, recent, sinks):
        for j in range(KV):
            rows = self.rows[layer][b][j]
            n = len(rows)
            if n > keep:
                order = sorted(range(n), key=lambda t: (sinks <= t < n - recent, -rows[t][2], t))
                self.rows[layer][b][j] = [rows[t] for t in sorted(order[:keep])]


def stored(cache, layer, rows):
    """Keys and values as the attention calls take them: 8-bit keys times their
    scale unrounded, values rounded to fp16."""
    keys, values = cache.gather(layer, rows)
    if cache.bits == 8:
        keys = (cache._pick(cache.keys[layer], rows).double()
                * cache._pick(cache.key_scales[layer], rows).double()[..., None])
    return keys.cpu(), values.cpu()


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("layout", ["pages", "rows"])
@pytest.mark.parametrize("shared", [False, True])
def test_steps_evict_steps(gpu, shared, layout, bits):
    g = torch.Generator().manual_seed(7)
    cache = KVCache([KVGroup("all", tuple(range(LAYERS)), KV, DIM)], page_size=PAGE,
                    capacities={"all": 40}, device=gpu, layout=layout, bits=bits)
    pool = cache.pools["all"]
    lengths = np.array([100, 20, 75])
    tables = [pool.allocate_many(-(-CAPACITY // PAGE) if b == 0 else 8, reserved=False)
              for b in range(3)]
    if shared:  # sequence 2 shares the first two pages of sequence 0
        pool.release(tables[2][:2])
        tables[2][:2] = tables[0][:2]
        pool.retain(tables[0][:2])
    model = Model(LAYERS, 3)
    credits = {i: torch.zeros((3, KV, CAPACITY), device=gpu) for i in range(LAYERS)}
    for layer in range(LAYERS):  # prompts: rows only
        new = torch.randn((2, int(lengths.sum()), KV, DIM), generator=g).half()
        at = 0
        for b, n in enumerate(lengths):
            k, v = new[0, at:at + n].clone(), new[1, at:at + n].clone()
            if shared and b == 2:
                k[:32], v[:32] = new[0, :32], new[1, :32]
            rows = torch.as_tensor(cache.rows(tables[b], 0, int(n)), device=gpu)
            cache.write(layer, rows, k.to(gpu), v.to(gpu))
            keys, values = stored(cache, layer, rows)
            for t in range(n):
                model.write(layer, b, keys[t], values[t])
            at += n

    positions, held = lengths.copy(), lengths.copy()

    def step():
        nonlocal positions, held
        batch = DecodeBatch(cache, torch.zeros(3), positions=positions, tables={"all": tables},
                            held=held, weights=credits)
        assert batch.offsets.tolist() == positions.tolist()
        assert batch.lengths.tolist() == (held + 1).tolist()
        for layer in range(LAYERS):
            q, k, v = (torch.randn((3, h, DIM), generator=g).half() for h in (HEADS, KV, KV))
            got = batch.attend(layer, q.to(gpu), k.to(gpu), v.to(gpu), scale=SCALE).cpu()
            for b in range(3):
                row = torch.as_tensor(cache.rows(tables[b], int(held[b]), int(held[b]) + 1),
                                      device=gpu)
                kk, vv = stored(cache, layer, row)
                model.write(layer, b, kk[0], vv[0])
                want = model.attend(layer, b, q[b])
                # fp16: weights and output rounded (2^-11 each), |v - out| of a few.
                assert (got[b].view(HEADS, DIM).double() - want).abs().max() < 2e-3
                for j in range(KV):
                    want_c = torch.tensor([r[2] for r in model.rows[layer][b][j]])
                    have = credits[layer][b, j, :len(want_c)].cpu()
                    assert torch.allclose(have, want_c, rtol=1e-4, atol=1e-5)
        positions, held = positions + 1, held + 1

    for _ in range(3):
        step()
    before = [t.copy() for t in tables]
    free = pool.free
    tables, held = cache.evict("all", tables, held, credits, keep=48, recent=8, sinks=2)
    assert held.tolist() == [48, 23, 48]
    for layer in range(LAYERS):
        for b in range(3):
            model.evict(layer, b, 48, 8, 2)
    front = 48 // PAGE
    assert np.array_equal(tables[1], before[1])
    if shared:
        assert not set(tables[0]) & set(before[0]) and not set(tables[2]) & set(before[2])
        assert pool.free == free + len(set(before[0]) | set(before[2])) - 2 * front
    else:
        assert np.array_equal(tables[0], before[0][:front])
        assert pool.free == free + len(before[0]) + len(before[2]) - 2 * front
    # Room for what follows.
    tables = [t if b == 1 else np.concatenate([t, pool.allocate_many(2, reserved=False)])
              for b, t in enumerate(tables)]
    for _ in range(2):
        step()


def test_captured(gpu):
    """Credit and select in a graph: every replay gives the eager results."""
    from instinct_amd.eviction import (attention_weights_workspace_bytes, evict_rows,
                                       paged_attention_weights)
    from instinct_amd.hip_kernels import new_workspace

    g = torch.Generator().manual_seed(1)
    keys, values = (torch.randn((24, 2, 16, 64), generator=g).half().to(gpu) for _ in range(2))
    tables = torch.randperm(24, generator=g).view(2, 12).int().to(gpu)
    to = tables[:, 8:].contiguous()
    lengths = torch.tensor([120, 70], dtype=torch.int32, device=gpu)
    q = torch.randn((2, 4, 64), generator=g).half().to(gpu)
    w = torch.rand((2, 2, 128), generator=g).to(gpu)
    out, packed = torch.zeros_like(w), torch.zeros_like(w)
    ws = new_workspace(attention_weights_workspace_bytes(2, 4, 128), gpu)

    def run():
        paged_attention_weights(q, keys, tables, lengths, w, page_size=16, longest=128, scale=0.1,
                                out=out, workspace=ws)
        return evict_rows(keys, values, out, tables, lengths, page_size=16, longest=128, keep=60,
                          recent=8, out_tables=to, out_weights=packed)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n, kept = run()
    for _ in range(3):
        q.copy_(torch.randn((2, 4, 64), generator=g).half())
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (n, kept, out, packed, keys, values)]
        eager = run()
        torch.cuda.synchronize()
        for a, b in zip(got, (*eager, out, packed, keys, values)):
            assert torch.equal(a, b)
