"""The calls of steps with many tokens a sequence together, as an engine makes them:
prompts packed into one step, trees verified and committed, single tokens, over caches
of both layouts and widths; against dense attention of the sequences' own tokens in
64 bits."""

import numpy as np
import pytest
import torch

from instinct_amd import drafts, paging
from instinct_amd.batches import DecodeBatch, DraftBatch, PackedPrefillBatch
from instinct_amd.hip_kernels import paged_decode_attention, rope_append
from instinct_amd.paged_kv import KVCache, KVGroup
from oracle import many_tokens as plain

pytestmark = pytest.mark.gpu

PAGE = 16


def projections(rng, n, heads, dtype):
    hq, hk, dim = heads
    return torch.as_tensor(rng.standard_normal((n, hq + 2 * hk, dim))).to(dtype).cuda()


def dense(q, k, v, *, scale, window):
    """The last query of q over all of k, v (float64), and the tolerance's size."""
    n, m = len(q), len(k)
    group = q.shape[1] // k.shape[1]
    out, size = np.zeros_like(q), np.zeros_like(q)
    at = np.arange(m)
    for h in range(q.shape[1]):
        keep = np.broadcast_to((at <= m - 1) & ((at > m - 1 - window) if window else True), (n, m))
        out[:, h], size[:, h] = plain._attend(q[:, h], k[:, h // group], v[:, h // group], keep,
                                              scale, 0.0)
    return out, size


@pytest.mark.parametrize("layout", ["pages", "rows"])
@pytest.mark.parametrize("dtype, bits", [(torch.float16, 16), (torch.bfloat16, 16),
                                         (torch.bfloat16, 8)])
def test_prefill_draft_commit_decode(gpu, layout, dtype, bits):
    rng = np.random.default_rng(bits)
    heads = (8, 2, 64)
    groups = [KVGroup("full", (0, 2), 2, 64), KVGroup("near", (1,), 2, 64, 40)]
    cache = KVCache(groups, page_size=PAGE, capacities={"full": 64, "near": 64}, dtype=dtype,
                    layout=layout, bits=bits)
    counts = np.array([37, 5, 90])
    need = (counts + 40) // PAGE + 1
    tables = {g: [cache.pools[g].allocate_many(int(n), reserved=False) for n in need]
              for g in ("full", "near")}
    # Every layer's keys and values of every sequence's tokens so far, and the tolerance
    # of what is read back from an 8-bit cache.
    kept = {layer: [np.zeros((2, 0, 2, 64)) for _ in counts] for layer in range(3)}

    def tolerance(want, size, values):
        rounded = plain.attention_tolerance(want, size, values, 200, dtype, bits == 8)
        return rounded

    # 1. The prompts, packed.
    step = PackedPrefillBatch(cache, torch.zeros(int(counts.sum()), dtype=torch.int64),
                              counts=counts, tables=tables)
    starts = np.concatenate([[0], np.cumsum(counts)])
    np.testing.assert_array_equal(step.starts.cpu().numpy(), starts)
    np.testing.assert_array_equal(step.offsets.cpu().numpy(),
                                  np.concatenate([np.arange(n) for n in counts]))
    assert step.ends.tolist() == [36, 41, 131]
    for layer in range(3):
        qkv = projections(rng, int(counts.sum()), heads, dtype)
        q, k, v = qkv.split([8, 2, 2], dim=1)
        out = step.attend(layer, q, k, v, scale=0.125).view(-1, 8, 64).double().cpu().numpy()
        window = cache.layer_group[layer].window
        host = [x.double().cpu().numpy() for x in (q, k, v)]
        want, size = plain.packed_prompts(*host, [int(s) for s in starts], scale=0.125,
                                          window=window)
        tol = plain.attention_tolerance(want, size, host[2], 200, dtype)
        assert np.all(np.abs(out - want) <= tol)

    def held_rows(layer, b, n):
        rows = cache.rows(tables[cache.layer_group[layer].name][b], 0, n)
        index = torch.as_tensor(rows, device="cuda")
        store = [cache._pick(s, index) for s in (cache.keys[layer], cache.values[layer])]
        if bits == 8:
            scales = [cache._pick(s, index) for s in cache.scales(layer)]
            return [(x.double() * s.double()[..., None]).cpu().numpy()
                    for x, s in zip(store, scales)]
        return [x.double().cpu().numpy() for x in store]

    for layer in range(3):
        for b, n in enumerate(counts):
            kept[layer][b] = np.stack(held_rows(layer, b, int(n)))
            if bits == 16:  # the rows are the prompt's own
                pass

    # 2. Trees, two steps; the model agrees with a side branch.
    lengths = counts.copy()
    for turn in range(2):
        trees = [[-1, 0, 1, 0, 3, 4], [-1], [-1, 0, 0, 2, 3, 2]]
        paths = [[0, 3, 4, 5], [0], [0, 2, 5]] if turn == 0 else [[0, 1], [0], [0, 2, 3, 4]]
        parents = np.concatenate(trees)
        nodes = np.array([len(t) for t in trees])
        first = np.concatenate([[0], np.cumsum(nodes)])
        tokens = torch.as_tensor(rng.permutation(100)[:len(parents)])
        targets = torch.full_like(tokens, 1000)
        for b, path in enumerate(paths):
            for i, j in zip(path, path[1:]):
                targets[first[b] + i] = tokens[first[b] + j]
        batch = DraftBatch(cache, tokens, counts=nodes, parents=parents, positions=lengths,
                           tables=tables)
        drafted = {}
        for layer in range(3):
            qkv = projections(rng, len(parents), heads, dtype)
            q, k, v = qkv.split([8, 2, 2], dim=1)
            out = batch.attend(layer, q, k, v, scale=0.125).view(-1, 8, 64).double().cpu().numpy()
            window = cache.layer_group[layer].window
            for b, tree in enumerate(trees):
                n = int(lengths[b])
                rows = np.stack(held_rows(layer, b, n + len(tree)))
                np.testing.assert_array_equal(rows[:, :n], kept[layer][b])
                drafted[layer, b] = rows[:, n:]
                for i in range(len(tree)):
                    line, j = [], i
                    while j >= 0:
                        line.insert(0, j)
                        j = tree[j]
                    assert int(batch.offsets[first[b] + i]) == n + len(line) - 1
                    seen = np.concatenate([kept[layer][b], rows[:, [n + j for j in line]]], axis=1)
                    at = first[b] + i
                    want, size = dense(q[at:at + 1].double().cpu().numpy(), *seen, scale=0.125,
                                       window=window)
                    assert np.all(np.abs(out[at:at + 1] - want) <= tolerance(want, size, seen[1]))
        done = batch.commit(targets.cuda())
        for name, got in done.items():
            assert got.accepted.tolist() == [len(p) for p in paths]
            assert got.lengths.tolist() == [n + len(p) for n, p in zip(lengths, paths)]
            assert got.following.tolist() == [1000] * 3
        for layer in range(3):
            for b, path in enumerate(paths):
                kept[layer][b] = np.concatenate([kept[layer][b], drafted[layer, b][:, path]], axis=1)
                np.testing.assert_array_equal(
                    np.stack(held_rows(layer, b, kept[layer][b].shape[1])), kept[layer][b])
        lengths = lengths + [len(p) for p in paths]

    # 3. A plain decode step goes on from there.
    batch = DecodeBatch(cache, torch.zeros(3), positions=lengths, tables=tables)
    for layer in range(3):
        qkv = projections(rng, 3, heads, dtype)
        q, k, v = qkv.split([8, 2, 2], dim=1)
        out = batch.attend(layer, q, k, v, scale=0.125).view(-1, 8, 64).double().cpu().numpy()
        for b in range(3):
            rows = np.stack(held_rows(layer, b, int(lengths[b]) + 1))
            np.testing.assert_array_equal(rows[:, :-1], kept[layer][b])
            want, size = dense(q[b:b + 1].double().cpu().numpy(), *rows, scale=0.125,
                               window=cache.layer_group[layer].window)
            assert np.abs(out[b:b + 1] - want).max() < 2e-2


def test_evicted_sequences(gpu):
    """Rows fewer than positions: nodes are rotated at their positions and lie behind
    the rows held."""
    cache = KVCache([KVGroup("g", (0,), 2, 64)], page_size=PAGE, capacities={"g": 16})
    tables = {"g": [cache.pools["g"].allocate_many(4, reserved=False) for _ in range(2)]}
    batch = DraftBatch(cache, torch.zeros(5), counts=[3, 2], parents=[-1, 0, 0, -1, 0],
                       positions=[1000, 20], held=[30, 20], tables=tables)
    assert batch.positions.tolist() == [1000, 1001, 1001, 20, 21]
    want = np.concatenate([cache.rows(t, s, s + n)
                           for t, s, n in zip(tables["g"], (30, 20), (3, 2))])
    np.testing.assert_array_equal(batch._steps["g"].rows.cpu().numpy(), want)


def test_captured_draft_steps(gpu):
    """A whole step in a graph: tables from the feed, append, tree attention, commit;
    replayed with other tokens, the state moving on in place, against eager steps."""
    heads, batch, most, layers = (8, 2, 64), 5, 8, 3
    rng = np.random.default_rng(3)
    trees = [np.concatenate([[-1], rng.integers(0, np.arange(1, most))]) for _ in range(batch)]
    parents = torch.as_tensor(np.concatenate(trees).astype(np.int32), device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")

    def fresh():
        gen = torch.Generator(device="cuda").manual_seed(9)
        cache = KVCache([KVGroup("g", tuple(range(layers)), 2, 64)], page_size=PAGE,
                        capacities={"g": 200})
        for store in cache._stores:
            for t in store.values():
                t.normal_(generator=gen)
        feed = paging.PageFeed(cache, "g", 150)
        state = dict(cache=cache, feed=feed, tables=torch.zeros((batch, 32), **i32),
                     lengths=torch.zeros(batch, **i32), pages=torch.zeros(batch, **i32),
                     counts=torch.full((batch,), most, **i32),
                     q=torch.zeros((layers, batch * most, 8, 64), dtype=torch.float16, device="cuda"),
                     k=torch.zeros((layers, batch * most, 2, 64), dtype=torch.float16, device="cuda"),
                     drafted=torch.zeros(batch * most, dtype=torch.int64, device="cuda"),
                     targets=torch.zeros(batch * most, dtype=torch.int64, device="cuda"),
                     ws=torch.empty(drafts.tree_workspace_bytes(64), dtype=torch.uint8,
                                    device="cuda"))
        return state

    def step(s):
        c = s["cache"]
        new = paging.extend_tables(s["tables"], s["lengths"], s["counts"], s["pages"],
                                   s["feed"].pages, s["feed"].drawn, page_size=PAGE,
                                   tokens=batch * most, parents=parents)
        s["pages"].copy_(new.pages)
        s["feed"].drawn.copy_(new.drawn)
        outs = []
        for i in range(layers):
            q = rope_append(s["q"][i], s["k"][i], s["k"][i], c.keys[i], c.values[i], new.positions,
                            new.rows, page_size=PAGE, dims=64, base=1e4)
            outs.append(drafts.tree_attention(q, c.keys[i], c.values[i], s["tables"], s["lengths"],
                                              new.starts, new.masks, page_size=PAGE, scale=0.125,
                                              workspace=s["ws"]))
        done = drafts.commit_drafts([(c.keys[i], c.values[i]) for i in range(layers)], s["tables"],
                                    s["lengths"], new.starts, parents, s["drafted"], s["targets"],
                                    page_size=PAGE)
        s["lengths"].copy_(done.lengths)
        return torch.stack(outs), done

    def feed_inputs(s, seed):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        s["q"].normal_(generator=gen)
        s["k"].normal_(generator=gen)
        for name in ("drafted", "targets"):
            s[name].copy_(torch.randint(0, 3, (batch * most,), generator=gen, device="cuda"))

    eager, captured = fresh(), fresh()
    warm = fresh()
    feed_inputs(warm, 0)
    step(warm)  # (rotary tables and the like, outside the capture)
    torch.cuda.synchronize()
    feed_inputs(captured, 0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, done = step(captured)
    for turn in range(6):
        feed_inputs(eager, turn)
        feed_inputs(captured, turn)
        want, want_done = step(eager)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for a, b in zip(done, want_done):
            assert torch.equal(a, b)
        for name in ("tables", "lengths", "pages"):
            assert torch.equal(captured[name], eager[name])
        assert torch.equal(captured["feed"].drawn, eager["feed"].drawn)
        for i in range(layers):
            assert torch.equal(captured["cache"].keys[i], eager["cache"].keys[i])
    assert int(eager["lengths"].min()) >= 6 and int(eager["lengths"].max()) > 10
    # And the single token's form of the same state: the decode call takes it as it is.
    c = eager["cache"]
    one = paged_decode_attention(eager["q"][0, :batch].contiguous(), c.keys[0], c.values[0],
                                 eager["tables"], eager["lengths"], page_size=PAGE,
                                 longest=int(eager["lengths"].max()), scale=0.125)
    assert torch.isfinite(one).all()
