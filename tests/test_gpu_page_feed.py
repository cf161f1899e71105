"""Steps that draw their pages from a PageFeed, one after the other."""

import numpy as np
import pytest
import torch

from instinct_amd.drafts import commit_drafts, tree_attention
from instinct_amd.hip_kernels import kv_write
from instinct_amd.paged_kv import KVCache, KVGroup
from instinct_amd.paging import PageFeed, StepRows, extend_tables

pytestmark = pytest.mark.gpu

P = 16
I32 = dict(dtype=torch.int32, device="cuda")


def make(pages=64):
    return KVCache([KVGroup("main", (0,), 2, 64)], page_size=P, capacities={"main": pages})


def in_tables(tables, pages):
    return [int(t) for row, n in zip(tables.tolist(), pages.tolist()) for t in row[:n]]


def test_the_documented_loop(gpu):
    """Trees drawn, written, committed, step after step past several pages, with a refill
    on the way: no page in two places, every kept row as it was written, and every page
    accounted for."""
    rng = np.random.default_rng(1)
    cache, batch = make(), 3
    keys, values = cache.keys[0], cache.values[0]
    pool = cache.pools["main"]
    counts = torch.tensor([9, 2, 20], **I32)
    n = int(counts.sum())
    tree = lambda m: np.concatenate([[-1], rng.integers(0, np.arange(1, m))])  # noqa: E731
    shapes = [tree(m) for m in counts.tolist()]
    parents = torch.as_tensor(np.concatenate(shapes).astype(np.int32), device="cuda")
    first = np.concatenate([[0], np.cumsum(counts.tolist())])
    tables = torch.zeros((batch, 20), **I32)
    lengths, pages = torch.zeros(batch, **I32), torch.zeros(batch, **I32)
    feed = PageFeed(cache, "main", 8)
    assert pool.free == 56
    kept_rows = [[] for _ in range(batch)]
    held = [0] * batch
    for turn in range(14):
        if turn and turn % 4 == 0:
            feed.refill(8)
        nodes = torch.as_tensor(rng.permutation(1000)[:n], device="cuda")
        targets = torch.full_like(nodes, -1)
        for b, parent in enumerate(shapes):  # the model agrees with the line of the last node
            node = len(parent) - 1
            while parent[node] >= 0:
                targets[first[b] + parent[node]] = nodes[first[b] + node]
                node = parent[node]
        k = torch.randn(n, 2, 64, device="cuda").half()
        step = extend_tables(tables, lengths, counts, pages, feed, page_size=P, tokens=n,
                             parents=parents)
        assert step.drawn is feed.drawn
        kv_write(keys, values, step.rows, k, -k, page_size=P)
        out = tree_attention(torch.randn(n, 4, 64, device="cuda").half(), keys, values, tables,
                             lengths, step.starts, step.masks, page_size=P, scale=0.1)
        assert torch.isfinite(out).all()
        kept = commit_drafts([(keys, values)], tables, lengths, step.starts, parents, nodes,
                             targets, page_size=P)
        lengths, pages = kept.lengths, step.pages
        for b in range(batch):
            path = [int(x) for x in kept.path[b] if x >= 0]
            kept_rows[b].append(k[[int(first[b]) + i for i in path]])
            held[b] += len(path)
        assert lengths.tolist() == held
        used = in_tables(tables, pages)
        assert len(set(used)) == len(used)
    assert sum(held) > 100 and len(used) > 8  # (of more than one refill)
    for b in range(batch):
        rows = torch.as_tensor(cache.rows(tables[b].cpu().numpy(), 0, held[b]), device="cuda")
        for store, want in ((keys, torch.cat(kept_rows[b])), (values, -torch.cat(kept_rows[b]))):
            assert torch.equal(cache._pick(store, rows), want)
    feed.close()
    assert pool.used == len(used)
    pool.release(used)
    assert pool.used == 0


def test_a_feed_that_runs_out_says_so(gpu):
    cache = make()
    feed = PageFeed(cache, "main", 2)
    tables, zero = torch.zeros((3, 4), **I32), torch.zeros(3, **I32)
    step = extend_tables(tables, zero, torch.full((3,), 5, **I32), zero, feed, page_size=P, tokens=15)
    assert step.rows.tolist()[10:] == [-1] * 5 and tables[2, 0] == -1
    for call in (lambda: feed.refill(4), feed.close):
        with pytest.raises(RuntimeError, match="3 pages of a feed of 2"):
            call()


def test_out_has_the_feeds_count(gpu):
    feed = PageFeed(make(), "main", 2)
    new = lambda n: torch.zeros(n, **I32)  # noqa: E731
    out = StepRows(new(2), new(1), new(1), new(2), new(3), new(3), None)
    args = (torch.zeros((1, 4), **I32), new(1), torch.full((1,), 3, **I32), new(1), feed)
    with pytest.raises(ValueError, match="the feed's"):
        extend_tables(*args, page_size=P, tokens=3, out=out)
    got = extend_tables(*args, page_size=P, tokens=3, out=out._replace(drawn=feed.drawn))
    assert got.drawn is feed.drawn and feed.drawn.tolist() == [1, 0]


def test_a_captured_step_goes_on_after_a_refill(gpu):
    """A graph that was captured when the feed held few pages draws what refills bring,
    each page once, and nothing from a closed feed."""
    cache, batch = make(256), 5
    pool = cache.pools["main"]
    feed = PageFeed(cache, "main", 12)
    feed.refill(12)
    feed.drawn[0] = 9
    taken = feed.pages[:9].tolist()
    feed.refill(4)  # (less than its room at the capture)
    tables, counts = torch.zeros((batch, 40), **I32), torch.tensor([7, 16, 0, 1, 20], **I32)
    new = lambda n: torch.zeros(n, **I32)  # noqa: E731
    tokens = int(counts.sum())
    out = StepRows(new(batch + 1), new(batch), new(batch), feed.drawn, new(tokens), new(tokens), None)
    step = lambda: extend_tables(tables, out.lengths, counts, out.pages, feed,  # noqa: E731
                                 page_size=P, tokens=tokens, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for turn in range(10):
        feed.refill(12 if turn % 3 else 5)
        graph.replay()
        torch.zeros(1000, device="cuda").sum()  # eager work between the replays
        used = in_tables(tables, out.pages)
        assert min(used) >= 0 and len(set(used + taken)) == len(used) + len(taken)
        assert int(out.rows.min()) >= 0
        assert pool.used == len(taken) + len(used) + len(feed._ids) - int(feed.drawn[0])
    assert len(used) > 25
    feed.close()
    assert pool.used == len(taken) + len(used)
    for _ in range(3):
        graph.replay()
    after = in_tables(tables, out.pages)
    assert set(after) == set(used) | {-1}


def test_steps_on_another_stream(gpu):
    """refill and close wait for steps of any stream, and what they put is there for a step
    that follows on one."""
    cache = make()
    pool = cache.pools["main"]
    feed = PageFeed(cache, "main", 8)
    tables, zero, counts = torch.zeros((2, 8), **I32), torch.zeros(2, **I32), torch.full((2,), 20, **I32)
    slow = torch.ones((4096, 4096), device="cuda") / 4096
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()

    def step():
        with torch.cuda.stream(stream):
            x = slow
            for _ in range(60):  # some tens of milliseconds
                x = slow @ x
            return extend_tables(tables, zero, counts, zero, feed, page_size=P, tokens=40)

    step()
    feed.refill(8)
    assert feed.pages.tolist() == list(range(4, 12))
    step()
    feed.close()
    assert pool.used == 8
    torch.cuda.synchronize()
    assert in_tables(tables, torch.full((2,), 2, **I32)) == [4, 5, 6, 7]


def test_a_captured_step_after_the_feed_outgrew_its_tensors(gpu):
    """It finds no page, whatever was allocated since."""
    feed = PageFeed(make(256), "main", 4)
    tables, counts = torch.zeros((2, 8), **I32), torch.full((2,), 5, **I32)
    new = lambda n: torch.zeros(n, **I32)  # noqa: E731
    out = StepRows(new(3), new(2), new(2), feed.drawn, new(10), new(10), None)
    zero = new(2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        extend_tables(tables, zero, counts, zero, feed, page_size=P, tokens=10, out=out)
    graph.replay()
    assert out.rows.tolist() == list(range(5)) + list(range(16, 21))
    feed.refill(100)
    others = [torch.full((4,), 7, **I32) for _ in range(64)]
    graph.replay()
    assert out.rows.tolist() == [-1] * 10 and tables[:, 0].tolist() == [-1, -1]
    assert feed.drawn.tolist() == [0, 0] and len(others) == 64
