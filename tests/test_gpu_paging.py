"""paging.extend_tables against the plain restatement: every value equal."""

import numpy as np
import pytest
import torch

from instinct_amd import paging
from oracle import many_tokens as plain

pytestmark = pytest.mark.gpu


def make(rng, batch, held, counts, page, *, tree, width=None, spare=8, room=None, extra=0.3):
    lengths = rng.integers(0, held + 1, batch)
    counts = rng.integers(0, counts + 1, batch) if np.isscalar(counts) else np.asarray(counts)
    pages = -(-lengths // page) + (rng.random(batch) < extra)
    need = np.maximum(pages, -(-(lengths + counts) // page))
    width = width or int(need.max()) + 2
    pages = np.minimum(pages, width)
    ids = rng.permutation(int(need.sum()) + spare + batch * width)
    tables = ids[:batch * width].reshape(batch, width)
    feed = ids[batch * width:]
    total = int(counts.sum())
    tokens = total + 5 if room is None else room
    parents = None
    if tree:
        parents = np.full(tokens, -1)
        at = 0
        for n in counts:
            for i in range(1, int(n)):
                if at + i < tokens:
                    parents[at + i] = rng.integers(-1, i) if rng.random() < 0.9 else rng.integers(-9, 99)
            at += int(n)
    return dict(tables=tables, lengths=lengths, counts=counts, pages=pages, feed=feed,
                drawn=np.array([3, 0]), parents=parents), dict(page_size=page, tokens=tokens)


def dev(a):
    return None if a is None else torch.as_tensor(np.asarray(a).astype(np.int32), device="cuda")


def check(arrays, kw, out=None):
    parents = arrays["parents"]
    put = {k: dev(v) for k, v in arrays.items()}
    if out == "in place":
        new = lambda n, t=torch.int32: torch.full((n,), -7, dtype=t, device="cuda")  # noqa: E731
        n, batch = kw["tokens"], len(arrays["lengths"])
        out = paging.StepRows(new(batch + 1), put["lengths"], put["pages"], put["drawn"], new(n),
                              new(n), None if parents is None else new(n, torch.int64))
    got = paging.extend_tables(put["tables"], put["lengths"], put["counts"], put["pages"],
                               put["feed"], put["drawn"], parents=put["parents"], out=out, **kw)
    want = plain.extend_tables(*(arrays[k] for k in ("tables", "lengths", "counts", "pages", "feed",
                                                     "drawn")), parents=parents, **kw)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(put["tables"].cpu().numpy(), want["tables"])
    for name in ("starts", "lengths", "pages", "drawn", "rows", "positions"):
        np.testing.assert_array_equal(getattr(got, name).cpu().numpy(), want[name], err_msg=name)
    if parents is None:
        assert got.masks is None
    else:
        np.testing.assert_array_equal(got.masks.cpu().numpy().view(np.uint64), want["masks"])
    assert put["drawn"].cpu().tolist()[1] == 0


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("batch, held, counts, page", [
    (1, 0, 1, 16), (1, 777, 16, 16), (3, 50, 64, 7), (17, 300, 9, 1), (64, 8192, 48, 16),
    (255, 100, 3, 32), (256, 40, 64, 64), (257, 1, 2, 16), (1000, 2000, 12, 16)])
def test_equals_plain(gpu, batch, held, counts, page, tree):
    rng = np.random.default_rng(batch * 1000 + counts)
    check(*make(rng, batch, held, counts, page, tree=tree))


def test_large_batch(gpu):
    check(*make(np.random.default_rng(1), 4096, 60, 5, 16, tree=True))


def test_long_prompts(gpu):
    rng = np.random.default_rng(2)
    check(*make(rng, 40, 0, rng.integers(0, 6000, 40), 16, tree=False))


def test_every_tree_is_a_chain_of_64(gpu):
    arrays, kw = make(np.random.default_rng(3), 9, 100, [64] * 9, 16, tree=True)
    arrays["parents"][:] = np.tile(np.arange(-1, 63), 10)[:kw["tokens"]]
    check(arrays, kw)


def test_nodes_past_the_64th(gpu):
    check(*make(np.random.default_rng(4), 3, 100, [70, 0, 200], 16, tree=True))


@pytest.mark.parametrize("tree", [False, True])
def test_in_place(gpu, tree):
    check(*make(np.random.default_rng(5), 300, 500, 20, 16, tree=tree), out="in place")
    check(*make(np.random.default_rng(6), 4, 500, 20, 16, tree=tree), out="in place")


def test_feed_runs_out(gpu):
    arrays, kw = make(np.random.default_rng(7), 30, 100, 40, 16, tree=False)
    arrays["feed"] = arrays["feed"][:17]
    check(arrays, kw)
    arrays["feed"] = arrays["feed"][:0]
    check(arrays, kw)
    arrays["drawn"] = np.array([2**31 - 2, 0])
    with np.errstate(over="ignore"):
        put = {k: dev(v) for k, v in arrays.items() if k != "parents"}
        got = paging.extend_tables(**put, **kw)
    assert got.drawn.tolist() == [2**31 - 1, 0]


def test_table_and_token_room_run_out(gpu):
    check(*make(np.random.default_rng(8), 30, 100, 400, 16, tree=False, width=9))
    check(*make(np.random.default_rng(9), 30, 100, 40, 16, tree=True, room=301))
    check(*make(np.random.default_rng(10), 5, 10, 4, 16, tree=False, room=0))


def test_negative_values(gpu):
    arrays, kw = make(np.random.default_rng(11), 20, 100, 12, 16, tree=True)
    arrays["counts"][3] = arrays["lengths"][5] = arrays["pages"][7] = -4
    check(arrays, kw)


def test_rows_past_32_bits_are_none(gpu):
    tables = dev([[5, 300_000_000, 0]])
    got = paging.extend_tables(tables, dev([14]), dev([4]), dev([2]), dev([1]), dev([0, 0]),
                               page_size=16, tokens=4)
    assert got.rows.tolist() == [94, 95, -1, -1]


def test_no_sequences(gpu):
    got = paging.extend_tables(dev(np.zeros((0, 4))), dev([]), dev([]), dev([]), dev([1]),
                               dev([2, 0]), page_size=16, tokens=3)
    assert got.starts.tolist() == [0] and got.rows.tolist() == [-1] * 3
    assert got.drawn.tolist() == [2, 0]


@pytest.mark.parametrize("batch", [3, 300])
def test_replayed_steps(gpu, batch):
    """A step captured once and replayed: lengths, pages and the feed move on."""
    rng = np.random.default_rng(batch)
    arrays, kw = make(rng, batch, 60, [2] * batch, 4, tree=False, width=40, spare=40 * batch)
    arrays["lengths"] = np.minimum(arrays["lengths"], arrays["pages"] * 4)
    put = {k: dev(v) for k, v in arrays.items() if k != "parents"}
    new = lambda n: torch.empty(n, dtype=torch.int32, device="cuda")  # noqa: E731
    out = paging.StepRows(new(batch + 1), put["lengths"], put["pages"], put["drawn"],
                          new(kw["tokens"]), new(kw["tokens"]), None)
    step = lambda: paging.extend_tables(put["tables"], put["lengths"], put["counts"],  # noqa: E731
                                        put["pages"], put["feed"], put["drawn"], out=out, **kw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    state = dict(arrays)
    for turn in range(6):
        graph.replay()
        torch.cuda.synchronize()
        want = plain.extend_tables(*(state[k] for k in ("tables", "lengths", "counts", "pages",
                                                        "feed", "drawn")), **kw)
        np.testing.assert_array_equal(put["tables"].cpu().numpy(), want["tables"])
        for name in ("starts", "lengths", "pages", "drawn", "rows", "positions"):
            np.testing.assert_array_equal(getattr(out, name).cpu().numpy(), want[name], name)
        state.update({k: want[k] for k in ("tables", "lengths", "pages", "drawn")})
        torch.zeros(1000, device="cuda").sum()  # eager work between the replays
