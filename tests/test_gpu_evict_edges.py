"""Calls of the eviction at the edges of what it takes."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def layer(gpu, pages, page=16, heads=2, dim=64, seed=0):
    g = torch.Generator().manual_seed(seed)
    keys, values = (torch.randn((pages, heads, page, dim), generator=g).half().to(gpu)
                    for _ in range(2))
    return keys, values, g


@pytest.mark.parametrize("in_place", [True, False])
def test_weights_and_tables_hold_the_longest(gpu, in_place):
    """Rows past either were lost without an error; nothing is touched."""
    from instinct_amd.eviction import evict_rows

    keys, values, _ = layer(gpu, 8)
    before = keys.clone(), values.clone()
    tables = torch.arange(4, dtype=torch.int32, device=gpu)[None]
    lengths = torch.tensor([60], dtype=torch.int32, device=gpu)
    kw = dict(page_size=16, longest=60, keep=32, recent=8,
              out_tables=None if in_place else tables + 4)
    for capacity in (59, 31):
        w = torch.ones((1, 2, capacity), device=gpu)
        with pytest.raises(ValueError, match=f"weights of {capacity} positions"):
            evict_rows(keys, values, w, tables, lengths, **kw)
    w = torch.ones((1, 2, 60), device=gpu)
    with pytest.raises(ValueError, match="tables of 3 pages"):
        evict_rows(keys, values, w, tables[:, :3], lengths, **kw)
    assert torch.equal(keys, before[0]) and torch.equal(values, before[1])
    n, kept = evict_rows(keys, values, w, tables, lengths, **kw)
    assert n.tolist() == [32] and kept[0, 0, -8:].tolist() == list(range(52, 60))


def test_tables_in_a_wider_one_are_in_place(gpu):
    """Columns of a wider table as both tables, or their first ones: rows move to the front of their own
    pages, as without out_tables."""
    from instinct_amd.eviction import evict_rows

    wide = torch.randperm(24, generator=torch.Generator().manual_seed(3)).int().view(2, 12).to(gpu)
    tables = wide[:, 2:10]
    lengths = torch.tensor([128, 90], dtype=torch.int32, device=gpu)
    kw = dict(page_size=16, longest=128, keep=70, recent=8, sinks=2)
    results = []
    for out_tables in (None, tables, wide[:, 2:10], wide[:, 2:7]):
        keys, values, g = layer(gpu, 24)
        w = torch.rand((2, 2, 128), generator=g).to(gpu)
        n, kept = evict_rows(keys, values, w, tables, lengths, out_tables=out_tables, **kw)
        results.append((n, kept, w, keys, values))
    assert results[0][0].tolist() == [70, 70]
    for got in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got, results[0]))


@pytest.mark.parametrize("in_place", [True, False])
def test_one_arena_as_keys_and_values(gpu, in_place):
    """Rows move once, as with the keys alone."""
    from instinct_amd.eviction import evict_rows

    tables = torch.randperm(80, generator=torch.Generator().manual_seed(4)).int().to(gpu)[None]
    lengths = torch.tensor([1000], dtype=torch.int32, device=gpu)
    stores = []
    for both in (False, True):
        keys, _, g = layer(gpu, 80, seed=5)
        w = torch.rand((1, 2, 1000), generator=g).to(gpu)
        evict_rows(keys, keys if both else None, w, tables[:, :63], lengths, page_size=16,
                   longest=1000, keep=260, out_tables=None if in_place else tables[:, 63:])
        stores.append(keys)
    assert torch.equal(*stores)


def test_hidden_keys_beside_a_nan(gpu):
    """A visible key of NaN makes the visible credits NaN; keys that the window or
    their page hides keep what they had."""
    from instinct_amd.eviction import paged_attention_weights

    keys, _, g = layer(gpu, 8)
    tables = torch.arange(8, dtype=torch.int32, device=gpu)[None].contiguous()
    tables[0, 5] = -1
    keys[6, 0, 3] = float("nan")  # position 99 of kv head 0
    q = torch.randn((1, 4, 64), generator=g).half().to(gpu)
    w = torch.rand((1, 2, 128), generator=g).to(gpu)
    lengths = torch.tensor([120], dtype=torch.int32, device=gpu)
    out = paged_attention_weights(q, keys, tables, lengths, w, page_size=16, longest=120, scale=0.1,
                                  window=60, out=torch.zeros_like(w))
    hidden = [t for t in range(119) if t < 60 or 80 <= t < 96]
    seen = [t for t in range(120) if t not in hidden]
    assert torch.equal(out[0, :, hidden], w[0, :, hidden])
    assert bool(out[0, 0, seen].isnan().all())
    # The other kv head's weights: two heads that each sum to 1.
    assert abs(float((out[0, 1, seen] - w[0, 1, seen]).sum() + w[0, 1, 119]) - 2) < 1e-4


@pytest.mark.parametrize("holes, in_place", [((5, 7), True), ((0, 2, 7), False)])
def test_no_kept_row_is_lost_to_released_pages(gpu, holes, in_place):
    """In place with the released pages past the kept rows, else on other pages with
    any released: every kept row is found at its place."""
    from instinct_amd.eviction import evict_rows

    keys, values, g = layer(gpu, 32)
    before = keys.cpu(), values.cpu()
    tables = torch.arange(16, dtype=torch.int32)[None]
    tables[0, list(holes)] = -1
    out = tables if in_place else torch.arange(16, 32, dtype=torch.int32)[None]
    w = torch.rand((1, 2, 200), generator=g).to(gpu)
    n, kept = evict_rows(keys, values, w, tables.to(gpu),
                         torch.tensor([200], dtype=torch.int32, device=gpu), page_size=16,
                         longest=200, keep=70, recent=6, sinks=3,
                         out_tables=None if in_place else out.to(gpu))
    assert n.tolist() == [70]
    for old, new in zip(before, (keys.cpu(), values.cpu())):
        for j in range(2):
            for i, t in enumerate(kept[0, j].tolist()):
                assert t // 16 not in holes
                assert torch.equal(new[out[0, i // 16], j, i % 16],
                                   old[tables[0, t // 16], j, t % 16])
