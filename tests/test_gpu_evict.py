"""Accumulated attention weights and eviction on the GPU against the oracle."""

import numpy as np
import pytest
import torch

from oracle import eviction as oracle

pytestmark = pytest.mark.gpu


def arena(layout, pages, page, heads, dim, dtype, g):
    shape = (pages * page, heads, dim) if layout == "rows" else (pages, heads, page, dim)
    return torch.randn(shape, generator=g).to(dtype)


def tables_for(lengths, page, pages, g):
    order = torch.randperm(pages, generator=g).tolist()
    width = max(1, max(-(-max(n, 0) // page) for n in lengths))
    t = torch.zeros((len(lengths), width), dtype=torch.int32)
    for b, n in enumerate(lengths):
        for i in range(-(-max(n, 0) // page)):
            t[b, i] = order.pop()
    return t


def check_weights(gpu, heads, lengths, *, page=16, layout="pages", dtype=torch.float16, window=0,
                  softcap=0.0, fresh=1, q8=False, change=None, capacity=None, scale=None):
    from instinct_amd.eviction import paged_attention_weights

    q_heads, kv_heads, dim = heads
    g = torch.Generator().manual_seed(dim + len(lengths))
    pages = sum(-(-max(n, 0) // page) for n in lengths) + 2
    keys = arena(layout, pages, page, kv_heads, dim, dtype, g)
    scales = None
    if q8:
        keys = (keys.float() * 40).round().clamp(-127, 127).to(torch.int8)
        scales = (torch.rand(keys.shape[:-1], generator=g) * 0.01 + 0.02).half()
    t = tables_for(lengths, page, pages, g)
    if change:
        change(keys, t)
    capacity = capacity or max(1, max(lengths)) + 5
    old = torch.rand((len(lengths), kv_heads, capacity), generator=g) * 3
    q = torch.randn((len(lengths), q_heads, dim), generator=g).to(dtype)
    scale = scale or dim ** -0.5
    kw = dict(page_size=page, scale=scale, window=window, softcap=softcap, fresh=fresh)
    want, bound = oracle.weights(q, keys, t, lengths, old, layout=layout, key_scales=scales, **kw)
    dev = [x.to(gpu) for x in (q, keys, t, torch.tensor(lengths, dtype=torch.int32), old)]
    dev_scales = None if scales is None else (scales.to(gpu), scales.to(gpu))
    out = old.to(gpu)
    for longest in (max(1, max(lengths)), 1):
        got = paged_attention_weights(*dev, longest=longest, scales=dev_scales, out=out, **kw)
        assert got is out
        over = (got.cpu().double() - want).abs() - bound
        assert bool((over <= 0).all()), f"past the bound by {over.max():.3e}"
    assert torch.equal(dev[4].cpu(), old)
    for b, n in enumerate(lengths):  # what lies past a sequence is left alone
        n = min(max(n, 0), t.shape[1] * page, capacity)
        assert torch.equal(out.cpu()[b, :, n:], old[b, :, n:])
    again = old.to(gpu)
    paged_attention_weights(*dev[:4], again, longest=max(1, max(lengths)), scales=dev_scales, **kw)
    assert torch.equal(again, out)  # in place, and the same bits


HEADS = [(14, 2, 64), (4, 4, 80), (12, 4, 96), (28, 4, 128), (8, 4, 256), (16, 2, 512), (40, 1, 72),
         (3, 1, 33), (2, 2, 7), (6, 2, 300), (66, 2, 16)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", HEADS)
def test_weights_shapes(gpu, heads, dtype):
    check_weights(gpu, heads, [1, 0, 17, 255, 256, 257, 600], dtype=dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128), (8, 4, 256), (3, 1, 33), (4, 2, 200)])
@pytest.mark.parametrize("layout", ["rows", "pages"])
def test_weights_int8(gpu, heads, layout, dtype):
    check_weights(gpu, heads, [1, 300, 40], layout=layout, q8=True, dtype=dtype)


@pytest.mark.parametrize("page, layout", [(1, "rows"), (7, "pages"), (48, "rows"), (64, "pages")])
def test_weights_pages(gpu, page, layout):
    check_weights(gpu, (28, 4, 128), [129, 2, 1100], page=page, layout=layout)


@pytest.mark.parametrize("window, softcap, fresh", [(1, 0.0, 1), (100, 0.0, 1), (256, 5.0, 3),
                                                    (0, 30.0, 0), (0, 0.0, 10 ** 9), (5000, 2.0, 7)])
def test_weights_options(gpu, window, softcap, fresh):
    check_weights(gpu, (8, 4, 64), [2500, 1, 100, 257], window=window, softcap=softcap, fresh=fresh)


def test_weights_long(gpu):
    """More chunks (256 keys) than a wave has lanes."""
    check_weights(gpu, (4, 1, 64), [17500])


def test_weights_masked_pages(gpu):
    """Hidden keys get nothing, whatever their rows hold; a sequence that sees
    none keeps what it had."""
    def change(keys, t):
        keys[0] = float("nan")
        t[t == 0] = -1
        t[0, 2] = -3
        t[0, 4] = 1 << 24
        t[1, :] = -1

    check_weights(gpu, (14, 2, 64), [300, 70, 20], change=change)


def test_weights_past_the_capacity(gpu):
    """A length past the capacity (or the table) is cut to it."""
    check_weights(gpu, (4, 2, 64), [300, 700], capacity=200)


def test_weights_large_scores(gpu):
    check_weights(gpu, (4, 2, 64), [900], scale=4.0)


def check_evict(gpu, lengths, *, keep, recent=0, sinks=0, page=16, layout="pages", heads=2, dim=64,
                dtype=torch.float16, in_place=True, q8=False, w=None, change=None, values=True):
    from instinct_amd.eviction import evict_rows

    g = torch.Generator().manual_seed(keep + page)
    need = sum(-(-max(n, 0) // page) for n in lengths)
    pages = 2 * need + 3
    stores = [arena(layout, pages, page, heads, dim, dtype, g) for _ in range(2 if values else 1)]
    if q8:
        stores = [(s.float() * 40).round().clamp(-127, 127).to(torch.int8) for s in stores]
        stores += [torch.rand(stores[0].shape[:-1], generator=g).half() for _ in range(2)]
    every = tables_for(list(lengths) * 2, page, pages, g)
    t, fresh = every[:len(lengths)].contiguous(), every[len(lengths):].contiguous()
    if change:
        change(t)
    to = t if in_place else fresh
    capacity = max(1, max(lengths)) + 3
    if w is None:
        w = torch.rand((len(lengths), heads, capacity), generator=g)
        w[w < 0.3] = 0.0  # alike
    rows = pages * page
    kept, new = oracle.select(w, t, lengths, page_size=page, arena_rows=rows, keep=keep,
                              recent=recent, sinks=sinks)
    dev = [s.to(gpu) for s in stores]
    out_w = w.to(gpu)
    dev_t = t.to(gpu)
    n, k = evict_rows(dev[0], dev[1] if values else None, out_w, dev_t,
                      torch.tensor(lengths, dtype=torch.int32, device=gpu), page_size=page,
                      longest=max(1, max(lengths)), keep=keep, recent=recent, sinks=sinks,
                      scales=tuple(dev[2:]) if q8 else None,
                      out_tables=None if in_place else to.to(gpu))
    assert n.tolist() == new.tolist()
    assert np.array_equal(k.cpu().numpy(), kept)
    want_w = w.clone()
    for b in range(len(lengths)):
        for j in range(heads):
            want_w[b, j, :new[b]] = w[b, j][torch.as_tensor(kept[b, j, :new[b]]).long()]
    assert torch.equal(out_w.cpu().view(torch.int32), want_w.view(torch.int32))
    for got, s in zip(dev, stores):
        want = oracle.move(s, kept, t, to, page_size=page, layout=layout)
        if not in_place:
            assert torch.equal(got.cpu(), want)
            continue
        # In place the places past the new length keep old rows: compare those
        # that count.
        for b in range(len(lengths)):
            for i in range(int(new[b])):
                page_id = int(t[b, i // page])
                if 0 <= page_id < pages:
                    at = (page_id * page + i % page if layout == "rows"
                          else (page_id, slice(None), i % page))
                    assert torch.equal(got[at].cpu(), want[at]), (b, i)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("layout", ["rows", "pages"])
@pytest.mark.parametrize("keep, recent, sinks", [(1, 0, 0), (1, 1, 0), (40, 10, 4), (64, 64, 0),
                                                 (200, 0, 8), (1000, 3, 2)])
def test_evict(gpu, keep, recent, sinks, layout, in_place):
    check_evict(gpu, [0, 1, 39, 40, 41, 333, 130], keep=keep, recent=recent, sinks=sinks,
                layout=layout, in_place=in_place)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("page, dim, heads", [(1, 64, 1), (7, 80, 3), (16, 33, 2), (64, 128, 4),
                                              (16, 1, 1), (32, 6, 2)])
def test_evict_shapes(gpu, page, dim, heads, in_place):
    check_evict(gpu, [100, 61], keep=50, recent=9, sinks=2, page=page, dim=dim, heads=heads,
                dtype=torch.bfloat16, in_place=in_place)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("layout", ["rows", "pages"])
@pytest.mark.parametrize("dim", [128, 31])
def test_evict_int8(gpu, layout, dim, in_place):
    check_evict(gpu, [90, 200], keep=77, recent=5, layout=layout, dim=dim, q8=True,
                in_place=in_place)


@pytest.mark.parametrize("in_place", [True, False])
def test_evict_long(gpu, in_place):
    """Positions beyond one stretch of rows (in place) and of threads."""
    check_evict(gpu, [3500, 2600], keep=2500, recent=100, sinks=4, heads=1, in_place=in_place)


def test_evict_one_arena(gpu):
    check_evict(gpu, [100], keep=64, recent=8, heads=1, dim=576, values=False)


@pytest.mark.parametrize("fill", [0.0, 1.0])
def test_evict_all_alike(gpu, fill):
    """Ties go to the lower positions, over several waves' stretches."""
    check_evict(gpu, [1100, 2100], keep=1024, recent=128, sinks=4, heads=1, dim=8,
                w=torch.full((2, 1, 2100), fill))


def test_evict_unusual_weights(gpu):
    """NaN below everything, -0 as 0, infinities, subnormals, negatives."""
    w = torch.randn((1, 2, 120))
    w[0, :, 3] = float("nan")
    w[0, :, 5] = float("inf")
    w[0, :, 7] = float("-inf")
    w[0, :, 20:30] = -0.0
    w[0, :, 30:40] = 0.0
    w[0, 0, 50:60] = 1e-42
    w[0, 1, 50:60] = -1e-42
    w[0, 1, 60:100] = float("nan")
    for keep in (1, 40, 60, 75, 90, 117, 119):
        check_evict(gpu, [120], keep=keep, w=w.clone())


@pytest.mark.parametrize("in_place", [True, False])
def test_evict_released_pages(gpu, in_place):
    """Positions on a page that is gone are not kept."""
    def change(t):
        t[0, 2] = -1
        t[0, 5] = 1 << 20
        t[1, :] = -1

    check_evict(gpu, [150, 40, 30], keep=60, recent=20, change=change, in_place=in_place)


def test_refusals(gpu):
    from instinct_amd import _lib
    from instinct_amd.eviction import evict_rows, paged_attention_weights

    keys = torch.zeros((4, 2, 16, 64), dtype=torch.float16, device=gpu)
    w = torch.zeros((1, 2, 64), device=gpu)
    t = torch.zeros((1, 4), dtype=torch.int32, device=gpu)
    n = torch.tensor([64], dtype=torch.int32, device=gpu)
    q = torch.zeros((1, 4, 64), dtype=torch.float16, device=gpu)
    kw = dict(page_size=16, longest=64)
    with pytest.raises(TypeError, match="keys"):
        paged_attention_weights(q.bfloat16(), keys, t, n, w, scale=1.0, **kw)
    with pytest.raises(TypeError, match="float32"):
        paged_attention_weights(q, keys, t, n, w.half(), scale=1.0, **kw)
    with pytest.raises(ValueError, match="weights must be"):
        paged_attention_weights(q, keys, t, n, w[:, :1], scale=1.0, **kw)
    with pytest.raises(ValueError, match="contiguous"):
        paged_attention_weights(q, keys, t, n, w[..., ::2], scale=1.0, **kw)
    with pytest.raises(ValueError, match="multiple of kv heads"):
        paged_attention_weights(q[:, :3].contiguous(), keys, t, n, w, scale=1.0, **kw)
    with pytest.raises(TypeError, match="int32"):
        paged_attention_weights(q, keys, t.long(), n, w, scale=1.0, **kw)
    with pytest.raises(_lib.PdaError):
        paged_attention_weights(q, keys, t, n, w, scale=float("inf"), **kw)
    with pytest.raises(_lib.PdaError, match="exceed keep"):
        evict_rows(keys, keys, w, t, n, keep=8, recent=9, **kw)
    with pytest.raises(_lib.PdaError, match="keep"):
        evict_rows(keys, keys, w, t, n, keep=0, **kw)
    with pytest.raises(ValueError, match="pages for the kept"):
        evict_rows(keys, keys, w, t, n, keep=40, out_tables=t[:, :2].contiguous(), **kw)
    with pytest.raises(ValueError, match="keys' shape"):
        evict_rows(keys, keys[:2], w, t, n, keep=8, **kw)
    with pytest.raises(ValueError, match="scales"):
        evict_rows(keys.to(torch.int8), keys.to(torch.int8), w, t, n, keep=8, **kw)
