"""Latent prefill of a chunk in which a token's row is not finite: queries before it
do not see it, and it does not reach them."""

import pytest
import torch
from test_gpu_latent import SMALL, THIN, TYPES, UNEVEN, WIDE, layer, pack

from oracle import latent as oracle

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


def check(gpu, shape, heads, start, count, poison, dtype, page=16):
    """``poison``: (position, latent or rotary dim, value)."""
    from instinct_amd.latent import latent_prefill_attention

    latent, rope, nope, value = shape
    pages = -(-(start + count) // page) + 2
    arena, kv_b, g = layer(shape, heads, pages * page, dtype, seed=count)
    table = pack([start + count], page, pages, g)[0]
    q = torch.randn((count, heads, nope + rope), generator=g).to(dtype)
    scale = (nope + rope) ** -0.5
    want, bound = oracle.prefill(q, arena, kv_b, table, start=start, page_size=page, scale=scale)
    for at, dim, x in poison:
        arena[int(table[at // page]) * page + at % page, dim] = x
    got = latent_prefill_attention(q.to(gpu), arena.to(gpu), kv_b.to(gpu), table.to(gpu),
                                   start=start, page_size=page, scale=scale).cpu().double()
    first = min(at for at, _, _ in poison) - start
    over = (got[:max(first, 0)] - want[:max(first, 0)]).abs() - bound[:max(first, 0)]
    assert bool((over <= 0).all()), f"past the bound by {over.max()}"
    seen = min([at for at, dim, _ in poison if dim < latent], default=start + count) - start
    assert bool(got[max(seen, 0):].isnan().all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("x", [INF, -INF, NAN])
@pytest.mark.parametrize("shape, heads", [(WIDE, 3), (SMALL, 14), (UNEVEN, 5), (THIN, 1),
                                          ((264, 16, 40, 24), 9)])
def test_shapes(gpu, shape, heads, x, dtype):
    check(gpu, shape, heads, 61, 150, [(150, 5, x)], dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_rotary_parts(gpu, dtype):
    check(gpu, SMALL, 3, 61, 150, [(150, 256 + 3, NAN), (170, 256 + 31, -INF)], dtype)
    check(gpu, WIDE, 2, 0, 1100, [(900, 512 + 60, INF)], dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("start, count, at", [
    (0, 1100, 1), (0, 1100, 1023), (0, 1100, 1099), (767, 257, 900),  # two blocks
    (4000, 300, 4100), (3000, 140, 3070), (3000, 140, 100)])           # split key ranges
def test_two_blocks_and_split_ranges(gpu, start, count, at, dtype):
    check(gpu, WIDE, 1, start, count, [(at, 511, NAN), (at, 3, INF)], dtype)


def test_last_range_holds_nothing_else(gpu):
    """The poisoned token alone in the part of a range that a query sees: the join
    takes its NaN for one, not for an empty range."""
    for at in range(3008, 3140, 64):
        check(gpu, SMALL, 2, 3000, 140, [(at, 9, NAN)], torch.float16)


def test_paired_tiles(gpu):
    check(gpu, (8, 16, 72, 8), 130, 0, 1030, [(640, 0, INF), (1000, 7, NAN)], torch.bfloat16,
          page=64)


def test_a_projection_that_is_not_finite(gpu):
    """A row of D_h with an infinity reaches its own dim alone."""
    from instinct_amd.latent import latent_prefill_attention

    arena, kv_b, g = layer(SMALL, 2, 128, torch.bfloat16)
    table = torch.arange(8, dtype=torch.int32)
    q = torch.randn((40, 2, 96), generator=g).bfloat16()
    want, bound = oracle.prefill(q, arena, kv_b, table, start=9, page_size=16, scale=0.1)
    kv_b[0, 64, 5] = INF
    got = latent_prefill_attention(q.to(gpu), arena.to(gpu), kv_b.to(gpu), table.to(gpu), start=9,
                                   page_size=16, scale=0.1).cpu().double()
    ok = (got - want).abs() <= bound
    assert not bool(got[:, 0, 0].isfinite().any())
    assert bool(ok[:, 0, 1:].all()) and bool(ok[:, 1].all())
