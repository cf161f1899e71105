"""Latent decode where queries into the latent pass fp16's range."""

import pytest
import torch
from test_gpu_latent import SMALL, THIN, UNEVEN, WIDE, layer, pack, run_decode

from oracle import latent as oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("shape, heads", [(WIDE, 16), (WIDE, 64), (WIDE, 128), (SMALL, 14),
                                          (SMALL, 40), (UNEVEN, 96), (THIN, 1), ((264, 0, 40, 24), 3)])
def test_absorbed_queries_past_fp16(gpu, shape, heads, sign):
    """Queries and projections inside fp16's range whose products are not: the
    scores, at a scale that keeps them a few units, and the result are as exact as
    any. Every third query is large, the others are ordinary ones of the same
    batch, whose scores at this scale are next to 0. (The bound's u A, with A the
    size of a score's terms, is below 0.1: 2^-11 of A up to 200.)"""
    latent, rope, nope, value = shape
    lengths, page = [1, 65, 0, 200, 33, 90], 16
    arena, kv_b, g = layer(shape, heads, 40 * page, torch.float16)
    kv_b = kv_b * 6
    tables = pack(lengths, page, 40, g)
    q = torch.randn((len(lengths), heads, nope + rope), generator=g).clamp(-4, 4)
    q[::3] *= 16000
    q = q.half()
    absorbed = torch.einsum("bhd,hdl->bhl", q[..., :nope].double(), kv_b[:, :nope].double())
    if nope > 8:
        assert absorbed.abs().max() > 1.5 * 65504 and bool(q.isfinite().all())
    # The terms of the largest score: absorbed queries and rotary parts times rows of
    # up to a few units.
    size = (absorbed.abs().sum(-1) + q[..., nope:].double().abs().sum(-1)).max()
    scale = sign * 100 / float(size)
    got = run_decode(gpu, q, arena, kv_b, tables, lengths, page, scale).cpu().double()
    want, bound = oracle.decode(q, arena, kv_b, tables, lengths, page_size=page, scale=scale)
    over = (got - want).abs() - bound
    assert bool((over <= 0).all()), f"past the bound by {over.max():.3e}"


def test_rows_of_one_key(gpu):
    """With one key the result is its value, whatever the score."""
    latent, rope, nope, value = WIDE
    arena, kv_b, g = layer(WIDE, 16, 16, torch.float16)
    q = torch.full((1, 16, nope + rope), 60000.0).half()
    tables = torch.zeros((1, 1), dtype=torch.int32)
    got = run_decode(gpu, q, arena, kv_b, tables, [1], 16, 0.07).cpu().double()
    want, bound = oracle.decode(q * 0, arena, kv_b, tables, [1], page_size=16, scale=0.07)
    assert bool(((got - want).abs() <= bound).all())
