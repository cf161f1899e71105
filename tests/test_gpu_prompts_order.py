"""Packed prompts of more items (128 queries of a head) than the GPU holds workgroups:
each takes several, in the order that the prompts' lengths give, the next one's first keys
and queries loaded beside the end of the last. Against 64 bits, with the tolerance of
oracle.many_tokens.attention_tolerance."""

import numpy as np
import pytest
import torch

from instinct_amd import prompts
from oracle import many_tokens as plain

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def make(seed, counts, q_heads, kv_heads, dim, dtype):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    qkv = torch.randn((int(sum(counts)), q_heads + 2 * kv_heads, dim), generator=gen,
                      device="cuda").to(dtype)
    starts = np.concatenate([[0], np.cumsum(counts)])
    return (*qkv.split([q_heads, kv_heads, kv_heads], dim=1), starts,
            torch.as_tensor(starts.astype(np.int32), device="cuda"))


def items(counts, q_heads):
    return sum(-(-int(n) // 128) for n in counts) * q_heads


def workgroups(dim):
    """That the GPU holds at once."""
    return 256 * (3 if dim <= 64 else 2 if dim <= 128 else 1)


def compare(got, q, k, v, starts, *, scale, window=0, rows=None):
    """Prompt by prompt and kv head by kv head; ``rows``: of each prompt only these."""
    group = q.shape[1] // k.shape[1]
    u = plain.half_step(q.dtype)
    bf16 = q.dtype == BF16
    worst = -float("inf")
    for a, z in zip(starts.tolist(), starts[1:].tolist()):
        if a == z:
            continue
        at = torch.arange(z - a, device="cuda") if rows is None else rows[rows < z - a]
        key = torch.arange(z - a, device="cuda")
        hidden = key[None] > at[:, None]
        if window:
            hidden |= key[None] <= at[:, None] - window
        for h in range(k.shape[1]):
            heads = slice(h * group, (h + 1) * group)
            kk, vv = k[a:z, h].double().contiguous(), v[a:z, h].double().contiguous()
            x = q[a + at, heads].double()  # [rows, group, dim]
            s = (x.reshape(-1, x.shape[-1]) @ kk.t().contiguous()).view(len(at), group, -1) * scale
            s.masked_fill_(hidden[:, None], -float("inf"))
            p = torch.softmax(s, dim=-1).view(-1, z - a)
            want, size = p @ vv, p @ vv.abs()
            # (oracle.many_tokens.attention_tolerance)
            tol = u * (size + 2 * want.abs()) + 2.0 ** -10.9 * size + 2.0 ** -24
            if not bf16:
                tol += (z - a) * 2.0 ** -25 * vv.abs().max()
            off = (got[a + at, heads].double().reshape(want.shape) - want).abs()
            # (A result that is not a number is off.)
            worst = max(worst, float(torch.nan_to_num(off - tol, nan=1e9).max()))
    assert worst <= 0, worst


MIXED = [700, 130, 1500, 257, 5, 900, 0, 1, 640, 1024, 64, 300]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("window", [0, 100, 700])
@pytest.mark.parametrize("heads", [(64, 4, 64), (40, 4, 96), (40, 2, 128), (32, 4, 256),
                                   (60, 2, 40), (40, 4, 112), (24, 2, 136)], ids=str)
def test_several_items_a_workgroup(gpu, heads, window, dtype):
    q, k, v, starts, dev = make(1, MIXED, *heads, dtype)
    assert items(MIXED, heads[0]) > 3 * workgroups(heads[2])
    got = prompts.packed_prompt_attention(q, k, v, dev, scale=0.1, window=window)
    compare(got, q, k, v, starts, scale=0.1, window=window)
    again = prompts.packed_prompt_attention(q, k, v, dev, scale=0.1, window=window)
    assert torch.equal(got, again)


@pytest.mark.parametrize("dtype, window", [(F16, 0), (BF16, 70)], ids=str)
@pytest.mark.parametrize("batch", [256, 300])  # with the order by lengths, and past it
def test_over_64_items_a_workgroup(gpu, batch, dtype, window):
    heads = (72, 2, 256)
    counts = np.random.default_rng(batch).integers(60, 160, batch)
    assert items(counts, heads[0]) > 65 * workgroups(256)
    q, k, v, starts, dev = make(2, counts, *heads, dtype)
    got = prompts.packed_prompt_attention(q, k, v, dev, scale=0.07, window=window)
    compare(got, q, k, v, starts, scale=0.07, window=window)


@pytest.mark.parametrize("counts", [[131072], [131073, 300], [40, 131200, 5000]], ids=str)
@pytest.mark.parametrize("window", [0, 3000])
def test_around_1024_tiles_a_prompt(gpu, counts, window):
    """The most tiles that the order by lengths takes, and more."""
    heads = (2, 1, 64)
    assert items(counts, heads[0]) > workgroups(64)
    q, k, v, starts, dev = make(3, counts, *heads, BF16)
    got = prompts.packed_prompt_attention(q, k, v, dev, scale=0.1, window=window)
    rows = torch.cat([torch.arange(0, 131200, 997), torch.arange(0, 300), torch.arange(4990, 5000),
                      torch.arange(131060, 131200)]).unique().cuda()
    compare(got, q, k, v, starts, scale=0.1, window=window, rows=rows)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")], ids=str)
@pytest.mark.parametrize("heads", [(64, 2, 64), (40, 2, 128), (32, 2, 256), (40, 2, 72)], ids=str)
@pytest.mark.parametrize("window", [0, 70])
def test_what_is_not_finite_stays_in_its_items(gpu, heads, window, bad):
    """Of one of several items that a workgroup takes, before and after others."""
    q, k, v, starts, dev = make(4, MIXED, *heads, F16)
    call = lambda: prompts.packed_prompt_attention(q, k, v, dev, scale=0.1, window=window)  # noqa: E731
    clean = call()
    group = heads[0] // heads[1]
    touched = torch.zeros(clean.shape[:2], dtype=torch.bool, device="cuda")
    for b, at in ((0, 131), (2, 1400), (5, 10), (9, 700), (11, 299)):
        a, z = int(starts[b]), int(starts[b + 1])
        v[a + at, 0, 3] = bad
        touched[a + at:min(z, a + at + window) if window else z, :group] = True
    got = call()
    assert torch.equal(got[~touched], clean[~touched])
    assert torch.equal(got[..., 4:], clean[..., 4:]) and torch.equal(got[..., :3], clean[..., :3])
    seen = got[..., 3][touched]
    assert torch.all(torch.isnan(seen) if bad != bad else seen == bad)
