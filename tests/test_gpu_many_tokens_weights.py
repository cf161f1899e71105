"""A row whose first key outweighs each of many others by some 2^25: together the others
still count, and where the first key's values are zeros they are all there is.

Weights are 16 bits wide where a row's maximum has the weight 2^7 or more; in fp16 one below
2^-14 is off by up to 2^-25, which is 2^-32 of the maximum's. So the tolerance is
u (sum p |v| + 2 |o|) for the rounding of weights and outputs, 2^-10.9 sum p |v| for the scores
(oracle.many_tokens.attention_tolerance), keys * 2^-32 (max |v| + |o|) for the small weights,
in the outputs and in their sum, and 2^-25 for an output below 2^-14."""

import numpy as np
import pytest
import torch

from instinct_amd import drafts, prompts
from oracle import many_tokens as plain

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def tolerance(want, size, keys, most, dtype, dequantized):
    u = plain.half_step(dtype)
    return (u * (size + 2 * want.abs()) + (2.0 ** -11 * size if dequantized else 0.0)
            + 2.0 ** -10.9 * size + keys * 2.0 ** -32 * (most + want.abs()) + 2.0 ** -25)


def keys_and_values(gen, n, dim):
    """Scores of a query of ones in element 0: 0 for the first key, -18.5 to -16.5 for the
    others (weights 2^-26.7 to 2^-23.8); values of one sign, the first key's zeros in the
    first half of the elements."""
    k = torch.zeros(n, dim, device="cuda")
    k[1:, 0] = -17.5 + 2 * (torch.rand(n - 1, generator=gen, device="cuda") - 0.5)
    v = torch.rand(n, dim, generator=gen, device="cuda") + 0.5
    v[0, :dim // 2] = 0
    return k, v


def exact(s, v):
    p = torch.softmax(s, dim=-1)
    return p @ v, p @ v.abs()


@pytest.mark.parametrize("n, dim", [(3000, 64), (3000, 128), (3000, 256), (131072, 64)], ids=str)
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
def test_packed_prompts(gpu, n, dim, dtype):
    gen = torch.Generator(device="cuda").manual_seed(n + dim)
    k, v = (x.to(dtype) for x in keys_and_values(gen, n, dim))
    q = torch.zeros(n, 2, dim, device="cuda", dtype=dtype)
    q[..., 0] = 1
    starts = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    got = prompts.packed_prompt_attention(q, k[:, None], v[:, None], starts, scale=1.0)
    for i in sorted({1, 63, 64, 700, 2999, n // 2, n - 1}):
        want, size = exact(k[:i + 1, 0].double()[None], v[:i + 1].double())
        tol = tolerance(want, size, i + 1, float(v.max()), dtype, False)
        off = (got[i].double() - want).abs()
        assert torch.all(off <= tol), (i, float((off - tol).max()), want[0, :2], got[i, 0, :2])


@pytest.mark.parametrize("n, dim, batch", [(3000, 64, 1), (3000, 64, 512), (3000, 128, 512),
                                           (3000, 256, 512), (131072, 128, 1),
                                           (40000, 128, 512)], ids=str)
@pytest.mark.parametrize("dtype, bits", [(F16, 16), (BF16, 16), (F16, 8), (BF16, 8)], ids=str)
def test_trees(gpu, n, dim, batch, dtype, bits):
    """512 sequences (over the same pages) are a workgroup each, whose pieces are whole."""
    gen = torch.Generator(device="cuda").manual_seed(n + dim + bits)
    page, nodes = 16, 3
    pages = -(-(n + nodes) // page)
    k, v = (x.view(pages, 1, page, dim) for x in keys_and_values(gen, pages * page, dim))
    scales = None
    if bits == 8:
        # (Keys in steps of 18.5 / 127; the values' scales, of 16 bits, are a step of each.)
        scales = tuple(torch.full((pages, 1, page), s, device="cuda").half()
                       for s in (18.5 / 127, 1.5 / 127))
        stores = [torch.round(x / s.float()[..., None]).clamp(-127, 127).to(torch.int8)
                  for x, s in zip((k, v), scales)]
        host = [x.double() * s.double()[..., None] for x, s in zip(stores, scales)]
    else:
        stores = [x.to(dtype) for x in (k, v)]
        host = [x.double() for x in stores]
    host = [x.reshape(-1, dim) for x in host]
    q = torch.zeros(batch * nodes, 4, dim, device="cuda", dtype=dtype)
    q[..., 0] = 1
    put = lambda x, t=np.int32: torch.as_tensor(np.asarray(x).astype(t), device="cuda")  # noqa: E731
    got = drafts.tree_attention(q, *stores, put([np.arange(pages)] * batch), put([n] * batch),
                                put(np.arange(batch + 1) * nodes), put([1, 3, 5] * batch, np.int64),
                                page_size=page, scale=1.0, scales=scales)
    got = got.view(batch, nodes, 4, dim)
    for i, line in enumerate(([0], [0, 1], [0, 2])):
        rows = list(range(n)) + [n + j for j in line]
        want, size = exact(host[0][rows, 0][None], host[1][rows])
        tol = tolerance(want, size, len(rows), float(host[1].max()), dtype, bits == 8)
        off = (got[:, i].double() - want).abs()
        assert torch.all(off <= tol), (i, float((off - tol).max()), want[0, :2], got[0, i, 0, :2])
