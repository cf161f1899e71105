"""What PackedPrefillBatch and DraftBatch write to the cache is what they were given:
every row of every sequence and layer against the projections, and the decode step that
reads those rows against 64 bits."""

import numpy as np
import pytest
import torch

from instinct_amd.batches import DecodeBatch, DraftBatch, PackedPrefillBatch
from instinct_amd.paged_kv import KVCache, KVGroup
from oracle import many_tokens as plain

pytestmark = pytest.mark.gpu

PAGE = 16


def check_rows(cache, layer, tables, b, start, k, v):
    """Rows start .. of sequence b hold k and v ``[n, kv_heads, dim]``: at 16 bits as they
    are. At 8 they were rounded to fp16 (x: 2^-11 of it, or 2^-25), their scale is fp16 of
    the largest / 127 (2^-11 of it again, and float32's division: in all 2^-10 + 2^-20) and
    the rows are within half a step of it (and a division's 127 * 2^-23 steps)."""
    rows = torch.as_tensor(cache.rows(tables[b], start, start + len(k)), device="cuda")
    for i, (store, x) in enumerate(((cache.keys[layer], k), (cache.values[layer], v))):
        got = cache._pick(store, rows)
        if cache.bits == 16:
            assert torch.equal(got, x)
            continue
        scale = cache._pick(cache.scales(layer)[i], rows).double()[..., None]
        x = x.double()
        top = x.abs().amax(-1, keepdim=True)
        assert torch.all((scale - top / 127).abs() <= (2 ** -10 + 2 ** -20) * top / 127)
        tol = (0.5 + 2.0 ** -16) * scale + 2.0 ** -11 * x.abs() + 2.0 ** -25
        assert torch.all((got.double() * scale - x).abs() <= tol)


@pytest.mark.parametrize("layout", ["pages", "rows"])
@pytest.mark.parametrize("dtype, bits", [(torch.float16, 16), (torch.bfloat16, 16),
                                         (torch.float16, 8), (torch.bfloat16, 8)], ids=str)
def test_rows_are_the_projections(gpu, layout, dtype, bits):
    gen = torch.Generator(device="cuda").manual_seed(bits)
    groups = [KVGroup("full", (0, 2), 2, 64), KVGroup("near", (1,), 2, 64, 40)]
    cache = KVCache(groups, page_size=PAGE, capacities={"full": 64, "near": 64}, dtype=dtype,
                    layout=layout, bits=bits)
    counts = np.array([37, 5, 90])
    need = (counts + 40) // PAGE + 1
    tables = {g: [cache.pools[g].allocate_many(int(n), reserved=False)[::-1].copy() for n in need]
              for g in ("full", "near")}

    def projections(n):
        qkv = torch.randn((n, 12, 64), generator=gen, device="cuda").to(dtype)
        return qkv.split([8, 2, 2], dim=1)

    of = lambda layer: tables[cache.layer_group[layer].name]  # noqa: E731
    written = {}
    step = PackedPrefillBatch(cache, torch.zeros(int(counts.sum()), dtype=torch.int64),
                              counts=counts, tables=tables)
    for layer in range(3):
        q, k, v = projections(int(counts.sum()))
        step.attend(layer, q, k, v, scale=0.125)
        written[layer] = [x.split(counts.tolist()) for x in (k, v)]
    for layer in range(3):  # (after all layers: none writes into another's rows)
        for b in range(3):
            check_rows(cache, layer, of(layer), b, 0, *(x[b] for x in written[layer]))

    nodes = np.array([6, 1, 30])
    parents = [[-1, 0, 1, 0, 3, 4], [-1], [-1] + [i // 2 for i in range(29)]]
    batch = DraftBatch(cache, torch.arange(int(nodes.sum())), counts=nodes,
                       parents=np.concatenate(parents), positions=counts, tables=tables)
    drafted = {}
    for layer in range(3):
        q, k, v = projections(int(nodes.sum()))
        batch.attend(layer, q, k, v, scale=0.125)
        drafted[layer] = [x.split(nodes.tolist()) for x in (k, v)]
    for layer in range(3):
        for b in range(3):
            check_rows(cache, layer, of(layer), b, 0, *(x[b] for x in written[layer]))
            check_rows(cache, layer, of(layer), b, int(counts[b]), *(x[b] for x in drafted[layer]))

    # The decode step behind the prompts (node 0's row is written again). It rounds at most
    # what oracle.many_tokens.attention_tolerance counts: weights, values, the output.
    step = DecodeBatch(cache, torch.zeros(3), positions=counts, tables=tables)
    for layer in range(3):
        q, k, v = projections(3)
        out = step.attend(layer, q, k, v, scale=0.125).view(3, 8, 64).double().cpu().numpy()
        window = cache.layer_group[layer].window
        for b in range(3):
            check_rows(cache, layer, of(layer), b, int(counts[b]), k[b:b + 1], v[b:b + 1])
            if bits == 16:
                kk, vv = (torch.cat([x[b], y[b:b + 1]]).double().cpu().numpy()
                          for x, y in zip(written[layer], (k, v)))
            else:
                rows = torch.as_tensor(cache.rows(of(layer)[b], 0, int(counts[b]) + 1),
                                       device="cuda")
                kk, vv = ((cache._pick(s, rows).double()
                           * cache._pick(c, rows).double()[..., None]).cpu().numpy()
                          for s, c in zip((cache.keys[layer], cache.values[layer]),
                                          cache.scales(layer)))
            n = len(kk)
            at = np.arange(n)
            keep = ((at > n - 1 - window) if window else at >= 0)[None]
            for h in range(8):
                want, size = plain._attend(q[b, h][None].double().cpu().numpy(), kk[:, h // 4],
                                           vv[:, h // 4], keep, 0.125, 0.0)
                tol = plain.attention_tolerance(want, size, vv, n, dtype, bits == 8)
                assert np.all(np.abs(out[b, h] - want[0]) <= tol[0])
