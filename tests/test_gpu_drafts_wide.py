"""Trees of more than 128 (node, query head) rows a sequence, which the kernels of eight
waves take at head dims 64, 96 and 128: every type against 64 bits."""

import numpy as np
import pytest
import torch

from test_gpu_drafts import BF16, F16, Case

pytestmark = pytest.mark.gpu

TYPES = pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
BITS = pytest.mark.parametrize("bits", [16, 8])
HEADS = pytest.mark.parametrize("heads", [(16, 2, 64), (12, 1, 96), (28, 4, 128)], ids=str)


def wide(case):
    """Whether the call has more rows than four waves hold for every sequence."""
    group = case.q.shape[1] // case.host[0].shape[1]
    return int(case.starts[-1]) * group > 128 * len(case.held)


@TYPES
@BITS
@HEADS
def test_against_64_bits(gpu, heads, dtype, bits):
    case = Case(21, [100, 0, 1333, 64], [64, 40, 64, 33], heads, dtype, bits=bits)
    assert wide(case)
    case.check()


@TYPES
@BITS
@HEADS
@pytest.mark.parametrize("kw", [dict(window=30), dict(window=200, softcap=20.0),
                                dict(scale=-0.2)], ids=str)
def test_windows_softcaps_scales(gpu, heads, dtype, bits, kw):
    case = Case(22, [400, 30, 1000], [64, 64, 47], heads, dtype, bits=bits, layout="rows", page=7)
    assert wide(case)
    case.check(**kw)


@TYPES
@BITS
@HEADS
def test_cut_units_and_released_pages(gpu, heads, dtype, bits):
    case = Case(23, [9000, 3000], [64, 64], heads, dtype, bits=bits)
    assert wide(case)
    case.tables[0, 3:9] = -1
    case.tables[1, 100] = 1 << 30
    case.tables[0, 400] = -7
    case.check()


@TYPES
@BITS
@HEADS
@pytest.mark.parametrize("bad", [float("nan"), float("inf")], ids=str)
def test_what_is_not_finite_reaches_those_that_see_it(gpu, heads, dtype, bits, bad):
    case = Case(24, [150, 90], [64, 60], heads, dtype, bits=bits, layout="rows")
    assert wide(case)
    clean = case.run(scale=0.1)
    node = 5
    row = case.tables[0, (150 + node) // 16] * 16 + (150 + node) % 16
    if bits == 8:
        case.scales[1][row] = bad
    else:
        case.stores[1][row, :, 1] = bad
    got = case.run(scale=0.1)
    sees = torch.tensor([bool(int(m) >> node & 1) for m in case.masks[:64]])
    assert 0 < int(sees.sum()) < 64
    assert torch.equal(got[:64][~sees], clean[:64][~sees]) and torch.equal(got[64:], clean[64:])
    assert not torch.isfinite(got[:64][sees][..., 1]).any()


@TYPES
@BITS
def test_repeated_and_captured(gpu, dtype, bits):
    from instinct_amd import drafts

    case = Case(25, [3000, 77, 512], [64, 64, 30], (28, 4, 128), dtype, bits=bits)
    assert wide(case)
    first = case.check()
    ws = torch.empty(drafts.tree_workspace_bytes(128), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(first)
    put = lambda a, t=np.int32: torch.as_tensor(np.asarray(a).astype(t), device="cuda")  # noqa: E731
    args = (case.q, *case.stores, put(case.tables), put(case.held), put(case.starts),
            put(case.masks.view(np.int64), np.int64))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        drafts.tree_attention(*args, page_size=16, scale=0.1, scales=tuple(case.scales) or None,
                              out=out, workspace=ws)
    for _ in range(4):
        out.zero_()
        ws.fill_(255)
        graph.replay()
        assert torch.equal(out, first)
        assert torch.equal(case.run(scale=0.1), first)
