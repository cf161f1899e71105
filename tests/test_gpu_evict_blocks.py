"""Evictions of sequences past 8192 positions, which the selection goes over in
blocks: what it carries from block to block, and weights packed in place from a
later block to the front."""

import pytest
import torch
from test_gpu_evict import check_evict

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("lengths, keep, recent, sinks", [
    ([8192, 8193, 8191], 300, 10, 4),        # one block and a position, exactly one, one less
    ([20000, 16384, 5], 8200, 100, 0),       # more kept than a block has
    ([24579], 24578, 0, 0),                  # all but one
    ([16385, 9000], 4000, 4000, 0),          # guarded positions alone
    ([17000], 17000, 1, 1),                  # nothing goes
])
def test_blocks(gpu, lengths, keep, recent, sinks, in_place):
    check_evict(gpu, lengths, keep=keep, recent=recent, sinks=sinks, heads=1, dim=8, page=64,
                in_place=in_place)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("keep", [1, 8192, 8193, 12000, 20000])
def test_ties_over_blocks(gpu, keep, in_place):
    """All alike, and alike but for a few heavier ones behind: the lower positions
    are kept, over the border of a block."""
    w = torch.full((2, 2, 20010), 0.5)
    w[:, 1, 8190:8200] = 0.75
    w[:, 1, 19000:19500] = 1.0
    check_evict(gpu, [20000, 10000], keep=keep, recent=1, heads=2, dim=8, page=64, w=w,
                in_place=in_place)


@pytest.mark.parametrize("in_place", [True, False])
def test_unusual_weights_over_blocks(gpu, in_place):
    """NaN last whichever block holds them, released pages in every block."""
    g = torch.Generator().manual_seed(2)
    w = torch.randn((1, 1, 20000), generator=g)
    w[..., 100:9000] = float("nan")
    w[..., 12000:12100] = float("inf")
    w[..., 15000:15100] = float("-inf")

    def change(t):
        t[0, 200:210] = -1
        t[0, 250] = 1 << 25

    for keep in (9000, 15000, 19000):
        check_evict(gpu, [20000], keep=keep, heads=1, dim=8, page=64, w=w.clone(), change=change,
                    in_place=in_place)
