"""Page tables and slot maps of a step, built on the GPU from the requests' lengths.

The reference gives a step's tokens their rows in host loops (``KVCache.rows``,
python/instinct/paged_kv.py:259-265; ``DecodeBatch.__init__``, batches.py:148-179)
after drawing the pages that they need one by one. Here the host sets pages aside
ahead of time (:class:`PageFeed`) and
:func:`extend_tables` does the rest of a step in one launch: it lengthens the page
tables out of that feed and gives every token its row and its position, and the nodes
of drafted trees the mask of their ancestors. Nothing crosses PCIe, so the launch can
sit in a captured graph and be replayed while the feed lasts.

The work happens in libpda.so (``csrc/pda_paging.hip``).
"""

from __future__ import annotations

from operator import attrgetter
from typing import TYPE_CHECKING, NamedTuple

import numpy as np
import torch

from . import _lib
from .eviction import _check_index
from .hip_kernels import on_device

if TYPE_CHECKING:
    from .paged_kv import KVCache

_contiguous, _device = torch.Tensor.is_contiguous, torch.Tensor.get_device
_dtype = attrgetter("dtype")


class PageFeed:
    """Pages of a group's pool set aside for steps that take them on the GPU.
    :func:`extend_tables` takes the feed and moves it on: ``pages`` are its page ids and
    ``drawn[0]`` how many of them were taken. The pages that were drawn belong
    to the sequences whose tables have them and go back with those
    (``PagePool.release``); :meth:`refill` and :meth:`close` read ``drawn`` (and wait
    for the GPU, whatever streams the steps run on). A step captured into a graph draws on
    the feed as it is at each replay, refilled or closed, up to as many pages as the feed
    had room for at the capture; the feed outlives the graph."""

    def __init__(self, cache: "KVCache", group: str, count: int) -> None:
        self._cache, self._pool = cache, cache.pools[group]
        self.page_size = cache.page_size
        self._ids = self._pool.allocate_many(count, reserved=False)
        self._outgrown: list[tuple[torch.Tensor, torch.Tensor]] = []
        self._make_room()
        self._put()

    def _make_room(self) -> None:
        device = self._cache.device
        self._room = torch.empty(len(self._ids), dtype=torch.int32, device=device)
        self.drawn = torch.empty(2, dtype=torch.int32, device=device)

    def _put(self) -> None:
        # (In place: steps that were captured read these tensors.)
        ids = np.full(len(self._room), -1, dtype=np.int32)
        ids[:len(self._ids)] = self._ids
        self._room.copy_(torch.from_numpy(ids))
        self.pages = self._room[:len(self._ids)]
        self.drawn.zero_()
        self._wait()

    def _wait(self) -> None:
        if self.drawn.is_cuda:
            torch.cuda.synchronize(self.drawn.device)

    def _left(self) -> np.ndarray:
        self._wait()
        drawn = int(self.drawn[0])
        if drawn > len(self._ids):
            raise RuntimeError(f"steps asked for {drawn} pages of a feed of {len(self._ids)}: "
                               "some of their tokens have no row")
        return self._ids[drawn:]

    def refill(self, count: int) -> None:
        """``count`` pages to draw again. Past the most that the feed held so far it takes
        new tensors, and a step that was captured before finds no page (row -1)."""
        left = self._left()
        more = max(0, count - len(left))
        self._ids = np.concatenate([left, self._pool.allocate_many(more, reserved=False)])
        if len(self._ids) > len(self._room):
            self._room.fill_(-1)
            self._outgrown.append((self._room, self.drawn))  # (graphs may still read them)
            self._make_room()
        self._put()

    def close(self) -> None:
        """Gives the pages that were not drawn back to the pool."""
        left = self._left()
        self._ids = self._ids[:0]
        self._put()
        self._pool.release(left)


class StepRows(NamedTuple):
    """What :func:`extend_tables` gives a step (int32 but for the masks)."""

    starts: torch.Tensor     # [batch + 1] first token of each sequence, and the end
    lengths: torch.Tensor    # [batch] rows held with the step's tokens
    pages: torch.Tensor      # [batch] pages held
    drawn: torch.Tensor      # [2] pages drawn from the feed, and 0 (a PageFeed's own)
    rows: torch.Tensor       # [tokens] arena row of each token
    positions: torch.Tensor  # [tokens]
    masks: torch.Tensor | None  # [tokens] int64, with parents


def extend_tables(tables: torch.Tensor, lengths: torch.Tensor, counts: torch.Tensor,
                  pages: torch.Tensor, feed: PageFeed | torch.Tensor,
                  drawn: torch.Tensor | None = None, *, page_size: int, tokens: int,
                  parents: torch.Tensor | None = None, out: StepRows | None = None) -> StepRows:
    """Lengthen the page tables ``[batch, width]`` (in place) for a step that brings
    ``counts[b]`` tokens to a sequence that holds ``lengths[b]`` rows on ``pages[b]``
    pages, taking what is missing from ``feed`` in the order of the sequences; and the
    step's slot map (:class:`StepRows`). A :class:`PageFeed` moves on by itself: the next
    step goes on behind the pages that this one took. Of a tensor of page ids the call
    takes those from entry ``drawn[0]`` on (int32 ``[2]``, zeros for a new one), which
    stays as it is: the next step's is the result's ``drawn``, or both take the same pages.

    ``tokens``: entries of the per-token results, at least ``counts.sum()``; those
    behind the last token have row -1 (the append writes nothing there), position 0
    and mask 0. ``parents`` (int32 ``[tokens]``): each sequence's tokens are a tree of
    up to 64 nodes and ``parents`` names each node's parent among them (-1: none); a
    node's position then goes by its depth and its mask has the bits of its ancestors
    and its own. A feed that runs out leaves -1 as page and row and ``drawn`` past its
    end. All are int32 on one GPU; ``out`` may hold ``lengths``, ``pages`` and ``drawn``
    themselves (a step replayed from a graph; of a :class:`PageFeed` it has ``drawn``). No
    counterpart in the reference."""
    own = feed if isinstance(feed, PageFeed) else None
    if own is not None:
        if drawn is not None:
            raise TypeError("a PageFeed counts for itself what was drawn")
        if page_size != own.page_size:
            raise ValueError(f"the feed's pages hold {own.page_size} rows")
        # (All of its room: a refilled feed's pages are there for a captured step.)
        feed, drawn = own._room, own.drawn
    elif drawn is None:
        raise TypeError("drawn goes with a feed of page ids")
    if not tables.is_cuda:
        raise ValueError("tables must be on a GPU")
    device = tables.device
    if tables.dtype != torch.int32 or tables.dim() != 2 or not tables.is_contiguous():
        raise ValueError("tables must be contiguous int32 [batch, width]")
    batch, width = tables.shape
    given = (lengths, counts, pages, feed, drawn)
    # (One test for what is all right: small steps wait for this code.)
    if (not all(map(_contiguous, given)) or set(map(_dtype, given)) != {torch.int32}
            or set(map(_device, given)) != {device.index} or feed.dim() != 1
            or not lengths.shape == counts.shape == pages.shape == (batch,)
            or drawn.shape != (2,)):
        for name, t, n in (("lengths", lengths, batch), ("counts", counts, batch),
                           ("pages", pages, batch), ("feed", feed, None), ("drawn", drawn, 2)):
            if t.dim() != 1:
                raise ValueError(f"{name} must have one dimension")
            if not _check_index(name, t, (t.shape[0] if n is None else n,), device) is t:
                raise ValueError(f"{name} must be contiguous")
    if tokens < 0:
        raise ValueError("tokens must not be negative")
    if parents is not None:
        parents = _check_index("parents", parents, (tokens,), device)
    if out is None:
        # (One allocation for the int32 results: seven took 9 us of a small step's 17.)
        parts = torch.empty(3 * batch + 3 + 2 * tokens, dtype=torch.int32, device=device
                            ).split_with_sizes((batch + 1, batch, batch, 2, tokens, tokens))
        masks = (None if parents is None
                 else torch.empty(tokens, dtype=torch.int64, device=device))
        out = StepRows(*parts, masks)
        if own is not None:
            out = out._replace(drawn=drawn)
    else:
        if own is not None and out.drawn is not drawn:
            raise ValueError("out.drawn must be the feed's: the next step goes by it")
        for name, t, n in zip(StepRows._fields, out, (batch + 1, batch, batch, 2, tokens, tokens,
                                                      tokens)):
            if t is None and name == "masks" and parents is None:
                continue
            dtype = torch.int64 if name == "masks" else torch.int32
            if (t is None or t.dtype != dtype or t.shape != (n,) or t.device != device
                    or not t.is_contiguous()):
                raise ValueError(f"out.{name} must be contiguous {dtype} [{n}] on {device}")
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    with on_device(device):
        rc = _lib.library().pda_extend_tables(
            tables.data_ptr(), width, lengths.data_ptr(), counts.data_ptr(), pages.data_ptr(),
            feed.data_ptr(), feed.shape[0], drawn.data_ptr(), ptr(parents), batch, page_size,
            tokens, out.starts.data_ptr(), out.lengths.data_ptr(), out.pages.data_ptr(),
            out.drawn.data_ptr(), out.rows.data_ptr(), out.positions.data_ptr(), ptr(out.masks),
            torch.cuda.current_stream(device).cuda_stream)
    _lib.check(rc)
    return out
