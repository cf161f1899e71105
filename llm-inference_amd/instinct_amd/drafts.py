"""Trees of drafted tokens over the paged cache, on MI355X.

A draft model proposes a tree of tokens for every sequence; the model runs all nodes
in one step, each seeing the rows that its sequence holds and its own ancestors
(:func:`tree_attention`, every layer), and afterwards the longest line of nodes that
it would have chosen itself is kept: :func:`commit_drafts` finds the line and packs
its rows behind those held, in all layers. Node 0 of a tree is the sequence's newest
token, the others are drafted. The rows, positions and ancestor masks come from
:func:`instinct_amd.paging.extend_tables`;
:class:`instinct_amd.batches.DraftBatch` makes a step's calls. The reference decodes
one token a sequence and step.

The work happens in libpda.so (``csrc/pda_drafts.hip``).
"""

from __future__ import annotations

from array import array
from collections.abc import Sequence
from operator import attrgetter
from typing import Any, NamedTuple

import torch

from . import _lib
from .eviction import _check_arena, _check_index
from .hip_kernels import _arena_geometry, _given_workspace, on_device, stream_workspace

NODES = 64  # of a tree: a mask has a bit for each

_contiguous, _device = torch.Tensor.is_contiguous, torch.Tensor.get_device
_size, _dtype = torch.Tensor.size, attrgetter("dtype")


def tree_workspace_bytes(head_dim: int) -> int:
    """Bytes of workspace :func:`tree_attention` needs, whatever its batch and lengths
    (``pda_tree_workspace_bytes``)."""
    return _lib.tree_workspace_bytes(int(head_dim))


def tree_attention(queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor,
                   tables: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor,
                   masks: torch.Tensor, *, page_size: int, scale: float, window: int = 0,
                   softcap: float = 0.0, scales: tuple[Any, Any] | None = None,
                   out: torch.Tensor | None = None,
                   workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of drafted trees: ``queries`` ``[tokens, q_heads, D]`` are the nodes,
    sequence b's ``starts[b] .. starts[b + 1] - 1`` (int32 ``[batch + 1]``, ascending
    from 0); node i sees the ``lengths[b]`` rows held before the tree and the nodes j
    whose bit ``masks`` (int64 ``[tokens]``) has; node j's keys and values are in row
    ``lengths[b] + j``, written before. A node that sees nothing gives zeros. Its
    position is ``lengths[b]`` plus its mask's bits less one; ``window`` hides what is
    that far behind it. Nodes past the 64th of a tree are seen by none. The arena, the
    tables (int32 ``[batch, width]``), ``scales`` (8-bit K/V) and ``softcap`` are those
    of :func:`instinct_amd.hip_kernels.paged_decode_attention`; ``D`` is a multiple of
    8 up to 256. Returns ``[tokens, q_heads, D]``, zeros behind the last sequence;
    repeated calls give the same bits. ``workspace``: a uint8 device tensor the caller
    owns (:func:`tree_workspace_bytes`), else the stream's cached one."""
    q8 = scales is not None
    if queries.dim() != 3 or queries.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("queries must be [tokens, q_heads, head_dim] float16 or bfloat16")
    if not queries.is_cuda or not queries.is_contiguous():
        raise ValueError("queries must be a contiguous GPU tensor")
    device = queries.device
    tokens, q_heads, head_dim = queries.shape
    layout, arena_rows, kv_heads, a_dim = _arena_geometry(keys, page_size)
    kind = torch.int8 if q8 else queries.dtype
    _check_arena("keys", keys, keys, kind)
    _check_arena("values", values, keys, kind)
    if keys.device != device or values.dim() != keys.dim():
        raise ValueError("keys and values must be arenas of one shape on the queries' device")
    if a_dim != head_dim:
        raise ValueError("keys must have the queries' head_dim")
    if q_heads == 0 or q_heads % kv_heads:
        raise ValueError("query heads must be a multiple of kv heads")
    if q8:
        for name, t in zip(("key_scales", "value_scales"), scales):
            _check_arena(name, t, keys, torch.float16)
            if t.dim() != keys.dim() - 1:
                raise ValueError(f"{name} must have one scale per row and kv head")
    if tables.dim() != 2:
        raise ValueError("tables must be [batch, width]")
    batch = tables.shape[0]
    tables = _check_index("tables", tables, (batch, None), device)
    lengths = _check_index("lengths", lengths, (batch,), device)
    starts = _check_index("starts", starts, (batch + 1,), device)
    if masks.dtype != torch.int64 or masks.dim() != 1 or masks.shape[0] < tokens:
        raise ValueError("masks must be int64 [tokens]")
    if masks.device != device:
        raise ValueError(f"masks must be on {device}")
    masks = masks.contiguous()
    if out is None:
        out = torch.empty_like(queries)
    elif (out.dtype != queries.dtype or out.shape != queries.shape or out.device != device
          or not out.is_contiguous()):
        raise ValueError("out must be contiguous and match the queries' shape, dtype and device")
    need = _lib.tree_workspace_bytes(head_dim)
    stream = int(torch.cuda.current_stream(device).cuda_stream)
    with on_device(device):
        ws = (stream_workspace(device, need, stream) if workspace is None
              else _given_workspace(workspace, device, need))
        entry = ("pda_tree_attention" + ("_q8" if q8 else "")
                 + ("_bf16" if queries.dtype == torch.bfloat16 else ""))
        extra = (scales[0].data_ptr(), scales[1].data_ptr()) if q8 else ()
        rc = getattr(_lib.library(), entry)(
            queries.data_ptr(), keys.data_ptr(), values.data_ptr(), *extra, tables.data_ptr(),
            lengths.data_ptr(), starts.data_ptr(), masks.data_ptr(), out.data_ptr(), tokens, batch,
            q_heads, kv_heads, head_dim, int(page_size), tables.shape[1], arena_rows, layout,
            float(scale), int(window), float(softcap), ws.data_ptr(), ws.numel(), stream)
    _lib.check(rc)
    return out


class Committed(NamedTuple):
    """What :func:`commit_drafts` found."""

    lengths: torch.Tensor    # [batch] int32: rows held now
    accepted: torch.Tensor   # [batch] int32: nodes kept
    path: torch.Tensor       # [batch, 64] int32: the kept nodes, then -1
    following: torch.Tensor  # [batch] int64: the model's choice after the last one


def commit_drafts(arenas: Sequence[tuple[torch.Tensor, ...]], tables: torch.Tensor,
                  lengths: torch.Tensor, starts: torch.Tensor, parents: torch.Tensor,
                  drafted: torch.Tensor, targets: torch.Tensor, *, page_size: int,
                  out: Committed | None = None) -> Committed:
    """Keep the drafted tokens that the model chose itself. A tree's node 0 is kept;
    after every kept node follows its first child whose ``drafted`` token equals
    ``targets`` there (the model's choice after that node: its best token, or one it
    sampled); all int64 or int32 ``[tokens]``, as ``parents`` (int32) and ``starts``
    are those of the step. The kept nodes' rows move behind the ``lengths[b]`` rows
    held before the step, in every arena: per layer ``(keys, values)`` or ``(keys,
    values, key_scales, value_scales)``, all of one shape and layout. Rows of other
    nodes stay as they are, to be overwritten; pages are kept (the next
    ``extend_tables`` takes as many fewer). A tree's rows lie on pages that no other
    sequence holds. ``out`` overlaps no input."""
    if not arenas:
        raise ValueError("no layers given")
    keys = arenas[0][0]
    layout, arena_rows, kv_heads, head_dim = _arena_geometry(keys, page_size)
    device = keys.device
    if len(arenas[0]) not in (2, 4) or any(len(a) != len(arenas[0]) for a in arenas):
        raise ValueError("a layer is (keys, values) or those and their scales")
    # (One test of a kind of store in all layers at once: with some dozens of stores the
    # call waits for this code.)
    shape = keys.shape
    for name, dtype, size, of_layers in zip(
            ("keys", "values", "key_scales", "value_scales"),
            (keys.dtype, keys.dtype, torch.float16, torch.float16),
            (shape, shape, shape[:-1], shape[:-1]), zip(*arenas)):
        if (not all(map(_contiguous, of_layers)) or set(map(_device, of_layers)) != {device.index}
                or set(map(_dtype, of_layers)) != {dtype}
                or list(map(_size, of_layers)) != [size] * len(arenas)):
            for t in of_layers:
                _check_arena(name, t, keys, dtype)
            raise ValueError(f"{name} must have the first layer's shape")
    stores = array("Q", [t.data_ptr() for arena in arenas for t in arena])
    if len(set(stores)) < len(stores):
        raise ValueError("a store given twice: its rows would move twice")
    if tables.dim() != 2:
        raise ValueError("tables must be [batch, width]")
    batch = tables.shape[0]
    tables = _check_index("tables", tables, (batch, None), device)
    lengths = _check_index("lengths", lengths, (batch,), device)
    starts = _check_index("starts", starts, (batch + 1,), device)
    parents = _check_index("parents", parents, (parents.shape[0],), device)
    tokens = parents.shape[0]
    for name, t in (("drafted", drafted), ("targets", targets)):
        if t.dtype not in (torch.int64, torch.int32) or t.dtype != drafted.dtype:
            raise TypeError("drafted and targets must both be int64 or int32")
        if t.dim() != 1 or t.shape[0] != tokens:
            raise ValueError(f"{name} must be [tokens] as parents")
        if t.device != device:
            raise ValueError(f"{name} must be on {device}")
    drafted, targets = drafted.contiguous(), targets.contiguous()
    if out is None:
        new, accepted, path = torch.empty(
            (2 + NODES) * batch, dtype=torch.int32, device=device
        ).split_with_sizes((batch, batch, NODES * batch))
        out = Committed(new, accepted, path.view(batch, NODES),
                        torch.empty(batch, dtype=torch.int64, device=device))
    else:
        for name, t, shape in zip(Committed._fields, out, ((batch,), (batch,), (batch, NODES),
                                                           (batch,))):
            dtype = torch.int64 if name == "following" else torch.int32
            if (t.dtype != dtype or t.shape != shape or t.device != device
                    or not t.is_contiguous()):
                raise ValueError(f"out.{name} must be contiguous {dtype} {list(shape)}")
    with on_device(device):
        rc = _lib.library().pda_commit_drafts(
            stores.buffer_info()[0], len(arenas), len(arenas[0]),
            head_dim * keys.element_size(), tables.data_ptr(), lengths.data_ptr(),
            starts.data_ptr(), parents.data_ptr(), drafted.data_ptr(), targets.data_ptr(),
            drafted.element_size(), out.lengths.data_ptr(), out.accepted.data_ptr(),
            out.path.data_ptr(), out.following.data_ptr(), tokens, batch, kv_heads,
            int(page_size), tables.shape[1], arena_rows, layout,
            torch.cuda.current_stream(device).cuda_stream)
    _lib.check(rc)
    return out
