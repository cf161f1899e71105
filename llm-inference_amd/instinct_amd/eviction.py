"""Eviction from the paged K/V cache by accumulated attention weight, on MI355X.

A cache that may not grow past a bound keeps the keys that attention uses: each
step credits every key of a sequence with the weights it was given
(:func:`paged_attention_weights`), and a sequence past its bound drops the keys
with the least credit and packs the rows of the others, per kv head
(:func:`evict_rows`). The credits are kept per sequence and logical position,
float32 ``[batch, kv_heads, capacity]``, so sequences that share a prefix's pages
do not share them. ``DecodeBatch(weights=...)`` makes the first call for every
layer, ``KVCache.evict`` the second for every layer of a group. The reference
bounds a cache by sliding windows alone.

The work happens in libpda.so (``csrc/pda_evict.hip``).
"""

from __future__ import annotations

from typing import Any

import torch

from . import _lib
from .hip_kernels import _arena_geometry, _given_workspace, on_device, stream_workspace


def _check_index(name: str, t: torch.Tensor, shape: tuple, device: torch.device) -> torch.Tensor:
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32")
    if t.dim() != len(shape) or t.shape[0] != shape[0]:  # (a second one may be anything)
        raise ValueError(f"{name} must be {list(shape)}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}")
    return t.contiguous()


def _same_columns(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two matrices of as many rows begin with the same columns in memory."""
    return (a.data_ptr() == b.data_ptr() and a.shape[0] == b.shape[0]
            and a.stride(-1) == b.stride(-1) and (a.shape[0] < 2 or a.stride(0) == b.stride(0)))


def check_weights(name: str, t: torch.Tensor, batch: int, kv_heads: int,
                  device: torch.device) -> int:
    """The capacity of float32 weights ``[batch, kv_heads, capacity]``."""
    if t.dtype != torch.float32:
        raise TypeError(f"{name} must be float32")
    if t.dim() != 3 or t.shape[0] != batch or t.shape[1] != kv_heads or t.shape[2] == 0:
        raise ValueError(f"{name} must be [batch, kv_heads, capacity]")
    if t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous and on {device}")
    return t.shape[2]


def _check_arena(name: str, t: torch.Tensor, keys: torch.Tensor, dtype: torch.dtype) -> None:
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_cuda or not t.is_contiguous() or t.device != keys.device:
        raise ValueError(f"{name} must be a contiguous GPU tensor beside the keys")
    if t is not keys and t.shape != keys.shape[:t.dim()]:
        raise ValueError(f"{name} must have the keys' shape")


def attention_weights_workspace_bytes(batch: int, q_heads: int, capacity: int) -> int:
    """Bytes of workspace :func:`paged_attention_weights` needs
    (``pda_attention_weights_workspace_bytes``)."""
    return _lib.attention_weights_workspace_bytes(int(batch), int(q_heads), int(capacity))


def paged_attention_weights(queries: torch.Tensor, keys: torch.Tensor, tables: torch.Tensor,
                            lengths: torch.Tensor, weights: torch.Tensor, *, page_size: int,
                            longest: int, scale: float, window: int = 0, softcap: float = 0.0,
                            scales: tuple[Any, Any] | None = None, fresh: int = 1,
                            out: torch.Tensor | None = None,
                            workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Credit a decode step's attention weights: for every position t below a
    sequence's length ``out[b, j, t] = weights[b, j, t] + sum over kv head j's
    query heads of softmax(scores)[t]``, the ``fresh`` newest positions starting
    from 0 (``fresh`` = the capacity takes nothing from ``weights``). The
    arguments up to ``scales`` are those of
    :func:`instinct_amd.hip_kernels.paged_decode_attention` (the keys alone;
    hidden keys get 0); ``weights`` is float32 ``[batch, kv_heads, capacity]``
    and no length may pass its capacity (a longer one is cut to it). ``out`` is
    ``weights`` unless given; entries from a sequence's length on are left as
    they were. Returns ``out``; repeated calls give the same bits."""
    q8 = scales is not None
    if queries.dim() != 3 or queries.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("queries must be [batch, q_heads, head_dim] float16 or bfloat16")
    batch, q_heads, head_dim = queries.shape
    layout, arena_rows, kv_heads, a_dim = _arena_geometry(keys, page_size)
    if not queries.is_cuda or not queries.is_contiguous():
        raise ValueError("queries must be a contiguous GPU tensor")
    device = queries.device
    _check_arena("keys", keys, keys, torch.int8 if q8 else queries.dtype)
    if keys.device != device:
        raise ValueError("keys must be on the queries' device")
    if a_dim != head_dim:
        raise ValueError("keys must have the queries' head_dim")
    if q_heads % kv_heads:
        raise ValueError("query heads must be a multiple of kv heads")
    if q8:
        _check_arena("key_scales", scales[0], keys, torch.float16)
        if scales[0].dim() != keys.dim() - 1:
            raise ValueError("key_scales must have one scale per row and kv head")
    tables = _check_index("tables", tables, (batch, None), device)
    lengths = _check_index("lengths", lengths, (batch,), device)
    capacity = check_weights("weights", weights, batch, kv_heads, device)
    if out is None:
        out = weights
    elif check_weights("out", out, batch, kv_heads, device) != capacity:
        raise ValueError("out must have the weights' shape")
    if batch == 0:
        return out
    need = _lib.attention_weights_workspace_bytes(batch, q_heads, capacity)
    stream = int(torch.cuda.current_stream(device).cuda_stream)
    ws = (stream_workspace(device, need, stream) if workspace is None
          else _given_workspace(workspace, device, need))
    entry = ("pda_attention_weights" + ("_q8" if q8 else "")
             + ("_bf16" if queries.dtype == torch.bfloat16 else ""))
    with on_device(device):
        rc = getattr(_lib.library(), entry)(
            queries.data_ptr(), keys.data_ptr(), *((scales[0].data_ptr(),) if q8 else ()),
            tables.data_ptr(), lengths.data_ptr(), weights.data_ptr(), out.data_ptr(), batch,
            q_heads, kv_heads, head_dim, int(page_size), int(tables.shape[1]), arena_rows, layout,
            capacity, int(longest), float(scale), int(window), float(softcap),
            min(int(fresh), capacity), ws.data_ptr(), ws.numel(), stream)
    _lib.check(rc)
    return out


def evict_rows(keys: torch.Tensor, values: torch.Tensor | None, weights: torch.Tensor,
               tables: torch.Tensor, lengths: torch.Tensor, *, page_size: int, longest: int,
               keep: int, recent: int = 0, sinks: int = 0,
               scales: tuple[Any, Any] | None = None, out_tables: torch.Tensor | None = None,
               out_weights: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Cut one layer's sequences down to ``keep`` rows a kv head: the first
    ``sinks``, the last ``recent`` and the heaviest other positions by
    ``weights`` (float32 ``[batch, kv_heads, capacity]``; of two alike the lower
    position, NaN last), in their order, packed to positions 0 .. of
    ``out_tables``; sequences of ``keep`` rows or fewer stay as they are.
    Positions on a negative or unknown page are gone.

    ``keys`` and ``values`` are a layer's arenas in either layout (``values``
    None: ``keys`` alone, as for one arena of latent rows), int8 with their
    ``scales`` at 8 bits. ``out_tables`` int32 ``[batch, width]`` names pages
    that no row is read from (a position that stays where it is excepted);
    without it, or where it is ``tables`` or its first columns, the rows move to
    the front of their own pages, which then must not be shared with another
    sequence; the first ``keep`` rows' pages must all be there then, since a kept
    row whose place lies on a page that is gone has nowhere to go and is lost
    (it still counts: its place is hidden like any on that page). Sequences that
    released their first pages need ``out_tables``. ``out_weights`` (``weights`` itself unless given) receives the kept
    positions' weights; its other entries are left. ``longest`` is the host-side
    largest length, which tables and weights must hold: rows past either could
    not be kept. Returns (new lengths int32 ``[batch]``, kept positions int32
    ``[batch, kv_heads, keep]``, -1 past a sequence's last)."""
    layout, arena_rows, kv_heads, head_dim = _arena_geometry(keys, page_size)
    dtype = torch.int8 if scales is not None else keys.dtype
    if dtype not in (torch.int8, torch.float16, torch.bfloat16):
        raise TypeError(f"keys must be float16, bfloat16 or int8, got {keys.dtype}")
    arenas = [("keys", keys)] + ([] if values is None else [("values", values)])
    for name, t in arenas:
        _check_arena(name, t, keys, dtype)
        if t.shape != keys.shape:
            raise ValueError(f"{name} must have the keys' shape")
    if scales is not None:
        for name, t in zip(("key_scales", "value_scales"), scales):
            _check_arena(name, t, keys, torch.float16)
            if t.dim() != keys.dim() - 1:
                raise ValueError(f"{name} must have one scale per row and kv head")
    elif keys.dtype == torch.int8:
        raise ValueError("an int8 cache needs its scales")
    device = keys.device
    batch = int(weights.shape[0])
    capacity = check_weights("weights", weights, batch, kv_heads, device)
    given = tables  # (the library compares addresses, which a copy would change)
    tables = _check_index("tables", tables, (batch, None), device)
    lengths = _check_index("lengths", lengths, (batch,), device)
    if int(longest) > capacity:
        raise ValueError(f"weights of {capacity} positions for a sequence of {int(longest)}")
    if int(longest) > tables.shape[1] * page_size:
        raise ValueError(f"tables of {tables.shape[1]} pages for a sequence of {int(longest)}")
    keep = int(keep)
    if out_tables is None:
        to = tables
    else:
        to = _check_index("out_tables", out_tables, (batch, None), device)
        if int(to.shape[1]) * page_size < min(keep, capacity, int(longest)):
            raise ValueError("out_tables must have pages for the kept rows")
        if _same_columns(out_tables, given):
            to = tables
    if out_weights is None:
        out_weights = weights
    out_capacity = check_weights("out_weights", out_weights, batch, kv_heads, device)
    kept = torch.empty((batch, kv_heads, max(keep, 0)), dtype=torch.int32, device=device)
    new_lengths = torch.empty(batch, dtype=torch.int32, device=device)
    lib = _lib.library()
    stride = int(tables.shape[1])
    stream = int(torch.cuda.current_stream(device).cuda_stream)
    with on_device(device):
        _lib.check(lib.pda_evict_select(
            weights.data_ptr(), out_weights.data_ptr(), tables.data_ptr(), lengths.data_ptr(),
            kept.data_ptr(), new_lengths.data_ptr(), batch, kv_heads, int(page_size), stride,
            arena_rows, capacity, out_capacity, keep, int(recent), int(sinks), stream))
        second = None if values is None else values.data_ptr()
        moves = [(keys.data_ptr(), second, head_dim * keys.element_size())]
        if scales is not None:
            moves.append((scales[0].data_ptr(), None if values is None else scales[1].data_ptr(),
                          2))
        for first, second, width in moves:
            _lib.check(lib.pda_evict_move(
                first, second, width, kept.data_ptr(), new_lengths.data_ptr(), tables.data_ptr(),
                to.data_ptr(), batch, kv_heads, int(page_size), stride, int(to.shape[1]),
                arena_rows, layout, keep, stream))
    return new_lengths, kept
