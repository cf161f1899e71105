"""Latent attention on MI355X: attention over one shared latent vector per token.

A layer of this kind caches per token one row ``[latent | rope]``: the
normalised latent, from which every head's keys and values are projected by
``kv_b`` ``[q_heads, nope + value, latent]``, and one rotated key that all heads
share. The reference has no such layer; paging, tables, lengths and the order
(write, then attend) are those of :mod:`instinct_amd.hip_kernels`.

* :func:`latent_append`: normalise, rotate and write a step's or a chunk's rows
  and rotate the queries, in one launch;
* :func:`latent_decode_attention`: one new token per sequence, absorbed form
  (the queries are projected into the latent and attend over the rows);
* :func:`latent_prefill_attention`: a chunk of one prompt, expanded form (every
  head's keys and values are projected out, then causal attention).

Head shapes: latents of 8..512 dims and nope and value dims of 8..128, in
eights; rotary parts of 0..64 dims in sixteens; any number of heads; fp16 or
bf16 throughout. The work happens in libpda.so (``csrc/pda_latent.hip``,
``csrc/pda_latent_prefill.hip``).
"""

from __future__ import annotations

from typing import Any

import torch

from . import _lib
from .hip_kernels import (_given_workspace, _int32_vector, on_device, rope_inv_freq,
                          stream_workspace)


def _check_16bit(name: str, t: torch.Tensor, dims: int, like: torch.Tensor,
                 rows_only: bool = False) -> None:
    """A GPU tensor of ``like``'s device and 16-bit type; contiguous, or with
    ``rows_only`` of contiguous rows any distance apart."""
    if (t is not like and t.dtype is like.dtype and t.dim() == dims and t.device == like.device
            and t.is_contiguous()):
        return  # (most tensors of most calls; `like` is checked itself)
    if t.dtype not in (torch.float16, torch.bfloat16) or t.dtype != like.dtype:
        raise TypeError(f"{name} must be {like.dtype} (float16 or bfloat16), got {t.dtype}")
    if not t.is_cuda or t.device != like.device:
        raise ValueError(f"{name} must be on the same GPU as the others")
    if t.dim() != dims:
        raise ValueError(f"{name} must have {dims} dimensions")
    if rows_only:
        if t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"{name} must have contiguous rows")
    elif not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _int32_on(name: str, t: torch.Tensor, n: int, device: torch.device) -> torch.Tensor:
    t = _int32_vector(name, t, n)
    if t.device != device:
        raise ValueError(f"{name} must be on {device}")
    return t


def _head_shape(q_width: int, arena: torch.Tensor, kv_b: torch.Tensor) -> tuple[int, ...]:
    """(q_heads, latent, rope, nope, value) of a layer from its tensors."""
    q_heads, out, latent = kv_b.shape
    rope = arena.shape[1] - latent
    nope = q_width - rope
    if rope < 0 or nope <= 0 or out - nope <= 0:
        raise ValueError("queries [.., q_heads, nope + rope], arena [rows, latent + rope] and "
                         "kv_b [q_heads, nope + value, latent] do not fit together")
    return q_heads, latent, rope, nope, out - nope


def latent_append(q: torch.Tensor | None, latent: torch.Tensor, k_rope: torch.Tensor,
                  arena: torch.Tensor, positions: torch.Tensor, rows: torch.Tensor, *,
                  dims: int, base: float | None = None, freqs: Any = None,
                  norm_weight: torch.Tensor | None = None, eps: float = 1e-6,
                  q_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Write ``n`` tokens' rows into the arena and rotate their queries, in one
    launch: ``arena[rows[i]] = [rms_norm(latent[i]) * norm_weight |
    rope(k_rope[i])]`` and the last ``rope`` elements of every query head
    rotated.

    ``latent`` ``[n, latent]`` and ``k_rope`` ``[n, rope]`` may be column slices
    of one projection's output (contiguous rows whose distance is a multiple of
    8 elements); ``arena`` ``[rows, latent + rope]``; ``q`` ``[n, q_heads, nope
    + rope]`` or None; ``positions`` and ``rows`` int32 ``[n]`` (rows outside
    the arena are not written; no two tokens may name one row). ``dims`` is
    ``rope`` (rotate, as :func:`instinct_amd.hip_kernels.rope`) or 0 (copy).
    ``norm_weight`` None stores the latents as they are. Returns the rotated
    queries (``q_out``, new unless given; it may be ``q``)."""
    _check_16bit("arena", arena, 2, arena)
    _check_16bit("latent", latent, 2, arena, rows_only=True)
    _check_16bit("k_rope", k_rope, 2, arena, rows_only=True)
    n, width = latent.shape
    rope = k_rope.shape[1]
    if k_rope.shape[0] != n or width + rope != arena.shape[1]:
        raise ValueError("latent and k_rope must be the arena's columns of n rows")
    if dims not in (0, rope):
        raise ValueError("dims must be 0 or the rotary width")
    q_heads = nope = 0
    if q is not None:
        _check_16bit("q", q, 3, arena)
        q_heads, nope = q.shape[1], q.shape[2] - rope
        if q.shape[0] != n or nope <= 0 or q_heads == 0:
            raise ValueError("q must be [n, q_heads, nope + rope]")
        if q_out is None:
            q_out = torch.empty_like(q)
        else:
            _check_16bit("q_out", q_out, 3, arena)
            if q_out.shape != q.shape:
                raise ValueError("q_out must have q's shape")
    elif q_out is not None:
        raise ValueError("q_out needs q")
    if norm_weight is not None:
        _check_16bit("norm_weight", norm_weight, 1, arena)
        if norm_weight.shape[0] != width:
            raise ValueError("norm_weight must be [latent]")
    rows = _int32_on("rows", rows, n, arena.device)
    if n == 0:
        return q_out
    table = None
    if dims:
        positions = _int32_on("positions", positions, n, arena.device)
        table = rope_inv_freq(dims, base=base, freqs=freqs, device=arena.device)
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    # (One row has no distance to a next one, whatever its stride says.)
    stride = lambda t, w: w if n == 1 else t.stride(0)  # noqa: E731
    entry = "pda_latent_append" + ("_bf16" if arena.dtype == torch.bfloat16 else "")
    with on_device(arena.device):
        rc = getattr(_lib.library(), entry)(
            ptr(q), ptr(q_out), ptr(latent), stride(latent, width), ptr(k_rope) if rope else None,
            stride(k_rope, rope), ptr(norm_weight), float(eps), ptr(arena),
            ptr(positions) if dims else None, ptr(rows), n, q_heads, width, rope, nope,
            arena.shape[0], ptr(table), torch.cuda.current_stream(arena.device).cuda_stream)
    _lib.check(rc)
    return q_out


def latent_decode_workspace_bytes(queries_shape: tuple[int, int, int], arena: torch.Tensor,
                                  kv_b: torch.Tensor, *, page_size: int, table_width: int,
                                  longest: int) -> int:
    """Bytes of workspace :func:`latent_decode_attention` needs for this shape
    (``pda_latent_decode_workspace_bytes``)."""
    batch, q_heads, _ = (int(x) for x in queries_shape)
    latent = int(kv_b.shape[2])
    return _lib.latent_decode_workspace_bytes(batch, q_heads, latent,
                                              int(arena.shape[1]) - latent, int(page_size),
                                              int(table_width), int(longest))


def latent_decode_attention(queries: torch.Tensor, arena: torch.Tensor, kv_b: torch.Tensor,
                            tables: torch.Tensor, lengths: torch.Tensor, *, page_size: int,
                            longest: int, scale: float, out: torch.Tensor | None = None,
                            workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention for one new token per sequence over its paged latent rows, in
    the absorbed form. ``queries`` ``[batch, q_heads, nope + rope]`` (rotated),
    ``arena`` ``[rows, latent + rope]``, ``kv_b`` ``[q_heads, nope + value,
    latent]``; ``tables`` ``[batch, width]`` and ``lengths`` ``[batch]`` int32,
    ``page_size`` and ``longest`` as for
    :func:`instinct_amd.hip_kernels.paged_decode_attention`. Returns ``[batch,
    q_heads, value]`` (zeros for a sequence with no key to see). Repeated calls
    give the same bits. ``workspace``: a uint8 device tensor the caller owns (at
    least :func:`latent_decode_workspace_bytes`; one per captured graph), else
    the stream's cached one."""
    _check_16bit("queries", queries, 3, queries)
    _check_16bit("arena", arena, 2, queries)
    _check_16bit("kv_b", kv_b, 3, queries)
    batch, q_heads, q_width = queries.shape
    heads, latent, rope, nope, value = _head_shape(q_width, arena, kv_b)
    if heads != q_heads:
        raise ValueError("kv_b must have the queries' heads")
    if tables.dtype != torch.int32 or lengths.dtype != torch.int32:
        raise TypeError("tables and lengths must be int32")
    if tables.dim() != 2 or tables.shape[0] != batch or lengths.shape != (batch,):
        raise ValueError("tables must be [batch, width] and lengths [batch]")
    device = queries.device
    if tables.device != device or lengths.device != device:
        raise ValueError(f"tables and lengths must be on {device}")
    tables, lengths = tables.contiguous(), lengths.contiguous()
    if out is None:
        out = torch.empty((batch, q_heads, value), dtype=queries.dtype, device=device)
    else:
        _check_16bit("out", out, 3, queries)
        if out.shape != (batch, q_heads, value):
            raise ValueError("out must be [batch, q_heads, value]")
    if batch == 0:
        return out
    stride = tables.shape[1]
    need = _lib.latent_decode_workspace_bytes(batch, q_heads, latent, rope, int(page_size), stride,
                                              int(longest))
    stream = int(torch.cuda.current_stream(device).cuda_stream)
    ws = (stream_workspace(device, need, stream) if workspace is None
          else _given_workspace(workspace, device, need))
    entry = "pda_latent_decode_attention" + ("_bf16" if queries.dtype == torch.bfloat16 else "")
    with on_device(device):
        rc = getattr(_lib.library(), entry)(
            queries.data_ptr(), arena.data_ptr(), kv_b.data_ptr(), tables.data_ptr(),
            lengths.data_ptr(), out.data_ptr(), batch, q_heads, latent, rope, nope, value,
            int(page_size), stride, arena.shape[0], int(longest), float(scale),
            ws.data_ptr(), ws.numel(), stream)
    _lib.check(rc)
    return out


def latent_prefill_workspace_bytes(start: int, queries_shape: tuple[int, int, int],
                                   arena: torch.Tensor, kv_b: torch.Tensor) -> int:
    """Bytes of workspace :func:`latent_prefill_attention` needs for this shape
    (``pda_latent_prefill_workspace_bytes``)."""
    count, q_heads, q_width = (int(x) for x in queries_shape)
    _, _, rope, nope, value = _head_shape(q_width, arena, kv_b)
    return _lib.latent_prefill_workspace_bytes(int(start), count, q_heads, rope, nope, value)


def latent_prefill_attention(queries: torch.Tensor, arena: torch.Tensor, kv_b: torch.Tensor,
                             table: torch.Tensor, *, start: int, page_size: int, scale: float,
                             out: torch.Tensor | None = None,
                             workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one prompt chunk over its sequence's latent rows, in the
    expanded form: ``queries`` ``[count, q_heads, nope + rope]`` (rotated) at
    positions ``start ..``, each over the keys up to its own, the chunk's rows
    already written; ``arena`` and ``kv_b`` as for
    :func:`latent_decode_attention`, ``table`` the sequence's int32 pages.
    Returns ``[count, q_heads, value]`` (zeros for a query with no key to see).
    ``workspace``: a uint8 device tensor the caller owns (at least
    :func:`latent_prefill_workspace_bytes`), else the stream's cached one."""
    _check_16bit("queries", queries, 3, queries)
    _check_16bit("arena", arena, 2, queries)
    _check_16bit("kv_b", kv_b, 3, queries)
    count, q_heads, q_width = queries.shape
    heads, latent, rope, nope, value = _head_shape(q_width, arena, kv_b)
    if heads != q_heads:
        raise ValueError("kv_b must have the queries' heads")
    device = queries.device
    if table.dtype != torch.int32 or table.dim() != 1 or table.device != device:
        raise ValueError(f"table must be an int32 vector on {device}")
    if int(table.shape[0]) == 0 and count > 0:
        raise ValueError("the table holds no pages")
    table = table.contiguous()
    if out is None:
        out = torch.empty((count, q_heads, value), dtype=queries.dtype, device=device)
    else:
        _check_16bit("out", out, 3, queries)
        if out.shape != (count, q_heads, value):
            raise ValueError("out must be [count, q_heads, value]")
    if count == 0:
        return out
    need = _lib.latent_prefill_workspace_bytes(int(start), count, q_heads, rope, nope, value)
    stream = int(torch.cuda.current_stream(device).cuda_stream)
    ws = (stream_workspace(device, need, stream) if workspace is None
          else _given_workspace(workspace, device, need))
    entry = "pda_latent_prefill_attention" + ("_bf16" if queries.dtype == torch.bfloat16 else "")
    with on_device(device):
        rc = getattr(_lib.library(), entry)(
            queries.data_ptr(), arena.data_ptr(), kv_b.data_ptr(), table.data_ptr(),
            int(table.shape[0]), int(start), count, out.data_ptr(), q_heads, latent, rope, nope,
            value, int(page_size), int(arena.shape[0]), float(scale), ws.data_ptr(), ws.numel(),
            stream)
    _lib.check(rc)
    return out
