"""What a model forward sees on a decode step: the op contract of the path.

Counterpart of ``DecodeBatch`` (python/instinct/batches.py:142-253) for the
MI355X kernel: one new token per sequence, page tables packed to
``[batch, width]`` int32 with zero padding (:170-179), ``lengths =
positions + 1`` (:162-164), write rows ``table[pos // P] * P + pos % P``
(:175-178), :meth:`DecodeBatch.rope` (:195-201) and
:meth:`DecodeBatch.attend`, which writes the new K/V first and then attends
over ``[first, length)`` (:203-226), returning ``[batch, q_heads *
head_dim]``. :meth:`DecodeBatch.rope_attend` does the model's two ``rope``
calls, the write and the attention with the rotation and the write fused into
one launch.

The packed tables, lengths and write rows are uploaded once per step and
shared by every layer of a group, as in the reference.
"""

from __future__ import annotations

from typing import Any

import numpy as np
import torch

from .eviction import paged_attention_weights
from .hip_kernels import (image_spans, paged_decode_attention, paged_prefill_attention, rope,
                          rope_append)
from .paged_kv import KVCache


def pack_tables(tables: list[np.ndarray] | list[list[int]], count: int) -> np.ndarray:
    """``[count, width]`` int32 with 0 padding (batches.py:171-174)."""
    width = max(1, max(len(t) for t in tables))
    packed = np.zeros((count, width), dtype=np.int32)
    for row, table in enumerate(tables):
        packed[row, : len(table)] = table
    return packed


def rows_by_group(cache: KVCache, held: Any, shape: tuple[int, ...]) -> dict[str, np.ndarray]:
    """The rows that sequences hold, int64 of ``shape``, by group name; one value
    for a cache of one group."""
    groups = cache.groups
    if not isinstance(held, dict):
        if len(groups) > 1:
            raise ValueError("held must name its groups in a cache of several")
        held = dict.fromkeys(groups, held)
    rows = {name: np.asarray(n).astype(np.int64) for name, n in held.items()}
    for name, n in rows.items():
        if name not in groups:
            raise ValueError(f"held names no group {name!r}")
        if n.shape != shape or np.any(n < 0):
            raise ValueError("held must be the rows of each sequence")
    return rows


class DecodeBatch:
    prefill = False

    def __init__(
        self,
        cache: KVCache,
        tokens: torch.Tensor,
        *,
        positions: np.ndarray,
        tables: dict[str, list[np.ndarray]],
        held: np.ndarray | dict[str, np.ndarray] | None = None,
        weights: dict[int, torch.Tensor] | None = None,
    ) -> None:
        """``held``: the rows each sequence's cache holds before this token,
        where rows were evicted (:meth:`KVCache.evict`) and it is no longer the
        token's position; by group name in a cache of several groups, of which
        those not named hold a row for every position. ``weights``: per layer
        float32 ``[batch, kv_heads, capacity]``, to which the step's attention
        weights are added in place (the new token's entry starts from them);
        the capacity holds every sequence with its new token.
        ``lengths`` and ``longest`` are those of the groups without evictions, or
        of the only group."""
        device = cache.device
        self.weights = weights or {}
        self.cache = cache
        self.tokens = tokens
        self.count = int(tokens.shape[0])
        positions = np.asarray(positions).astype(np.int64)
        self.offsets = torch.as_tensor(positions.astype(np.int32), device=device)
        by_group = {} if held is None else rows_by_group(cache, held, (self.count,))
        if len(cache.groups) == 1:
            positions = by_group.get(next(iter(cache.groups)), positions)
        put = lambda n: torch.as_tensor((n + 1).astype(np.int32), device=device)  # noqa: E731
        self.lengths = put(positions)
        self.longest = int(positions.max()) + 1
        page = cache.page_size
        self._lengths: dict[str, torch.Tensor] = {}
        self._longest: dict[str, int] = {}
        self._write: dict[str, torch.Tensor] = {}
        self._tables: dict[str, torch.Tensor] = {}
        for name in cache.groups:
            at = by_group.get(name, positions)
            past = at // page >= np.array([len(table) for table in tables[name]])
            if np.any(past):
                b = int(np.argmax(past))
                raise ValueError(f"group {name!r}: no page for row {at[b]} of sequence {b}")
            self._lengths[name] = self.lengths if at is positions else put(at)
            self._longest[name] = int(at.max()) + 1
            packed = pack_tables(tables[name], self.count)
            pages = packed[np.arange(self.count), at // page]
            rows = (pages.astype(np.int64) * page + at % page).astype(np.int32)
            self._write[name] = torch.as_tensor(rows, device=device)
            self._tables[name] = torch.as_tensor(packed, device=device)
        for layer, w in self.weights.items():
            group = cache.layer_group.get(layer)
            if group is None or w.shape[-1] < self._longest[group.name]:
                raise ValueError(f"weights of layer {layer} must hold its longest sequence")

    @property
    def positions(self) -> torch.Tensor:
        return self.offsets

    def rope(self, x: torch.Tensor, dims: int, *, base: float | None = None,
             freqs: Any = None) -> torch.Tensor:
        """Rotary embedding of ``[batch, heads, head_dim]`` at each
        sequence's position (batches.py:195-201, portable.py:88-132)."""
        return rope(x.to(self.cache.dtype).contiguous(), self.offsets, dims, base=base,
                    freqs=freqs)

    def rope_attend(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                    dims: int, scale: float, base: float | None = None, freqs: Any = None,
                    softcap: float = 0.0) -> torch.Tensor:
        """``attend(layer, rope(q), rope(k), v)`` with the rotation of q and k
        and the K/V write in one launch (the model calls of
        backends/dense.py:99-102 and DecodeBatch.attend, batches.py:203-226).
        A bf16 model over an 8-bit cache takes the three steps apart: its
        rotated keys are rounded to bf16 before they are quantized, as the
        reference's are, while the fused 8-bit write rounds them to fp16."""
        group = self.cache.layer_group[layer]
        cache = self.cache
        dtype = cache.compute_dtype
        if dtype != cache.dtype:
            rot = dict(base=base, freqs=freqs)
            return self.attend(layer, self.rope(q, dims, **rot), self.rope(k, dims, **rot), v,
                               scale=scale, softcap=softcap)
        q_rot = rope_append(q.to(dtype).contiguous(), k.to(dtype).contiguous(),
                            v.to(dtype).contiguous(), cache.keys[layer],
                            cache.values[layer], self.offsets, self._write[group.name],
                            page_size=cache.page_size, dims=dims, base=base, freqs=freqs,
                            scales=cache.scales(layer))
        return self._attend_written(layer, q_rot, scale=scale, softcap=softcap)

    def attend(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
               scale: float, softcap: float = 0.0) -> torch.Tensor:
        """Write this step's K/V, then paged decode attention
        (batches.py:203-226). ``q`` is ``[batch, q_heads, head_dim]``; ``k``,
        ``v`` are ``[batch, kv_heads, head_dim]``."""
        group = self.cache.layer_group[layer]
        self.cache.write(layer, self._write[group.name], k, v)
        return self._attend_written(layer, q, scale=scale, softcap=softcap)

    def _attend_written(self, layer: int, q: torch.Tensor, *, scale: float,
                        softcap: float) -> torch.Tensor:
        group = self.cache.layer_group[layer]
        q = q.to(self.cache.decode_dtype).contiguous()
        if layer in self.weights:
            paged_attention_weights(
                q, self.cache.keys[layer], self._tables[group.name], self._lengths[group.name],
                self.weights[layer], page_size=self.cache.page_size,
                longest=self._longest[group.name], scale=scale, window=group.window,
                softcap=softcap,
                scales=self.cache.scales(layer))
        out = paged_decode_attention(
            q,
            self.cache.keys[layer],
            self.cache.values[layer],
            self._tables[group.name],
            self._lengths[group.name],
            page_size=self.cache.page_size,
            longest=self._longest[group.name],
            scale=scale,
            window=group.window,
            softcap=softcap,
            scales=self.cache.scales(layer),
        )
        return out.reshape(self.count, -1).to(self.cache.dtype)


class PrefillBatch:
    """A chunk of one sequence's prompt (batches.py:26-132): positions
    ``start .. start + count - 1``, the chunk's K/V written to the cache
    first, then causal attention over the sequence's pages on the GPU
    (``pda_paged_prefill_attention``, ``_q8`` for an 8-bit cache),
    ``[count, q_heads * head_dim]`` out. ``images``: (at, embeddings) as the
    reference takes them (or (at, length)); their tokens also see the rest of
    their image (batches.py:107-118)."""

    prefill = True

    def __init__(self, cache: KVCache, tokens: torch.Tensor, *, start: int,
                 tables: dict[str, np.ndarray], images: Any = (),
                 held: int | dict[str, int] | None = None) -> None:
        """``held``: the rows that the sequence's cache holds before the chunk,
        where rows were evicted and it is no longer ``start``; by group name as
        for :class:`DecodeBatch`. The chunk is rotated at its positions and
        written behind the rows held, all of which it sees."""
        device = cache.device
        self.cache = cache
        self.tokens = tokens
        self.count = int(tokens.shape[0])
        self.start = int(start)
        self.images = list(images)
        end = self.start + self.count
        rows = {} if held is None else rows_by_group(cache, held, ())
        # First row of the chunk in each group.
        self._starts = {name: int(rows.get(name, self.start)) for name in cache.groups}
        if self.images and set(self._starts.values()) != {self.start}:
            raise ValueError("images need a cache from which no rows were evicted")
        self._spans = image_spans(
            [(at, x if isinstance(x, int) else int(x.shape[0])) for at, x in self.images], device)
        self.offsets = torch.arange(self.start, end, dtype=torch.int32, device=device)
        self._write: dict[str, torch.Tensor] = {}
        self._tables: dict[str, torch.Tensor] = {}
        for name, first in self._starts.items():
            table = np.asarray(tables[name])
            self._write[name] = torch.as_tensor(cache.rows(table, first, first + self.count),
                                                device=device)
            self._tables[name] = torch.as_tensor(table.astype(np.int32), device=device)

    @property
    def positions(self) -> torch.Tensor:
        return self.offsets

    def inject(self, x: torch.Tensor) -> torch.Tensor:
        """Put image embeddings in place of their placeholder tokens
        (batches.py:63-68)."""
        for at, embeddings in self.images:
            if isinstance(embeddings, int):
                continue
            offset = at - self.start
            x[offset:offset + int(embeddings.shape[0])] = embeddings.to(x.dtype)
        return x

    def rope(self, x: torch.Tensor, dims: int, *, base: float | None = None,
             freqs: Any = None) -> torch.Tensor:
        """Rotate ``[tokens, heads, head_dim]`` at the chunk's positions
        (batches.py:70-81)."""
        return rope(x.to(self.cache.dtype).contiguous(), self.offsets, dims, base=base,
                    freqs=freqs)

    def attend(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
               scale: float, softcap: float = 0.0) -> torch.Tensor:
        """Write the chunk's K/V (quantized in an 8-bit cache), then its
        attention over the dequantized rows (batches.py:84-132,
        paged_kv.py:285-292)."""
        group = self.cache.layer_group[layer]
        self.cache.write(layer, self._write[group.name], k, v)
        out = paged_prefill_attention(
            q.to(self.cache.compute_dtype).contiguous(), self.cache.keys[layer],
            self.cache.values[layer],
            self._tables[group.name], start=self._starts[group.name],
            page_size=self.cache.page_size,
            scale=scale, window=group.window, softcap=softcap,
            scales=self.cache.scales(layer),
            images=self._spans if self._spans is not None else ())
        return out.reshape(self.count, -1).to(self.cache.dtype)
