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

from .drafts import NODES, Committed, commit_drafts, tree_attention
from .eviction import paged_attention_weights
from .hip_kernels import (image_spans, paged_decode_attention, paged_prefill_attention, rope,
                          rope_append)
from .paged_kv import KVCache
from .paging import StepRows, extend_tables
from .prompts import packed_prompt_attention


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


class _ManyTokens:
    """What steps that bring several tokens of several sequences have in common: the
    rows of the new tokens in every group, made on the GPU, and the calls that write
    them. ``held``: rows of each sequence before the step, by group."""

    prefill = True

    def _place(self, cache: KVCache, counts: np.ndarray, held: dict[str, np.ndarray],
               tables: dict[str, list[np.ndarray]], parents: torch.Tensor | None,
               tokens: int) -> None:
        device, page = cache.device, cache.page_size
        for name, group in cache.groups.items():  # (before any layer's K/V are written)
            if group.head_dim % 8 or group.head_dim > 256:
                raise ValueError(f"group {name!r}: steps of many tokens a sequence serve head dims "
                                 f"that are multiples of 8 up to 256, not {group.head_dim}")
        pages = {name: np.array([len(t) for t in tables[name]], dtype=np.int64)
                 for name in cache.groups}
        for name, have in pages.items():
            if have.shape != counts.shape:
                raise ValueError(f"group {name!r}: a table for each sequence")
            short = (-(-(held[name] + counts) // page) > have) & (counts > 0)
            if np.any(short):
                b = int(np.argmax(short))
                raise ValueError(f"group {name!r}: no page for row {held[name][b] + counts[b] - 1} "
                                 f"of sequence {b}")
            for b in np.flatnonzero(counts):
                first = int(held[name][b]) // page
                new = np.asarray(tables[name][b])[first:-(-int(held[name][b] + counts[b]) // page)]
                if np.any(new < 0):
                    row = max(int(held[name][b]), (first + int(np.argmax(new < 0))) * page)
                    raise ValueError(f"group {name!r}: no page for row {row} of sequence {b}")
        put = lambda a: torch.as_tensor(np.asarray(a).astype(np.int32), device=device)  # noqa: E731
        self._tables: dict[str, torch.Tensor] = {}
        self._held: dict[str, torch.Tensor] = {}
        self._steps: dict[str, StepRows] = {}
        none, drawn = put([]), put([0, 0])
        for name, have in pages.items():
            packed = pack_tables(tables[name], len(counts)) if len(counts) else np.zeros((0, 1))
            self._tables[name], self._held[name] = put(packed), put(held[name])
            self._steps[name] = extend_tables(
                self._tables[name], self._held[name], put(counts), put(have), none, drawn,
                page_size=page, tokens=tokens, parents=parents)

    @property
    def positions(self) -> torch.Tensor:
        return self.offsets

    def rope(self, x: torch.Tensor, dims: int, *, base: float | None = None,
             freqs: Any = None) -> torch.Tensor:
        """Rotate ``[tokens, heads, head_dim]`` at the tokens' positions
        (batches.py:70-81)."""
        return rope(x.to(self.cache.dtype).contiguous(), self.offsets, dims, base=base,
                    freqs=freqs)

    def _check_queries(self, layer: int, q: torch.Tensor) -> None:
        group = self.cache.layer_group[layer]
        if (q.dim() != 3 or q.shape[0] != self.count or q.shape[2] != group.head_dim
                or q.shape[1] == 0 or q.shape[1] % group.kv_heads):
            raise ValueError(f"q must be [{self.count}, a multiple of {group.kv_heads}, "
                             f"{group.head_dim}], got {list(q.shape)}")

    def _write(self, layer: int, k: torch.Tensor, v: torch.Tensor) -> str:
        group = self.cache.layer_group[layer]
        self.cache.write(layer, self._steps[group.name].rows, k, v)
        return group.name


class PackedPrefillBatch(_ManyTokens):
    """Whole prompts of several sequences in one step: ``tokens`` holds them one behind
    the other, ``counts[b]`` of sequence b, which holds nothing yet. Their keys and
    values go to the cache, and every prompt attends to itself as it was projected (in
    an 8-bit cache too: what later steps read is rounded, what the prompt sees is not).
    ``tables``: per group the pages of each sequence. Outputs ``[tokens, q_heads *
    head_dim]``; ``ends`` are the rows of the prompts' last tokens. The reference
    prefills one sequence a step (``PrefillBatch``, batches.py:26-132)."""

    def __init__(self, cache: KVCache, tokens: torch.Tensor, *, counts: np.ndarray,
                 tables: dict[str, list[np.ndarray]]) -> None:
        counts = np.asarray(counts).astype(np.int64)
        if counts.ndim != 1 or np.any(counts < 0) or int(counts.sum()) != int(tokens.shape[0]):
            raise ValueError("counts must be the tokens of each prompt")
        self.cache, self.tokens, self.count = cache, tokens, int(tokens.shape[0])
        zero = np.zeros_like(counts)
        self._place(cache, counts, dict.fromkeys(cache.groups, zero), tables, None, self.count)
        step = next(iter(self._steps.values()))
        self.offsets, self.starts = step.positions, step.starts
        self.ends = torch.as_tensor(np.cumsum(counts)[counts > 0] - 1, device=cache.device)

    def attend(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
               scale: float, softcap: float = 0.0) -> torch.Tensor:
        """Write the prompts' K/V, then their attention. ``q`` ``[tokens, q_heads,
        head_dim]``, ``k`` and ``v`` ``[tokens, kv_heads, head_dim]``; slices of one
        projection are read where they are."""
        self._check_queries(layer, q)
        self._write(layer, k, v)
        dtype = self.cache.dtype
        out = packed_prompt_attention(
            q.to(dtype), k.to(dtype), v.to(dtype), self.starts, scale=scale,
            window=self.cache.layer_group[layer].window, softcap=softcap)
        return out.reshape(self.count, -1)


class DraftBatch(_ManyTokens):
    """A step that verifies a tree of drafted tokens for every sequence: ``tokens``
    holds the trees one behind the other, ``counts[b]`` nodes (up to 64) of sequence b,
    node 0 its newest token, and ``parents`` each node's parent among its sequence's
    nodes (-1: none). ``positions``: of each sequence's node 0. ``held``: the rows held
    before the step where rows were evicted, as for :class:`DecodeBatch`. ``tables``:
    per group the pages of each sequence, with room for all nodes. After the layers,
    :meth:`commit` keeps the nodes that the model agrees with. No counterpart in the
    reference."""

    def __init__(self, cache: KVCache, tokens: torch.Tensor, *, counts: np.ndarray,
                 parents: np.ndarray, positions: np.ndarray,
                 tables: dict[str, list[np.ndarray]],
                 held: np.ndarray | dict[str, np.ndarray] | None = None) -> None:
        counts = np.asarray(counts).astype(np.int64)
        parents = np.asarray(parents).astype(np.int64)
        positions = np.asarray(positions).astype(np.int64)
        if counts.ndim != 1 or np.any(counts < 0) or int(counts.sum()) != int(tokens.shape[0]):
            raise ValueError("counts must be the nodes of each tree")
        if np.any(counts > NODES):
            raise ValueError(f"a tree holds up to {NODES} nodes")
        if positions.shape != counts.shape or np.any(positions < 0):
            raise ValueError("positions must be those of each sequence's first node")
        index = np.arange(len(tokens)) - np.repeat(np.cumsum(counts) - counts, counts)
        if parents.shape != index.shape or np.any((parents < -1) | (parents >= index)):
            raise ValueError("a node's parent is an earlier node of its tree, or -1")
        self.cache, self.tokens, self.count = cache, tokens, int(tokens.shape[0])
        self._moved: set[int] = set()  # layers committed since they were written
        rows = {} if held is None else rows_by_group(cache, held, counts.shape)
        for name, n in rows.items():
            if cache.groups[name].window and np.any(n != positions):
                raise ValueError("a windowed group releases its pages by position")
        self.parents = torch.as_tensor(parents.astype(np.int32), device=cache.device)
        self._place(cache, counts, {name: rows.get(name, positions) for name in cache.groups},
                    tables, self.parents, self.count)
        name, step = next(iter(self._steps.items()))
        self.starts, self.masks, self.offsets = step.starts, step.masks, step.positions
        if name in rows:  # (positions count on where rows were evicted)
            ahead = np.repeat(positions - rows[name], counts).astype(np.int32)
            self.offsets = self.offsets + torch.as_tensor(ahead, device=cache.device)

    def attend(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
               scale: float, softcap: float = 0.0) -> torch.Tensor:
        """Write the nodes' K/V behind the rows held, then attention over those and the
        nodes' ancestors, ``[tokens, q_heads * head_dim]``."""
        self._check_queries(layer, q)
        name = self._write(layer, k, v)
        self._moved.discard(layer)
        cache = self.cache
        out = tree_attention(
            q.to(cache.decode_dtype).contiguous(), cache.keys[layer], cache.values[layer],
            self._tables[name], self._held[name], self.starts, self.masks,
            page_size=cache.page_size, scale=scale, window=cache.groups[name].window,
            softcap=softcap, scales=cache.scales(layer))
        return out.reshape(self.count, -1).to(cache.dtype)

    def commit(self, targets: torch.Tensor) -> dict[str, Committed]:
        """Keep each tree's line of nodes that the model agrees with: ``targets`` is its
        choice after every node, of the tokens' type. Moves the kept rows in every
        layer; returns what was kept by group (the same but for ``lengths``, the rows
        held now). The sequences' pages stay theirs. Rows that have moved do not move
        again: a step is committed once, or once more when every layer was attended
        again."""
        if self._moved:
            raise RuntimeError(f"the rows of layers {sorted(self._moved)} have moved already")
        done = {}
        for name, group in self.cache.groups.items():
            arenas = [(self.cache.keys[i], self.cache.values[i], *(self.cache.scales(i) or ()))
                      for i in group.layers]
            done[name] = commit_drafts(
                arenas, self._tables[name], self._held[name], self.starts, self.parents,
                self.tokens.to(self.cache.device), targets, page_size=self.cache.page_size)
            self._moved.update(group.layers)
        return done
