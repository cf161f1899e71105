"""Float64 restatement of the accumulated attention weights and of the eviction
that follows them, on the CPU (test infrastructure)."""

from __future__ import annotations

import numpy as np
import torch

from .latent import rows_of


def rows_view(arena, page_size, layout):
    """[rows, kv_heads, ..] copy of an arena in either layout."""
    if layout == "rows":
        return arena.clone()
    return arena.transpose(1, 2).reshape(-1, arena.shape[1], *arena.shape[3:])


def weights(q, keys, tables, lengths, old, *, page_size, layout, scale, window=0, softcap=0.0,
            key_scales=None, fresh=1):
    """(out, bound): [batch, kv_heads, capacity] float64.

    The bound: a score is summed in float32 over the head dim, 32 products at a
    time, and scaled: (D / 32 + 36) 2^-24 of its terms' size, and with softcap
    or without a few 2^-23 of its own; a weight is off by as much relatively,
    twice (its own score and the sum's), plus 2^-21 for the exponentials, the
    chunk factors and the sums; the output adds one rounding."""
    rows = rows_view(keys, page_size, layout).double()
    if key_scales is not None:
        rows = rows * rows_view(key_scales, page_size, layout).double()[..., None]
    kv_heads, dim = rows.shape[1:]
    group = q.shape[1] // kv_heads
    out = old.double().clone()
    bound = torch.zeros_like(out)
    for b in range(q.shape[0]):
        n = min(max(int(lengths[b]), 0), len(tables[b]) * page_size, old.shape[2])
        at = rows_of(tables[b], page_size, n, rows.shape[0])
        if window:
            at[:max(0, n - window)] = -1
        good = torch.as_tensor(at >= 0)
        k = rows[torch.as_tensor(np.maximum(at, 0))]
        k[~good] = 0.0
        for j in range(kv_heads):
            x = q[b, j * group:(j + 1) * group].double()
            s = scale * (x @ k[:, j].t())
            err = abs(scale) * (x.abs() @ k[:, j].abs().t()) * (dim / 32 + 36) * 2.0 ** -24
            if softcap:
                s = softcap * torch.tanh(s / softcap)
                err = err + 8 * 2.0 ** -23 * softcap
            err = err + 4 * 2.0 ** -23 * s.abs()
            s[:, ~good] = -np.inf
            p = torch.softmax(s, dim=-1) if bool(good.any()) else torch.zeros_like(s)
            worst = err[:, good].amax(-1, keepdim=True) if bool(good.any()) else err[:, :0].sum()
            credit = p.sum(0)
            base = out[b, j, :n].clone()
            base[max(0, n - fresh):] = 0.0
            out[b, j, :n] = base + credit
            bound[b, j, :n] = (p * (err + worst + 2.0 ** -21)).sum(0) + 2.0 ** -24 * (base + credit)
    return out, 1.01 * bound + 1e-30


def select(w, tables, lengths, *, page_size, arena_rows, keep, recent, sinks):
    """(kept [batch, kv_heads, keep] with -1 padding, lengths): the rule itself,
    by ranking every position."""
    w = np.asarray(w, dtype=np.float64)
    batch, kv_heads, capacity = w.shape
    kept = np.full((batch, kv_heads, keep), -1, dtype=np.int32)
    new = np.zeros(batch, dtype=np.int32)
    for b in range(batch):
        n = min(max(int(lengths[b]), 0), len(tables[b]) * page_size, capacity)
        held = rows_of(tables[b], page_size, n, arena_rows) >= 0
        for j in range(kv_heads):
            rank = []
            for t in range(n):
                if held[t]:
                    guard = t < sinks or t >= n - recent
                    x = w[b, j, t]
                    # Heaviest first; NaN below everything, -0 as 0.
                    rank.append((not guard, bool(np.isnan(x)), 0.0 if np.isnan(x) else -x + 0.0, t))
            pick = sorted(t for *_, t in sorted(rank)[:keep])
            kept[b, j, :len(pick)] = pick
            new[b] = len(pick)
    return kept, new


def move(arena, kept, tables, out_tables, *, page_size, layout):
    """The arena with every kept row copied to its place."""
    src = arena.clone()
    dst = arena.clone()
    pages = arena.shape[0] // page_size if layout == "rows" else arena.shape[0]

    def cell(t, table, j):
        page = int(table[t // page_size]) if t // page_size < len(table) else -1
        if not 0 <= page < pages:
            return None
        return (page * page_size + t % page_size, j) if layout == "rows" else (page, j, t % page_size)

    for b in range(kept.shape[0]):
        for j in range(kept.shape[1]):
            for i, t in enumerate(kept[b, j].tolist()):
                if t >= 0:
                    a, z = cell(t, tables[b], j), cell(i, out_tables[b], j)
                    if a is not None and z is not None:
                        dst[z] = src[a]
    return dst
