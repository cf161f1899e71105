"""Float64 restatement of latent attention on the CPU (test infrastructure).

Written from the definitions, every head's keys and values projected out
(expanded form): key(t) = [U_h c_t ; k_t], value(t) = D_h c_t, softmax of
scale * q . key over the keys a query sees. Beside the result each attention
function returns a bound of the error that a 16-bit computation of it may
have, element by element.
"""

from __future__ import annotations

import numpy as np
import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def rows_of(table, page_size: int, n: int, arena_rows: int):
    """Arena rows of positions 0 .. n - 1; -1 where the page is negative, not in
    the arena or past the table."""
    at = np.arange(n)
    page = at // page_size
    table = np.asarray(table, dtype=np.int64)
    ids = np.where(page < len(table), table[np.minimum(page, max(len(table) - 1, 0))], -1)
    good = (ids >= 0) & (ids < arena_rows // page_size)
    return np.where(good, ids * page_size + at % page_size, -1)


def _attend(q, arena, kv_b, rows, scale):
    """One query [heads, nope + rope] over given rows: (out, spread, off, terms),
    all [heads, value]: spread = sum of p (1 + A) |v - out|, with A the sum of
    the magnitudes in the latent part of the score; off = sum of |v - out|;
    terms = |D_h| times the weighted |latents|, the size of what the output is
    summed from."""
    heads, width, latent = kv_b.shape
    rope = arena.shape[1] - latent
    nope = q.shape[1] - rope
    value = width - nope
    zeros = torch.zeros((heads, value), dtype=torch.float64)
    rows = rows[rows >= 0]
    if len(rows) == 0:
        return zeros, zeros, zeros, zeros
    x = arena[torch.as_tensor(rows)].double()
    c, k = x[:, :latent], x[:, latent:]
    q, w = q.double(), kv_b.double()
    keys = torch.einsum("hdl,tl->htd", w[:, :nope], c)
    values = torch.einsum("hdl,tl->htd", w[:, nope:], c)
    s = scale * (torch.einsum("hd,htd->ht", q[:, :nope], keys) + q[:, nope:] @ k.t())
    p = torch.softmax(s, dim=-1)
    out = torch.einsum("ht,htd->hd", p, values)
    q_lat = torch.einsum("hd,hdl->hl", q[:, :nope], w[:, :nope])
    a = abs(scale) * (q_lat.abs() @ c.abs().t())
    off = (values - out[:, None]).abs()
    terms = torch.einsum("hdl,hl->hd", w[:, nope:].abs(), p @ c.abs())
    return out, torch.einsum("ht,htd->hd", p * (1 + a), off), off.sum(1), terms


def decode(q, arena, kv_b, tables, lengths, *, page_size, scale):
    """(out, bound) of the decode call, [batch, heads, value] float64.

    The bound, with u half a step of the type: the output's rounding u |out|;
    the weights' u p and the absorbed queries' (scores off by u A at most), both
    to first order in u, each times |v - out| since the weights' sum has the
    same errors; a fp16 weight below the normal range is off by half its
    smallest step, 2^-25, instead. 1.1 for the second order (u A is below 0.1
    where this is used) and 2e-5 for the scores' and weights' float32 steps.
    Sums in float32 are off by 2^-24 a step of the size of their terms, which
    may cancel: n keys and 512 latent dims go 16 at a time, so n / 16 + 16 and
    32 + 16 steps; the joined latents are two 16-bit numbers, off by u^2."""
    u = HALF_STEP[q.dtype]
    out, bound = [], []
    for b in range(q.shape[0]):
        n = min(max(int(lengths[b]), 0), len(tables[b]) * page_size)
        rows = rows_of(tables[b], page_size, n, arena.shape[0])
        o, spread, off, terms = _attend(q[b], arena, kv_b, rows, scale)
        out.append(o)
        tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
        bound.append(1.1 * u * (o.abs() + spread) + tiny * (1 + off) + 2e-5 * (o.abs() + spread)
                     + ((n / 16 + 64) * 2.0 ** -24 + u * u) * terms)
    return torch.stack(out), torch.stack(bound)


def append(q, latent, k_rope, arena, positions, rows, *, inv_freq, norm_weight, eps):
    """(rotated queries, arena) in float64; ``inv_freq`` None: no rotation."""
    def turn(x):
        if inv_freq is None:
            return x.double()
        half = x.shape[-1] // 2
        angle = (positions.numpy().astype(np.float32)[:, None]
                 * inv_freq.numpy().astype(np.float32)).astype(np.float64)
        shape = (x.shape[0],) + (1,) * (x.dim() - 2) + (half,)
        c, s = torch.as_tensor(np.cos(angle)).view(shape), torch.as_tensor(np.sin(angle)).view(shape)
        a, b = x[..., :half].double(), x[..., half:].double()
        return torch.cat([a * c - b * s, b * c + a * s], dim=-1)

    c = latent.double()
    if norm_weight is not None:
        c = c / torch.sqrt((c * c).mean(-1, keepdim=True) + eps) * norm_weight.double()
    new = torch.cat([c, turn(k_rope)], dim=-1)
    arena = arena.double()
    for i, row in enumerate(rows.tolist()):
        if 0 <= row < arena.shape[0]:
            arena[row] = new[i]
    if q is None:
        return None, arena
    rope = k_rope.shape[1]
    q = q.double()
    if rope:
        q = torch.cat([q[..., :-rope], turn(q[..., -rope:])], dim=-1)
    return q, arena


def prefill(q, arena, kv_b, table, *, start, page_size, scale):
    """(out, bound) of the prefill call, [count, heads, value] float64.

    The bound, with u half a step of the type: the output's rounding u |out|;
    the weights' u p and the keys' (scores off by u A, A = scale * |q| . |key|),
    to first order, each times |v - out|; the values' u p |v|; a fp16 weight
    below the normal range by half its smallest step. 1.1, 2e-5 and 2^-24 a step
    of the terms' size as for the decode call; the keys' and values' own sums
    over 512 latent dims take 32 + 16 steps of the size of |U_h| |c|, |D_h| |c|."""
    u = HALF_STEP[q.dtype]
    heads, width, latent = kv_b.shape
    count = q.shape[0]
    rope = arena.shape[1] - latent
    nope = q.shape[2] - rope
    end = start + count
    rows = rows_of(table, page_size, end, arena.shape[0])
    good = torch.as_tensor(rows >= 0)
    x = arena[torch.as_tensor(np.maximum(rows, 0))].double()
    x[~good] = 0.0
    c, k = x[:, :latent], x[:, latent:]
    hidden = (torch.arange(end)[None] > start + torch.arange(count)[:, None]) | ~good[None]
    none = hidden.all(-1)
    out = torch.zeros((count, heads, width - nope), dtype=torch.float64)
    bound = torch.zeros_like(out)
    step = 48 * 2.0 ** -24
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    for h in range(heads):
        w = kv_b[h].double()
        key, v = c @ w[:nope].t(), c @ w[nope:].t()
        key_terms, v_terms = c.abs() @ w[:nope].abs().t(), c.abs() @ w[nope:].abs().t()
        qh = q[:, h].double()
        s = scale * (qh[:, :nope] @ key.t() + qh[:, nope:] @ k.t())
        p = torch.softmax(s.masked_fill(hidden, -np.inf), dim=-1)
        p[none] = 0.0
        a = abs(scale) * (qh[:, :nope].abs() @ key.abs().t())
        b = abs(scale) * (qh[:, :nope].abs() @ key_terms.t()) * step
        o = p @ v
        part = max(1, (1 << 24) // (end * (width - nope)))
        for i in range(0, count, part):
            z = slice(i, min(i + part, count))
            off = (v[None] - o[z, None]).abs()  # [queries, keys, value]
            weigh = lambda x, off=off: torch.matmul(x[:, None], off)[:, 0]  # noqa: E731
            spread = weigh(p[z] * (1 + a[z]))
            bound[z, h] = (1.1 * u * (o[z].abs() + spread + p[z] @ v.abs())
                           + 1.1 * weigh(p[z] * b[z]) + step * (p[z] @ v_terms)
                           + (end / 16 + 64) * 2.0 ** -24 * (p[z] @ v.abs())
                           + tiny * (1 + weigh((~hidden[z]).double()))
                           + 2e-5 * (o[z].abs() + spread))
        out[:, h] = o
    return out, bound
