"""Plain restatements, on the CPU and in 64 bits, of the calls of a step that takes
many tokens of every sequence: page tables and slot maps, attention of packed prompts
and of drafted trees, and the commitment of accepted nodes. Test infrastructure."""

import numpy as np

NODES = 64


def ancestors(parents):
    """Mask of every node of one tree (Python integers), 0 past the 64th."""
    masks = []
    for i, parent in enumerate(parents):
        up = masks[parent] if 0 <= parent < i else 0
        masks.append(up | 1 << i if i < NODES else 0)
    return masks


def extend_tables(tables, lengths, counts, pages, feed, drawn, *, page_size, tokens,
                  parents=None):
    """The arrays of ``paging.extend_tables`` as a dict (``tables`` among them)."""
    tables = np.array(tables, dtype=np.int64)
    width = tables.shape[1]
    starts, out_lengths, out_pages = [0], [], []
    rows, positions, masks = [-1] * tokens, [0] * tokens, [0] * tokens
    taken = int(drawn[0])
    for b, (held, n, have) in enumerate(zip(lengths, counts, pages)):
        held, have = max(0, int(held)), min(max(0, int(have)), width)
        first = starts[-1]
        n = min(max(0, int(n)), tokens - first)
        if n:
            need = min(-(-(held + n) // page_size), width)
            while have < need:
                tables[b, have] = feed[taken] if 0 <= taken < len(feed) else -1
                have, taken = have + 1, taken + 1
        tree = None if parents is None else ancestors([int(x) for x in parents[first:first + n]])
        for i in range(n):
            j = (held + i) // page_size
            page = tables[b, j] if j < have else -1
            row = page * page_size + (held + i) % page_size
            rows[first + i] = int(row) if page >= 0 and row < 1 << 31 else -1
            positions[first + i] = held + i
            if tree is not None:
                masks[first + i] = tree[i]
                positions[first + i] = held + max(0, bin(tree[i]).count("1") - 1)
        starts.append(first + n)
        out_lengths.append(held + n)
        out_pages.append(have)
    return dict(tables=tables, starts=np.array(starts), lengths=np.array(out_lengths),
                pages=np.array(out_pages), drawn=np.array([taken, 0]), rows=np.array(rows),
                positions=np.array(positions), masks=np.array(masks, dtype=np.uint64))


def _attend(q, k, v, keep, scale, softcap):
    """One head: outputs, and the weighted sum of absolute values (for tolerances)."""
    s = q @ k.T * scale
    if softcap > 0:
        s = softcap * np.tanh(s / softcap)
    s = np.where(keep, s, -np.inf)
    top = s.max(axis=-1, keepdims=True, initial=-np.inf)
    with np.errstate(invalid="ignore"):
        w = np.exp(s - np.where(top == -np.inf, 0.0, top))
    total = w.sum(axis=-1, keepdims=True)
    p = np.divide(w, total, out=np.zeros_like(w), where=total != 0)
    # (Hidden values take no part, whatever they are.)
    out = np.zeros((q.shape[0], v.shape[1]))
    size = np.zeros_like(out)
    for i in range(q.shape[0]):
        seen = keep[i]
        out[i] = p[i, seen] @ v[seen]
        size[i] = p[i, seen] @ np.abs(v[seen])
    return out, size


def packed_prompts(q, k, v, starts, *, scale, window=0, softcap=0.0):
    """[tokens, q_heads, D] float64 outputs and sums of weighted absolute values;
    zeros in rows of no prompt."""
    q, k, v = (np.asarray(x, dtype=np.float64) for x in (q, k, v))
    group = q.shape[1] // k.shape[1]
    out, size = np.zeros_like(q), np.zeros_like(q)
    for a, z in zip(starts, starts[1:]):
        at = np.arange(z - a)
        keep = at[None] <= at[:, None]
        if window:
            keep &= at[None] > at[:, None] - window
        for h in range(q.shape[1]):
            out[a:z, h], size[a:z, h] = _attend(q[a:z, h], k[a:z, h // group], v[a:z, h // group],
                                                keep, scale, softcap)
    return out, size


def trees(q, keys, values, tables, lengths, starts, masks, *, page_size, scale, window=0,
          softcap=0.0):
    """As ``packed_prompts`` for ``drafts.tree_attention``; ``keys``/``values`` float64
    ``[rows, kv_heads, D]`` (dequantized). ``masks``: unsigned."""
    q = np.asarray(q, dtype=np.float64)
    pages = keys.shape[0] // page_size
    group = q.shape[1] // keys.shape[1]
    out, size = np.zeros_like(q), np.zeros_like(q)
    for b, held in enumerate(lengths):
        a, z = int(starts[b]), int(starts[b + 1])
        n, held = z - a, int(held)
        end = held + min(n, NODES)
        at = np.arange(end)
        page = np.array([tables[b][j] if j < len(tables[b]) else -1 for j in at // page_size],
                        dtype=np.int64).reshape(-1)
        usable = (page >= 0) & (page < pages)
        rows = np.where(usable, page, 0) * page_size + at % page_size
        keep = np.zeros((n, end), dtype=bool)
        for i in range(n):
            line = [j for j in range(min(n, NODES)) if int(masks[a + i]) >> j & 1]
            bits = bin(int(masks[a + i])).count("1")
            first = max(0, held + max(0, bits - 1) - window + 1) if window else 0
            keep[i, min(first, held):held] = True
            if window and bits > window:  # the last of the mask's bits, whether nodes or not
                all_bits = [j for j in range(NODES) if int(masks[a + i]) >> j & 1][-window:]
                line = [j for j in line if j in all_bits]
            keep[i, [held + j for j in line]] = True
        keep &= usable[None]
        for h in range(q.shape[1]):
            out[a:z, h], size[a:z, h] = _attend(q[a:z, h], keys[rows, h // group],
                                                values[rows, h // group], keep, scale, softcap)
    return out, size


def commit(lengths, starts, parents, drafted, targets):
    """(lengths, accepted, path, following) of ``drafts.commit_drafts``."""
    out_lengths, accepted, paths, following = [], [], [], []
    for b, held in enumerate(lengths):
        a = int(starts[b])
        n = min(int(starts[b + 1]) - a, NODES)
        path = [0] if n else []
        while path:
            last = path[-1]
            fits = [i for i in range(last + 1, n)
                    if parents[a + i] == last and drafted[a + i] == targets[a + last]]
            if not fits:
                break
            path.append(fits[0])
        out_lengths.append(int(held) + len(path))
        accepted.append(len(path))
        paths.append(path + [-1] * (NODES - len(path)))
        following.append(int(targets[a + path[-1]]) if path else -1)
    return (np.array(out_lengths), np.array(accepted), np.array(paths).reshape(-1, NODES),
            np.array(following))


def half_step(dtype):
    """Largest relative error of one rounding to a 16-bit type (by its name)."""
    return 2.0 ** -8 if "bfloat16" in str(dtype) else 2.0 ** -11


def attention_tolerance(out, size, values, keys_seen, dtype, dequantized=False):
    """How far attention in these kernels may be from 64 bits, element by element.

    Weights are rounded to the element type (u, relative) and divided by the sum of
    the rounded ones: u (sum p |v| + |o|). The output is rounded once: u |o|. 8-bit
    values are rounded once when their scale is taken: u sum p |v|. Scores are sums of
    up to 256 products in float32, times log2 e, capped and exponentiated there: for
    unit-variance inputs |score| stays below 2^4 and its error below 260 * 2^-24 *
    2^4 < 2^-11.9, on both the weight and the sum: 2^-10.9 sum p |v|. fp16 weights
    that are subnormal have an absolute error of at most 2^-25 of the largest each
    (2^-32 where the largest has the weight 2^7)."""
    u = half_step(dtype)
    small = 0.0 if "bfloat16" in str(dtype) else keys_seen * 2.0 ** -25 * np.abs(values).max()
    return (u * (size + 2 * np.abs(out)) + (u * size if dequantized else 0.0)
            + 2.0 ** -10.9 * size + small + 2.0 ** -24)
