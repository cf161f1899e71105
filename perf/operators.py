"""The operators of latent attention and of cache eviction, to be timed and checked.

A model whose attention keeps one latent vector a token calls the library three
times a layer: the append (normalise the latents, rotate, write the rows), the
decode attention of a step over the paged latent rows (absorbed form) and the
prefill attention of a prompt's chunk (expanded form). An engine that bounds its
cache adds two calls over the ordinary paged K/V: the weights that a step's
attention gives every key, accumulated per sequence and kv head, and the
eviction, which keeps the heaviest keys and packs their rows.

``own`` selects the library's calls; without it the same mathematics runs in
elementary torch operations in float32, rounded once at the end. Lengths belong
to a case (a seed of their own draws them), so that its work is known; tables
and all values come from the seed of the preparation.
"""

import math
import sys
from pathlib import Path

import numpy as np
import torch

ROOT = Path(__file__).resolve().parent.parent
if str(ROOT / "llm-inference_amd") not in sys.path:
    sys.path.insert(0, str(ROOT / "llm-inference_amd"))

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
BASE = 1e6

# (query heads, latent width, rotary dims, nope dims, value dims) of a layer.
WIDE = (512, 64, 128, 128)
SMALL = (256, 32, 64, 64)
UNEVEN = (384, 48, 96, 80)


def _named(name, case):
    return dict(case, name=name) if name else case


def _latent(heads, shape):
    latent, rope, nope, value = shape
    return dict(heads=heads, latent=latent, rope=rope, nope=nope, value=value)


def _append(name, heads, shape, *, count, dtype):
    return _named(name, dict(_latent(heads, shape), kind="append", count=count, dtype=dtype))


def _decode(name, heads, shape, *, batch, low, high, dtype, page=16, lengths_seed=1):
    return _named(name, dict(_latent(heads, shape), kind="decode", batch=batch, low=low, high=high,
                             dtype=dtype, page=page, lengths_seed=lengths_seed))


def _prefill(name, heads, shape, *, start, count, dtype, page=16):
    return _named(name, dict(_latent(heads, shape), kind="prefill", start=start, count=count,
                             dtype=dtype, page=page))


def _weights(name, heads, *, batch, low, high, dtype, page=16, layout="pages", window=0,
             softcap=0.0, lengths_seed=1):
    q_heads, kv_heads, head_dim = heads
    return _named(name, dict(kind="weights", q_heads=q_heads, kv_heads=kv_heads,
                             head_dim=head_dim, batch=batch, low=low, high=high, dtype=dtype,
                             page=page, layout=layout, window=window, softcap=softcap,
                             lengths_seed=lengths_seed))


def _evict(name, heads, *, batch, low, high, keep, recent, sinks, dtype, page=16, layout="pages",
           lengths_seed=1):
    _, kv_heads, head_dim = heads
    return _named(name, dict(kind="evict", kv_heads=kv_heads, head_dim=head_dim, batch=batch,
                             low=low, high=high, keep=keep, recent=recent, sinks=sinks,
                             dtype=dtype, page=page, layout=layout, lengths_seed=lengths_seed))


def listed():
    return [
        # The append of a small batch's decode step: the smallest call, all latency.
        _append("append-step", 16, WIDE, count=8, dtype="bf16"),
        # The append of a whole prompt in a layer of 128 heads.
        _append("append-prompt", 128, WIDE, count=4096, dtype="fp16"),
        # One user early in a chat.
        _decode("decode-one-short", 16, WIDE, batch=1, low=777, high=777, dtype="bf16"),
        # A full batch of mixed contexts in a layer of 128 heads.
        _decode("decode-batch64", 128, WIDE, batch=64, low=512, high=8192, dtype="bf16", page=64,
                lengths_seed=2),
        # Two users with long documents: few sequences spread over the GPU.
        _decode("decode-long", 32, WIDE, batch=2, low=100000, high=131072, dtype="fp16",
                lengths_seed=3),
        # A prompt's chunk after a cached prefix, as a scheduler cuts it.
        _prefill("prefill-chunk", 16, WIDE, start=7777, count=512, dtype="bf16"),
        # A fresh prompt in a layer of 128 heads: the largest call.
        _prefill("prefill-prompt", 128, WIDE, start=0, count=4096, dtype="bf16", page=64),
        # A prompt of odd length after a short prefix on a small model.
        _prefill("prefill-ragged-small", 14, SMALL, start=389, count=1531, dtype="fp16"),
        # The weights of one short step of a small model.
        _weights("weights-short", (14, 2, 64), batch=4, low=200, high=700, dtype="fp16"),
        # The weights of a full batch on a 7B shape.
        _weights("weights-batch64", (28, 4, 128), batch=64, low=512, high=8192, dtype="bf16",
                 lengths_seed=2),
        # A sequence that has just passed its bound, on a small model.
        _evict("evict-one", (14, 2, 64), batch=1, low=1100, high=1100, keep=1024, recent=128,
               sinks=4, dtype="fp16"),
        # A batch cut to a quarter of its longest context on a 7B shape.
        _evict("evict-batch32", (28, 4, 128), batch=32, low=1024, high=8192, keep=2048,
               recent=512, sinks=4, dtype="bf16", lengths_seed=4),
    ]


HEADS = [(14, 2, 64), (16, 16, 64), (32, 32, 80), (32, 8, 96), (28, 4, 128), (32, 8, 128),
         (40, 8, 128), (8, 4, 256), (16, 2, 512)]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """Any of the five calls, over the ranges that the listed ones stand for;
    bounded so that none costs more than the largest listed one."""
    kind = rng.choice(["append", "decode", "decode", "prefill", "prefill", "weights", "evict"])
    dtype = rng.choice(["fp16", "bf16"])
    page = rng.choice([16, 16, 32, 64])
    heads = rng.choice([8, 12, 16, 20, 32, 64, 96, 128])
    shape = rng.choice([WIDE, WIDE, SMALL, UNEVEN])
    seed = rng.randrange(1 << 20)
    if kind == "append":
        return _append(None, heads, shape, count=_log(rng, 1, 4096), dtype=dtype)
    if kind == "decode":
        batch = _log(rng, 1, 64)
        high = _log(rng, 1, 131072)
        while batch * high * heads > 64 * 8192 * 128 or batch * high > 64 * 8192:
            high = max(1, high // 2)
        return _decode(None, heads, shape, batch=batch, low=max(1, high // rng.randint(1, 16)),
                       high=high, dtype=dtype, page=page, lengths_seed=seed)
    if kind == "prefill":
        count = _log(rng, 1, 4096)
        start = rng.choice([0, _log(rng, 1, 32768)])
        while ((start + count) * count * heads > 4096 * 4096 * 64
               or (start + count) * heads > 4096 * 128):
            if start > count:
                start //= 2
            else:
                count = max(1, count // 2)
        return _prefill(None, heads, shape, start=start, count=count, dtype=dtype, page=page)
    shape = rng.choice(HEADS)
    layout = rng.choice(["pages", "pages", "rows"])
    batch = _log(rng, 1, 64)
    high = _log(rng, 2, 65536)
    limit = 64 * 8192 * 4 * 128 if kind == "weights" else 32 * 8192 * 4 * 128
    while batch * high * shape[1] * shape[2] > limit:
        high = max(2, high // 2)
    low = max(1, high // rng.randint(1, 8))
    if kind == "weights":
        return _weights(None, shape, batch=batch, low=low, high=high, dtype=dtype, page=page,
                        layout=layout, window=rng.choice([0, 0, 0, 512]),
                        softcap=rng.choice([0.0, 0.0, 30.0]), lengths_seed=seed)
    keep = rng.randint(max(1, high // 8), high)
    recent = rng.randint(0, keep // 2)
    return _evict(None, shape, batch=batch, low=low, high=high, keep=keep, recent=recent,
                  sinks=rng.randint(0, min(8, keep - recent)), dtype=dtype, page=page,
                  layout=layout, lengths_seed=seed)


# ---------------------------------------------------------------------------
# Inputs.

def _lengths(case):
    rng = np.random.default_rng(case["lengths_seed"])
    return rng.integers(case["low"], case["high"] + 1, case["batch"]).astype(np.int64)


def _tables(lengths, page, rng, first=0):
    """Page tables of sequences that hold the pages of a full arena in any
    order, 0 past a sequence's last page, and the pages' number."""
    need = -(-lengths // page)
    order = first + rng.permutation(int(need.sum())).astype(np.int32)
    tables = np.zeros((len(lengths), int(need.max())), dtype=np.int32)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = order[at:at + n]
        at += n
    return tables, first + int(need.sum())


def _normal(gen, shape, dtype, std=1.0):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=gen)


def _int(a):
    return torch.as_tensor(np.ascontiguousarray(a).astype(np.int32), device="cuda")


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    state = dict(case=case)
    if case["kind"] in ("append", "decode", "prefill"):
        heads, latent, rope = case["heads"], case["latent"], case["rope"]
        nope, value = case["nope"], case["value"]
        state["scale"] = (nope + rope) ** -0.5
        if case["kind"] == "append":
            n = case["count"]
            # The down projection's output: latent and rotary key side by side.
            down = _normal(gen, (n, latent + rope), dtype)
            rows = rng.permutation(2 * n)[:n]
            return dict(state, q=_normal(gen, (n, heads, nope + rope), dtype),
                        c=down[:, :latent], k=down[:, latent:],
                        norm=(1.0 + _normal(gen, (latent,), torch.float32, 0.1)).to(dtype),
                        arena=_normal(gen, (2 * n, latent + rope), dtype),
                        positions=_int(rng.integers(0, 65536, n)), rows=_int(rows))
        # Normalised latents, rotated keys of the same size; projections that
        # give keys, values and scores of about unit variance.
        state["kv_b"] = _normal(gen, (heads, nope + value, latent), dtype, latent ** -0.5)
        if case["kind"] == "decode":
            lengths = _lengths(case)
            tables, pages = _tables(lengths, case["page"], rng)
            return dict(state, arena=_normal(gen, (pages * case["page"], latent + rope), dtype),
                        q=_normal(gen, (case["batch"], heads, nope + rope), dtype),
                        tables=_int(tables), lengths=_int(lengths), longest=int(lengths.max()))
        end = np.array([case["start"] + case["count"]])
        tables, pages = _tables(end, case["page"], rng)
        return dict(state, arena=_normal(gen, (pages * case["page"], latent + rope), dtype),
                    q=_normal(gen, (case["count"], heads, nope + rope), dtype),
                    table=_int(tables[0]))
    lengths = _lengths(case)
    page, kv_heads, dim = case["page"], case["kv_heads"], case["head_dim"]
    tables, pages = _tables(lengths, page, rng)
    capacity = int(lengths.max())
    out_tables = None
    if case["kind"] == "evict":
        # The kept rows go to fresh pages (the old ones may be shared).
        out_tables, pages = _tables(np.minimum(lengths, case["keep"]), page, rng, first=pages)
    shape = ((pages * page, kv_heads, dim) if case["layout"] == "rows"
             else (pages, kv_heads, page, dim))
    state.update(keys=_normal(gen, shape, dtype), tables=_int(tables), lengths=_int(lengths),
                 longest=capacity)
    # Accumulated weights: many small, few large, and some that never were
    # above zero (those are alike).
    w = torch.empty((case["batch"], kv_heads, capacity), device="cuda")
    w.exponential_(generator=gen).pow_(3)
    state["weights"] = torch.where(w < 0.01, torch.zeros_like(w), w)
    if case["kind"] == "weights":
        return dict(state, q=_normal(gen, (case["batch"], case["q_heads"], dim), dtype),
                    scale=dim ** -0.5, out=torch.zeros_like(w))
    return dict(state, values=_normal(gen, shape, dtype), out_tables=_int(out_tables),
                out_weights=torch.zeros_like(w))


# ---------------------------------------------------------------------------
# One pass.

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    case = state["case"]
    if case["kind"] in ("append", "decode", "prefill"):
        from instinct_amd import latent

        if case["kind"] == "append":
            q = latent.latent_append(state["q"], state["c"], state["k"], state["arena"],
                                     state["positions"], state["rows"], dims=case["rope"],
                                     base=BASE, norm_weight=state["norm"], eps=EPS)
            return {"q": q, "arena": state["arena"]}
        if case["kind"] == "decode":
            return latent.latent_decode_attention(
                state["q"], state["arena"], state["kv_b"], state["tables"], state["lengths"],
                page_size=case["page"], longest=state["longest"], scale=state["scale"])
        return latent.latent_prefill_attention(
            state["q"], state["arena"], state["kv_b"], state["table"], start=case["start"],
            page_size=case["page"], scale=state["scale"])
    from instinct_amd import eviction

    if case["kind"] == "weights":
        return eviction.paged_attention_weights(
            state["q"], state["keys"], state["tables"], state["lengths"], state["weights"],
            page_size=case["page"], longest=state["longest"], scale=state["scale"],
            window=case["window"], softcap=case["softcap"], out=state["out"])
    lengths, kept = eviction.evict_rows(
        state["keys"], state["values"], state["weights"], state["tables"], state["lengths"],
        page_size=case["page"], longest=state["longest"], keep=case["keep"],
        recent=case["recent"], sinks=case["sinks"], out_tables=state["out_tables"],
        out_weights=state["out_weights"])
    return {"lengths": lengths, "kept": kept, "keys": state["keys"], "values": state["values"],
            "weights": state["out_weights"]}


def _positions_rows(pages, page, n):
    at = torch.arange(n, device="cuda")
    return pages[at // page].long() * page + at % page


def _angles(positions, dims):
    """Cosine and sine of each token's angles: position times inverse
    frequency, both and their product float32, as the append defines them."""
    half = dims // 2
    power = (-np.arange(half, dtype=np.float32) * np.float32(2)) / np.float32(dims)
    freq = torch.as_tensor(np.power(np.float32(BASE), power, dtype=np.float32), device="cuda")
    angle = (positions.float()[:, None] * freq).double()
    return angle.cos(), angle.sin()


def _run_plain(state):
    case = state["case"]
    return {"append": _plain_append, "decode": _plain_decode, "prefill": _plain_prefill,
            "weights": _plain_weights, "evict": _plain_evict}[case["kind"]](state)


def _plain_append(state):
    case = state["case"]
    dtype, half, nope = state["q"].dtype, case["rope"] // 2, case["nope"]
    cos, sin = (t.float() for t in _angles(state["positions"], case["rope"]))

    def rotate(x, cos, sin):
        a, b = x[..., :half].float(), x[..., half:].float()
        return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1).to(dtype)

    c = state["c"].float()
    c = c * torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS) * state["norm"].float()
    state["arena"][state["rows"].long()] = torch.cat(
        [c.to(dtype), rotate(state["k"], cos, sin)], dim=-1)
    q = torch.cat([state["q"][..., :nope], rotate(state["q"][..., nope:], cos[:, None],
                                                  sin[:, None])], dim=-1)
    return {"q": q, "arena": state["arena"]}


def _plain_decode(state):
    case = state["case"]
    nope, latent = case["nope"], case["latent"]
    up = state["kv_b"][:, :nope].float()
    down = state["kv_b"][:, nope:].float().transpose(1, 2).contiguous()
    q = state["q"].float()
    q_lat = torch.matmul(q[..., :nope].transpose(0, 1).contiguous(), up).transpose(0, 1)
    q_all = torch.cat([q_lat, q[..., nope:]], dim=-1) * state["scale"]
    o = torch.empty((case["batch"], case["heads"], latent), device="cuda")
    for b, n in enumerate(_lengths(case).tolist()):
        rows = state["arena"][_positions_rows(state["tables"][b], case["page"], n)].float()
        s = q_all[b] @ rows.t()
        p = torch.exp(s - s.amax(-1, keepdim=True))
        o[b] = (p @ rows[:, :latent].contiguous()) / p.sum(-1, keepdim=True)
    out = torch.matmul(o.transpose(0, 1).contiguous(), down).transpose(0, 1)
    return out.contiguous().to(state["q"].dtype)


def _plain_prefill(state):
    case = state["case"]
    nope, latent, start, count = case["nope"], case["latent"], case["start"], case["count"]
    end = start + count
    rows = state["arena"][_positions_rows(state["table"], case["page"], end)].float()
    c, k_rope = rows[:, :latent].contiguous(), rows[:, latent:].contiguous()
    hidden = (torch.arange(end, device="cuda")[None]
              > start + torch.arange(count, device="cuda")[:, None])
    out = torch.empty((count, case["heads"], case["value"]), dtype=state["q"].dtype,
                      device="cuda")
    for h in range(case["heads"]):
        kv = c @ state["kv_b"][h].float().t()
        q = state["q"][:, h].float() * state["scale"]
        s = q[:, :nope] @ kv[:, :nope].t() + q[:, nope:] @ k_rope.t()
        s.masked_fill_(hidden, -math.inf)
        p = torch.exp_(s.sub_(s.amax(-1, keepdim=True)))
        out[:, h] = ((p @ kv[:, nope:].contiguous()) / p.sum(-1, keepdim=True)).to(out.dtype)
    return out


def _rows_of(store, pages, page, n):
    at = torch.arange(n, device="cuda")
    ids = pages[at // page].long()
    if store.dim() == 3:
        return store[ids * page + at % page]
    return store[ids, :, at % page]


def _plain_weights(state):
    case = state["case"]
    kv_heads, group = case["kv_heads"], case["q_heads"] // case["kv_heads"]
    out = state["out"]
    for b, n in enumerate(_lengths(case).tolist()):
        keys = _rows_of(state["keys"], state["tables"][b], case["page"], n).float()
        q = state["q"][b].float().view(kv_heads, group, -1)
        s = torch.matmul(q, keys.permute(1, 2, 0).contiguous()) * state["scale"]
        if case["softcap"] > 0:
            s = case["softcap"] * torch.tanh(s / case["softcap"])
        if case["window"]:
            s[..., :max(0, n - case["window"])] = -math.inf
        p = torch.exp(s - s.amax(-1, keepdim=True))
        p = (p / p.sum(-1, keepdim=True)).sum(1)
        # The newest key's entry starts here.
        out[b, :, :n - 1] = state["weights"][b, :, :n - 1] + p[:, :-1]
        out[b, :, n - 1] = p[:, -1]
    return out


def _choose(weights, n, keep, recent, sinks):
    """[kv heads, min(n, keep)] positions to keep, ascending: the first
    ``sinks``, the last ``recent`` and the heaviest others, the lower of two
    alike."""
    w = weights[:, :n]
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices
    at = torch.arange(n, device=w.device)
    rest = ~((at < sinks) | (at >= n - recent))
    order = order.gather(-1, torch.sort(rest[order].to(torch.int8), dim=-1, stable=True).indices)
    return order[:, :keep].sort(-1).values


def _plain_evict(state):
    case = state["case"]
    page, keep = case["page"], case["keep"]
    lengths = _lengths(case)
    kept = torch.full((case["batch"], case["kv_heads"], keep), -1, dtype=torch.int32,
                      device="cuda")
    heads = torch.arange(case["kv_heads"], device="cuda")[:, None]
    for b, n in enumerate(lengths.tolist()):
        pick = _choose(state["weights"][b], n, keep, case["recent"], case["sinks"])
        m = pick.shape[1]
        kept[b, :, :m] = pick.int()
        state["out_weights"][b, :, :m] = state["weights"][b].gather(-1, pick)
        to = torch.arange(m, device="cuda")
        src, dst = state["tables"][b][pick // page].long(), state["out_tables"][b][to // page].long()
        for store in (state["keys"], state["values"]):
            if case["layout"] == "rows":
                store[dst * page + to % page, heads] = store[src * page + pick % page, heads]
            else:
                store[dst, heads, to % page] = store[src, heads, pick % page]
    return {"lengths": torch.as_tensor(np.minimum(lengths, keep).astype(np.int32), device="cuda"),
            "kept": kept, "keys": state["keys"], "values": state["values"],
            "weights": state["out_weights"]}


# ---------------------------------------------------------------------------
# What a pass cannot do without.

def work(case):
    kind = case["kind"]
    if kind in ("append", "decode", "prefill"):
        heads, latent, rope = case["heads"], case["latent"], case["rope"]
        nope, value = case["nope"], case["value"]
        row = 2 * (latent + rope)
        query, result = 2 * heads * (nope + rope), 2 * heads * value
        up = 2 * heads * (nope + value) * latent
        if kind == "append":
            n = case["count"]
            return {"bytes": n * (2 * query + 2 * row + 8) + 2 * latent,
                    "flops": n * (4 * latent + 3 * rope * (heads + 1))}
        if kind == "decode":
            lengths, batch = _lengths(case), case["batch"]
            keys = int(lengths.sum())
            tables = 4 * int((-(-lengths // case["page"])).sum()) + 4 * batch
            return {"bytes": keys * row + batch * (query + result) + up + tables,
                    "flops": 2 * keys * heads * (2 * latent + rope) + batch * up}
        end = case["start"] + case["count"]
        seen = int((case["start"] + 1 + np.arange(case["count"], dtype=np.int64)).sum())
        return {"bytes": end * row + case["count"] * (query + result) + up
                + 4 * -(-end // case["page"]),
                "flops": end * up + 2 * seen * heads * (nope + rope + value)}
    lengths, kv_heads, dim = _lengths(case), case["kv_heads"], case["head_dim"]
    tables = 4 * int((-(-lengths // case["page"])).sum()) + 4 * case["batch"]
    if kind == "weights":
        seen = np.minimum(lengths, case["window"]) if case["window"] else lengths
        keys = int(seen.sum())
        return {"bytes": keys * kv_heads * 2 * dim + 8 * kv_heads * int(lengths.sum()) + tables
                + 2 * case["batch"] * case["q_heads"] * dim,
                "flops": keys * case["q_heads"] * (2 * dim + 4)}
    kept = int(np.minimum(lengths, case["keep"]).sum())
    return {"bytes": 4 * kv_heads * int(lengths.sum()) + kv_heads * kept * (2 * 2 * 2 * dim + 8)
            + tables, "flops": kv_heads * int(lengths.sum())}


# ---------------------------------------------------------------------------
# The definitions in 64 bits.

def exact(case, seed):
    state = prepare(case, seed)
    return {"append": _exact_append, "decode": _exact_decode, "prefill": _exact_prefill,
            "weights": _exact_weights, "evict": _exact_evict}[case["kind"]](state)


def _exact_append(state):
    case = state["case"]
    latent, nope, half = case["latent"], case["nope"], case["rope"] // 2
    cos, sin = _angles(state["positions"], case["rope"])
    turn = torch.complex(cos, sin)
    arena = state["arena"].double()
    c = state["c"].double()
    rms = torch.sqrt(c.pow(2).sum(-1, keepdim=True) / latent + EPS)
    rows = state["rows"].long()
    k = state["k"].double()
    k = torch.complex(k[:, :half].contiguous(), k[:, half:].contiguous()) * turn
    arena[rows, :latent] = c / rms * state["norm"].double()
    arena[rows, latent:latent + half] = k.real
    arena[rows, latent + half:] = k.imag
    q = state["q"].double()
    r = torch.complex(q[..., nope:nope + half].contiguous(),
                      q[..., nope + half:].contiguous()) * turn[:, None]
    q[..., nope:nope + half], q[..., nope + half:] = r.real, r.imag
    return {"q": q, "arena": arena}


def _latent_rows(state, pages, n):
    page = state["case"]["page"]
    store = state["arena"].view(-1, page, state["arena"].shape[1])
    return store[pages[:-(-n // page)].long()].flatten(0, 1)[:n].double()


def _exact_decode(state):
    """Expanded: every head's own keys and values from the latents."""
    case = state["case"]
    nope, latent = case["nope"], case["latent"]
    lengths = _lengths(case)
    out = torch.empty((case["batch"], case["heads"], case["value"]), dtype=torch.float64,
                      device="cuda")
    if int(lengths.sum()) * case["heads"] > 1 << 26:
        # (Expanded in 64 bits this would take too long: the same sums taken
        # over the latent instead.)
        for b, n in enumerate(lengths.tolist()):
            rows = _latent_rows(state, state["tables"][b], n)
            w = state["kv_b"].double()
            q = state["q"][b].double()
            lat = (q[:, :nope, None] * w[:, :nope]).sum(1)
            s = torch.cat([lat, q[:, nope:]], -1) @ rows.t().contiguous()
            p = torch.softmax(s * state["scale"], dim=-1)
            mean = p @ rows[:, :latent].contiguous()
            out[b] = (w[:, nope:] * mean[:, None]).sum(-1)
        return out
    for b, n in enumerate(lengths.tolist()):
        rows = _latent_rows(state, state["tables"][b], n)
        for h in range(case["heads"]):
            kv = rows[:, :latent].contiguous() @ state["kv_b"][h].double().t().contiguous()
            k = torch.cat([kv[:, :nope], rows[:, latent:]], dim=-1)
            p = torch.softmax(k @ state["q"][b, h].double() * state["scale"], dim=0)
            out[b, h] = p @ kv[:, nope:].contiguous()
    return out


def _exact_prefill(state):
    case = state["case"]
    nope, latent, start, count = case["nope"], case["latent"], case["start"], case["count"]
    rows = _latent_rows(state, state["table"], start + count)
    out = torch.empty((count, case["heads"], case["value"]), dtype=torch.float64, device="cuda")
    for h in range(case["heads"]):
        kv = rows[:, :latent].contiguous() @ state["kv_b"][h].double().t().contiguous()
        k = torch.cat([kv[:, :nope], rows[:, latent:]], dim=-1)
        v = kv[:, nope:].contiguous()
        for a in range(0, count, 1024):
            z = min(a + 1024, count)
            s = state["q"][a:z, h].double() @ k[:start + z].t().contiguous() * state["scale"]
            s = s.tril_(start + a).masked_fill_(
                torch.ones_like(s, dtype=torch.bool).triu_(start + a + 1), -math.inf)
            out[a:z, h] = torch.softmax(s, dim=-1) @ v[:start + z]
    return out


def _exact_weights(state):
    case = state["case"]
    group = case["q_heads"] // case["kv_heads"]
    out = state["out"].double()
    old = state["weights"].double()
    for b, n in enumerate(_lengths(case).tolist()):
        first = max(0, n - case["window"]) if case["window"] else 0
        keys = _rows_of(state["keys"], state["tables"][b], case["page"], n)[first:].double()
        out[b, :, :n - 1] = old[b, :, :n - 1]
        for h in range(case["q_heads"]):
            s = keys[:, h // group].contiguous() @ state["q"][b, h].double() * state["scale"]
            if case["softcap"] > 0:
                s = case["softcap"] * torch.tanh(s / case["softcap"])
            out[b, h // group, first:n] += torch.softmax(s, dim=0)
    return out


def _exact_evict(state):
    """The chosen positions by ranking every key; the packed rows are copies."""
    case = state["case"]
    page, keep = case["page"], case["keep"]
    lengths = _lengths(case)
    kept = np.full((case["batch"], case["kv_heads"], keep), -1, dtype=np.int32)
    weights = state["weights"].cpu().numpy()
    packed = np.zeros_like(weights)
    for b, n in enumerate(lengths.tolist()):
        at = np.arange(n)
        rest = (at >= case["sinks"]) & (at < n - case["recent"])
        for j in range(case["kv_heads"]):
            order = np.lexsort((at, -weights[b, j, :n], rest))
            pick = np.sort(order[:keep])
            kept[b, j, :len(pick)] = pick
            packed[b, j, :len(pick)] = weights[b, j, pick]
    moved = []
    for store in (state["keys"], state["values"]):
        store = store.clone()
        tiles = store if case["layout"] == "pages" else store.view(
            -1, page, *store.shape[1:]).transpose(1, 2)
        for b, n in enumerate(lengths.tolist()):
            for j in range(case["kv_heads"]):
                pick = torch.as_tensor(kept[b, j, :min(n, keep)], device="cuda").long()
                to = torch.arange(len(pick), device="cuda")
                tiles[state["out_tables"][b][to // page].long(), j, to % page] = tiles[
                    state["tables"][b][pick // page].long(), j, pick % page]
        moved.append(store.double())
    return {"lengths": torch.as_tensor(np.minimum(lengths, keep).astype(np.int32), device="cuda"),
            "kept": torch.as_tensor(kept, device="cuda"), "keys": moved[0], "values": moved[1],
            "weights": torch.as_tensor(packed, device="cuda").double()}
