"""Latent attention on the GPU against the float64 oracle: append and decode."""

import pytest
import torch

from oracle import latent as oracle

pytestmark = pytest.mark.gpu

WIDE, SMALL, UNEVEN, THIN = (512, 64, 128, 128), (256, 32, 64, 64), (384, 48, 96, 80), (8, 0, 8, 8)
TYPES = [torch.float16, torch.bfloat16]


def layer(shape, heads, rows, dtype, seed=0):
    """Arena of unit latents and keys and the projection that keeps them so."""
    latent, rope, nope, value = shape
    g = torch.Generator().manual_seed(seed)
    arena = torch.randn((rows, latent + rope), generator=g).to(dtype)
    kv_b = (torch.randn((heads, nope + value, latent), generator=g) * latent ** -0.5).to(dtype)
    return arena, kv_b, g


def pack(lengths, page, pages, g):
    """Tables of distinct random pages, 0 past a sequence's last page."""
    order = torch.randperm(pages, generator=g).tolist()
    width = max(1, max(-(-max(n, 0) // page) for n in lengths))
    tables = torch.zeros((len(lengths), width), dtype=torch.int32)
    for b, n in enumerate(lengths):
        for i in range(-(-max(n, 0) // page)):
            tables[b, i] = order.pop()
    return tables


def run_decode(gpu, q, arena, kv_b, tables, lengths, page, scale, **kw):
    from instinct_amd.latent import latent_decode_attention

    return latent_decode_attention(q.to(gpu), arena.to(gpu), kv_b.to(gpu), tables.to(gpu),
                                   torch.tensor(lengths, dtype=torch.int32, device=gpu),
                                   page_size=page, longest=max(1, max(lengths)), scale=scale, **kw)


def check_decode(gpu, shape, heads, lengths, page, dtype, change=None, seed=0):
    latent, rope, nope, value = shape
    pages = sum(-(-max(n, 0) // page) for n in lengths) + 3
    arena, kv_b, g = layer(shape, heads, pages * page, dtype, seed)
    tables = pack(lengths, page, pages, g)
    if change:
        change(arena, tables)
    q = torch.randn((len(lengths), heads, nope + rope), generator=g).to(dtype)
    scale = (nope + rope) ** -0.5
    got = run_decode(gpu, q, arena, kv_b, tables, lengths, page, scale).cpu().double()
    want, bound = oracle.decode(q, arena, kv_b, tables, lengths, page_size=page, scale=scale)
    over = (got - want).abs() - bound
    assert bool((over <= 0).all()), f"past the bound by {over.max():.3e}"
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape, heads", [(WIDE, 16), (WIDE, 33), (WIDE, 128), (WIDE, 130),
                                          (SMALL, 14), (SMALL, 64), (UNEVEN, 20), (UNEVEN, 96),
                                          (THIN, 1), ((264, 16, 40, 24), 3)])
def test_decode_shapes(gpu, shape, heads, dtype):
    check_decode(gpu, shape, heads, [1, 31, 32, 33, 0, 200, 65], 16, dtype)


@pytest.mark.parametrize("page", [1, 7, 16, 48, 64])
@pytest.mark.parametrize("heads", [16, 64, 128])
def test_decode_pages(gpu, page, heads):
    """Pages that end inside a tile, and one key a page."""
    check_decode(gpu, SMALL, heads, [129, 2, 77], page, torch.bfloat16)


@pytest.mark.parametrize("heads", [16, 64, 128])
def test_decode_long(gpu, heads):
    """A sequence over many workgroups and chunks of rows (2048 keys), beside
    short ones."""
    check_decode(gpu, SMALL, heads, [4500, 3, 2048, 2049], 16, torch.float16)


@pytest.mark.parametrize("heads", [3, 256])
@pytest.mark.parametrize("batch", [1, 2, 3, 4, 5, 7, 8, 9, 31, 33, 70])
def test_decode_batches(gpu, batch, heads):
    """Any number of sequences in the join, one to 32 of them a workgroup, empty
    ones first, last and between."""
    g = torch.Generator().manual_seed(batch)
    lengths = torch.randint(0, 180, (batch,), generator=g).tolist()
    lengths[0] = 0 if batch > 2 else 77
    lengths[-1] = 0 if batch > 3 else 130
    lengths[batch // 2] = 0 if batch > 4 else lengths[batch // 2]
    check_decode(gpu, (32, 16, 24, 40), heads, lengths, 16, torch.float16)


def test_decode_many_parts(gpu):
    """A sequence in more parts than a wave has lanes."""
    check_decode(gpu, (72, 16, 16, 128), 5, [21000, 40], 64, torch.bfloat16)


def test_decode_one_key_is_its_value(gpu):
    check_decode(gpu, WIDE, 16, [1], 16, torch.float16)


@pytest.mark.parametrize("heads", [16, 128])
def test_decode_masked_pages(gpu, heads):
    """Released and unknown pages hide their keys whatever the rows hold; a
    sequence with none left gives zeros."""
    def change(arena, tables):
        arena[0] = float("nan")  # row 0 is page 0, that -1 must not lead to
        tables[tables == 0] = -1
        tables[0, 1] = -1
        tables[0, 3] = 1 << 20
        tables[2, :] = -7

    got = check_decode(gpu, WIDE, heads, [150, 70, 40], 16, torch.bfloat16, change)
    assert bool((got[2] == 0).all())


def test_decode_rows_past_the_length(gpu):
    """What a sequence's last page holds past its length is not used."""
    def change(arena, tables):
        arena.view(-1, 16, arena.shape[1])[tables[0, 1].long(), 5:] = float("inf")

    check_decode(gpu, WIDE, 16, [21], 16, torch.float16, change)


def test_decode_large_scores(gpu):
    """Scores far apart move the running maximum within a sequence."""
    latent, rope, nope, value = SMALL
    arena, kv_b, g = layer(SMALL, 16, 64 * 16, torch.float16)
    arena *= torch.linspace(0.1, 3.0, 64 * 16)[:, None].to(arena.dtype)
    tables = torch.arange(64, dtype=torch.int32)[None]
    q = torch.randn((1, 16, nope + rope), generator=g).to(torch.float16)
    scale = 3 * (nope + rope) ** -0.5
    got = run_decode(gpu, q, arena, kv_b, tables, [1000], 16, scale).cpu().double()
    want, bound = oracle.decode(q, arena, kv_b, tables, [1000], page_size=16, scale=scale)
    assert bool(((got - want).abs() <= bound).all())


def test_decode_repeats_and_hint(gpu):
    """Same bits again; `longest` too small or too large changes rounding only."""
    from instinct_amd.latent import latent_decode_attention

    arena, kv_b, g = layer(WIDE, 32, 200 * 16, torch.bfloat16)
    lengths = [1500, 20, 900]
    tables = pack(lengths, 16, 200, g)
    q = torch.randn((3, 32, 192), generator=g).to(torch.bfloat16)
    want, bound = oracle.decode(q, arena, kv_b, tables, lengths, page_size=16, scale=0.07)
    dev = [x.to(gpu) for x in (q, arena, kv_b, tables)]
    n = torch.tensor(lengths, dtype=torch.int32, device=gpu)
    for longest in (1, 1500, 1 << 20):
        a = latent_decode_attention(*dev, n, page_size=16, longest=longest, scale=0.07)
        b = latent_decode_attention(*dev, n, page_size=16, longest=longest, scale=0.07)
        assert torch.equal(a, b)
        assert bool(((a.cpu().double() - want).abs() <= bound).all())


@pytest.mark.parametrize("heads", [16, 64, 128])
def test_decode_past_the_caches(gpu, heads):
    """A `longest` whose rows would pass what the caches hold: their rows are
    copied the other way, over chunks of rows and in the middle of one."""
    from instinct_amd.latent import latent_decode_attention

    lengths, page = [2500, 1, 0, 130], 16
    arena, kv_b, g = layer(WIDE, heads, 200 * page, torch.float16)
    tables = pack(lengths, page, 200, g)
    q = torch.randn((4, heads, 192), generator=g).to(torch.float16)
    got = latent_decode_attention(*(x.to(gpu) for x in (q, arena, kv_b, tables)),
                                  torch.tensor(lengths, dtype=torch.int32, device=gpu),
                                  page_size=page, longest=1 << 17, scale=0.07)
    want, bound = oracle.decode(q, arena, kv_b, tables, lengths, page_size=page, scale=0.07)
    assert bool(((got.cpu().double() - want).abs() <= bound).all())


def test_decode_far_rows(gpu):
    """Rows whose element offset passes 2^31."""
    latent, rope, nope, value = WIDE
    rows = (1 << 31) // 576 // 16 * 16 + 4096
    arena = torch.zeros((rows, 576), dtype=torch.bfloat16, device=gpu)
    near, kv_b, g = layer(WIDE, 16, 64, torch.bfloat16)
    arena[-64:] = near.to(gpu)
    q = torch.randn((1, 16, nope + rope), generator=g).to(torch.bfloat16)
    pages = rows // 16
    tables = torch.arange(pages - 4, pages, dtype=torch.int32)[None]
    got = run_decode(gpu, q, arena, kv_b, tables, [60], 16, 0.07).cpu().double()
    want, bound = oracle.decode(q, near, kv_b, tables - (pages - 4), [60], page_size=16,
                                scale=0.07)
    assert bool(((got - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape, heads, n", [(WIDE, 16, 1), (WIDE, 128, 5), (SMALL, 17, 9),
                                             (UNEVEN, 3, 70), (THIN, 2, 4)])
@pytest.mark.parametrize("norm", [True, False])
def test_append(gpu, shape, heads, n, dtype, norm):
    """One rounding per element: the float32 value is off by a few 2^-24 of
    its terms (512 squares summed, two products)."""
    from instinct_amd.hip_kernels import rope_inv_freq
    from instinct_amd.latent import latent_append

    latent, rope, nope, _ = shape
    g = torch.Generator().manual_seed(3)
    down = torch.randn((n, latent + rope + 8), generator=g).to(dtype)
    c, k = down[:, :latent], down[:, latent:latent + rope]
    weight = (1 + 0.1 * torch.randn(latent, generator=g)).to(dtype) if norm else None
    q = torch.randn((n, heads, nope + rope), generator=g).to(dtype)
    arena = torch.randn((2 * n + 1, latent + rope), generator=g).to(dtype)
    rows = torch.randperm(2 * n + 1, generator=g)[:n].int()
    positions = torch.randint(0, 100000, (n,), generator=g).int()
    inv = rope_inv_freq(rope, base=1e6, device="cpu") if rope else None
    want_q, want_a = oracle.append(q, c, k, arena, positions, rows, inv_freq=inv,
                                   norm_weight=weight, eps=1e-6)
    dev = down.to(gpu)
    store, dq = arena.to(gpu), q.to(gpu)
    args = (dev[:, :latent], dev[:, latent:latent + rope], store, positions.to(gpu), rows.to(gpu))
    kw = dict(dims=rope, base=1e6, norm_weight=None if weight is None else weight.to(gpu))
    got_q = latent_append(dq, *args, **kw)
    assert torch.equal(dq.cpu(), q)
    u = oracle.HALF_STEP[dtype]
    for got, want in ((got_q, want_q), (store, want_a)):
        bound = 1.01 * u * want.abs() + 2.0 ** -25 + 4e-6
        assert bool(((got.cpu().double() - want).abs() <= bound).all())
    untouched = sorted(set(range(2 * n + 1)) - set(rows.tolist()))
    assert torch.equal(store.cpu()[untouched], arena[untouched])
    # In place, and the write alone.
    again = arena.to(gpu)
    assert latent_append(dq, *args[:2], again, *args[3:], q_out=dq, **kw) is dq
    assert torch.equal(dq, got_q) and torch.equal(again, store)
    alone = arena.to(gpu)
    assert latent_append(None, *args[:2], alone, *args[3:], **kw) is None
    assert torch.equal(alone, store)


def test_append_drops_rows_outside(gpu):
    from instinct_amd.latent import latent_append

    arena = torch.zeros((4, 72), dtype=torch.float16, device=gpu)
    c = torch.ones((3, 64), dtype=torch.float16, device=gpu)
    k = torch.ones((3, 8 * 2), dtype=torch.float16, device=gpu)[:, :0]
    arena = torch.zeros((4, 64), dtype=torch.float16, device=gpu)
    rows = torch.tensor([-1, 2, 4], dtype=torch.int32, device=gpu)
    latent_append(None, c, k, arena, rows, rows, dims=0)
    assert arena.sum(1).tolist() == [0, 0, 64, 0]


def test_append_copies_without_rotation(gpu):
    from instinct_amd.latent import latent_append

    g = torch.Generator().manual_seed(5)
    down = torch.randn((6, 576), generator=g).half().to(gpu)
    q = torch.randn((6, 4, 192), generator=g).half().to(gpu)
    arena = torch.zeros((6, 576), dtype=torch.float16, device=gpu)
    rows = torch.arange(6, dtype=torch.int32, device=gpu)
    out = latent_append(q, down[:, :512], down[:, 512:], arena, rows, rows, dims=0)
    assert torch.equal(out, q) and torch.equal(arena, down)


def test_refusals(gpu):
    from instinct_amd import _lib
    from instinct_amd.latent import latent_append, latent_decode_attention

    q = torch.zeros((2, 4, 192), dtype=torch.float16, device=gpu)
    arena = torch.zeros((64, 576), dtype=torch.float16, device=gpu)
    kv_b = torch.zeros((4, 256, 512), dtype=torch.float16, device=gpu)
    tables = torch.zeros((2, 4), dtype=torch.int32, device=gpu)
    n = torch.ones(2, dtype=torch.int32, device=gpu)
    kw = dict(page_size=16, longest=1, scale=0.1)
    call = latent_decode_attention
    with pytest.raises(TypeError):
        call(q, arena.bfloat16(), kv_b, tables, n, **kw)
    with pytest.raises(ValueError, match="contiguous"):
        call(q.transpose(0, 1), arena, kv_b, tables, n, **kw)
    with pytest.raises(ValueError, match="heads"):
        call(q, arena, kv_b[:3].contiguous(), tables, n, **kw)
    with pytest.raises(ValueError, match="fit together"):
        call(q, arena[:, :500].contiguous(), kv_b, tables, n, **kw)
    with pytest.raises(TypeError, match="int32"):
        call(q, arena, kv_b, tables.long(), n, **kw)
    with pytest.raises(ValueError, match="lengths"):
        call(q, arena, kv_b, tables, n[:1], **kw)
    with pytest.raises(ValueError, match="same GPU|must be on"):
        call(q, arena, kv_b, tables.cpu(), n, **kw)
    with pytest.raises(ValueError, match="out must"):
        call(q, arena, kv_b, tables, n, out=q, **kw)
    with pytest.raises(ValueError, match="workspace"):
        call(q, arena, kv_b, tables, n, workspace=torch.empty(8, dtype=torch.uint8, device=gpu),
             **kw)
    with pytest.raises(_lib.PdaError):
        call(q, arena[:8].contiguous(), kv_b, tables, n, **kw)
    c, k = arena[:2, :512], arena[:2, 512:]
    with pytest.raises(ValueError, match="dims"):
        latent_append(q, c, k, arena, n, n, dims=32, base=1e6)
    with pytest.raises(ValueError, match="contiguous rows"):
        latent_append(None, c.t().contiguous().t(), k, arena, n, n, dims=64, base=1e6)
    with pytest.raises(ValueError, match="arena's columns"):
        latent_append(None, c[:, :256], k, arena, n, n, dims=64, base=1e6)
