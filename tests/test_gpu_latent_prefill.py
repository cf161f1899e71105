"""Latent prefill attention on the GPU against the float64 oracle, and the
latent calls as a model makes them."""

import pytest
import torch
from test_gpu_latent import SMALL, THIN, TYPES, UNEVEN, WIDE, layer, pack

from oracle import latent as oracle

pytestmark = pytest.mark.gpu


def check(gpu, shape, heads, start, count, *, page=16, dtype=torch.bfloat16, change=None,
          scale=None, **kw):
    from instinct_amd.latent import latent_prefill_attention

    latent, rope, nope, value = shape
    end = start + count
    pages = -(-end // page) + 2
    arena, kv_b, g = layer(shape, heads, pages * page, dtype, seed=count)
    table = pack([end], page, pages, g)[0]
    if change:
        change(arena, table)
    q = torch.randn((count, heads, nope + rope), generator=g).to(dtype)
    scale = scale or (nope + rope) ** -0.5
    got = latent_prefill_attention(q.to(gpu), arena.to(gpu), kv_b.to(gpu), table.to(gpu),
                                   start=start, page_size=page, scale=scale, **kw)
    want, bound = oracle.prefill(q, arena, kv_b, table, start=start, page_size=page, scale=scale)
    over = (got.cpu().double() - want).abs() - bound
    assert bool((over <= 0).all()), f"past the bound by {over.max():.3e}"
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape, heads", [(WIDE, 3), (WIDE, 9), (SMALL, 14), (UNEVEN, 5), (THIN, 1),
                                          ((264, 16, 40, 24), 17), ((512, 0, 128, 64), 2),
                                          ((72, 64, 8, 128), 2)])
def test_shapes(gpu, shape, heads, dtype):
    check(gpu, shape, heads, 61, 150, dtype=dtype)


@pytest.mark.parametrize("start, count", [(0, 1), (0, 2), (63, 1), (64, 1), (0, 64), (0, 65),
                                          (1, 127), (0, 128), (0, 129), (700, 3), (300, 257)])
def test_lengths(gpu, start, count):
    check(gpu, SMALL, 2, start, count, dtype=torch.float16)


@pytest.mark.parametrize("page", [1, 7, 48, 64])
def test_pages(gpu, page):
    check(gpu, SMALL, 3, 100, 90, page=page)


def test_split_key_ranges(gpu):
    """Few query tiles over a long prefix: the key ranges are split and joined;
    the first queries' last ranges are empty."""
    check(gpu, SMALL, 2, 3000, 140)
    check(gpu, WIDE, 1, 1500, 20, dtype=torch.float16)


# The kernel of two query blocks a wave: wide heads, 256 queries and 1024 keys at
# least.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape, heads, start, count", [
    (WIDE, 2, 0, 1100), (WIDE, 1, 767, 257), (UNEVEN, 9, 801, 256), ((512, 0, 72, 128), 2, 300, 800)])
def test_two_blocks(gpu, shape, heads, start, count, dtype):
    check(gpu, shape, heads, start, count, dtype=dtype)


def test_two_blocks_split(gpu):
    """Key ranges that no query of a wave sees, and ones that some do."""
    check(gpu, WIDE, 1, 4000, 300, dtype=torch.float16)


@pytest.mark.parametrize("count", [1030, 1300])
def test_two_blocks_paired(gpu, count):
    """Two query tiles a workgroup, an odd number of tiles and an even one."""
    check(gpu, (8, 16, 72, 8), 130, 0, count, page=64)


def test_two_blocks_masked(gpu):
    def change(arena, table):
        arena[:16] = float("inf")  # page 0, that -1 must not lead to
        table[table == 0] = -1
        table[0], table[1], table[30], table[40] = -1, 1 << 20, -9, 1 << 30
        table[-2] = -1

    got = check(gpu, (64, 16, 96, 40), 2, 0, 1100, change=change)
    assert bool((got[:32] == 0).all())


@pytest.mark.parametrize("scale", [-0.05, 0.6])
def test_two_blocks_scales(gpu, scale):
    """A negative scale, and scores that move the running maximum."""
    check(gpu, (256, 32, 128, 72), 2, 500, 530, scale=scale, dtype=torch.float16)


def test_head_groups(gpu):
    """More heads than fit the bound on expanded rows: groups of heads in turn."""
    from instinct_amd import _lib

    start, count, heads = 32900, 3, 130
    per_head = -(-(start + count) // 64) * 64 * 2 * (64 + 64)
    assert per_head * heads > 1 << 30 > per_head * 8
    assert _lib.latent_prefill_workspace_bytes(start, count, heads, 0, 8, 8) < per_head * heads
    check(gpu, THIN, heads, start, count)


def test_far_prefix(gpu):
    """More tiles of tokens than a launch's second dimension holds, most of them
    on released pages: the same as the pages that are left alone."""
    from instinct_amd.latent import latent_prefill_attention

    page, start, count = 64, 65536 * 128 + 100, 3
    arena, kv_b, g = layer(THIN, 2, 4 * page, torch.float16)
    table = torch.full((-(-(start + count) // page),), -1, dtype=torch.int32)
    table[0], table[1000], table[-1] = 2, 0, 3
    q = torch.randn((count, 2, 8), generator=g).to(torch.float16)
    got = latent_prefill_attention(q.to(gpu), arena.to(gpu), kv_b.to(gpu), table.to(gpu),
                                   start=start, page_size=page, scale=0.35)
    want, bound = oracle.prefill(q, arena, kv_b, torch.tensor([2, 0, 3]),
                                 start=2 * page + start % page, page_size=page, scale=0.35)
    assert bool(((got.cpu().double() - want).abs() <= bound).all())


def test_masked_pages(gpu):
    """Released and unknown pages hide their keys whatever the rows hold;
    queries with nothing left give zeros."""
    def change(arena, table):
        arena[:16] = float("nan")  # page 0, that -1 must not lead to
        table[table == 0] = -1
        table[0], table[1], table[4] = -1, 1 << 20, -9

    got = check(gpu, SMALL, 3, 0, 150, change=change)
    assert bool((got[:32] == 0).all())


def test_short_table(gpu):
    """Keys past the table are hidden."""
    check(gpu, SMALL, 2, 20, 100, change=lambda arena, table: table.resize_(4))


def test_rows_past_the_chunk(gpu):
    def change(arena, table):
        arena.view(-1, 16, arena.shape[1])[table[-1].long(), 15:] = float("inf")

    check(gpu, WIDE, 2, 40, 103, change=change)


@pytest.mark.parametrize("scale", [-0.05, 0.4])
def test_scales(gpu, scale):
    check(gpu, SMALL, 2, 50, 100, scale=scale, dtype=torch.float16)


def test_repeats(gpu):
    assert torch.equal(check(gpu, WIDE, 3, 900, 60), check(gpu, WIDE, 3, 900, 60))


def test_refusals(gpu):
    from instinct_amd import _lib
    from instinct_amd.latent import latent_prefill_attention as call

    q = torch.zeros((2, 4, 192), dtype=torch.float16, device=gpu)
    arena = torch.zeros((64, 576), dtype=torch.float16, device=gpu)
    kv_b = torch.zeros((4, 256, 512), dtype=torch.float16, device=gpu)
    table = torch.zeros(4, dtype=torch.int32, device=gpu)
    kw = dict(start=0, page_size=16, scale=0.1)
    with pytest.raises(TypeError):
        call(q, arena, kv_b.bfloat16(), table, **kw)
    with pytest.raises(ValueError, match="heads"):
        call(q[:, :2].contiguous(), arena, kv_b, table, **kw)
    with pytest.raises(ValueError, match="table"):
        call(q, arena, kv_b, table.long(), **kw)
    with pytest.raises(ValueError, match="no pages"):
        call(q, arena, kv_b, table[:0], **kw)
    with pytest.raises(ValueError, match="out must"):
        call(q, arena, kv_b, table, out=q, **kw)
    with pytest.raises(ValueError, match="workspace"):
        call(q, arena, kv_b, table, workspace=torch.empty(8, dtype=torch.uint8, device=gpu), **kw)
    with pytest.raises(_lib.PdaError):
        call(q, arena, kv_b, table, start=-1, page_size=16, scale=0.1)
    assert call(q[:0], arena, kv_b, table, **kw).shape == (0, 4, 128)


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_then_steps(gpu, dtype):
    """A prompt in two chunks, then decode steps of a batch, append and
    attention each, against float64 over what the arena holds; and the prompt's
    last token in both forms."""
    from instinct_amd.latent import (latent_append, latent_decode_attention,
                                     latent_prefill_attention)

    latent, rope, nope, value = WIDE
    heads, page = 6, 16
    arena, kv_b, g = layer(WIDE, heads, 40 * page, dtype)
    store, up = arena.to(gpu), kv_b.to(gpu)
    weight = (1 + 0.1 * torch.randn(latent, generator=g)).to(dtype).to(gpu)
    order = torch.randperm(40, generator=g).int()
    tables = order[:30].view(2, 15).contiguous()
    scale = (nope + rope) ** -0.5

    def append(positions, table_rows, count):
        down = torch.randn((count, latent + rope), generator=g).to(dtype).to(gpu)
        q = torch.randn((count, heads, nope + rope), generator=g).to(dtype).to(gpu)
        rows = torch.tensor([int(t[p // page]) * page + p % page
                             for t, p in zip(table_rows, positions)], dtype=torch.int32)
        return latent_append(q, down[:, :latent], down[:, latent:], store,
                             torch.tensor(positions, dtype=torch.int32, device=gpu), rows.to(gpu),
                             dims=rope, base=1e6, norm_weight=weight, q_out=q)

    held = [0, 0]
    for b, chunks in enumerate(([70, 41], [100])):
        for count in chunks:
            q = append(list(range(held[b], held[b] + count)), [tables[b]] * count, count)
            got = latent_prefill_attention(q, store, up, tables[b].to(gpu), start=held[b],
                                           page_size=page, scale=scale).cpu().double()
            want, bound = oracle.prefill(q.cpu(), store.cpu(), kv_b, tables[b], start=held[b],
                                         page_size=page, scale=scale)
            assert bool(((got - want).abs() <= bound).all())
            held[b] += count
        n = torch.tensor([held[b]], dtype=torch.int32, device=gpu)
        other = latent_decode_attention(q[-1:].contiguous(), store, up, tables[b:b + 1].to(gpu), n,
                                        page_size=page, longest=held[b], scale=scale)
        _, near = oracle.decode(q[-1:].cpu(), store.cpu(), kv_b, tables[b:b + 1], [held[b]],
                                page_size=page, scale=scale)
        assert bool(((other[0].cpu().double() - got[-1]).abs() <= near[0] + bound[-1]).all())
    for _ in range(3):
        q = append(held, tables, 2)
        held = [n + 1 for n in held]
        got = latent_decode_attention(q, store, up, tables.to(gpu),
                                      torch.tensor(held, dtype=torch.int32, device=gpu),
                                      page_size=page, longest=max(held), scale=scale)
        want, bound = oracle.decode(q.cpu(), store.cpu(), kv_b, tables, held, page_size=page,
                                    scale=scale)
        assert bool(((got.cpu().double() - want).abs() <= bound).all())


def test_captured_step(gpu):
    """Append and both attentions in a graph: every replay gives the eager
    results, with eager calls on the same stream workspace between them."""
    from instinct_amd.hip_kernels import new_workspace
    from instinct_amd.latent import (latent_append, latent_decode_attention,
                                     latent_decode_workspace_bytes, latent_prefill_attention,
                                     latent_prefill_workspace_bytes)

    latent, rope, nope, value = SMALL
    arena, kv_b, g = layer(SMALL, 8, 40 * 16, torch.float16)
    store, up = arena.to(gpu), kv_b.to(gpu)
    tables = torch.randperm(40, generator=g).int().view(2, 20).to(gpu)
    positions = torch.tensor([299, 77], dtype=torch.int32, device=gpu)
    lengths = positions + 1
    rows = (tables[torch.arange(2), (positions // 16).long()] * 16 + positions % 16).int()
    down = torch.randn((2, latent + rope), generator=g).half().to(gpu)
    q = torch.randn((2, 8, nope + rope), generator=g).half().to(gpu)
    q2 = torch.randn((40, 8, nope + rope), generator=g).half().to(gpu)
    rot, out = torch.empty_like(q), torch.empty((2, 8, value), dtype=torch.float16, device=gpu)
    out2 = torch.empty((40, 8, value), dtype=torch.float16, device=gpu)
    ws = new_workspace(latent_decode_workspace_bytes((2, 8, nope + rope), store, up, page_size=16,
                                                     table_width=20, longest=320), gpu)
    ws2 = new_workspace(latent_prefill_workspace_bytes(260, (40, 8, nope + rope), store, up), gpu)

    def run(**kw):
        latent_append(q, down[:, :latent], down[:, latent:], store, positions, rows, dims=rope,
                      base=1e6, q_out=rot)
        latent_decode_attention(rot, store, up, tables, lengths, page_size=16, longest=320,
                                scale=0.1, out=out, workspace=kw.get("a"))
        latent_prefill_attention(q2, store, up, tables[0], start=260, page_size=16, scale=0.1,
                                 out=out2, workspace=kw.get("b"))

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(a=ws, b=ws2)
    for _ in range(3):
        q.copy_(torch.randn(q.shape, generator=g).half())
        down.copy_(torch.randn(down.shape, generator=g).half())
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (rot, out, out2, store)]
        run()
        torch.cuda.synchronize()
        for a, b in zip(got, (rot, out, out2, store)):
            assert torch.equal(a, b)


def test_two_streams(gpu):
    """Calls of two shapes under way on two streams at once."""
    from instinct_amd.latent import latent_decode_attention

    cases = []
    for shape, heads, n in ((WIDE, 64, 3000), (SMALL, 16, 5000)):
        arena, kv_b, g = layer(shape, heads, 320 * 16, torch.bfloat16)
        q = torch.randn((1, heads, shape[1] + shape[2]), generator=g).bfloat16()
        dev = [t.to(gpu) for t in (q, arena, kv_b, torch.randperm(320, generator=g).int()[None])]
        cases.append((dev, torch.tensor([n], dtype=torch.int32, device=gpu), n))
    call = lambda dev, n, longest: latent_decode_attention(  # noqa: E731
        *dev, n, page_size=16, longest=longest, scale=0.08)
    want = [call(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(5):
        for i, c in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i].append(call(*c))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(w, x) for x in outs)
