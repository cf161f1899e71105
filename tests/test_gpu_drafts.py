"""drafts.tree_attention and drafts.commit_drafts against plain restatements in 64
bits, with the tolerance of oracle.many_tokens.attention_tolerance."""

import numpy as np
import pytest
import torch

from instinct_amd import drafts
from oracle import many_tokens as plain

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def dev(a, dtype=np.int32):
    return torch.as_tensor(np.asarray(a).astype(dtype), device="cuda")


def random_tree(rng, n):
    return [-1] + [int(rng.integers(max(0, i - 9), i)) for i in range(1, n)] if n else []


class Case:
    def __init__(self, seed, held, nodes, heads, dtype, *, page=16, layout="pages", bits=16,
                 behind=0, masks=None):
        rng = np.random.default_rng(seed)
        gen = torch.Generator().manual_seed(seed)
        hq, hk, dim = heads
        need = [-(-(h + min(n, 64)) // page) for h, n in zip(held, nodes)]
        pages = sum(need) + 3
        order = rng.permutation(pages)
        self.tables = np.zeros((len(held), max(need, default=0) + 2), dtype=np.int64)
        at = 0
        for b, n in enumerate(need):
            self.tables[b, :n] = order[at:at + n]
            at += n
        shape = (pages * page, hk, dim)
        self.page, self.layout, self.bits, self.dtype = page, layout, bits, dtype
        self.host, self.stores, self.scales = [], [], []
        for _ in range(2):
            if bits == 8:
                rows = torch.randint(-127, 128, shape, generator=gen, dtype=torch.int8)
                scale = ((torch.rand(shape[:2], generator=gen) + 0.5) / 64).half()
                self.host.append((rows.double() * scale.double()[..., None]).numpy())
                self.scales.append(self._lay(scale))
            else:
                rows = torch.randn(shape, generator=gen).to(dtype)
                self.host.append(rows.double().numpy())
            self.stores.append(self._lay(rows))
        self.held, self.nodes = np.asarray(held), np.asarray(nodes)
        self.starts = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int64)
        total = int(self.starts[-1])
        self.parents = [p for n in nodes for p in random_tree(rng, n)]
        if masks is None:
            masks = [m for a, z in zip(self.starts, self.starts[1:])
                     for m in plain.ancestors(self.parents[a:z])]
        self.masks = np.array(list(masks) + [0] * behind, dtype=np.uint64)
        self.q = torch.randn((total + behind, hq, dim), generator=gen).to(dtype).cuda()

    def _lay(self, rows):
        if self.layout == "rows":
            return rows.cuda()
        tiles = rows.view(-1, self.page, *rows.shape[1:]).transpose(1, 2)
        return tiles.contiguous().cuda()

    def run(self, **kw):
        return drafts.tree_attention(
            self.q, *self.stores, dev(self.tables), dev(self.held), dev(self.starts),
            dev(self.masks.view(np.int64), np.int64), page_size=self.page,
            scales=tuple(self.scales) or None, **kw)

    def check(self, got=None, **kw):
        kw = dict(dict(scale=0.1), **kw)
        got = self.run(**kw) if got is None else got
        want, size = plain.trees(self.q.double().cpu().numpy(), *self.host, self.tables, self.held,
                                 self.starts, [int(m) for m in self.masks], page_size=self.page,
                                 **kw)
        tol = plain.attention_tolerance(want, size, self.host[1], int(self.held.max()) + 64,
                                        self.dtype, self.bits == 8)
        off = np.abs(got.double().cpu().numpy() - want)
        worst = np.unravel_index(np.argmax(off - tol), off.shape)
        assert np.all(off <= tol), (worst, off[worst], tol[worst], want[worst])
        return got


HEADS = [(14, 2, 64), (28, 4, 128), (8, 8, 96), (6, 2, 256), (4, 1, 80), (3, 1, 8)]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_against_64_bits(gpu, heads, dtype, bits):
    Case(1, [100, 0, 333, 64, 1], [16, 3, 1, 9, 0], heads, dtype, bits=bits).check()


@pytest.mark.parametrize("page, layout", [(1, "pages"), (7, "rows"), (16, "rows"), (64, "pages"),
                                          (100, "pages"), (256, "rows")])
@pytest.mark.parametrize("bits", [16, 8])
def test_pages_and_layouts(gpu, page, layout, bits):
    Case(2, [130, 63, 257], [20, 5, 64], (8, 2, 64), BF16, page=page, layout=layout,
         bits=bits).check()


@pytest.mark.parametrize("held, nodes, heads", [
    ([0], [1], (4, 4, 64)), ([0, 0], [64, 2], (8, 2, 128)), ([63], [2], (4, 2, 64)),
    ([64], [1], (4, 2, 64)), ([65], [64], (16, 1, 64)), ([5000], [12], (14, 2, 64)),
    ([9000, 10, 4000], [64, 1, 33], (8, 1, 128)), ([1500], [64], (32, 1, 64)),
    ([20000], [4], (2, 2, 256)), ([0, 700, 0, 3], [0, 8, 0, 0], (4, 2, 64)),
    ([700], [150], (4, 2, 64)), ([40], [100], (28, 4, 128))], ids=str)
def test_lengths(gpu, held, nodes, heads):
    Case(3, held, nodes, heads, F16).check()


def test_many_sequences(gpu):
    rng = np.random.default_rng(4)
    Case(4, rng.integers(0, 300, 400), rng.integers(0, 10, 400), (2, 2, 64), F16).check()


@pytest.mark.parametrize("kw", [
    dict(window=1), dict(window=3), dict(window=50), dict(window=64), dict(window=300),
    dict(window=1 << 30), dict(softcap=3.0), dict(softcap=30.0, window=20), dict(scale=-0.2),
    dict(scale=0.0)], ids=str)
@pytest.mark.parametrize("bits", [16, 8])
def test_windows_softcaps_scales(gpu, kw, bits):
    Case(5, [400, 30, 1000], [40, 64, 7], (8, 2, 128), F16, bits=bits).check(**kw)


def test_any_mask(gpu):
    """Masks that are no tree's: nothing, everything, later nodes, nodes that are not there."""
    masks = [0, (1 << 64) - 1, 1 << 63, 0b1010, 0, (1 << 64) - 1, 7, 1]
    case = Case(6, [70, 0], [4, 4], (4, 2, 64), F16, masks=masks)
    got = case.check()
    assert not got[4].any()  # sees nothing
    case.check(window=2)


def test_rows_behind_the_last_sequence_are_zeros(gpu):
    case = Case(7, [70, 200], [4, 9], (4, 2, 80), F16, behind=50)
    out = torch.full_like(case.q, float("nan"))
    assert case.run(scale=0.1, out=out) is out
    assert not out[13:].any()
    case.check(got=out)
    empty = Case(7, [], [], (4, 2, 64), F16, behind=5)
    assert not empty.run(scale=0.1).any()


def test_released_and_foreign_pages(gpu):
    """Pages that are negative or past the arena hide their keys, whatever is in row 0."""
    for bits in (16, 8):
        case = Case(8, [200, 40], [6, 6], (4, 2, 64), F16, bits=bits)
        case.tables[0, 2:5] = -1
        case.tables[0, 7] = 1 << 30
        case.tables[1, 0] = -5
        case.check()
        case.tables[:] = -1
        assert not case.run(scale=0.1).any()


def test_table_shorter_than_the_length(gpu):
    case = Case(9, [200, 40], [6, 6], (4, 2, 64), F16)
    case.held[0] = 10_000  # the table's pages are what there is
    got = case.run(scale=0.1)
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")], ids=str)
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dim", [64, 128, 256, 80])
def test_what_is_not_finite_reaches_those_that_see_it(gpu, dim, bits, bad):
    """Neither a node that is not seen, nor a row behind the last node, nor one out of
    the window changes anything, whatever its key and value hold."""
    case = Case(10, [150, 90], [8, 3], (4, 2, dim), F16, bits=bits, layout="rows")
    clean = case.run(scale=0.1, window=64)

    def spoil(b, position, where):
        row = case.tables[b, position // 16] * 16 + position % 16
        if bits == 8:
            case.scales[where][row] = bad
        else:
            case.stores[where][row, :, 1] = bad
        return case.run(scale=0.1, window=64)

    for where in (0, 1):
        # Out of the window, and behind the last node.
        assert torch.equal(spoil(0, 3, where), clean)
        assert torch.equal(spoil(0, 158, where), clean)
        assert torch.equal(spoil(1, 93, where), clean)
    node = 3
    sees = torch.tensor([bool(int(m) >> node & 1) for m in case.masks[:8]])
    got = spoil(0, 150 + node, 1)
    assert torch.equal(got[:8][~sees], clean[:8][~sees]) and torch.equal(got[8:], clean[8:])
    assert not torch.isfinite(got[:8][sees][..., 1]).any()
    if bits == 16:
        assert torch.equal(got[..., 2:], clean[..., 2:])
    got = spoil(0, 150 + node, 0)
    assert torch.equal(got[:8][~sees], clean[:8][~sees]) and torch.equal(got[8:], clean[8:])


def test_repeated_captured_and_other_streams(gpu):
    case = Case(11, [3000, 77, 512], [16, 64, 3], (28, 4, 128), BF16)
    args = (case.q, *case.stores, dev(case.tables), dev(case.held), dev(case.starts),
            dev(case.masks.view(np.int64), np.int64))
    kw = dict(page_size=16, scale=0.09)
    first = drafts.tree_attention(*args, **kw)
    ws = torch.empty(drafts.tree_workspace_bytes(128), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        drafts.tree_attention(*args, out=out, workspace=ws, **kw)
    for _ in range(4):
        out.zero_()
        ws.fill_(255)
        graph.replay()
        assert torch.equal(out, first)
        assert torch.equal(drafts.tree_attention(*args, **kw), first)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = drafts.tree_attention(*args, **kw)
    stream.synchronize()
    assert torch.equal(again, first)


def test_one_node_is_a_decode_step(gpu):
    """A tree of the newest token alone is what the decode call computes."""
    from instinct_amd.hip_kernels import paged_decode_attention

    case = Case(12, [300, 0, 4000], [1, 1, 1], (28, 4, 128), F16)
    want = paged_decode_attention(case.q, *case.stores, dev(case.tables), dev(case.held + 1),
                                  page_size=16, longest=4001, scale=0.09)
    got = case.check(scale=0.09)
    assert (got - want).abs().max() < 4e-3


def test_refusals(gpu):
    case = Case(13, [20], [4], (4, 2, 64), F16)
    base = dict(queries=case.q, keys=case.stores[0], values=case.stores[1], tables=dev(case.tables),
                lengths=dev(case.held), starts=dev(case.starts),
                masks=dev(case.masks.view(np.int64), np.int64), page_size=16, scale=0.1)

    def refuses(kind, **kw):
        with pytest.raises(kind):
            drafts.tree_attention(**dict(base, **kw))

    refuses(TypeError, queries=case.q.float())
    refuses(TypeError, queries=case.q.bfloat16())
    refuses(ValueError, queries=case.q[:, :3].contiguous())
    refuses(ValueError, queries=case.q.transpose(0, 1))
    refuses(ValueError, masks=base["masks"].int())
    refuses(ValueError, masks=base["masks"][:2])
    refuses(TypeError, lengths=base["lengths"].long())
    refuses(ValueError, starts=base["starts"][:1])
    refuses(ValueError, page_size=32)
    refuses(ValueError, out=torch.empty(4, 4, 32, dtype=F16, device="cuda"))
    refuses(ValueError, workspace=torch.empty(100, dtype=torch.uint8, device="cuda"))
    refuses(ValueError, tables=base["tables"].cpu())


# ---------------------------------------------------------------------------
# Commitment.

def commit_case(seed, held, nodes, *, vocabulary, int64=True):
    rng = np.random.default_rng(seed)
    parents = [p for n in nodes for p in random_tree(rng, n)] + [-1, 0, 5]
    drafted = rng.integers(0, vocabulary, len(parents))
    targets = rng.integers(0, vocabulary, len(parents))
    starts = np.concatenate([[0], np.cumsum(nodes)])
    for a, n in zip(starts, nodes):  # the model agrees with the line of a late node
        node = min(n, 64) - 1
        while node > 0 and parents[a + node] >= 0:
            targets[a + parents[a + node]] = drafted[a + node]
            node = parents[a + node]
    kind = np.int64 if int64 else np.int32
    return (np.asarray(held), starts, parents, drafted.astype(kind), targets.astype(kind))


@pytest.mark.parametrize("layout", ["pages", "rows"])
@pytest.mark.parametrize("heads, bits, page", [
    ((2, 64), 16, 16), ((4, 128), 16, 16), ((2, 64), 8, 16), ((3, 80), 16, 7), ((8, 256), 16, 32),
    ((1, 8), 8, 1), ((5, 7), 16, 16), ((2, 9), 8, 5), ((1, 512), 16, 16)])
@pytest.mark.parametrize("layers", [1, 3])
def test_commit(gpu, heads, bits, page, layout, layers):
    held, nodes = [0, 5, 77, 300, 31, 9], [64, 1, 20, 0, 70, 33]
    kv_heads, dim = heads
    case = commit_case(dim + page, held, nodes, vocabulary=9, int64=layers == 1)
    rng = np.random.default_rng(dim)
    need = [-(-(h + n) // page) + 1 for h, n in zip(held, nodes)]
    order = rng.permutation(sum(need))
    tables = np.full((len(held), max(need)), -1)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = order[at:at + n]
        at += n
    tables[4, -1] = -1
    rows = sum(need) * page
    host, arenas = [], []
    for _ in range(layers):
        layer = []
        for s in range(2 if bits == 16 else 4):
            shape = (rows, kv_heads, dim) if s < 2 else (rows, kv_heads)
            kind = torch.int8 if bits == 8 and s < 2 else F16
            layer.append(torch.as_tensor(rng.integers(-100, 100, shape)).to(kind))
        host.append(layer)
        lay = lambda x: x if layout == "rows" else x.view(  # noqa: E731
            -1, page, *x.shape[1:]).transpose(1, 2).contiguous()
        arenas.append(tuple(lay(x).cuda() for x in layer))
    got = drafts.commit_drafts(arenas, dev(tables), dev(held), dev(case[1]), dev(case[2]),
                               torch.as_tensor(case[3]).cuda(), torch.as_tensor(case[4]).cuda(),
                               page_size=page)
    want = plain.commit(*case)
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        np.testing.assert_array_equal(x.cpu().numpy(), y)
    assert sorted(want[1])[-2] > 3  # (lines of some length)
    for layer, arena in zip(host, arenas):
        for x, store in zip(layer, arena):
            rows = x.clone()
            for b, path in enumerate(want[2]):
                for i, node in enumerate(path):
                    if node >= 0:
                        place = lambda p: tables[b, p // page] * page + p % page  # noqa: E731
                        rows[place(held[b] + i)] = x[place(held[b] + node)]
            flat = store if layout == "rows" else store.transpose(1, 2).flatten(0, 1)
            assert torch.equal(flat.cpu(), rows)


def test_commit_past_48_layers(gpu):
    case = commit_case(1, [3], [6], vocabulary=1)
    arenas = [tuple(torch.randn(4, 2, 16, 64, device="cuda").half() for _ in range(2))
              for _ in range(50)]
    before = [tuple(x.clone() for x in a) for a in arenas]
    got = drafts.commit_drafts(arenas, dev([[2, 0]]), dev([3]), dev(case[1]), dev(case[2]),
                               torch.as_tensor(case[3]).cuda(), torch.as_tensor(case[4]).cuda(),
                               page_size=16)
    path = [int(x) for x in got.path[0] if x >= 0]
    assert len(path) > 1
    for a, b in zip(arenas, before):
        for x, y in zip(a, b):
            y[2, :, 3:3 + len(path)] = y[2, :, [3 + n for n in path]]
            assert torch.equal(x, y)


def test_commit_refusals_and_bad_pages(gpu):
    case = commit_case(2, [3], [6], vocabulary=1)
    arena = tuple(torch.randn(4, 2, 16, 64, device="cuda").half() for _ in range(2))
    base = dict(arenas=[arena], tables=dev([[2, 0]]), lengths=dev([3]), starts=dev(case[1]),
                parents=dev(case[2]), drafted=torch.as_tensor(case[3]).cuda(),
                targets=torch.as_tensor(case[4]).cuda(), page_size=16)

    def refuses(kind, **kw):
        with pytest.raises(kind):
            drafts.commit_drafts(**dict(base, **kw))

    refuses(ValueError, arenas=[])
    refuses(ValueError, arenas=[arena, arena])
    refuses(ValueError, arenas=[arena[:1]])
    refuses(TypeError, targets=base["targets"].int())
    refuses(TypeError, drafted=base["drafted"].float())
    refuses(ValueError, targets=base["targets"][:2])
    refuses(ValueError, starts=dev([0]))
    good = drafts.commit_drafts(**base)
    with pytest.raises(Exception, match="out_lengths"):
        drafts.commit_drafts(**dict(base, out=good._replace(lengths=base["lengths"])))
    before = arena[0].clone()
    for tables in ([[-1, 0]], [[4, 0]]):
        got = drafts.commit_drafts(**dict(base, tables=dev(tables)))
        assert torch.equal(got.path, good.path) and torch.equal(arena[0], before)
