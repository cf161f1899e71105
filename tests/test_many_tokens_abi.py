"""The calls of steps with many tokens a sequence validate their arguments on the host
(every rejected call returns before touching HIP); what they share with the plain
restatements is checked on small cases by hand."""

import ctypes

import numpy as np
import pytest

from instinct_amd import _lib
from oracle import many_tokens as plain

FAKE = 0x10000
BAD, ALIGN, LONG = (_lib.PDA_ERR_INVALID_ARGUMENT, _lib.PDA_ERR_ALIGNMENT, _lib.PDA_ERR_TOO_LONG)


def rejected(code, want):
    assert code == want
    assert _lib.library().pda_last_error().decode() != ""


def extend(**overrides):
    args = dict(tables=FAKE, table_stride=64, lengths=FAKE, counts=FAKE, pages=FAKE, feed=FAKE,
                feed_len=10, drawn=FAKE, parents=FAKE, batch=2, page_size=16, tokens=100,
                starts=FAKE, out_lengths=FAKE, out_pages=FAKE, out_drawn=FAKE, rows=FAKE,
                positions=FAKE, masks=FAKE, stream=None)
    args.update(overrides)
    return _lib.library().pda_extend_tables(*args.values())


@pytest.mark.parametrize("overrides, code", [
    (dict(batch=-1), BAD), (dict(batch=4097), LONG), (dict(table_stride=0), BAD),
    (dict(feed_len=-1), BAD), (dict(page_size=0), BAD), (dict(tokens=-1), BAD),
    (dict(tables=None), BAD), (dict(feed=None), BAD), (dict(drawn=None), BAD),
    (dict(starts=None), BAD), (dict(rows=None), BAD), (dict(positions=None), BAD),
    (dict(masks=None), BAD), (dict(out_pages=None), BAD), (dict(counts=FAKE + 2), ALIGN),
    (dict(rows=FAKE + 1), ALIGN), (dict(masks=FAKE + 4), ALIGN)])
def test_extend_rejects(overrides, code):
    rejected(extend(**overrides), code)


def packed(**overrides):
    args = dict(q=FAKE, q_token=3584, q_head=128, k=FAKE, k_token=512, k_head=128, v=FAKE,
                v_token=512, v_head=128, starts=FAKE, out=FAKE, tokens=100, batch=2, q_heads=28,
                kv_heads=4, head_dim=128, scale=0.1, window=0, softcap=0.0, stream=None)
    args.update(overrides)
    return _lib.library().pda_packed_prompt_attention(*args.values())


@pytest.mark.parametrize("overrides, code", [
    (dict(tokens=-1), BAD), (dict(batch=-1), BAD), (dict(q_heads=0), BAD), (dict(kv_heads=0), BAD),
    (dict(q_heads=30), _lib.PDA_ERR_HEAD_RATIO), (dict(head_dim=0), _lib.PDA_ERR_HEAD_DIM),
    (dict(head_dim=100), _lib.PDA_ERR_HEAD_DIM), (dict(head_dim=264), _lib.PDA_ERR_HEAD_DIM),
    (dict(window=-1), BAD), (dict(scale=float("nan")), BAD), (dict(scale=float("inf")), BAD),
    (dict(softcap=-1.0), BAD), (dict(q=None), BAD), (dict(v=None), BAD), (dict(starts=None), BAD),
    (dict(out=None), BAD), (dict(q=FAKE + 8), ALIGN), (dict(out=FAKE + 2), ALIGN),
    (dict(k_token=516), ALIGN), (dict(v_head=-128), ALIGN), (dict(starts=FAKE + 2), ALIGN),
    (dict(tokens=(1 << 31) - 1), LONG)])
def test_packed_rejects(overrides, code):
    rejected(packed(**overrides), code)


def tree(**overrides):
    args = dict(q=FAKE, k=FAKE, v=FAKE, tables=FAKE, lengths=FAKE, starts=FAKE, masks=FAKE,
                out=FAKE, tokens=100, batch=2, q_heads=28, kv_heads=4, head_dim=128, page_size=16,
                table_stride=64, arena_rows=4096, layout=_lib.PDA_LAYOUT_PAGES, scale=0.1,
                window=0, softcap=0.0, workspace=FAKE, workspace_bytes=1 << 32, stream=None)
    args.update(overrides)
    return _lib.library().pda_tree_attention(*args.values())


@pytest.mark.parametrize("overrides, code", [
    (dict(tokens=-1), BAD), (dict(batch=-1), BAD), (dict(q_heads=0), BAD), (dict(page_size=0), BAD),
    (dict(q_heads=30), _lib.PDA_ERR_HEAD_RATIO), (dict(head_dim=12), _lib.PDA_ERR_HEAD_DIM),
    (dict(head_dim=512), _lib.PDA_ERR_HEAD_DIM), (dict(window=-1), BAD), (dict(layout=2), BAD),
    (dict(arena_rows=8), BAD), (dict(table_stride=0), BAD), (dict(scale=float("nan")), BAD),
    (dict(softcap=float("inf")), BAD), (dict(page_size=1 << 24), BAD), (dict(k=None), BAD),
    (dict(masks=None), BAD), (dict(q=FAKE + 8), ALIGN), (dict(masks=FAKE + 4), ALIGN),
    (dict(lengths=FAKE + 2), ALIGN), (dict(workspace=None), _lib.PDA_ERR_WORKSPACE),
    (dict(workspace_bytes=1000), _lib.PDA_ERR_WORKSPACE),
    (dict(workspace=FAKE + 16), _lib.PDA_ERR_WORKSPACE), (dict(tokens=1 << 30), LONG)])
def test_tree_rejects(overrides, code):
    rejected(tree(**overrides), code)


def test_tree_workspace():
    size = ctypes.c_size_t(0)
    call = _lib.library().pda_tree_workspace_bytes
    assert call(128, ctypes.byref(size)) == 0 and size.value % 256 == 0
    rejected(call(10, ctypes.byref(size)), _lib.PDA_ERR_HEAD_DIM)
    rejected(call(128, None), BAD)


def commit(**overrides):
    stores = overrides.pop("stores", [FAKE, 2 * FAKE])
    args = dict(stores=None if stores is None else (ctypes.c_void_p * len(stores))(*stores),
                layers=1, stores_per_layer=2, width=256, tables=FAKE, lengths=FAKE, starts=FAKE,
                parents=FAKE, drafted=FAKE, targets=FAKE, token_bytes=8, out_lengths=2 * FAKE,
                accepted=FAKE, path=FAKE, following=FAKE, tokens=10, batch=2, kv_heads=4,
                page_size=16, table_stride=8, arena_rows=4096, layout=_lib.PDA_LAYOUT_ROWS,
                stream=None)
    args.update(overrides)
    return _lib.library().pda_commit_drafts(*args.values())


@pytest.mark.parametrize("overrides, code", [
    (dict(layers=0), BAD), (dict(stores_per_layer=3), BAD), (dict(width=0), BAD),
    (dict(tokens=-1), BAD), (dict(batch=-1), BAD), (dict(kv_heads=0), BAD), (dict(page_size=0), BAD),
    (dict(table_stride=0), BAD), (dict(token_bytes=2), BAD), (dict(layout=2), BAD),
    (dict(arena_rows=8), BAD), (dict(stores=None), BAD), (dict(stores=[FAKE, None]), BAD),
    (dict(parents=None), BAD), (dict(following=None), BAD), (dict(out_lengths=FAKE), BAD),
    (dict(path=FAKE + 2), ALIGN), (dict(drafted=FAKE + 4), ALIGN), (dict(batch=1 << 18), LONG)])
def test_commit_rejects(overrides, code):
    rejected(commit(**overrides), code)


def test_nothing_to_do_is_accepted():
    assert packed(tokens=0) == 0 and tree(tokens=0) == 0 and commit(batch=0) == 0


def test_plain_tables_by_hand():
    got = plain.extend_tables([[7, 9, 0], [4, 0, 0]], [20, 3], [14, 2], [2, 1], [30, 31, 32],
                              [1, 0], page_size=16, tokens=18)
    assert got["tables"].tolist() == [[7, 9, 31], [4, 0, 0]]
    assert got["starts"].tolist() == [0, 14, 16] and got["drawn"].tolist() == [2, 0]
    assert got["rows"].tolist() == [9 * 16 + i for i in range(4, 16)] + [496, 497, 67, 68, -1, -1]
    assert got["positions"].tolist() == list(range(20, 34)) + [3, 4, 0, 0]


def test_plain_tree_by_hand():
    #   0 - 1 - 2
    #    \- 3 - 4
    parents = [-1, 0, 1, 0, 3]
    assert plain.ancestors(parents) == [1, 3, 7, 9, 25]
    lengths, accepted, path, following = plain.commit(
        [10], [0, 5], parents, [50, 51, 52, 51, 53], [51, 9, 9, 53, 77])
    # Of two children with the same token the first is kept.
    assert (lengths[0], accepted[0], path[0, :3].tolist(), following[0]) == (12, 2, [0, 1, -1], 9)
    lengths, accepted, path, following = plain.commit(
        [10], [0, 5], parents, [50, 51, 52, 54, 53], [54, 9, 9, 53, 77])
    assert (lengths[0], accepted[0], path[0, :4].tolist(), following[0]) == (13, 3, [0, 3, 4, -1], 77)


def test_plain_attention_by_hand():
    one = np.ones((3, 1, 8))
    v = np.arange(3.0)[:, None, None] * one
    out, _ = plain.packed_prompts(one, one, v, [0, 3], scale=1.0)
    np.testing.assert_allclose(out[:, 0, 0], [0.0, 0.5, 1.0])
    out, _ = plain.packed_prompts(one, one, v, [0, 3], scale=1.0, window=2)
    np.testing.assert_allclose(out[:, 0, 0], [0.0, 0.5, 1.5])
    # Two held rows and a tree of two siblings under node 0.
    rows = np.concatenate([one, one, one])[:5]
    v = np.arange(5.0)[:, None, None] * np.ones((5, 1, 8))
    out, _ = plain.trees(one, rows, v, [[0, 1, 2, 3, 4]], [2], [0, 3], [1, 3, 5], page_size=1,
                         scale=1.0)
    np.testing.assert_allclose(out[:, 0, 0], [1.0, 6 / 4, 7 / 4])
