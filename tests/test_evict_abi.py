"""The eviction calls validate their arguments on the host (no GPU call is
made: every rejected call returns before touching HIP), and KVCache.evict checks
what it is asked on the CPU."""

import numpy as np
import pytest
import torch

from instinct_amd import _lib, eviction
from instinct_amd.paged_kv import KVCache, KVGroup

FAKE = 0x10000


def weights(**overrides):
    args = dict(queries=FAKE, keys=FAKE, tables=FAKE, lengths=FAKE, weights=FAKE, out=FAKE, batch=2,
                q_heads=28, kv_heads=4, head_dim=128, page_size=16, table_stride=64,
                arena_rows=4096, layout=_lib.PDA_LAYOUT_PAGES, capacity=1024, longest=1000,
                scale=0.09, window=0, softcap=0.0, fresh=1, workspace=FAKE,
                workspace_bytes=1 << 30, stream=None)
    args.update(overrides)
    return _lib.library().pda_attention_weights(*args.values())


def select(**overrides):
    args = dict(weights=FAKE, out_weights=FAKE, tables=FAKE, lengths=FAKE, kept=FAKE,
                new_lengths=FAKE, batch=2, kv_heads=4, page_size=16, table_stride=64,
                arena_rows=4096, capacity=1024, out_capacity=1024, keep=512, recent=64, sinks=4,
                stream=None)
    args.update(overrides)
    return _lib.library().pda_evict_select(*args.values())


def move(**overrides):
    args = dict(arena=FAKE, arena2=FAKE, width=256, kept=FAKE, new_lengths=FAKE, tables=FAKE,
                out_tables=FAKE, batch=2, kv_heads=4, page_size=16, table_stride=64, out_stride=64,
                arena_rows=4096, layout=_lib.PDA_LAYOUT_PAGES, keep=512, stream=None)
    args.update(overrides)
    return _lib.library().pda_evict_move(*args.values())


BAD, ALIGN = _lib.PDA_ERR_INVALID_ARGUMENT, _lib.PDA_ERR_ALIGNMENT


@pytest.mark.parametrize("overrides, code", [
    (dict(batch=-1), BAD), (dict(batch=65536), BAD), (dict(kv_heads=0), BAD),
    (dict(q_heads=30), _lib.PDA_ERR_HEAD_RATIO), (dict(head_dim=0), _lib.PDA_ERR_HEAD_DIM),
    (dict(head_dim=513), _lib.PDA_ERR_HEAD_DIM), (dict(page_size=0), BAD),
    (dict(capacity=0), BAD), (dict(capacity=(1 << 31) - 1), _lib.PDA_ERR_TOO_LONG),
    (dict(window=-1), BAD), (dict(fresh=-1), BAD), (dict(layout=2), BAD),
    (dict(arena_rows=8), BAD), (dict(scale=float("nan")), BAD), (dict(softcap=-1.0), BAD),
    (dict(queries=None), BAD), (dict(out=None), BAD), (dict(keys=FAKE + 8), ALIGN),
    (dict(weights=FAKE + 2), ALIGN), (dict(workspace=None), _lib.PDA_ERR_WORKSPACE),
    (dict(workspace_bytes=100), _lib.PDA_ERR_WORKSPACE), (dict(workspace=FAKE + 16), ALIGN),
])
def test_weights_rejects(overrides, code):
    assert weights(**overrides) == code
    assert _lib.library().pda_last_error().decode() != ""


@pytest.mark.parametrize("overrides, code", [
    (dict(batch=65536), BAD), (dict(kv_heads=0), BAD), (dict(keep=0), BAD), (dict(recent=-1), BAD),
    (dict(sinks=-1), BAD), (dict(recent=510), BAD), (dict(capacity=0), BAD),
    (dict(out_capacity=100, out_weights=2 * FAKE), BAD), (dict(out_capacity=512), BAD),
    (dict(arena_rows=8), BAD), (dict(kept=None), BAD), (dict(weights=None), BAD),
    (dict(lengths=FAKE + 1), ALIGN), (dict(table_stride=0), BAD),
    (dict(capacity=(1 << 31) - 1, out_weights=None), _lib.PDA_ERR_TOO_LONG),
])
def test_select_rejects(overrides, code):
    assert select(**overrides) == code
    assert _lib.library().pda_last_error().decode() != ""


@pytest.mark.parametrize("overrides, code", [
    (dict(batch=-1), BAD), (dict(kv_heads=40000), BAD), (dict(width=0), BAD), (dict(keep=0), BAD),
    (dict(out_stride=0), BAD), (dict(arena=None), BAD), (dict(out_tables=None), BAD),
    (dict(layout=7), BAD), (dict(arena_rows=8), BAD), (dict(kept=FAKE + 2), ALIGN),
])
def test_move_rejects(overrides, code):
    assert move(**overrides) == code
    assert _lib.library().pda_last_error().decode() != ""


def test_empty_calls_are_no_ops():
    assert weights(batch=0) == select(batch=0) == move(batch=0) == _lib.PDA_OK


def test_python_checks_on_the_cpu():
    q = torch.zeros((1, 2, 8), dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        eviction.paged_attention_weights(q, q, q, q, q, page_size=16, longest=1, scale=1.0)
    with pytest.raises(TypeError, match="queries"):
        eviction.paged_attention_weights(q.float(), q, q, q, q, page_size=16, longest=1, scale=1.0)


def cache(window=0):
    return KVCache([KVGroup("g", (0,), 1, 8, window)], page_size=4, capacities={"g": 8},
                   device="cpu")


def test_cache_evict_refuses_before_it_changes_anything():
    store = cache()
    table = store.pools["g"].allocate_many(5, reserved=False)
    with pytest.raises(ValueError, match="windowed"):
        cache(window=8).evict("g", [table], np.array([20]), {}, keep=8)
    for bad in (dict(keep=0), dict(keep=8, recent=9), dict(keep=8, sinks=-1)):
        with pytest.raises(ValueError, match="keep"):
            store.evict("g", [table], np.array([20]), {}, **bad)
    with pytest.raises(RuntimeError, match="all its pages"):
        store.evict("g", [np.array([0, -1, 2, 3, 4])], np.array([20]), {}, keep=8)
    with pytest.raises(RuntimeError, match="all its pages"):
        store.evict("g", [table[:3]], np.array([20]), {}, keep=8)
    # A shared page needs fresh ones, and there are not enough.
    store.pools["g"].retain(table[:1])
    with pytest.raises(RuntimeError, match="exhausted"):
        store.evict("g", [table], np.array([20]), {}, keep=16)
    assert store.pools["g"].free == 3


def test_cache_evict_leaves_short_sequences():
    store = cache()
    table = store.pools["g"].allocate_many(2, reserved=False)
    tables, lengths = store.evict("g", [table], np.array([7]), {}, keep=8)
    assert tables[0].tolist() == table.tolist() and lengths.tolist() == [7]
    assert store.pools["g"].free == 6
