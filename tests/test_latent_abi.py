"""The latent calls validate their arguments on the host (no GPU call is made:
every rejected call returns before touching HIP)."""

import pytest
import torch

from instinct_amd import _lib, latent

FAKE = 0x10000  # an aligned, never-dereferenced address


def append(**overrides):
    args = dict(q=FAKE, q_out=FAKE, latent=FAKE, latent_stride=576, k_rope=FAKE, k_stride=576,
                norm_weight=FAKE, eps=1e-6, arena=FAKE, positions=FAKE, rows=FAKE, n=4,
                q_heads=16, latent_dim=512, rope_dim=64, nope_dim=128, arena_rows=64,
                inv_freq=FAKE, stream=None)
    args.update(overrides)
    return _lib.library().pda_latent_append(*args.values())


def decode(**overrides):
    args = dict(queries=FAKE, arena=FAKE, kv_b=FAKE, tables=FAKE, lengths=FAKE, out=FAKE, batch=4,
                q_heads=16, latent_dim=512, rope_dim=64, nope_dim=128, value_dim=128,
                page_size=16, table_stride=64, arena_rows=4096, longest=1000, scale=0.07,
                workspace=FAKE, workspace_bytes=1 << 30, stream=None)
    args.update(overrides)
    return _lib.library().pda_latent_decode_attention_bf16(*args.values())


def prefill(**overrides):
    args = dict(queries=FAKE, arena=FAKE, kv_b=FAKE, table=FAKE, table_len=64, start=100, count=50,
                out=FAKE, q_heads=16, latent_dim=512, rope_dim=64, nope_dim=128, value_dim=128,
                page_size=16, arena_rows=4096, scale=0.07, workspace=FAKE,
                workspace_bytes=1 << 31, stream=None)
    args.update(overrides)
    return _lib.library().pda_latent_prefill_attention(*args.values())


SHAPES = [
    (dict(q_heads=0), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(q_heads=65536), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(latent_dim=0), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(latent_dim=520), _lib.PDA_ERR_HEAD_DIM),
    (dict(latent_dim=500), _lib.PDA_ERR_HEAD_DIM),
    (dict(rope_dim=-16), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(rope_dim=24), _lib.PDA_ERR_HEAD_DIM),
    (dict(rope_dim=80), _lib.PDA_ERR_HEAD_DIM),
    (dict(nope_dim=136), _lib.PDA_ERR_HEAD_DIM),
    (dict(nope_dim=100), _lib.PDA_ERR_HEAD_DIM),
    (dict(arena=None), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(arena=FAKE + 8), _lib.PDA_ERR_ALIGNMENT),
]


@pytest.mark.parametrize("overrides, code", SHAPES + [
    (dict(n=-1), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(q=None), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(rows=None), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(k_rope=None), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(positions=None), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(q=None, q_out=None, latent=None, k_rope=None, arena=None, rows=None),
     _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(latent_stride=504), _lib.PDA_ERR_ALIGNMENT),
    (dict(latent_stride=513), _lib.PDA_ERR_ALIGNMENT),
    (dict(k_stride=60), _lib.PDA_ERR_ALIGNMENT),
    (dict(eps=-1.0), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(eps=float("nan")), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(rows=FAKE + 2), _lib.PDA_ERR_ALIGNMENT),
    (dict(n=1 << 30, q_heads=64), _lib.PDA_ERR_INVALID_ARGUMENT),
])
def test_append_rejects(overrides, code):
    assert append(**overrides) == code
    assert _lib.library().pda_last_error().decode() != ""


@pytest.mark.parametrize("overrides, code", SHAPES + [
    (dict(value_dim=0), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(value_dim=132), _lib.PDA_ERR_HEAD_DIM),
    (dict(batch=-1), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(batch=8185), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(page_size=0), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(table_stride=0), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(batch=8184, table_stride=1 << 28), _lib.PDA_ERR_TOO_LONG),
    (dict(arena_rows=8), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(arena_rows=1 << 31), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(scale=float("inf")), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(tables=None), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(lengths=FAKE + 2), _lib.PDA_ERR_ALIGNMENT),
    (dict(workspace=None), _lib.PDA_ERR_WORKSPACE),
    (dict(workspace_bytes=1024), _lib.PDA_ERR_WORKSPACE),
    (dict(workspace=FAKE + 64), _lib.PDA_ERR_ALIGNMENT),
])
def test_decode_rejects(overrides, code):
    assert decode(**overrides) == code
    assert _lib.library().pda_last_error().decode() != ""


@pytest.mark.parametrize("overrides, code", SHAPES + [
    (dict(value_dim=0), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(count=-1), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(start=-1), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(start=(1 << 31) - 60), _lib.PDA_ERR_TOO_LONG),
    (dict(table_len=0), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(page_size=0), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(arena_rows=8), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(arena_rows=1 << 31), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(scale=float("nan")), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(table=None), _lib.PDA_ERR_INVALID_ARGUMENT),
    (dict(table=FAKE + 2), _lib.PDA_ERR_ALIGNMENT),
    (dict(workspace=None), _lib.PDA_ERR_WORKSPACE),
    (dict(workspace_bytes=1024), _lib.PDA_ERR_WORKSPACE),
    (dict(workspace=FAKE + 64), _lib.PDA_ERR_ALIGNMENT),
])
def test_prefill_rejects(overrides, code):
    assert prefill(**overrides) == code
    assert _lib.library().pda_last_error().decode() != ""


def test_prefill_workspace_is_bounded():
    """The expanded rows of as many heads as fit in 1 GiB, not of all."""
    some = _lib.latent_prefill_workspace_bytes(0, 4096, 128, 64, 128, 128)
    assert some >= 4096 * 128 * 256 * 2
    far = _lib.latent_prefill_workspace_bytes(130000, 1024, 128, 64, 128, 128)
    assert far < (1 << 30) + (1 << 29)


def test_empty_calls_are_no_ops():
    assert prefill(count=0) == _lib.PDA_OK
    assert append(n=0) == _lib.PDA_OK
    assert decode(batch=0, workspace=None, workspace_bytes=0) == _lib.PDA_OK
    assert _lib.latent_decode_workspace_bytes(0, 16, 512, 64, 16, 4, 1) == 0


def test_workspace_is_bounded():
    """Two partial slots a workgroup at most, whatever the context."""
    need = _lib.latent_decode_workspace_bytes(4, 16, 512, 64, 16, 64, 1024)
    far = _lib.latent_decode_workspace_bytes(4, 16, 512, 64, 16, 1 << 20, 1 << 24)
    assert need <= far <= (256 + 4 + 1) * 16 * (512 * 4 + 8) + 4 * 16 * 576 * 2 + 2048


def test_python_checks():
    q = torch.zeros((1, 16, 192), dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        latent.latent_decode_attention(q, q, q, q, q, page_size=16, longest=1, scale=1.0)
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        latent.latent_append(None, q.float(), q, q.float(), q, q, dims=0)
