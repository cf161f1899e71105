"""Latent calls past what one launch takes (2^32 threads) are refused on the host,
before anything is launched."""

from test_latent_abi import append, prefill

from instinct_amd import _lib


def test_append():
    """2^24 workgroups of queries; one of rows and 2^24 - 1 of queries."""
    assert append(n=1 << 24) == _lib.PDA_ERR_INVALID_ARGUMENT
    assert "workgroups" in _lib.library().pda_last_error().decode()
    assert append(n=1 << 20, q_heads=256) == _lib.PDA_ERR_INVALID_ARGUMENT
    assert "workgroups" in _lib.library().pda_last_error().decode()


def test_prefill_join():
    """A long prefix whose heads go one at a time in split key ranges: count x heads
    x value dims in the join."""
    overrides = dict(start=1 << 22, count=1 << 15, q_heads=16384, workspace_bytes=1 << 62)
    assert prefill(**overrides) == _lib.PDA_ERR_INVALID_ARGUMENT
    assert "workgroups" in _lib.library().pda_last_error().decode()
