"""prompts.packed_prompt_attention against the plain restatement in 64 bits, with the
tolerance of oracle.many_tokens.attention_tolerance."""

import numpy as np
import pytest
import torch

from instinct_amd import prompts
from oracle import many_tokens as plain

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def make(seed, counts, q_heads, kv_heads, dim, dtype, *, fused=True, behind=0):
    gen = torch.Generator().manual_seed(seed)
    total = int(sum(counts)) + behind
    shape = lambda h: (total, h, dim)  # noqa: E731
    if fused:
        qkv = torch.randn(shape(q_heads + 2 * kv_heads), generator=gen).to(dtype).cuda()
        q, k, v = qkv.split([q_heads, kv_heads, kv_heads], dim=1)
    else:
        q, k, v = (torch.randn(shape(h), generator=gen).to(dtype).cuda()
                   for h in (q_heads, kv_heads, kv_heads))
    starts = np.concatenate([[0], np.cumsum(counts)])
    return q, k, v, starts, torch.as_tensor(starts.astype(np.int32), device="cuda")


def compare(got, q, k, v, starts, **kw):
    host = lambda t: t.double().cpu().numpy()  # noqa: E731
    want, size = plain.packed_prompts(host(q), host(k), host(v), [int(x) for x in starts], **kw)
    longest = int(np.diff(starts).max(initial=0))
    tol = plain.attention_tolerance(want, size, host(v), longest, got.dtype)
    off = np.abs(host(got) - want)
    worst = np.unravel_index(np.argmax(off - tol), off.shape)
    assert np.all(off <= tol), (worst, off[worst], tol[worst], want[worst])


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("counts, heads", [
    ([1], (14, 2, 64)), ([1, 1, 1], (4, 4, 128)), ([20, 200, 33, 5], (14, 2, 64)),
    ([64], (28, 4, 128)), ([65, 0, 127], (28, 4, 128)), ([128, 129, 1], (32, 8, 96)),
    ([300], (32, 32, 80)), ([257, 31], (24, 8, 112)), ([190, 7, 70], (16, 8, 256)),
    ([400, 3], (2, 1, 8)), ([150], (5, 1, 136)), ([0, 90, 0, 0, 31, 0], (8, 8, 72))],
    ids=lambda x: "-".join(map(str, x)))
def test_against_64_bits(gpu, counts, heads, dtype):
    q, k, v, starts, dev = make(1, counts, *heads, dtype)
    scale = heads[2] ** -0.5
    compare(prompts.packed_prompt_attention(q, k, v, dev, scale=scale), q, k, v, starts,
            scale=scale)


@pytest.mark.parametrize("counts", [[1100], [70, 900, 513, 2], [2049]], ids=str)
@pytest.mark.parametrize("heads", [(4, 2, 64), (4, 1, 128), (2, 1, 256), (2, 2, 96)], ids=str)
def test_longer_prompts(gpu, counts, heads):
    q, k, v, starts, dev = make(2, counts, *heads, BF16)
    compare(prompts.packed_prompt_attention(q, k, v, dev, scale=0.11), q, k, v, starts, scale=0.11)


@pytest.mark.parametrize("kw", [dict(window=1), dict(window=7), dict(window=64), dict(window=100),
                                dict(window=100000), dict(softcap=5.0), dict(softcap=30.0, window=33),
                                dict(scale=-0.2), dict(scale=0.0), dict(scale=0.5)], ids=str)
@pytest.mark.parametrize("heads", [(6, 2, 64), (4, 2, 128), (2, 2, 256)], ids=str)
def test_windows_softcaps_scales(gpu, heads, kw):
    q, k, v, starts, dev = make(3, [140, 333, 9], *heads, F16)
    kw = dict(dict(scale=0.1), **kw)
    compare(prompts.packed_prompt_attention(q, k, v, dev, **kw), q, k, v, starts, **kw)


@pytest.mark.parametrize("heads", [(4, 2, 128), (4, 4, 80)], ids=str)
def test_strides(gpu, heads):
    """Heads and tokens in other orders and distances than the tested ones."""
    q, k, v, starts, dev = make(4, [77, 150], *heads, BF16, fused=False)
    by_head = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    wide = torch.zeros(227, heads[1], heads[2] + 24, dtype=BF16, device="cuda")
    wide[..., 8:8 + heads[2]] = k
    got = prompts.packed_prompt_attention(by_head(q), wide[..., 8:8 + heads[2]], by_head(v), dev,
                                          scale=0.1)
    assert torch.equal(got, prompts.packed_prompt_attention(q, k, v, dev, scale=0.1))
    compare(got, q, k, v, starts, scale=0.1)
    # One key and value for all tokens' heads: a stride of 0.
    one = k[:, :1].expand(-1, heads[0] // 2, -1)
    got = prompts.packed_prompt_attention(q, one, one, dev, scale=0.1)
    compare(got, q, one, one, starts, scale=0.1)


def test_strides_of_dimensions_of_one(gpu):
    """What a tensor's stride says of one token or one head does not matter."""
    q, k, v, starts, dev = make(12, [70], 1, 1, 64, F16, fused=False)
    odd = lambda t: t.as_strided(t.shape, (64, 3, 1))  # noqa: E731
    got = prompts.packed_prompt_attention(odd(q), odd(k), odd(v), dev, scale=0.1)
    compare(got, q, k, v, starts, scale=0.1)
    q, k, v, starts, dev = make(13, [1], 4, 2, 64, F16, fused=False)
    odd = lambda t: t.as_strided(t.shape, (5, 64, 1))  # noqa: E731
    got = prompts.packed_prompt_attention(odd(q), odd(k), odd(v), dev, scale=0.1)
    compare(got, q, k, v, starts, scale=0.1)


def test_rows_behind_the_last_prompt_are_zeros(gpu):
    for behind in (1, 130, 300):
        q, k, v, starts, dev = make(5, [100, 60], 4, 2, 64, F16, behind=behind)
        out = torch.full((160 + behind, 4, 64), float("nan"), dtype=F16, device="cuda")
        got = prompts.packed_prompt_attention(q, k, v, dev, scale=0.1, out=out)
        assert got is out and not out[160:].any()
        compare(out, q, k, v, starts, scale=0.1)


def test_no_tokens_and_no_prompts(gpu):
    q, k, v, starts, dev = make(6, [0, 0], 4, 2, 64, F16)
    assert prompts.packed_prompt_attention(q, k, v, dev, scale=0.1).shape == (0, 4, 64)
    q, k, v, _, _ = make(6, [30], 4, 2, 64, F16)
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert not prompts.packed_prompt_attention(q, k, v, none, scale=0.1).any()


@pytest.mark.parametrize("heads", [(4, 2, 64), (2, 1, 128), (2, 2, 256), (2, 1, 80)], ids=str)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")], ids=str)
@pytest.mark.parametrize("which", ["keys", "values", "queries"])
def test_what_is_not_finite_reaches_those_that_see_it(gpu, heads, bad, which):
    """A token that is not finite changes no row in front of it, of other prompts, or
    past its window."""
    counts, at, window = [50, 260, 40], 50 + 131, 70
    q, k, v, starts, dev = make(7, counts, *heads, F16, fused=False)
    clean = prompts.packed_prompt_attention(q, k, v, dev, scale=0.1, window=window)
    x = dict(keys=k, values=v, queries=q)[which]
    x[at, 0, 3] = bad
    got = prompts.packed_prompt_attention(q, k, v, dev, scale=0.1, window=window)
    group = heads[0] // heads[1]
    touched = torch.zeros(got.shape[:2], dtype=torch.bool, device="cuda")
    if which == "queries":
        touched[at, 0] = True
    else:
        touched[at:at + window, :group] = True
    assert torch.equal(got[~touched], clean[~touched])
    if which == "values":
        # The one element, in every row that sees it.
        assert torch.equal(got[..., 4:], clean[..., 4:])
        seen = got[at:at + window, :group, 3]
        assert torch.all(torch.isnan(seen) if bad != bad else seen == bad)
    elif which == "queries":
        assert not torch.isfinite(got[at, 0]).any() or abs(bad) == float("inf")


def test_repeated_and_captured(gpu):
    """The same bits every time, also from a graph replayed between eager calls, and
    with a current stream of its own."""
    q, k, v, starts, dev = make(8, [300, 20, 511], 14, 2, 64, F16)
    first = prompts.packed_prompt_attention(q, k, v, dev, scale=0.125)
    out = torch.empty_like(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        prompts.packed_prompt_attention(q, k, v, dev, scale=0.125, out=out)
    for _ in range(4):
        out.zero_()
        graph.replay()
        assert torch.equal(out, first)
        assert torch.equal(prompts.packed_prompt_attention(q, k, v, dev, scale=0.125), first)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = prompts.packed_prompt_attention(q, k, v, dev, scale=0.125)
    stream.synchronize()
    assert torch.equal(again, first)


def test_many_prompts(gpu):
    rng = np.random.default_rng(9)
    counts = rng.integers(0, 12, 700)
    q, k, v, starts, dev = make(9, counts, 2, 1, 64, F16)
    compare(prompts.packed_prompt_attention(q, k, v, dev, scale=0.1), q, k, v, starts, scale=0.1)


def test_refusals(gpu):
    q, k, v, _, dev = make(10, [30], 4, 2, 64, F16)
    call = prompts.packed_prompt_attention
    with pytest.raises(TypeError):
        call(q.float(), k, v, dev, scale=0.1)
    with pytest.raises(TypeError):
        call(q, k.bfloat16(), v, dev, scale=0.1)
    with pytest.raises(TypeError):
        call(q, k, v, dev.long(), scale=0.1)
    with pytest.raises(ValueError):
        call(q, k[:, :, :32], v, dev, scale=0.1)
    with pytest.raises(ValueError):
        call(q[:, :3], k, v, dev, scale=0.1)
    with pytest.raises(ValueError):
        call(q, k, v[:20], dev, scale=0.1)
    with pytest.raises(ValueError):
        call(q.transpose(1, 2), k, v, dev, scale=0.1)
    with pytest.raises(ValueError):
        call(q, k, v, dev.cpu(), scale=0.1)
    with pytest.raises(ValueError):
        call(q, k, v, dev, scale=0.1, out=torch.empty(30, 4, 32, dtype=F16, device="cuda"))
