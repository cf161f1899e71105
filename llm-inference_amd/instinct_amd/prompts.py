"""Attention of whole prompts packed one behind the other, on MI355X.

The reference prefills one sequence a call, from the paged cache it has written the
keys and values to (``PrefillBatch.attend``, python/instinct/batches.py:84-132).
Fresh prompts need no cache to attend to themselves: their queries, keys and values
lie side by side as the projection left them, and :func:`packed_prompt_attention`
serves any number of prompts of any lengths in one call
(:class:`instinct_amd.batches.PackedPrefillBatch` writes the cache as well).

The work happens in libpda.so (``csrc/pda_prompts.hip``).
"""

from __future__ import annotations

import torch

from . import _lib
from .eviction import _check_index
from .hip_kernels import on_device


def packed_prompt_attention(queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor,
                            starts: torch.Tensor, *, scale: float, window: int = 0,
                            softcap: float = 0.0, out: torch.Tensor | None = None
                            ) -> torch.Tensor:
    """Causal attention of packed prompts: ``queries`` ``[tokens, q_heads, D]``,
    ``keys`` and ``values`` ``[tokens, kv_heads, D]``, fp16 or bf16; prompt b's tokens
    are ``starts[b] .. starts[b + 1] - 1`` (int32 ``[batch + 1]`` on the GPU, ascending
    from 0). A token attends to itself and the tokens before it in its prompt, with
    the window and softcap of the decode call. The elements of a head lie side by
    side; tokens and heads may be any multiple of 8 elements apart (slices of one
    projection's output are read where they are). ``D`` is a multiple of 8 up to 256.
    Returns ``[tokens, q_heads, D]`` (``out``, contiguous, where given); rows behind
    the last prompt are zeros."""
    if queries.dim() != 3 or queries.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("queries must be [tokens, q_heads, head_dim] float16 or bfloat16")
    if not queries.is_cuda:
        raise ValueError("queries must be on a GPU")
    device = queries.device
    tokens, q_heads, head_dim = queries.shape
    kv_heads = keys.shape[1] if keys.dim() == 3 else 0
    size = (tokens, kv_heads, head_dim)
    for name, t in (("keys", keys), ("values", values)):
        if t.dtype is not queries.dtype:
            raise TypeError(f"{name} must be {queries.dtype}, got {t.dtype}")
        if t.device != device:
            raise ValueError(f"{name} must be on {device}")
        if t.shape != size or not kv_heads:
            raise ValueError(f"{name} must be [tokens, kv_heads, head_dim] beside the queries")
    if q_heads == 0 or q_heads % kv_heads:
        raise ValueError("query heads must be a multiple of kv heads")
    q_token, q_head, q_one = queries.stride()
    k_token, k_head, k_one = keys.stride()
    v_token, v_head, v_one = values.stride()
    # (A tensor's stride says nothing where its size is one.)
    if tokens == 1:
        q_token = k_token = v_token = 0
    if q_heads == 1:
        q_head = 0
    if kv_heads == 1:
        k_head = v_head = 0
    if head_dim > 1 and (q_one != 1 or k_one != 1 or v_one != 1):
        raise ValueError("the elements of a head must lie side by side")
    if starts.dim() != 1 or starts.shape[0] == 0:
        raise ValueError("starts must be int32 [batch + 1]")
    starts = _check_index("starts", starts, (starts.shape[0],), device)
    if out is None:
        out = torch.empty_like(queries, memory_format=torch.contiguous_format)
    elif (out.dtype != queries.dtype or out.shape != queries.shape or out.device != device
          or not out.is_contiguous()):
        raise ValueError("out must be contiguous and match the queries' shape, dtype and device")
    entry = ("pda_packed_prompt_attention_bf16" if queries.dtype == torch.bfloat16
             else "pda_packed_prompt_attention")
    with on_device(device):
        rc = getattr(_lib.library(), entry)(
            queries.data_ptr(), q_token, q_head, keys.data_ptr(), k_token, k_head,
            values.data_ptr(), v_token, v_head, starts.data_ptr(), out.data_ptr(),
            tokens, starts.shape[0] - 1, q_heads, kv_heads, head_dim, float(scale), int(window),
            float(softcap), torch.cuda.current_stream(device).cuda_stream)
    _lib.check(rc)
    return out
