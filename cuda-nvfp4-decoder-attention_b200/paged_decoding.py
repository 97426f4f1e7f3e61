"""Serving drafted tokens from a paged KV cache: one decoder-attention step, and the accepted path.

``cuda_decoder_attention_paged_forward_`` composes the framework's operators:
input RMSNorm, Q/K/V projections of the NVFP4 weights, per-head norms, rotary
positions, the append into the slots that ``cuda_reserve_pages_`` gave, attention
through the block table, the O projection.  A step that verifies drafted tokens::

    cache = PagedKVCache.allocate(N, Hkv, 64, D, "nvfp4")
    table = PageTable.allocate(B, 32768 // 64, N, 64)
    slots, granted = cuda_reserve_pages_(table, past, T)
    y, k, v = cuda_decoder_attention_paged_forward_(
        x, g_in, wq, wk, wv, g_q, g_k, wo, cache, table.pages, slots, depths=depths, tree_mask=mask,
        inv_freq=inv_freq, past_lengths=past, max_past_length=bound, counts=granted)
    path, counts, token = cuda_verify_drafted(target, drafted, uniforms, draft_probs=draft, parents=parents,
                                              counts=granted)
    accept_drafted_paged_(cache, k, v, path, slots, counts=counts)
    past += counts
    cuda_release_pages_(table, past)   # what only rejected tokens held

A sequence that got no pages (``granted`` 0) goes through all of it untouched.  No
call reads anything back, so a step can be captured into a CUDA graph.  (No
counterpart in the reference, whose cache reserves C slots a sequence:
decoder_attention_cuda.py:149-417.)
"""

from __future__ import annotations

import torch

from cuda_primitives import (cuda_apply_rope_qk, cuda_paged_attention, cuda_paged_kv_append_, cuda_rms_norm,
                             cuda_w4a16_linear)


def cuda_decoder_attention_paged_forward_(x, input_norm_weight, q_weight, k_weight, v_weight, q_norm_weight,
                                          k_norm_weight, out_weight, cache, block_table: torch.Tensor,
                                          slots: torch.Tensor, *, past_lengths: torch.Tensor, max_past_length: int,
                                          inv_freq: torch.Tensor, depths: torch.Tensor | None = None,
                                          tree_mask: torch.Tensor | None = None, counts: torch.Tensor | None = None,
                                          attention_factor: float = 1.0, interleaved: bool = True,
                                          rms_eps: float = 1.0e-6):
    """One step for T tokens x ``[B, T, H]`` of every sequence over a ``PagedKVCache``; returns ``(y, new_k, new_v)``.

    Token t of sequence b sits at position ``P_b + depths[.., t]`` (int64 ``[T]``
    or ``[B, T]``; t without them), its row goes to ``slots[b, t]``, and it sees
    the committed positions and what its row of ``tree_mask`` names (without a
    mask the tokens up to itself).  Tokens ``t >= counts[b]`` are padding.
    ``new_k`` and ``new_v`` ``[B, T, Hkv, D]`` are the rows as they went in, for
    ``accept_drafted_paged_``.
    """
    if not isinstance(x, torch.Tensor) or x.ndim != 3:
        raise TypeError("x must be a rank-3 torch.Tensor")
    b, t, hidden = x.shape
    hkv, d = cache.k_codes.shape[1], cache.head_dim
    if hidden % d:
        raise ValueError(f"hidden size must be divisible by the cache's head dimension ({hidden} % {d} != 0)")
    xn = cuda_rms_norm(x, input_norm_weight, rms_eps)
    q = cuda_rms_norm(cuda_w4a16_linear(xn, q_weight).view(b, t, hidden // d, d), q_norm_weight, rms_eps)
    k = cuda_rms_norm(cuda_w4a16_linear(xn, k_weight).view(b, t, hkv, d), k_norm_weight, rms_eps)
    v = cuda_w4a16_linear(xn, v_weight).view(b, t, hkv, d)
    if depths is None:
        depths = torch.arange(t, device=x.device)
    q, k = cuda_apply_rope_qk(q, k, depths + past_lengths[:, None], inv_freq, interleaved=interleaved,
                              attention_factor=attention_factor)
    cuda_paged_kv_append_(cache, k, v, slots, counts=counts)
    ctx = cuda_paged_attention(q, cache, block_table, tree_mask=tree_mask, past_lengths=past_lengths,
                               max_past_length=max_past_length, counts=counts)
    return cuda_w4a16_linear(ctx.view(b, t, hidden), out_weight), k, v


def accept_drafted_paged_(cache, new_k: torch.Tensor, new_v: torch.Tensor, path: torch.Tensor, slots: torch.Tensor, *,
                          counts: torch.Tensor | None = None) -> None:
    """Commit the drafted tokens ``path`` (int64 ``[B, n]``, node indices from the root on) in the first slots.

    The i-th accepted token's row goes to ``slots[b, i]``, the slot of position
    ``P_b + i``, from BF16 as it did before.  Only the first ``counts[b]`` (CUDA
    int64 ``[B]``) nodes of a path are committed; a number that is no node is not
    (so ``cuda_verify_drafted``'s -1 behind a path needs no counts).
    """
    cuda_paged_kv_append_(cache, new_k, new_v, slots, source=path, counts=counts)


__all__ = ["accept_drafted_paged_", "cuda_decoder_attention_paged_forward_"]
