"""Verifying a tree of drafted tokens: one decoder-attention step over a quantised (or BF16) cache.

``cuda_decoder_attention_tree_forward_`` composes the framework's operators:
input RMSNorm, Q/K/V projections of the NVFP4 weights, per-head norms, rotary
positions at each node's depth, the append (quantised as it is written) into the
slots after the P_b committed positions, tree attention, the O projection.
``accept_drafted_`` then commits one path of the tree per sequence.  A step::

    cache = QuantizedKVCache.allocate(B, Hkv, 32768, D, "nvfp4")
    inv_freq, factor = rope_frequencies(D, scaling="yarn", factor=4.0, original_length=8192)
    y, k, v = cuda_decoder_attention_tree_forward_(
        x, g_in, wq, wk, wv, g_q, g_k, wo, cache, depths=depths, tree_mask=mask, inv_freq=inv_freq,
        attention_factor=factor, past_lengths=past, max_past_length=bound)
    accept_drafted_(cache, k, v, path, past_lengths=past, counts=counts)   # path: int64 [B, n]
    past += counts

(No counterpart in the reference, whose step appends and attends causally:
decoder_attention_cuda.py:149-417.)
"""

from __future__ import annotations

import torch

from cuda_primitives import (cuda_apply_rope_qk, cuda_kv_cache_append_, cuda_quantized_kv_append_, cuda_rms_norm,
                             cuda_tree_attention_cached, cuda_w4a16_linear)


def cuda_decoder_attention_tree_forward_(x, input_norm_weight, q_weight, k_weight, v_weight, q_norm_weight,
                                         k_norm_weight, out_weight, cache, past_length: int = 0, *, depths,
                                         inv_freq, tree_mask=None, past_lengths: torch.Tensor | None = None,
                                         max_past_length: int | None = None, attention_factor: float = 1.0,
                                         interleaved: bool = True, rms_eps: float = 1.0e-6):
    """One step for T drafted tokens x ``[B, T, H]`` of every sequence; returns ``(y, new_k, new_v)``.

    Token t of sequence b sits at position ``P_b + depths[.., t]`` (int64 ``[T]``
    or ``[B, T]``) and sees the committed positions and the drafted tokens its
    row of ``tree_mask`` names (ancestors and itself; without a mask the causal
    chain).  ``cache`` is a ``QuantizedKVCache`` or a pair of BF16 caches; slots
    ``P_b .. P_b + T - 1`` are written.  ``new_k`` and ``new_v`` ``[B, T, Hkv, D]`` are the rows as they
    went in, for ``accept_drafted_``.
    """
    if not isinstance(x, torch.Tensor) or x.ndim != 3:
        raise TypeError("x must be a rank-3 torch.Tensor")
    bf16 = isinstance(cache, (tuple, list))
    b, t, hidden = x.shape
    hkv = cache[0].shape[1] if bf16 else cache.k_codes.shape[1]
    d = cache[0].shape[3] if bf16 else cache.head_dim
    if hidden % d:
        raise ValueError(f"hidden size must be divisible by the cache's head dimension ({hidden} % {d} != 0)")
    xn = cuda_rms_norm(x, input_norm_weight, rms_eps)
    q = cuda_rms_norm(cuda_w4a16_linear(xn, q_weight).view(b, t, hidden // d, d), q_norm_weight, rms_eps)
    k = cuda_rms_norm(cuda_w4a16_linear(xn, k_weight).view(b, t, hkv, d), k_norm_weight, rms_eps)
    v = cuda_w4a16_linear(xn, v_weight).view(b, t, hkv, d)
    positions = depths + past_length if past_lengths is None else depths + past_lengths[:, None]
    q, k = cuda_apply_rope_qk(q, k, positions, inv_freq, interleaved=interleaved, attention_factor=attention_factor)
    if bf16:
        cuda_kv_cache_append_(cache[0], cache[1], k, v, past_length, past_lengths=past_lengths)
    else:
        cuda_quantized_kv_append_(cache, k, v, past_length, past_lengths=past_lengths)
    ctx = cuda_tree_attention_cached(q, cache, past_length, tree_mask=tree_mask, past_lengths=past_lengths,
                                     max_past_length=max_past_length)
    return cuda_w4a16_linear(ctx.view(b, t, hidden), out_weight), k, v


def accept_drafted_(cache, new_k: torch.Tensor, new_v: torch.Tensor, path: torch.Tensor, past_length: int = 0, *,
                    past_lengths: torch.Tensor | None = None, counts: torch.Tensor | None = None) -> None:
    """Commit the drafted tokens ``path`` (int64 ``[B, n]``, node indices from the root on) in slots ``P_b ..``.

    ``cache`` as in ``cuda_decoder_attention_tree_forward_``.  ``counts`` (CUDA
    int64 ``[B]``): only the first ``counts[b]`` nodes of a sequence's path; what
    stands after them may be any number (-1, say).  Rows go in as they did
    before, from BF16: a quantised cache gets the same bytes, now in consecutive
    slots.
    """
    # A gather outside would stop the device: a number that is no node is taken as the nearest one.
    index = path.clamp(0, new_k.shape[1] - 1)[:, :, None, None].expand(-1, -1, *new_k.shape[2:])
    rows = [torch.gather(x, 1, index) for x in (new_k, new_v)]
    if not isinstance(cache, (tuple, list)):
        cuda_quantized_kv_append_(cache, *rows, past_length, past_lengths=past_lengths, counts=counts)
        return
    if counts is not None:  # past a sequence's count the slots keep what they hold
        t = torch.arange(path.shape[1], device=path.device)
        slot = (t + (past_length if past_lengths is None else past_lengths[:, None])).clamp(0, cache[0].shape[2] - 1)
        slot = slot.expand(path.shape)[:, None, :, None].expand(-1, new_k.shape[2], -1, new_k.shape[3])
        kept = (t < counts[:, None])[:, :, None, None]
        rows = [torch.where(kept, x, torch.gather(c, 2, slot).transpose(1, 2)) for x, c in zip(rows, cache)]
    cuda_kv_cache_append_(cache[0], cache[1], *(x.contiguous() for x in rows), past_length, past_lengths=past_lengths)


def check_tree_wait_status(stream: torch.cuda.Stream | None = None) -> None:
    """Raise ``RuntimeError`` if a wait inside tree attention gave up on the stream's device since the last check.

    The kernels' warps hand tiles to one another over barriers in shared memory;
    every such wait is bounded, and one that runs out records a flag and lets the
    kernel end with garbage instead of hanging.  The call itself does not read
    the flag back; this function does, synchronises ``stream`` (default: the
    current one) and clears it.  The flag is the device's: calls on other streams
    are covered as far as they come before ``stream``'s work or have ended.
    """
    import nvfp4da_capi

    stream = stream if stream is not None else torch.cuda.current_stream()
    with torch.cuda.device(stream.device):
        flags = nvfp4da_capi.tree_sync_status(stream)
    if flags:
        raise RuntimeError(f"a bounded wait of tree attention timed out (flags 0x{flags:x}); the contexts since the "
                           "last check are not valid")


__all__ = ["accept_drafted_", "check_tree_wait_status", "cuda_decoder_attention_tree_forward_"]
