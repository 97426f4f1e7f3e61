"""Python boundary of the B200 operator library (drop-in for the reference's
``cuda_primitives.py``, reference cuda_primitives.py:1-222).

Loads ``lib/cuda_primitives.so`` (or ``$CUDA_PRIMITIVES_LIBRARY``) with
``torch.ops.load_library``; a missing library raises ``ImportError`` — there is
no fallback implementation.  The wrappers have the reference's names,
arguments and error behaviour.  Weight arguments accept this package's
``NVFP4Tensor`` or the reference's (same four fields).
"""

from __future__ import annotations

import os
from pathlib import Path

import torch

from nvfp4_tensor import NVFP4Tensor, is_nvfp4_tensor, quantize_nvfp4  # noqa: F401
from quantized_kv_cache import QuantizedKVCache, rope_frequencies  # noqa: F401

_PACKAGE_DIR = Path(__file__).resolve().parent
_LIBRARY_PATH = Path(os.environ.get("CUDA_PRIMITIVES_LIBRARY", _PACKAGE_DIR / "lib" / "cuda_primitives.so"))

if not _LIBRARY_PATH.is_file():
    raise ImportError(
        f"CUDA primitives library not found at {_LIBRARY_PATH}; "
        "run `python cuda-nvfp4-decoder-attention_b200/build.py` from the repository root"
    )

torch.ops.load_library(str(_LIBRARY_PATH))
_ops = torch.ops.cuda_nvfp4_decoder_attention
LIBRARY_PATH = _LIBRARY_PATH


def _require_weight(name: str, weight: object) -> None:
    if not is_nvfp4_tensor(weight):
        raise TypeError(f"{name} must be an NVFP4Tensor")
    derived = (weight.packed_values.shape[0], weight.packed_values.shape[1] * 2)
    if tuple(weight.logical_shape) != derived:
        raise ValueError(f"{name}.logical_shape must match packed_values-derived shape "
                         f"({tuple(weight.logical_shape)} != {derived})")


def _require_int(name: str, value: object) -> None:
    if isinstance(value, bool) or not isinstance(value, int):
        raise TypeError(f"{name} must be an integer")


def cuda_unpack_e2m1_codes(packed_values: torch.Tensor) -> torch.Tensor:
    """Unpack even-low, odd-high E2M1 bytes (reference cuda_primitives.py:30-36)."""
    return _ops.cuda_unpack_e2m1_codes(packed_values)


def cuda_dequantize_nvfp4(quantized) -> torch.Tensor:
    """Decode NVFP4 storage to FP32 ``(q * beta) * gamma`` (reference cuda_primitives.py:39-62)."""
    _require_weight("quantized", quantized)
    return _ops.cuda_dequantize_nvfp4(quantized.packed_values, quantized.block_scales,
                                      quantized.global_decode_scale)


def cuda_w4a16_linear(x: torch.Tensor, weight) -> torch.Tensor:
    """BF16 ``x @ W_hat.T`` with in-kernel NVFP4 decode (reference cuda_primitives.py:65-91)."""
    _require_weight("weight", weight)
    return _ops.cuda_w4a16_linear(x, weight.packed_values, weight.block_scales, weight.global_decode_scale)


def cuda_w4a16_linear_grouped_decode(x: torch.Tensor, weight) -> torch.Tensor:
    """Same projection under the reference's grouped-decode name (reference cuda_primitives.py:94-120)."""
    _require_weight("weight", weight)
    return _ops.cuda_w4a16_linear_grouped_decode(x, weight.packed_values, weight.block_scales,
                                                 weight.global_decode_scale)


def cuda_rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    """RMSNorm over the last dimension (reference cuda_primitives.py:123-130)."""
    return _ops.cuda_rms_norm(x, weight, eps)


def cuda_apply_rope(x: torch.Tensor, past_length: int, rope_theta: float = 10000.0) -> torch.Tensor:
    """Adjacent-pair RoPE at positions ``past_length + t`` (reference cuda_primitives.py:133-144)."""
    return _ops.cuda_apply_rope(x, past_length, rope_theta)


def cuda_gqa_attention(q: torch.Tensor, present_k: torch.Tensor, present_v: torch.Tensor,
                       past_length: int) -> torch.Tensor:
    """Causal GQA over compact ``[B, Hkv, P+T, D]`` caches (reference cuda_primitives.py:147-161)."""
    _require_int("past_length", past_length)
    return _ops.cuda_gqa_attention(q, present_k, present_v, past_length)


def cuda_gqa_attention_cached(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                              past_length: int) -> torch.Tensor:
    """Causal GQA over physical ``[B, Hkv, C, D]`` caches (reference cuda_primitives.py:164-183)."""
    _require_int("past_length", past_length)
    return _ops.cuda_gqa_attention_cached(q, k_cache, v_cache, past_length)


def cuda_kv_cache_append_(k_cache: torch.Tensor, v_cache: torch.Tensor, new_k: torch.Tensor,
                          new_v: torch.Tensor, past_length: int = 0, *,
                          past_lengths: torch.Tensor | None = None) -> None:
    """Write token-major K/V into slots ``past_length ..`` in place (reference cuda_primitives.py:186-207).

    ``past_lengths`` (CUDA int64 ``[B]``; no reference counterpart) replaces the
    common past length; a slot outside the cache is not written.
    """
    _require_int("past_length", past_length)
    if past_lengths is None:
        _ops.cuda_kv_cache_append_(k_cache, v_cache, new_k, new_v, past_length)
    else:
        _ops.cuda_kv_cache_append_varlen_(k_cache, v_cache, new_k, new_v, past_lengths)


# ------------------------------------------------------------------ drafted-token verification
def cuda_apply_rope_qk(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *,
                       interleaved: bool = True, attention_factor: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """Rotary positions of q ``[B, T, Hq, D]`` and k ``[B, T, Hkv, D]`` in one launch (no reference counterpart).

    ``positions``: int64 ``[T]`` or ``[B, T]``, one per token (a drafted token
    sits at past length + its depth in the tree).  ``inv_freq``: float32
    ``[rotary_dim / 2]`` (``rope_frequencies`` makes it, scaled for long
    contexts); the first ``rotary_dim`` elements of each head turn, in adjacent
    pairs (``interleaved``) or as halves, the others are copied.  q and k may be
    strided views that are contiguous in their last dimension.
    """
    return _ops.cuda_apply_rope_qk(q, k, positions, inv_freq, interleaved, attention_factor)


def cuda_quantized_kv_append_(cache, new_k: torch.Tensor, new_v: torch.Tensor, past_length: int = 0, *,
                              past_lengths: torch.Tensor | None = None, counts: torch.Tensor | None = None) -> None:
    """Quantise ``[B, T, Hkv, D]`` BF16 rows into slots ``past_length ..`` of a ``QuantizedKVCache`` in place.

    ``past_lengths`` (CUDA int64 ``[B]``) replaces the common past length;
    tokens ``t >= counts[b]`` (CUDA int64 ``[B]``) are not written, nor is a
    slot outside the cache.  A row with an infinity or NaN reads back as NaN.
    """
    _require_int("past_length", past_length)
    _ops.cuda_quantized_kv_append_(cache.k_codes, cache.v_codes, cache.k_row_scales, cache.v_row_scales,
                                   cache.k_block_scales, cache.v_block_scales, new_k, new_v, past_length,
                                   past_lengths, counts)


def cuda_quantized_kv_read(cache, start: int = 0, length: int | None = None, *,
                           starts: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Slots ``[start, start + length)`` of a ``QuantizedKVCache`` as BF16 K and V ``[B, Hkv, length, D]``.

    ``starts`` (CUDA int64 ``[B]``) gives each sequence a window of its own;
    slots outside the cache then read as zeros.  ``length`` defaults to the
    slots from ``start`` on.
    """
    _require_int("start", start)
    if length is None:
        length = cache.k_codes.shape[2] - start
    _require_int("length", length)
    return _ops.cuda_quantized_kv_read(cache.k_codes, cache.v_codes, cache.k_row_scales, cache.v_row_scales,
                                       cache.k_block_scales, cache.v_block_scales, start, length, starts)


def cuda_tree_attention_cached(q: torch.Tensor, cache, past_length: int = 0, *, tree_mask: torch.Tensor | None = None,
                               past_lengths: torch.Tensor | None = None,
                               max_past_length: int | None = None) -> torch.Tensor:
    """Attention of T drafted tokens q ``[B, T, Hq, D]`` over a cache that holds them after its P_b positions.

    ``cache``: a ``QuantizedKVCache``, read in its own format, or a pair of BF16
    caches ``(k_cache, v_cache)``.  Token t sees slots below P_b and slot
    ``P_b + u`` where ``tree_mask[b, t, u]`` (bool ``[T, T]`` or ``[B, T, T]``;
    without one ``u <= t``); a query that sees nothing gets zeros.  With
    ``past_lengths`` (CUDA int64 ``[B]``) ``max_past_length`` is a host bound on
    them.  T = 1 is single-token decode.
    """
    _require_int("past_length", past_length)
    if past_lengths is None:
        max_past_length = past_length
    else:
        _require_int("max_past_length", max_past_length)
    if isinstance(cache, (tuple, list)):
        k_cache, v_cache = cache
        return _ops.cuda_tree_attention_cached(q, k_cache, v_cache, None, None, None, None, tree_mask, past_length,
                                               past_lengths, max_past_length)
    return _ops.cuda_tree_attention_cached(q, cache.k_codes, cache.v_codes, cache.k_row_scales, cache.v_row_scales,
                                           cache.k_block_scales, cache.v_block_scales, tree_mask, past_length,
                                           past_lengths, max_past_length)


__all__ = [
    "cuda_apply_rope",
    "cuda_apply_rope_qk",
    "cuda_dequantize_nvfp4",
    "cuda_gqa_attention",
    "cuda_gqa_attention_cached",
    "cuda_kv_cache_append_",
    "cuda_quantized_kv_append_",
    "cuda_quantized_kv_read",
    "cuda_rms_norm",
    "cuda_tree_attention_cached",
    "cuda_unpack_e2m1_codes",
    "cuda_w4a16_linear",
    "cuda_w4a16_linear_grouped_decode",
    "quantize_nvfp4",
    "rope_frequencies",
    "NVFP4Tensor",
    "QuantizedKVCache",
]
