"""Plain 64-bit (and, for the quantiser's bytes, FP32) restatements of the
operators that verify drafted tokens over a quantised cache, in numpy/torch on
the CPU.  The tests' oracle; written from the definitions."""

from __future__ import annotations

import math

import numpy as np
import torch

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E4M3 = np.array([m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
                 for e in range(16) for m in range(8)][:127])
F32_MAX = np.finfo(np.float32).max


def nearest_code(x: np.ndarray, levels: np.ndarray) -> np.ndarray:
    """Index of the nearest level to x >= 0 (the even index of two as near), saturating."""
    hi = np.clip(np.searchsorted(levels, x), 0, len(levels) - 1)
    lo = np.clip(hi - 1, 0, None)
    up, down = np.abs(levels[hi] - x), np.abs(x - levels[lo])
    return np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo).astype(np.uint8)


def quantize_rows(fmt: str, rows: torch.Tensor):
    """(codes, row scales, block scales or None) with the FP32 operation order of the definition."""
    x = rows.float().cpu().numpy()
    f = np.float32
    bad = ~np.isfinite(x).all(-1)
    x = np.where(bad[..., None], f(0), x)
    amax = np.abs(x).max(-1)
    top = f(448 if fmt == "fp8" else 2688)
    with np.errstate(divide="ignore", over="ignore", invalid="ignore"):
        enc = np.where(amax == 0, f(1), np.minimum((f(1) / amax) * top, F32_MAX)).astype(f)
    gamma = np.where(bad, f("nan"), amax * f(1.0 / float(top))).astype(f)
    sign = np.signbit(x)
    if fmt == "fp8":
        code = nearest_code(np.abs(x * enc[..., None]).astype(np.float64), E4M3)
        codes = np.where(bad[..., None], 0, code | (sign * 128)).astype(np.uint8)
        return codes, gamma, None
    blocks = x.reshape(*x.shape[:-1], -1, 16)
    cand = (np.abs(blocks).max(-1) * (enc * f(1.0 / 6.0))[..., None]).astype(f)
    beta = nearest_code(cand.astype(np.float64), E4M3)
    value = E4M3[beta].astype(f)
    with np.errstate(divide="ignore", over="ignore"):
        factor = np.where(value > 0, np.minimum(f(1) / (value * (f(1) / enc)[..., None]), F32_MAX), f(0)).astype(f)
    y = (blocks * factor[..., None]).astype(f)
    code = nearest_code(np.abs(y).astype(np.float64), E2M1) | (np.signbit(blocks) * 8).astype(np.uint8)
    code = np.where(value[..., None] > 0, code, 0).reshape(x.shape).astype(np.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), gamma, beta


def stored_values(fmt: str, codes, gamma, beta=None) -> torch.Tensor:
    """FP64 values of stored rows (numpy or tensors)."""
    codes, gamma = np.asarray(codes), np.asarray(gamma).astype(np.float64)
    if fmt == "fp8":
        table = np.append(E4M3, np.nan)
        v = table[codes & 127] * np.where(codes > 127, -1.0, 1.0)
    else:
        v = np.stack((E2M1[codes & 7] * np.where(codes & 8, -1.0, 1.0),
                      E2M1[(codes >> 4) & 7] * np.where(codes & 128, -1.0, 1.0)), -1)
        v = v.reshape(*codes.shape[:-1], -1, 16) * np.append(E4M3, np.nan)[np.asarray(beta)][..., None]
        v = v.reshape(*codes.shape[:-1], -1)
    return torch.from_numpy(v * gamma[..., None])


def cache_values(cache) -> tuple[torch.Tensor, torch.Tensor]:
    """FP64 K and V of a QuantizedKVCache, or of a pair of BF16 caches."""
    if isinstance(cache, (tuple, list)):
        return tuple(x.cpu().double() for x in cache)
    out = []
    for n in "kv":
        fields = [getattr(cache, f"{n}_{f}") for f in ("codes", "row_scales", "block_scales")]
        out.append(stored_values(cache.format, *(None if x is None else x.cpu().numpy() for x in fields)))
    return tuple(out)


def rope(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, interleaved: bool, factor: float):
    x, r = x.cpu().double(), 2 * inv_freq.numel()
    angle = positions.cpu().double()[..., None] * inv_freq.cpu().double()
    angle = angle.expand(x.shape[0], x.shape[1], r // 2)[:, :, None]
    c, s = torch.cos(angle) * factor, torch.sin(angle) * factor
    e, o = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    y = x.clone()
    y[..., e] = x[..., e] * c - x[..., o] * s
    y[..., o] = x[..., e] * s + x[..., o] * c
    return y


def tree_attention(q, k, v, pasts, mask=None):
    """FP64 context, and sum_j p_j |v_j| (the size that rounding errors of p scale with).

    q [B, T, Hq, D]; k, v [B, Hkv, C, D] FP64; keys a query does not see are left out before any arithmetic."""
    q = q.cpu().double()
    b, t, hq, d = q.shape
    group = hq // k.shape[1]
    ctx, size = torch.zeros_like(q), torch.zeros_like(q)
    for i in range(b):
        p = int(pasts[i])
        for u in range(t):
            row = torch.arange(t) <= u if mask is None else (mask if mask.ndim == 2 else mask[i])[u].cpu().bool()
            seen = torch.cat((torch.arange(p), p + row.nonzero().flatten()))
            if seen.numel() == 0:
                continue
            for h in range(hq):
                kk, vv = k[i, h // group, seen], v[i, h // group, seen]
                w = torch.softmax(kk @ q[i, u, h] / math.sqrt(d), 0)
                ctx[i, u, h], size[i, u, h] = w @ vv, w @ vv.abs()
    return ctx, size


def random_tree(batch: int, tokens: int, seed: int):
    """Ancestor masks [B, T, T] and depths [B, T] of random trees, ancestors first."""
    g = torch.Generator().manual_seed(seed)
    mask, depth = torch.zeros((batch, tokens, tokens), dtype=torch.bool), torch.zeros((batch, tokens), dtype=torch.int64)
    for b in range(batch):
        for t in range(tokens):
            if t:
                parent = int(torch.randint(0, t, (1,), generator=g))
                mask[b, t], depth[b, t] = mask[b, parent], depth[b, parent] + 1
            mask[b, t, t] = True
    return mask, depth
