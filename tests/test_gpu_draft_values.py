"""GPU checks of tree attention at the values that hide faults: infinities and NaN in committed rows of V, and keys
that carry nearly all of the weight while their V rows are small.

Tolerances as in test_gpu_draft_ops.py: 2^-8 |o| for the rounding of the result to BF16, 2^-10 sum_j p_j |v_j| for
the probabilities and scores.  Where rows of V differ by more than FP16 spans, what the header of the kernels states
besides: over codes a weight has steps of 2^-28 of the largest p_j gamma_j (gamma_j: the row scale), so that every
key may add half a step times its code.
"""

from __future__ import annotations

import math

import pytest
import torch

import draft_reference as ref
from test_gpu_draft_ops import FORMATS, check_context, filled, randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cp():
    import cuda_primitives

    return cuda_primitives


# Tokens of four query heads a KV head: 8, 24, 40 and 160 query rows, so that every kernel and both of its forms run.
TOKENS = [2, 6, 10, 40]


# ------------------------------------------------------------------ infinities and NaN in committed rows of V
def spoil(fmt, cache, slot, d0):
    """An infinity or NaN into V of every head at `slot`, around element d0; the elements it reaches."""
    if fmt == "bf16":
        cache[1][:, :, slot, d0] = float("nan" if slot % 2 else "-inf")
        return [d0]
    if fmt == "fp8":
        cache.v_codes[:, :, slot, d0] = 0x7F
        return [d0]
    cache.v_block_scales[:, :, slot, d0 // 16] = 0x7F
    return list(range(d0 // 16 * 16, d0 // 16 * 16 + 16))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("t", TOKENS)
def test_infinities_and_nan_in_committed_rows_reach_every_query(cp, fmt, d, t):
    """Just before P_b, at the start of the tile that holds P_b, and a tile earlier: wherever P_b falls."""
    for p in (64, 127, 1000):
        for slot in {p - 1, p // 64 * 64 - (p % 64 == 0), max(0, p // 64 * 64 - 1), p - 50}:
            cache = filled(cp, fmt, 1, 2, 1088, d, 11)
            q = randn((1, t, 8, d), 12)
            wild = spoil(fmt, cache, slot, 37)
            got = cp.cuda_tree_attention_cached(q.cuda(), cache, p).cpu()
            assert not torch.isfinite(got[..., wild]).any(), (p, slot)
            rest = [i for i in range(d) if i not in wild]
            exact, size = ref.tree_attention(q, *ref.cache_values(cache), [p])
            check_context(got[..., rest], exact[..., rest], size[..., rest])


# ------------------------------------------------------------------ heavy keys with small rows of V
def check_shares(cache, q, got, past):
    """A causal chain's context, with the steps of the weights over codes in the tolerance."""
    k, v = (x.cuda() for x in ref.cache_values(cache))
    q = q.cuda().double()
    b, t, hq, d = q.shape
    group = hq // k.shape[1]
    quantised = not isinstance(cache, tuple)
    for u in range(t):
        n = past + u + 1
        for h in range(k.shape[1]):
            heads = slice(h * group, (h + 1) * group)
            w = torch.softmax(torch.einsum("bjd,bgd->bgj", k[:, h, :n], q[:, u, heads]) / math.sqrt(d), -1)
            exact, size = torch.einsum("bgj,bjd->bgd", w, v[:, h, :n]), torch.einsum("bgj,bjd->bgd", w, v[:, h, :n].abs())
            if quantised:
                gamma = cache.v_row_scales[:, h, :n].double()
                codes = (v[:, h, :n] / gamma.clamp(min=1e-300)[..., None]).abs().sum(1)
                size = size + 2.0 ** 10 * 2.0 ** -29 * (w * gamma[:, None]).amax(-1)[..., None] * codes[:, None]
            check_context(got[:, u, heads], exact.cpu(), size.cpu())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("t", TOKENS)
@pytest.mark.parametrize("small,lead", [(24, 40), (30, 60), (60, 90)])
def test_heavy_keys_whose_rows_of_v_are_small(cp, fmt, d, t, small, lead):
    """One key has 2^lead times the weight of any other and a row of V 2^-small times theirs, at the start, in the
    middle, at the end of the committed rows, and among the drafted ones."""
    p, cap = 1000, 1088
    g = torch.Generator().manual_seed(7)
    u = torch.where(torch.rand((d,), generator=g) < 0.5, -1.0, 1.0)
    for heavy in (0, 500, p - 1, p):
        k = 0.05 * torch.randn((1, cap, 2, d), generator=g)
        v = torch.randn((1, cap, 2, d), generator=g)
        k[:, heavy] = u * lead * math.log(2.0) / math.sqrt(d)  # q = u: a score of lead ln 2
        v[:, heavy] *= 2.0 ** -small
        q = (u * (1.0 + 0.02 * torch.randn((1, t, 8, 1), generator=g))).to(torch.bfloat16)
        k, v = k.to(torch.bfloat16), v.to(torch.bfloat16)
        if fmt == "bf16":
            cache = (k.transpose(1, 2).contiguous().cuda(), v.transpose(1, 2).contiguous().cuda())
        else:
            cache = cp.QuantizedKVCache.allocate(1, 2, cap, d, fmt)
            cp.cuda_quantized_kv_append_(cache, k.cuda(), v.cuda(), 0)
        got = cp.cuda_tree_attention_cached(q.cuda(), cache, p)
        check_shares(cache, q, got, p)


@pytest.mark.parametrize("fmt", ["fp8", "nvfp4"])
@pytest.mark.parametrize("t", TOKENS)
@pytest.mark.parametrize("order", ["rising", "falling", "rising in 64", "shuffled"])
def test_sizes_of_v_that_change_along_the_cache(cp, fmt, t, order):
    """Rows of V from 2^-50 to 2^50 against scores that make every row's share alike, and rows of zeros before the
    first that counts; enough units that a CTA walks several tiles of each."""
    b, p, cap, d = 40, 1000, 1088, 128
    g = torch.Generator().manual_seed(8)
    u = torch.where(torch.rand((d,), generator=g) < 0.5, -1.0, 1.0)
    j = torch.arange(cap)
    at = {"rising": j, "falling": cap - 1 - j, "rising in 64": j % 64 * 17, "shuffled": j * 389 % cap}[order]
    size = 100.0 * at / (cap - 1) - 50.0  # log2
    k = (-size[:, None, None] * math.log(2.0) / math.sqrt(d) * u).expand(b, cap, 2, d).to(torch.bfloat16)
    v = torch.randn((b, cap, 2, d), generator=g) * torch.exp2(size)[:, None, None]
    v[:, ::200] = 0
    v = v.to(torch.bfloat16)
    q = u.expand(b, t, 8, d).to(torch.bfloat16)
    cache = cp.QuantizedKVCache.allocate(b, 2, cap, d, fmt)
    cp.cuda_quantized_kv_append_(cache, k.cuda(), v.cuda(), 0)
    got = cp.cuda_tree_attention_cached(q.cuda(), cache, p)
    check_shares(cache, q, got, p)
