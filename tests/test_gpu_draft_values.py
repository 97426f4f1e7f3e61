"""GPU checks of tree attention at the values that hide faults: infinities and NaN in committed rows of V.

Tolerances as in test_gpu_draft_ops.py: 2^-8 |o| for the rounding of the result to BF16, 2^-10 sum_j p_j |v_j| for
the probabilities and scores.
"""

from __future__ import annotations

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
