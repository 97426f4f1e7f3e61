"""GPU checks of tree attention at shapes past the small ones: many sequences, on both sides of where the general kernel
takes over, prompts of many passes of query rows, and every one of many repeated calls."""

from __future__ import annotations

import pytest
import torch

import draft_reference as ref
from test_gpu_draft_ops import FORMATS, check_tree, filled, randn
from test_gpu_draft_values import check_shares

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cp():
    import cuda_primitives

    return cuda_primitives


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("b", [31, 32, 33, 65, 1023, 1024, 1025])
@pytest.mark.parametrize("t,hq", [(1, 2), (9, 4)])
def test_many_sequences(cp, fmt, b, t, hq):
    """Lengths from 0 up; the prefix of tiles over more sequences than a warp has lanes."""
    if b > 100 and t > 1:
        hq = 1
    pasts = [(i * 37) % (128 - t) for i in range(b)]
    check_tree(cp, fmt, b, t, hq, 1, 64 if t == 1 else 128, pasts, 128, seed=b)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d,t,group", [(64, 600, 4), (128, 600, 4), (128, 257, 1), (256, 150, 2), (96, 100, 2)])
@pytest.mark.parametrize("p", [0, 70])
def test_prompts(cp, fmt, d, t, group, p):
    """A causal prompt: up to ten passes of 256 rows, whose last tokens see tiles that the first do not."""
    cache = filled(cp, fmt, 1, 1, -(-(p + t) // 64) * 64, d, 21)
    q = randn((1, t, group, d), 22)
    check_shares(cache, q, cp.cuda_tree_attention_cached(q.cuda(), cache, p), p)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("t", [2, 3, 6, 16, 40])  # 8, 12, 24, 64 and 160 query rows a KV head
@pytest.mark.parametrize("d", [64, 128])
def test_every_repeated_call_gives_the_same_bits(cp, fmt, t, d):
    """Uneven units that many CTAs share, whichever warp or CTA comes first."""
    from tree_decoding import check_tree_wait_status

    b, hkv, group, cap = 3, 3, 4, 6144
    cache = filled(cp, fmt, b, hkv, cap, d, 41)
    q = randn((b, t, hkv * group, d), 42).cuda()
    mask = ref.random_tree(b, t, 43)[0].cuda()
    past = torch.tensor([cap - t, 1717, 70]).cuda()

    def call():
        return cp.cuda_tree_attention_cached(q, cache, tree_mask=mask, past_lengths=past, max_past_length=cap - t)

    check_tree_wait_status()
    first = call().view(torch.int16)
    other = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(300):
        other += (call().view(torch.int16) != first).any()
    assert int(other) == 0 and torch.isfinite(first.view(torch.bfloat16).float()).all()
    check_tree_wait_status()
