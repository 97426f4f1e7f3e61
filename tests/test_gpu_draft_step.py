"""GPU checks of the drafted-token step over BF16 caches: acceptance of a path of the tree."""

from __future__ import annotations

import pytest
import torch

import draft_reference as ref
from test_gpu_draft_ops import randn, step_inputs

pytestmark = pytest.mark.gpu

B, T, H, HKV, D, CAP = 2, 6, 512, 2, 64, 64


@pytest.fixture(scope="module")
def cp():
    import cuda_primitives

    return cuda_primitives


def paths(mask):
    """The path to the last node of every sequence, padded with -1, and its length."""
    path = torch.full((mask.shape[0], mask.shape[1]), -1, dtype=torch.int64)
    counts = torch.zeros((mask.shape[0],), dtype=torch.int64)
    for i, m in enumerate(mask):
        nodes = m[-1].nonzero().flatten()
        path[i, :len(nodes)], counts[i] = nodes, len(nodes)
    return path, counts


@pytest.mark.parametrize("kind", [tuple, list])
def test_accepting_a_path_over_bf16_caches(cp, kind):
    """The accepted tokens' rows, bit for bit, in consecutive slots, and nothing else changed."""
    from tree_decoding import accept_drafted_, cuda_decoder_attention_tree_forward_

    past = 40
    x, (g_in, g_q, g_k), (wq, wk, wv, wo) = step_inputs(cp, B, T, H, HKV, D, 6)
    mask, depths = ref.random_tree(B, T, 12)
    cache = kind(randn((B, HKV, CAP, D), s).cuda() for s in (1, 2))
    _, k, v = cuda_decoder_attention_tree_forward_(
        x, g_in, wq, wk, wv, g_q, g_k, wo, cache, past, depths=depths.cuda(), tree_mask=mask.cuda(),
        inv_freq=cp.rope_frequencies(D)[0])
    path, counts = paths(mask)
    assert len(set(counts.tolist())) > 1 and (counts < T).any()  # trees that branch, paths of different lengths
    want = [c.clone() for c in cache]
    for i in range(B):
        n = int(counts[i])
        for w, rows in zip(want, (k, v)):
            w[i, :, past:past + n] = rows[i, path[i, :n].cuda()].transpose(0, 1)
    accept_drafted_(cache, k, v, path.cuda(), past, counts=counts.cuda())
    assert all(torch.equal(c, w) for c, w in zip(cache, want))
    whole = [c.clone() for c in want]
    nodes = torch.tensor([[0, 2], [1, 3]]).cuda()
    for w, rows in zip(whole, (k, v)):
        w[:, :, past:past + 2] = torch.stack([rows[i, nodes[i]] for i in range(B)]).transpose(1, 2)
    accept_drafted_(cache, k, v, nodes, past)
    assert all(torch.equal(c, w) for c, w in zip(cache, whole))
    with pytest.raises(RuntimeError, match="exceeds cache capacity"):
        accept_drafted_(cache, k, v, path.cuda(), CAP - 2, counts=counts.cuda())
    with pytest.raises(ValueError, match="per-sequence past_lengths need"):
        accept_drafted_(cache, k, v, nodes, past_lengths=counts.cuda())
