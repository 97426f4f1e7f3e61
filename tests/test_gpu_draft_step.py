"""GPU checks of the drafted-token step over BF16 caches: sequences of their own lengths, and acceptance of a path."""

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


def test_appending_at_each_sequence_s_own_length(cp):
    """Slots outside a cache are not written, and what no host check sees is refused where it can be."""
    cache = [randn((3, HKV, CAP, D), s).cuda() for s in (3, 4)]
    want = [c.clone() for c in cache]
    k, v = (randn((3, 5, HKV, D), s).cuda() for s in (5, 6))
    past = torch.tensor([7, CAP - 2, -1])
    for w, rows in zip(want, (k, v)):
        w[0, :, 7:12] = rows[0].transpose(0, 1)
        w[1, :, CAP - 2:] = rows[1, :2].transpose(0, 1)
    assert cp.cuda_kv_cache_append_(*cache, k, v, past_lengths=past.cuda()) is None
    assert all(torch.equal(c, w) for c, w in zip(cache, want))
    for lengths, text in ((past.cuda()[:2], "shape"), (past.cuda().int(), "dtype"), (past, "CUDA tensor")):
        with pytest.raises(RuntimeError, match=text):
            cp.cuda_kv_cache_append_(*cache, k, v, past_lengths=lengths)
    with pytest.raises(RuntimeError, match="must match cache"):
        cp.cuda_kv_cache_append_(*cache, k[:2], v[:2], past_lengths=past.cuda())


def test_tree_step_over_bf16_caches_with_lengths_of_their_own(cp):
    """Every sequence gets what it would at a common length, and accepts its own path."""
    from tree_decoding import accept_drafted_, cuda_decoder_attention_tree_forward_

    past = torch.tensor([40, 9])
    x, (g_in, g_q, g_k), (wq, wk, wv, wo) = step_inputs(cp, B, T, H, HKV, D, 7)
    mask, depths = ref.random_tree(B, T, 12)
    start = [randn((B, HKV, CAP, D), s).cuda() for s in (1, 2)]
    args = dict(depths=depths.cuda(), tree_mask=mask.cuda(), inv_freq=cp.rope_frequencies(D)[0])

    def step(cache, *a, **kw):
        return cuda_decoder_attention_tree_forward_(x, g_in, wq, wk, wv, g_q, g_k, wo, cache, *a, **args, **kw)

    cache = tuple(c.clone() for c in start)
    y, k, v = step(cache, past_lengths=past.cuda(), max_past_length=58)
    path, counts = paths(mask)
    accept_drafted_(cache, k, v, path.cuda(), past_lengths=past.cuda(), counts=counts.cuda())
    for i in range(B):  # the whole batch at this sequence's length
        p, n = int(past[i]), int(counts[i])
        alone = tuple(c.clone() for c in start)
        z, ka, va = step(alone, p)
        assert torch.equal(k[i], ka[i]) and torch.equal(v[i], va[i])
        # parts of the cache fall to other CTAs: the context's sums may round differently
        assert (y[i].float() - z[i].float()).abs().max() <= 2.0 ** -6 * float(z.abs().max())
        for c, a, s, rows in zip(cache, alone, start, (k, v)):
            assert torch.equal(a[i, :, p:p + T], rows[i].transpose(0, 1))
            want = a[i].clone()
            want[:, p:p + n] = rows[i, path[i, :n].cuda()].transpose(0, 1)
            assert torch.equal(c[i], want)
            assert torch.equal(want[:, :p], s[i, :, :p]) and torch.equal(want[:, p + T:], s[i, :, p + T:])
