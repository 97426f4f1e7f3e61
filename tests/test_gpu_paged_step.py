"""GPU checks of the paged operators together, as a server uses them: steps of drafted trees, whole and captured."""

from __future__ import annotations

import pytest
import torch

import draft_reference
import paged_reference as ref
from test_gpu_draft_ops import randn, step_inputs

pytestmark = pytest.mark.gpu

B, T, H, HKV, D, SIZE, VOCAB = 4, 6, 512, 2, 64, 16, 500


@pytest.fixture(scope="module")
def cp():
    import cuda_primitives

    return cuda_primitives


def trees(seed):
    """Parents [B, T], masks and depths of random trees."""
    g = torch.Generator().manual_seed(seed)
    parents = (torch.rand((B, T), generator=g) * torch.arange(T)).long()
    parents[:, 0] = -1
    mask, depth = torch.zeros((B, T, T), dtype=torch.bool), torch.zeros((B, T), dtype=torch.int64)
    for b in range(B):
        for t in range(T):
            if t:
                mask[b, t], depth[b, t] = mask[b, parents[b, t]], depth[b, parents[b, t]] + 1
            mask[b, t, t] = True
    return parents, mask, depth


def probabilities(seed):
    g = torch.Generator().manual_seed(seed)
    logits = 2.0 * torch.randn((B, T, VOCAB), generator=g)
    target = torch.softmax(logits, -1)
    draft = torch.softmax(logits + 0.3 * torch.randn((B, T, VOCAB), generator=g), -1)
    return target, draft, torch.rand((B, T), generator=g), g


@pytest.mark.parametrize("format", ["bf16", "fp8", "nvfp4"])
def test_steps_of_drafted_trees(cp, format):
    """Five steps beside the same ones over a cache of whole sequences: paths, tokens, lengths, rows and outputs."""
    from paged_decoding import accept_drafted_paged_, cuda_decoder_attention_paged_forward_
    from tree_decoding import accept_drafted_, check_tree_wait_status, cuda_decoder_attention_tree_forward_

    _, (g_in, g_q, g_k), (wq, wk, wv, wo) = step_inputs(cp, B, T, H, HKV, D, 6)
    pages = 40
    cache = cp.PagedKVCache.allocate(pages, HKV, SIZE, D, format)
    table = cp.PageTable.allocate(B, 9, pages, SIZE)
    if format == "bf16":
        whole = tuple(torch.zeros((B, HKV, 128, D), dtype=torch.bfloat16, device="cuda") for _ in "kv")
    else:
        whole = cp.QuantizedKVCache.allocate(B, HKV, 128, D, format)
    freq = cp.rope_frequencies(D)[0]
    past = torch.tensor([0, 13, 30, 15]).cuda()
    # what the sequences hold at the start
    slots, granted = cp.cuda_reserve_pages_(table, torch.zeros_like(past), 30, counts=past)
    assert granted.tolist() == past.tolist()
    k0, v0 = randn((B, 30, HKV, D), 1).cuda(), randn((B, 30, HKV, D), 2).cuda()
    cp.cuda_paged_kv_append_(cache, k0, v0, slots, counts=past)
    if format == "bf16":
        cp.cuda_kv_cache_append_(*whole, k0, v0, 0)
    else:
        cp.cuda_quantized_kv_append_(whole, k0, v0, 0, counts=past)
    for step in range(5):
        parents, mask, depth = trees(step)
        target, draft, u, g = probabilities(50 + step)
        tokens = torch.zeros((B, T), dtype=torch.int64)
        for t in range(1, T):
            tokens[:, t] = torch.multinomial(draft[torch.arange(B), parents[:, t]], 1, generator=g)[:, 0]
        x = randn((B, T, H), 90 + step).cuda()
        args = dict(depths=depth.cuda(), tree_mask=mask.cuda(), inv_freq=freq, past_lengths=past, max_past_length=100)
        slots, granted = cp.cuda_reserve_pages_(table, past, T)
        assert granted.tolist() == [T] * B
        y, k, v = cuda_decoder_attention_paged_forward_(x, g_in, wq, wk, wv, g_q, g_k, wo, cache, table.pages, slots,
                                                        counts=granted, **args)
        z, ka, va = cuda_decoder_attention_tree_forward_(x, g_in, wq, wk, wv, g_q, g_k, wo, whole, **args)
        assert torch.equal(k, ka) and torch.equal(v, va)
        # the parts of a sum fall to other CTAs: the contexts may round differently
        assert (y.float() - z.float()).abs().max() <= 2.0 ** -6 * float(z.abs().max())
        path, counts, nexts = cp.cuda_verify_drafted(target.cuda(), tokens.cuda(), u.cuda(), draft_probs=draft.cuda(),
                                                     parents=parents.cuda(), counts=granted)
        assert (path.tolist(), counts.tolist(), nexts.tolist()) == ref.verify(target, tokens, u, draft, parents)
        accept_drafted_paged_(cache, k, v, path, slots, counts=counts)
        accept_drafted_(whole, k, v, path, past_lengths=past, counts=counts)
        past += counts
        cp.cuda_release_pages_(table, past)
        held = table.held.tolist()
        assert held == [-(-int(p) // SIZE) for p in past] and int(table.free_count) == pages - sum(held)
        # the committed rows, byte for byte as the whole cache holds them
        n = int(past.max())
        at = torch.arange(n).cuda()
        slot = table.pages.gather(1, (at // SIZE).expand(B, n)).long() * SIZE + at % SIZE
        slot = torch.where(at < past[:, None], slot, -1)
        got = cp.cuda_paged_kv_read(cache, slot)
        want = [c[:, :, :n] for c in whole] if format == "bf16" else cp.cuda_quantized_kv_read(whole, 0, n)
        live = (at < past[:, None])[:, None, :, None]
        assert all(torch.equal(a, torch.where(live, b, 0)) for a, b in zip(got, want))
    check_tree_wait_status()
    cp.cuda_release_pages_(table, torch.zeros_like(past))
    assert sorted(table.free_pages.tolist()) == list(range(pages)) and int(table.free_count) == pages


def test_a_sequence_that_gets_no_pages_is_left_as_it_is(cp):
    """Out of pages: its rows, lengths and table stay, its context and outputs are zeros, the others go on."""
    from paged_decoding import accept_drafted_paged_, cuda_decoder_attention_paged_forward_

    x, (g_in, g_q, g_k), (wq, wk, wv, wo) = step_inputs(cp, B, T, H, HKV, D, 7)
    cache = cp.PagedKVCache.allocate(6, HKV, SIZE, D)
    for c in (cache.k_codes, cache.v_codes):
        c.fill_(7.0)
    table = cp.PageTable.allocate(B, 4, 6, SIZE)
    past = torch.tensor([0, 14, 16, 12]).cuda()
    _, granted = cp.cuda_reserve_pages_(table, torch.zeros_like(past), 16, counts=past)
    assert granted.tolist() == past.tolist()  # a page each for three
    cp.cuda_reserve_pages_(table, torch.zeros_like(past), 64, counts=torch.tensor([0, 64, 0, 0]).cuda())
    before = table.pages.clone()
    slots, granted = cp.cuda_reserve_pages_(table, past, T)  # none left: who needs one goes without
    assert granted.tolist() == [0, T, 0, 0] and torch.equal(table.pages, before)
    rows = cache.k_codes.clone()
    y, k, v = cuda_decoder_attention_paged_forward_(
        x, g_in, wq, wk, wv, g_q, g_k, wo, cache, table.pages, slots, inv_freq=cp.rope_frequencies(D)[0],
        past_lengths=past, max_past_length=40, counts=granted)
    assert (y[granted == 0] == 0).all() and (y[1] != 0).any()
    target, draft, u, _ = probabilities(3)
    path, counts, nexts = cp.cuda_verify_drafted(target.cuda(), torch.zeros((B, T), dtype=torch.int64).cuda(), u.cuda(),
                                                 draft_probs=draft.cuda(), counts=granted)
    assert counts[granted == 0].tolist() == [0, 0, 0] and nexts[granted == 0].tolist() == [-1] * 3
    accept_drafted_paged_(cache, k, v, path, slots, counts=counts)
    changed = (cache.k_codes != rows).any(dim=3).any(dim=1)  # [N, S]
    own = slots[1]
    assert set(changed.flatten().nonzero().flatten().tolist()) <= set(own.tolist())


def test_a_captured_step_follows_lengths_and_tables(cp):
    """One graph of a whole step, replayed as the sequences grow, beside the same steps launched one by one."""
    from paged_decoding import accept_drafted_paged_, cuda_decoder_attention_paged_forward_

    _, (g_in, g_q, g_k), (wq, wk, wv, wo) = step_inputs(cp, B, T, H, HKV, D, 8)
    freq, steps = cp.rope_frequencies(D)[0], 12
    parents, mask, depth = (t.cuda() for t in trees(3))
    xs = randn((steps, B, T, H), 4).cuda()
    us = torch.rand((steps, B, T), generator=torch.Generator().manual_seed(5)).cuda()
    target, draft, _, g = probabilities(9)
    target, draft = target.cuda(), draft.cuda()
    tokens = torch.randint(0, VOCAB, (B, T), generator=g).cuda()

    def state():
        return (cp.PagedKVCache.allocate(60, HKV, SIZE, D, "nvfp4"), cp.PageTable.allocate(B, 12, 60, SIZE),
                torch.zeros((B,), dtype=torch.int64, device="cuda"))

    def step(s, x, u):
        cache, table, past = s
        slots, granted = cp.cuda_reserve_pages_(table, past, T)
        y, k, v = cuda_decoder_attention_paged_forward_(
            x, g_in, wq, wk, wv, g_q, g_k, wo, cache, table.pages, slots, depths=depth, tree_mask=mask, inv_freq=freq,
            past_lengths=past, max_past_length=12 * SIZE - T, counts=granted)
        path, counts, nexts = cp.cuda_verify_drafted(target, tokens, u, draft_probs=draft, parents=parents, counts=granted)
        accept_drafted_paged_(cache, k, v, path, slots, counts=counts)
        past += counts
        cp.cuda_release_pages_(table, past)
        return y, path, counts, nexts

    a, b = state(), state()
    x, u = xs[0].clone(), us[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(b, x, u)
    for i in range(steps):
        want = step(a, xs[i], us[i])
        x.copy_(xs[i])
        u.copy_(us[i])
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip(out, want))
        assert torch.equal(a[2], b[2]) and torch.equal(a[1].pages, b[1].pages)
    assert torch.equal(a[0].k_codes, b[0].k_codes) and torch.equal(a[0].v_row_scales, b[0].v_row_scales)
    assert (a[2] >= steps).all()


def test_two_streams_and_another_current_stream(cp):
    """Calls on two streams at once, each with its own pool and table, give what they give one after another."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    sets = []
    for i in range(2):
        g = torch.Generator().manual_seed(i)
        table = torch.randperm(64, generator=g).int().view(4, 16).cuda()
        cache = cp.PagedKVCache.allocate(64, 2, 16, 128, "fp8")
        k, v = randn((4, 256, 2, 128), 2 * i).cuda(), randn((4, 256, 2, 128), 2 * i + 1).cuda()
        at = torch.arange(256).cuda()
        slots = table[:, at // 16].long() * 16 + at % 16
        cp.cuda_paged_kv_append_(cache, k, v, slots)
        sets.append((cache, table, randn((4, 1, 8, 128), 9 + i).cuda(), torch.tensor([255, 100, 17, 0]).cuda()))

    def call(s):
        cache, table, q, past = s
        return cp.cuda_paged_attention(q, cache, table, past_lengths=past, max_past_length=255)

    want = [call(s) for s in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(30):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(call(sets[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])
