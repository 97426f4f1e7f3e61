"""GPU check of sequences that share a prefix's pages, as the documentation says to do it."""

from __future__ import annotations

import pytest
import torch

import paged_reference as ref
from test_gpu_draft_ops import check_context, randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cp():
    import cuda_primitives

    return cuda_primitives


@pytest.mark.parametrize("format", ["bf16", "nvfp4"])
def test_a_shared_prefix_is_held_by_one_row(cp, format):
    """Row 0 holds the prefix; the others what comes behind it, with lengths that start there.  One ends, its pages are
    handed out and written again, and the other still reads the prefix; at the end every page is free once."""
    size, n_prefix, hkv, d, t = 16, 3, 2, 128, 20
    prefix = n_prefix * size
    cache = cp.PagedKVCache.allocate(12, hkv, size, d, format)
    table = cp.PageTable.allocate(3, 6, 12, size)
    own = torch.zeros((3,), dtype=torch.int64, device="cuda")  # lengths behind the prefix; row 0: of the prefix

    def grow(counts, seed):
        slots, granted = cp.cuda_reserve_pages_(table, own, t, counts=counts)
        assert torch.equal(granted, counts)
        k, v = (randn((3, t, hkv, d), s).cuda() for s in (seed, seed + 1))
        cp.cuda_paged_kv_append_(cache, k, v, slots, counts=granted)

    def attend(seed):
        """The last token of rows 1 and 2 over the prefix and their own pages."""
        rows = torch.cat((table.pages[:1, :n_prefix].expand(2, -1), table.pages[1:]), 1)
        past = prefix + own[1:] - 1
        q = randn((2, 1, 4 * hkv, d), seed)
        got = cp.cuda_paged_attention(q.cuda(), cache, rows, past_lengths=past, max_past_length=rows.shape[1] * size - 1)
        check_context(got, *ref.attention(q, cache, rows, past.tolist()))

    for at in range(0, prefix, 16):
        grow(torch.tensor([16, 0, 0]).cuda(), at)
        own[0] += 16
    counts = torch.tensor([0, 20, 13]).cuda()
    grow(counts, 100)
    own += counts
    attend(1)
    own[1] = 0  # sequence 1 ends
    cp.cuda_release_pages_(table, own)
    held = table.pages[0, :n_prefix].tolist()
    assert not set(held) & set(table.free_pages[:int(table.free_count)].tolist())
    for seed in (200, 300):  # a new sequence in its place, and sequence 2 goes on
        counts = torch.tensor([0, 17, 18]).cuda()
        grow(counts, seed)
        own += counts
        attend(seed)
    cp.cuda_release_pages_(table, torch.zeros_like(own))
    assert int(table.free_count) == 12 and sorted(table.free_pages.tolist()) == list(range(12))
