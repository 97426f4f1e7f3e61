"""GPU checks of the paged KV cache's operators against their definitions.

Tolerances: pages, slots and stored rows bit for bit; attention as for the
attention over whole caches (test_gpu_draft_ops): the result's rounding to BF16,
and probabilities kept to 11 bits at least.
"""

from __future__ import annotations

import pytest
import torch

import draft_reference
import paged_reference as ref
from test_gpu_draft_ops import check_context, randn, rows_of_all_sizes

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cp():
    import cuda_primitives

    return cuda_primitives


def state(table):
    n = int(table.free_count)
    return table.pages.tolist(), table.held.tolist(), table.free_pages[:n].tolist()


def table_of(cp, batch, most, pool, size, held, seed=0):
    """A table whose sequences hold ``held`` pages of a pool in no order; the rest are free."""
    g = torch.Generator().manual_seed(seed)
    t = cp.PageTable.allocate(batch, most, pool, size)
    order = torch.randperm(pool, generator=g).int()
    at = 0
    for b, n in enumerate(held):
        t.pages[b, :n] = order[at:at + n].cuda()
        at += n
    t.held.copy_(torch.tensor(held))
    t.free_pages[:pool - at] = order[at:].cuda()
    t.free_count.fill_(pool - at)
    return t


# ------------------------------------------------------------------ pages and slots
@pytest.mark.parametrize("batch,most,size,tokens,seed", [
    (1, 1, 16, 1, 1), (3, 5, 16, 7, 2), (8, 40, 16, 1, 3), (33, 9, 48, 100, 4), (5, 200, 32, 2048, 5),
    (1024, 6, 16, 3, 6), (1025, 6, 16, 20, 7), (2500, 3, 64, 1, 8), (64, 130, 16, 2000, 9),
])
def test_reserve_and_release(cp, batch, most, size, tokens, seed):
    """Ragged lengths and counts, a pool that runs out, and what was taken given back."""
    g = torch.Generator().manual_seed(seed)
    room = most * size
    pasts = torch.randint(0, max(1, room - tokens + 1), (batch,), generator=g)
    pasts[torch.rand((batch,), generator=g) < 0.1] = room  # does not fit the table
    pasts[torch.rand((batch,), generator=g) < 0.1] = 0
    pasts[torch.rand((batch,), generator=g) < 0.05] = -3
    counts = torch.randint(-1, tokens + 3, (batch,), generator=g)
    held = [min(most, max(0, -(-int(p) // size) + int(torch.randint(0, 2, (1,), generator=g)))) for p in pasts]
    need = sum(max(0, -(-(int(p) + tokens) // size) - h) for p, h in zip(pasts, held))
    for spare, n in ((need + 3, None), (need // 2, counts), (1, None)):
        t = table_of(cp, batch, most, sum(held) + max(1, spare), size, held, seed)
        before = state(t)
        want = ref.reserve(*before, size, t.free_pages.numel(), pasts.tolist(), n, tokens)
        slots, granted = cp.cuda_reserve_pages_(t, pasts.cuda(), tokens, counts=None if n is None else n.cuda())
        assert state(t) == want[:3]
        assert slots.tolist() == want[3] and granted.tolist() == want[4]
        after = state(t)
        kept = pasts + torch.randint(-20, tokens + 1, (batch,), generator=g)
        cp.cuda_release_pages_(t, kept.cuda())
        assert state(t) == ref.release(*after, size, t.free_pages.numel(), kept.tolist())
        cp.cuda_release_pages_(t, torch.zeros((batch,), dtype=torch.int64).cuda())
        assert (t.pages == -1).all() and (t.held == 0).all()
        assert sorted(t.free_pages.tolist()) == list(range(t.free_pages.numel()))


def test_release_undoes_reserve_also_in_a_graph(cp):
    past = torch.tensor([5, 100, 31, 0]).cuda()
    t = table_of(cp, 4, 20, 40, 16, [1, 7, 2, 0])
    before = state(t)
    cp.cuda_reserve_pages_(t, past, 33)
    cp.cuda_release_pages_(t, past)
    assert state(t) == before
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        slots, granted = cp.cuda_reserve_pages_(t, past, 33)
    for _ in range(2):
        past += 33
        cp.cuda_reserve_pages_(t, past - 33, 33)
        graph.replay()  # a second time at once: nothing more is needed
        a = slots.clone()
        assert granted.tolist() == [33] * 4
        # the replay reads the lengths as they are now
        assert torch.equal(a[0] % 16, (past[0] + torch.arange(33).cuda()) % 16)
    held = t.held.tolist()
    assert held == [-(-(int(p) + 33) // 16) for p in past]


def test_tables_that_were_damaged_stay_inside(cp):
    """Entries, counts and lengths no call would leave: nothing is written outside, nothing named twice by them."""
    t = table_of(cp, 3, 4, 6, 16, [2, 1, 1])
    guard = torch.full((3, 4), 77, dtype=torch.int32, device="cuda")
    t.free_count.fill_(1 << 40)
    t.held.copy_(torch.tensor([1 << 50, -9, 3]))
    slots, granted = cp.cuda_reserve_pages_(t, torch.tensor([60, 0, (1 << 62)]).cuda(), 4)
    assert granted.tolist() == [4, 4, 0] and (slots < 6 * 16).all() and (slots[2] == -1).all()
    t.free_count.fill_(6)  # a full stack takes nothing more
    t.held.copy_(torch.tensor([4, 4, 4]))
    t.pages.copy_(torch.tensor([[0, 1, -1, 9], [2, 1 << 30, 3, 4], [-5, 5, 0, 1]]))
    free = t.free_pages.clone()
    cp.cuda_release_pages_(t, torch.tensor([-(1 << 60), 16, 1 << 60]).cuda())
    assert torch.equal(free, t.free_pages) and t.free_count.item() == 6
    assert t.held.tolist() == [0, 1, 4] and t.pages[0].tolist() == [-1] * 4 and t.pages[1].tolist() == [2, -1, -1, -1]
    assert t.pages[2].tolist() == [-5, 5, 0, 1] and (guard == 77).all()


def test_page_refusals(cp):
    t, n = cp.PageTable.allocate(2, 3, 5, 16), torch.zeros((2,), dtype=torch.int64).cuda()
    for past, kw, text in ((n[:1], {}, "shape"), (n.int(), {}, "dtype"), (n.cpu(), {}, "CUDA tensor"),
                           (n, dict(counts=n[:1]), "counts must have shape")):
        with pytest.raises(RuntimeError, match=text):
            cp.cuda_reserve_pages_(t, past, 1, **kw)
    with pytest.raises(RuntimeError, match="tokens must be positive"):
        cp.cuda_reserve_pages_(t, n, 0)
    with pytest.raises(RuntimeError, match="at most 2\\^20 tokens"):
        cp.cuda_reserve_pages_(t, n, (1 << 20) + 1)
    with pytest.raises(RuntimeError, match="lengths must have shape"):
        cp.cuda_release_pages_(t, n[:1])


# ------------------------------------------------------------------ rows by slots
def stored(cache):
    return [x for n in "kv" for x in (getattr(cache, f"{n}_{f}") for f in ("codes", "row_scales", "block_scales"))
            if x is not None]


@pytest.mark.parametrize("format", ["bf16", "fp8", "nvfp4"])
@pytest.mark.parametrize("b,t,hkv,d,size", [(1, 1, 1, 16, 16), (3, 7, 5, 64, 48), (5, 33, 2, 96, 16), (2, 5, 3, 128, 64),
                                            (17, 1, 8, 256, 32), (2, 300, 1, 80, 128)])
def test_rows_written_and_read_by_slots(cp, format, b, t, hkv, d, size):
    """Every stored byte, at given slots and nowhere else, and the rows back."""
    pages = -(-b * t // size) + 2
    cache = cp.PagedKVCache.allocate(pages, hkv, size, d, format)
    for x in stored(cache):
        x.view(torch.uint8).fill_(0x5a)
    before = [x.clone() for x in stored(cache)]
    g = torch.Generator().manual_seed(b * t)
    slots = torch.randperm(pages * size, generator=g)[:b * t].view(b, t)
    k, v = rows_of_all_sizes((b, t, hkv, d), 1), rows_of_all_sizes((b, t, hkv, d), 2)
    if t > 2:  # slots that are none: not written, read as zeros
        slots[0, 1], slots[-1, 2] = -1, pages * size
    cp.cuda_paged_kv_append_(cache, k.cuda(), v.cuda(), slots.cuda())
    inside = (slots >= 0) & (slots < pages * size)
    page, at = slots[inside] // size, slots[inside] % size
    i = 0
    for rows in (k, v):
        parts = (rows, None, None) if format == "bf16" else draft_reference.quantize_rows(format, rows)
        for part in parts:
            if part is None:
                continue
            want = before[i].clone()
            part = torch.as_tensor(part)
            want[page.cuda(), :, at.cuda()] = part[inside].cuda()
            assert torch.equal(stored(cache)[i].view(torch.uint8), want.view(torch.uint8))
            i += 1
    got = cp.cuda_paged_kv_read(cache, slots.cuda())
    for x, values in zip(got, ref.pool_values(cache)):
        back = values[slots.clamp(0, pages * size - 1) // size, :, slots.clamp(min=0) % size].to(torch.bfloat16)
        back[~inside] = 0
        assert torch.equal(x.cpu(), back.transpose(1, 2))


def test_rows_by_source_counts_and_strides(cp):
    """A path's rows, cut out of a projection's output; rows behind a count and numbers that are no token stay out."""
    b, t, hkv, d, size = 2, 6, 2, 64, 16
    flat = randn((b, t, 3 * hkv * d + 4), 3).cuda()
    for extra in (0, 1, 4):
        k, v = (flat[..., extra + i * hkv * d:extra + (i + 1) * hkv * d].unflatten(-1, (hkv, d)) for i in (0, 2))
        slots = torch.tensor([[3, 4, 5, 6, 7], [40, 41, 42, 43, 44]]).cuda()
        source = torch.tensor([[0, 2, 5], [1, -1, 9]]).cuda()
        cache = cp.PagedKVCache.allocate(3, hkv, size, d)
        cp.cuda_paged_kv_append_(cache, k, v, slots, source=source, counts=torch.tensor([2, 3]).cuda())
        want = torch.zeros_like(cache.k_codes)
        want[0, :, 3], want[0, :, 4], want[2, :, 8] = k[0, 0], k[0, 2], k[1, 1]
        assert torch.equal(cache.k_codes, want)
        assert torch.equal(cache.v_codes[0, :, 4], v[0, 2]) and (cache.v_codes[0, :, 5] == 0).all()


def test_row_refusals(cp):
    cache, x = cp.PagedKVCache.allocate(3, 2, 16, 64), randn((2, 3, 2, 64), 1).cuda()
    slots = torch.zeros((2, 3), dtype=torch.int64).cuda()
    for args, kw, text in (((x, x[:1], slots), {}, "same shape"), ((x[..., :32], x[..., :32], slots), {}, "matching the cache"),
                           ((x, x, slots[:, :2].contiguous()), {}, "n >= 3"), ((x, x, slots.int()), {}, "dtype"),
                           ((x, x, slots), dict(source=slots[:1]), "source must have shape"),
                           ((x, x, slots), dict(counts=slots[:, 0]), "counts must be contiguous"),
                           ((x.float(), x.float(), slots), {}, "dtype")):
        with pytest.raises(RuntimeError, match=text):
            cp.cuda_paged_kv_append_(cache, *args, **kw)
    with pytest.raises(RuntimeError, match="slots must have shape"):
        cp.cuda_paged_kv_read(cache, slots[0])


# ------------------------------------------------------------------ attention
def filled_pool(cp, format, pages, hkv, size, d, seed):
    """A pool of which every row is written, and its allocation."""
    cache = cp.PagedKVCache.allocate(pages, hkv, size, d, format)
    k, v = randn((pages, size, hkv, d), seed).cuda(), randn((pages, size, hkv, d), seed + 1).cuda()
    slots = torch.arange(pages * size).view(pages, size).cuda()
    cp.cuda_paged_kv_append_(cache, k, v, slots)
    return cache


def poison(cache, seen_slots):
    """Infinities, NaN and codes that stand for NaN in every row that no sequence has."""
    n, _, size = cache.k_codes.shape[:3]
    left = torch.ones((n * size,), dtype=torch.bool)
    left[seen_slots] = False
    page, at = left.nonzero().flatten() // size, left.nonzero().flatten() % size
    for x in stored(cache):
        bad = {torch.bfloat16: float("nan"), torch.float32: float("inf"), torch.uint8: 0x7f}[x.dtype]
        x[page.cuda(), :, at.cuda()] = bad


def sequences(cp, format, pasts, t, hkv, size, d, seed):
    """A pool and the table of sequences with these lengths and t tokens behind them; all else poisoned."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-(p + t) // size) for p in pasts]
    pages = sum(need) + 2
    cache = filled_pool(cp, format, pages, hkv, size, d, seed)
    order = torch.randperm(pages, generator=g).int()
    table = torch.randint(-(1 << 31), 1 << 31, (len(pasts), max(need) + 1), generator=g).int()  # junk behind the lengths
    slots, at = [], 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
        slots += [int(table[b, j // size]) * size + j % size for j in range(pasts[b] + t)]
    poison(cache, torch.tensor(slots))
    return cache, table


CASES = [
    # hkv, group, d, size, t, pasts
    (1, 1, 64, 16, 1, [0]),
    (2, 4, 128, 16, 1, [511, 0, 15, 16, 17]),
    (6, 4, 128, 64, 1, [63, 64, 700]),
    (3, 8, 128, 48, 1, [300, 1, 47, 95]),
    (2, 1, 256, 32, 1, [200, 31]),
    (1, 8, 64, 128, 1, [1000, 127]),
    (2, 16, 128, 256, 1, [400]),
    (1, 2, 96, 16, 1, [77, 130]),          # the general kernel's head dimensions
    (2, 3, 16, 80, 3, [100, 3]),
    (2, 4, 64, 32, 5, [90, 0, 31]),
    (2, 2, 128, 16, 8, [120, 250, 9]),
    (1, 8, 128, 16, 5, [333]),
    (2, 8, 256, 16, 3, [60, 5]),
    (1, 1, 128, 1024, 2, [1500, 20]),
    (1, 4, 64, 16, 33, [50]),
]


@pytest.mark.parametrize("format", ["bf16", "fp8", "nvfp4"])
@pytest.mark.parametrize("hkv,group,d,size,t,pasts", CASES)
def test_paged_attention(cp, format, hkv, group, d, size, t, pasts):
    cache, table = sequences(cp, format, pasts, t, hkv, size, d, 11)
    q = randn((len(pasts), t, hkv * group, d), 3)
    past, bound = torch.tensor(pasts), max(pasts) + 3
    bound = min(bound, table.shape[1] * size - t)
    for mask in (None, draft_reference.random_tree(len(pasts), t, 4)[0]):
        got = cp.cuda_paged_attention(q.cuda(), cache, table.cuda(), past_lengths=past.cuda(), max_past_length=bound,
                                      tree_mask=None if mask is None else mask.cuda())
        check_context(got, *ref.attention(q, cache, table, pasts, mask))


@pytest.mark.parametrize("format", ["bf16", "fp8", "nvfp4"])
@pytest.mark.parametrize("d,size", [(128, 16), (64, 64), (256, 48), (80, 32)])
def test_padded_batches_and_pages_that_are_gone(cp, format, d, size):
    """Rows past a count are zeros whatever q holds there; positions of pages that are not named are not seen."""
    pasts, t, hkv, group = [130, 40, 0, 65], 4, 2, 4
    cache, table = sequences(cp, format, pasts, t, hkv, size, d, 21)
    counts = torch.tensor([4, 2, 0, 9])
    table[0, 1], table[3, 0] = -1, cache.pages + 5  # the second page of one, the first of another
    q = randn((4, t, hkv * group, d), 3)
    q[1, 2:], q[2] = float("nan"), float("inf")
    got = cp.cuda_paged_attention(q.cuda(), cache, table.cuda(), past_lengths=torch.tensor(pasts).cuda(),
                                  max_past_length=130, counts=counts.cuda())
    check_context(got, *ref.attention(q.nan_to_num(0, 0, 0), cache, table, pasts, None, counts))
    assert (got[1, 2:] == 0).all() and (got[2] == 0).all()
    table[:] = -1
    got = cp.cuda_paged_attention(q.cuda(), cache, table.cuda(), past_lengths=torch.tensor(pasts).cuda(),
                                  max_past_length=130)
    assert (got == 0).all()


@pytest.mark.parametrize("format", ["bf16", "fp8", "nvfp4"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [8, 9, 12, 13, 16, 17, 24, 25, 32, 33, 64, 65, 128, 129, 256, 257, 600])
def test_rows_on_both_sides_of_every_kernel_rule(cp, format, d, rows):
    """Ragged sequences, one of them padding, pages that are gone, trees; every number of query rows a rule looks at."""
    group = next(g for g in (4, 3, 2, 1) if rows % g == 0) if rows != 600 else 8
    t, pasts, size = rows // group, [0, 333, 64, 201], {64: 32, 128: 16}[d]
    cache, table = sequences(cp, format, pasts, t, 2, size, d, rows)
    counts = torch.tensor([t, t, 0, max(1, t // 2)])
    table[1, 2], table[1, 5], table[3, 0] = -1, cache.pages, -7
    mask = draft_reference.random_tree(4, t, rows)[0]
    q = randn((4, t, 2 * group, d), 3)
    q[2], q[3, counts[3]:] = float("nan"), float("inf")
    got = cp.cuda_paged_attention(q.cuda(), cache, table.cuda(), past_lengths=torch.tensor(pasts).cuda(),
                                  max_past_length=333, counts=counts.cuda(), tree_mask=mask.cuda())
    check_context(got, *ref.attention(q.nan_to_num(0, 0, 0), cache, table, pasts, mask, counts))
    assert (got[2] == 0).all() and (got[3, counts[3]:] == 0).all()


@pytest.mark.parametrize("format", ["bf16", "fp8", "nvfp4"])
@pytest.mark.parametrize("t", [2, 5, 40])
def test_many_rows_of_wide_heads(cp, format, t):
    """Head dimension 256 keeps the streaming kernel, whatever the rows."""
    cache, table = sequences(cp, format, [70, 5], t, 2, 16, 256, 51)
    q = randn((2, t, 16, 256), 3)
    got = cp.cuda_paged_attention(q.cuda(), cache, table.cuda(), past_lengths=torch.tensor([70, 5]).cuda(),
                                  max_past_length=70)
    check_context(got, *ref.attention(q, cache, table, [70, 5]))


@pytest.mark.parametrize("format", ["bf16", "fp8", "nvfp4"])
@pytest.mark.parametrize("t", [1, 8, 40])
def test_infinities_in_rows_that_are_seen(cp, format, t):
    """Rows of V with an infinity or NaN reach the queries that see them, and no other."""
    pasts, size, d = [100, 70], 16, 128
    cache, table = sequences(cp, format, pasts, t, 1, size, d, 41)
    rows = randn((2, 1, 1, d), 9).cuda()
    rows[0, 0, 0, 5] = float("inf")
    wild = torch.tensor([[int(table[0, 37 // size]) * size + 37 % size],
                         [int(table[1, (70 + t - 1) // size]) * size + (70 + t - 1) % size]])
    cp.cuda_paged_kv_append_(cache, randn((2, 1, 1, d), 8).cuda(), rows, wild.cuda())
    q = randn((2, t, 4, d), 3)
    got = cp.cuda_paged_attention(q.cuda(), cache, table.cuda(), past_lengths=torch.tensor(pasts).cuda(),
                                  max_past_length=100)
    bad = ~torch.isfinite(got)
    assert bad[0, :, :, 5].all() and not bad[1].any()
    if format == "bf16":  # a quantised row with an infinity is NaN throughout
        bad[0, :, :, 5] = False
        assert not bad.any()
    else:
        assert bad[0].all()


@pytest.mark.parametrize("format", ["bf16", "fp8", "nvfp4"])
def test_masks_that_leave_a_row_empty(cp, format):
    cache, table = sequences(cp, format, [0, 0], 3, 2, 16, 64, 5)
    mask = torch.tensor([[[0, 0, 0], [1, 1, 0], [0, 0, 0]], [[1, 0, 0], [0, 0, 0], [0, 0, 1]]]).bool()
    q = randn((2, 3, 4, 64), 3)
    got = cp.cuda_paged_attention(q.cuda(), cache, table.cuda(), past_lengths=torch.zeros(2, dtype=torch.int64).cuda(),
                                  max_past_length=0, tree_mask=mask.cuda())
    check_context(got, *ref.attention(q, cache, table, [0, 0], mask))
    assert (got[0, 0] == 0).all() and (got[0, 2] == 0).all() and (got[1, 1] == 0).all()


@pytest.mark.parametrize("format", ["bf16", "fp8", "nvfp4"])
def test_many_ragged_sequences(cp, format):
    """Units that several CTAs share and CTAs that hold several units; two sequences that share pages."""
    g = torch.Generator().manual_seed(3)
    pasts = torch.randint(1, 900, (67,), generator=g).tolist()
    cache, table = sequences(cp, format, pasts, 1, 2, 16, 128, 31)
    n = min(pasts[0], pasts[1]) // 16
    table[1, :n] = table[0, :n]  # a common prefix
    q = randn((67, 1, 8, 128), 3)
    got = cp.cuda_paged_attention(q.cuda(), cache, table.cuda(), past_lengths=torch.tensor(pasts).cuda(),
                                  max_past_length=max(pasts))
    check_context(got, *ref.attention(q, cache, table, pasts))


@pytest.mark.parametrize("format,b", [("bf16", 1024), ("nvfp4", 1024), ("fp8", 1025)])
def test_as_many_sequences_as_the_streaming_kernel_takes_and_one_more(cp, format, b):
    g = torch.Generator().manual_seed(b)
    pasts = torch.randint(0, 60, (b,), generator=g).tolist()
    cache, table = sequences(cp, format, pasts, 1, 1, 16, 64, 61)
    q = randn((b, 1, 2, 64), 3)
    got = cp.cuda_paged_attention(q.cuda(), cache, table.cuda(), past_lengths=torch.tensor(pasts).cuda(),
                                  max_past_length=60)
    check_context(got, *ref.attention(q, cache, table, pasts))


@pytest.mark.parametrize("format", ["bf16", "fp8"])
def test_offsets_past_32_bits(cp, format):
    """A pool of more than 2^31 elements; the sequence lives on its last pages."""
    pages, hkv, size, d, n = 17000, 8, 64, 256, 150
    cache = cp.PagedKVCache.allocate(pages, hkv, size, d, format)
    assert cache.k_codes.numel() > 1 << 31
    table = torch.tensor([[pages - 1, pages - 3, pages - 2]], dtype=torch.int32)
    at = torch.arange(n)
    slots = (table[0, at // size].long() * size + at % size)[None].cuda()
    k, v = (randn((1, n, hkv, d), s).cuda() for s in (1, 2))
    cp.cuda_paged_kv_append_(cache, k, v, slots)
    got = cp.cuda_paged_kv_read(cache, slots)
    tail = cp.PagedKVCache(format, d, *(getattr(cache, f"{n}_{f}")[-3:].clone() if getattr(cache, f"{n}_{f}") is not None
                                        else None for f in ("codes", "row_scales", "block_scales") for n in "kv"))
    tail_table = table - (pages - 3)
    want = cp.cuda_paged_kv_read(tail, (tail_table[0, at // size].long() * size + at % size)[None].cuda())
    assert all(torch.equal(x, y) for x, y in zip(got, want)) and (got[0] != 0).any()
    for rows in (1, 3):  # the streaming kernel, and with a head dimension of 256 many rows of it
        q = randn((1, rows, 4 * hkv, d), 3)
        past = torch.tensor([n - rows]).cuda()
        got = cp.cuda_paged_attention(q.cuda(), cache, table.cuda(), past_lengths=past, max_past_length=n)
        check_context(got, *ref.attention(q, tail, tail_table, [n - rows]))


@pytest.mark.parametrize("format", ["bf16", "fp8", "nvfp4"])
@pytest.mark.parametrize("t", [1, 5])
def test_paged_is_the_whole_cache_s_attention(cp, format, t):
    """The same rows in a cache of whole sequences: the same context but for the order of sums."""
    b, hkv, d, size, cap = 3, 2, 128, 16, 4096
    pasts = torch.tensor([4000, 77, 2049])
    k, v = (randn((b, cap, hkv, d), s).cuda() for s in (1, 2))
    if format == "bf16":
        whole = tuple(x.transpose(1, 2).contiguous() for x in (k, v))
    else:
        whole = cp.QuantizedKVCache.allocate(b, hkv, cap, d, format)
        cp.cuda_quantized_kv_append_(whole, k, v, 0)
    g = torch.Generator().manual_seed(1)
    table = torch.randperm(b * cap // size, generator=g).int().view(b, -1).cuda()
    pool = cp.PagedKVCache.allocate(b * cap // size, hkv, size, d, format)
    at = torch.arange(cap).cuda()
    cp.cuda_paged_kv_append_(pool, k, v, table[:, at // size].long() * size + at % size)
    q = randn((b, t, 4 * hkv, d), 3).cuda()
    mask = draft_reference.random_tree(b, t, 2)[0].cuda()
    want = cp.cuda_tree_attention_cached(q, whole, tree_mask=mask, past_lengths=pasts.cuda(), max_past_length=4000)
    got = cp.cuda_paged_attention(q, pool, table, past_lengths=pasts.cuda(), max_past_length=4000, tree_mask=mask)
    # two results of the same values, each within a BF16 rounding and 2^-10 of the weighted |v| (at most max |v|)
    tol = 2.0 ** -7 * want.abs().float() + 2.0 ** -9 * 5.0
    assert ((got.float() - want.float()).abs() <= tol).all()


@pytest.mark.parametrize("d", [96, 128])
@pytest.mark.parametrize("bound", [0, 100])
def test_lengths_past_the_bound_that_a_call_is_planned_for(cp, d, bound):
    pasts = [1500, 90]
    cache, table = sequences(cp, "fp8", pasts, 1, 2, 16, d, 71)
    q = randn((2, 1, 4, d), 3)
    got = cp.cuda_paged_attention(q.cuda(), cache, table.cuda(), past_lengths=torch.tensor(pasts).cuda(),
                                  max_past_length=bound)
    check_context(got, *ref.attention(q, cache, table, pasts))


def test_attention_refusals(cp):
    cache, q = cp.PagedKVCache.allocate(3, 2, 16, 64, "fp8"), randn((2, 1, 4, 64), 1).cuda()
    table, past = torch.zeros((2, 2), dtype=torch.int32).cuda(), torch.zeros((2,), dtype=torch.int64).cuda()

    def call(q=q, cache=cache, table=table, past=past, bound=0, **kw):
        return cp.cuda_paged_attention(q, cache, table, past_lengths=past, max_past_length=bound, **kw)

    for kw, text in ((dict(table=table[:1]), "block_table must have shape"), (dict(table=table.long()), "dtype"),
                     (dict(past=past[:1]), "past_lengths must have shape"), (dict(q=q[..., :32].contiguous()), "head dimensions"),
                     (dict(q=q[:, :, :3].contiguous()), "divisible"), (dict(bound=32), "exceeds the block table"),
                     (dict(bound=-1), "nonnegative"), (dict(counts=past[:1]), "counts must have shape"),
                     (dict(tree_mask=torch.ones((2, 2)).bool().cuda()), "tree_mask must have shape")):
        with pytest.raises(RuntimeError, match=text):
            call(**kw)
