"""GPU checks of the paged attention on sizes that a server has: many tiles a CTA, the most sequences a kernel takes,
prompts, and what stands in rows that some queries see.  The oracle is FP64 on the device, a sequence at a time.

Tolerances are test_gpu_draft_ops.check_context's: the result's rounding to BF16, and probabilities to 11 bits.
"""

from __future__ import annotations

import math

import pytest
import torch

import draft_reference
from test_gpu_draft_ops import randn

pytestmark = pytest.mark.gpu

FORMATS = ["bf16", "fp8", "nvfp4"]


@pytest.fixture(scope="module")
def cp():
    import cuda_primitives

    return cuda_primitives


def values(cache, rows, head):
    """FP64 K and V [n, D] of one head's rows (page, row) of a pool, from the stored bytes."""
    out = []
    for n in "kv":
        codes, scales, blocks = (getattr(cache, f"{n}_{f}") for f in ("codes", "row_scales", "block_scales"))
        x = codes[rows[0], head, rows[1]]
        if cache.format == "bf16":
            out.append(x.double())
            continue
        if cache.format == "fp8":
            x = x.view(torch.float8_e4m3fn).double()
        else:
            levels = torch.from_numpy(draft_reference.E2M1).cuda()
            x = torch.stack((x & 15, x >> 4), -1).flatten(-2).long()
            x = levels[x & 7] * (1 - 2 * (x >> 3))
            x = x.unflatten(-1, (-1, 16)) * blocks[rows[0], head, rows[1]].view(torch.float8_e4m3fn).double()[..., None]
            x = x.flatten(-2)
        out.append(x * scales[rows[0], head, rows[1]].double()[:, None])
    return out


def attention(q, cache, table, pasts, mask=None, counts=None):
    """FP64 context and sum_j p_j |v_j|; a key that a query does not see has weight 0 and value 0 in its sums."""
    b, t, hq, d = q.shape
    n, hkv, size = cache.k_codes.shape[:3]
    group = hq // hkv
    ctx = torch.zeros((b, t, hq, d), dtype=torch.float64, device="cuda")
    weight = torch.zeros_like(ctx)
    causal = torch.ones((t, t), dtype=torch.bool, device="cuda").tril()
    for i in range(b):
        live = t if counts is None else max(0, min(int(counts[i]), t))
        if live == 0:
            continue
        j = torch.arange(pasts[i] + live, device="cuda")
        page = table[i, j // size].long()
        there = (page >= 0) & (page < n)
        rows, j = (page[there], j[there] % size), j[there]
        if not len(j):
            continue
        m = causal if mask is None else (mask if mask.ndim == 2 else mask[i])
        new = j >= pasts[i]
        sees = torch.ones((live, len(j)), dtype=torch.bool, device="cuda")
        sees[:, new] = m[:live][:, j[new] - pasts[i]]
        for h in range(hkv):
            k, v = values(cache, rows, h)
            for g in range(h * group, (h + 1) * group):
                s = (q[i, :live, g].double() @ k.T) / math.sqrt(d)
                s = torch.where(sees, s, -math.inf)
                w = torch.where(sees, torch.exp(s - s.amax(-1, keepdim=True)), 0.0)
                w = w / w.sum(-1, keepdim=True)
                w = torch.where(sees.any(-1, keepdim=True), w, 0.0)
                odd = ~torch.isfinite(v).all(-1)
                ctx[i, :live, g] = w[:, ~odd] @ v[~odd]
                weight[i, :live, g] = w[:, ~odd] @ v[~odd].abs()
                for x in odd.nonzero().flatten().tolist():  # rows with infinities or NaN, for the queries that see them
                    ctx[i, :live, g] += torch.where(sees[:, x:x + 1], w[:, x:x + 1] * v[x], 0.0)
                    weight[i, :live, g] += torch.where(sees[:, x:x + 1], w[:, x:x + 1] * v[x].abs(), 0.0)
    return ctx, weight


def check(got, ctx, weight, more=0.0):
    err = (got.double() - ctx).abs()
    tol = 2.0 ** -8 * (1 + 2.0 ** -6) * ctx.abs() + 2.0 ** -10 * weight + more
    finite = torch.isfinite(ctx)
    assert torch.equal(torch.isfinite(got), finite)
    assert (err <= tol)[finite].all(), float((err - tol)[finite].max())


def sequences(cp, format, pasts, t, hkv, size, d, seed, spare=2):
    """A pool of written rows and the table of sequences with t tokens behind these lengths; junk behind what they hold."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-(p + t) // size) for p in pasts]
    pages = sum(need) + spare
    cache = cp.PagedKVCache.allocate(pages, hkv, size, d, format)
    gc = torch.Generator(device="cuda").manual_seed(seed)
    for at in range(0, pages, 4096):
        n = min(4096, pages - at)
        k, v = (torch.randn((n, size, hkv, d), generator=gc, device="cuda").to(torch.bfloat16) for _ in "kv")
        cp.cuda_paged_kv_append_(cache, k, v, torch.arange(at * size, (at + n) * size, device="cuda").view(n, size))
    order = torch.randperm(pages, generator=g).int()
    table = torch.randint(-(1 << 31), 1 << 31, (len(pasts), max(need) + 1), generator=g).int()
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return cache, table


def call(cp, q, cache, table, pasts, **kw):
    bound = kw.pop("bound", max(pasts))
    return cp.cuda_paged_attention(q, cache, table, past_lengths=torch.tensor(pasts).cuda(), max_past_length=bound, **kw)


# ------------------------------------------------------------------ many tiles a CTA
@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("d,size", [(128, 16), (64, 48), (64, 16)])
@pytest.mark.parametrize("t", [1, 5, 16, 40])
def test_many_tiles_a_cta(cp, format, d, size, t):
    """Dozens of tiles a CTA: rings of stages and of missing pages go round, and tables are looked up again and again.
    4, 20, 64 and 160 query rows a KV head; pages that are gone all over the sequences; padding."""
    b, hkv, group = 32, 4, 4
    g = torch.Generator().manual_seed(t)
    pasts = torch.randint(1500, 4001, (b,), generator=g).tolist()
    pasts[3], pasts[17] = 0, 90
    cache, table = sequences(cp, format, pasts, t, hkv, size, d, t)
    for i in range(b):  # single pages, and a run of some hundred positions
        n = -(-(pasts[i] + t) // size)
        if n > 20:
            table[i, torch.randint(0, n, (6,), generator=g)] = -1
            at = int(torch.randint(0, n - 16, (1,), generator=g))
            table[i, at:at + 16] = cache.pages + i
    counts = torch.randint(1, t + 1, (b,), generator=g)
    counts[5] = 0
    mask = draft_reference.random_tree(b, t, t)[0].cuda()
    q = randn((b, t, hkv * group, d), 3).cuda()
    for kw in (dict(counts=counts.cuda(), tree_mask=mask), dict()):
        got = call(cp, q, cache, table.cuda(), pasts, **kw)
        check(got, *attention(q, cache, table.cuda(), pasts, kw.get("tree_mask"), counts if kw else None))
        again = [call(cp, q, cache, table.cuda(), pasts, **kw) for _ in range(3)]
        assert all(torch.equal(got, x) for x in again)
        if kw:
            dead = torch.arange(t)[None] >= counts[:, None]
            assert (got[dead.cuda()] == 0).all()


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("d,t,group", [(64, 1, 2), (128, 1, 4), (256, 1, 2), (64, 11, 4), (128, 11, 3)])
def test_the_most_sequences(cp, format, d, t, group):
    """1,024 sequences: the largest prefix that the streaming and the tcgen05 kernels hold."""
    g = torch.Generator().manual_seed(d + t)
    pasts = torch.randint(0, 150, (1024,), generator=g).tolist()
    cache, table = sequences(cp, format, pasts, t, 1, 16, d, 5)
    q = randn((1024, t, group, d), 3).cuda()
    check(call(cp, q, cache, table.cuda(), pasts), *attention(q, cache, table.cuda(), pasts))


# ------------------------------------------------------------------ prompts
@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("d,t,size", [(128, 1100, 64), (64, 2043, 16), (96, 1030, 48), (256, 517, 32)])
def test_prompts(cp, format, d, t, size):
    """Prompts of a thousand tokens and more through the block table, one of them after a prefix, one shorter."""
    pasts, counts = [0, 333], torch.tensor([t, t - 77])
    cache, table = sequences(cp, format, pasts, t, 2, size, d, 9)
    q = randn((2, t, 8, d), 3).cuda()
    got = call(cp, q, cache, table.cuda(), pasts, counts=counts.cuda())
    check(got, *attention(q, cache, table.cuda(), pasts, None, counts))
    assert (got[1, t - 77:] == 0).all()


# ------------------------------------------------------------------ other head dimensions, several splits
@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("bound", [0, 1000, 5000])
def test_splits_and_a_last_one_past_the_bound(cp, format, bound):
    pasts = [5000, 90, 1001]
    cache, table = sequences(cp, format, pasts, 3, 2, 16, 96, 13)
    table[0, 100:180] = -1
    q = randn((3, 3, 8, 96), 3).cuda()
    got = call(cp, q, cache, table.cuda(), pasts, bound=bound)
    check(got, *attention(q, cache, table.cuda(), pasts))


# ------------------------------------------------------------------ infinities and NaN
@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("d", [64, 80, 96, 128, 256])
@pytest.mark.parametrize("t", [3, 12])
def test_wild_drafted_rows_reach_the_queries_that_see_them(cp, format, d, t):
    """Infinities (BF16) and NaN codes or block scales in drafted rows of V: in the elements they stand in, for the
    queries whose mask names the row, and for no other."""
    pasts, size = [150, 64, 0], 16
    cache, table = sequences(cp, format, pasts, t, 2, size, d, 17)
    mask = draft_reference.random_tree(3, t, 29)[0]
    for i in range(3):
        for u, e in ((1, 5), (t - 1, 17)):
            pos = pasts[i] + u
            at = (int(table[i, pos // size]), i % 2, pos % size)
            if format == "bf16":
                cache.v_codes[at][e] = float("inf") if u == 1 else float("nan")
            elif format == "fp8":
                cache.v_codes[at][e] = 0x7f if u == 1 else 0xff
            else:
                cache.v_block_scales[at][e // 16] = 0x7f
    q = randn((3, t, 8, d), 3).cuda()
    got = call(cp, q, cache, table.cuda(), pasts, tree_mask=mask.cuda())
    ctx, weight = attention(q, cache, table.cuda(), pasts, mask.cuda())
    assert 0 < int((~torch.isfinite(ctx)).sum()) < ctx.numel() // 4
    check(got, ctx, weight)


# ------------------------------------------------------------------ the range of a query's elements
@pytest.mark.parametrize("format", ["fp8", "nvfp4"])
@pytest.mark.parametrize("d,t", [(64, 1), (96, 1), (128, 1), (128, 9)])
@pytest.mark.parametrize("size", [30, 36])
def test_a_query_whose_elements_span_more_than_16_bits(cp, format, d, t, size):
    """The largest element is 2^size of the others and meets keys that are 0 there, so the others make the scores.

    Over codes a query is scaled so that its largest element is 2^14 and goes to FP16, whose steps end at 2^-24: an
    element of 2^(14 - size) and 8 significant bits is exact for size = 30 (its last bit is at least 2^-23).  For
    size = 36 it is off by half of 2^-24 at most, 2^-25 2^(size - 14) = 2^-3 as an element of q, so a score by
    e = 2^-3 sum_d |k_d| / sqrt(D), a weight by a factor within exp(+-2 e), and the context by
    (exp(2 e) - 1)(weight + |context|)."""
    pasts = [70, 300]
    cache, table = sequences(cp, format, pasts, t, 1, 16, d, 19)
    g = torch.Generator(device="cuda").manual_seed(3)
    k = 2.0 ** -6 * torch.randn((cache.pages, 16, 1, d), generator=g, device="cuda")
    k[..., 0] = 0.0
    v = torch.randn((cache.pages, 16, 1, d), generator=g, device="cuda").to(torch.bfloat16)
    cp.cuda_paged_kv_append_(cache, k.to(torch.bfloat16), v, torch.arange(cache.pages * 16, device="cuda").view(-1, 16))
    q = randn((2, t, 4, d), 5).cuda()
    q = (torch.sign(q) * (1 + q.abs().clamp(max=0.99))).to(torch.bfloat16)
    q[..., 0] = 2.0 ** size
    ctx, weight = attention(q, cache, table.cuda(), pasts)
    e = 0.0 if size == 30 else 2.0 ** -3 * float(k.abs().sum(-1).max()) * 1.1 / math.sqrt(d)  # 1.1: codes' rounding
    check(call(cp, q, cache, table.cuda(), pasts), ctx, weight, math.expm1(2 * e) * (weight + ctx.abs()))


# ------------------------------------------------------------------ the table's end, masks over many tokens
@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("t", [8, 24])
def test_padding_past_the_table_s_end(cp, format, d, t):
    """P_b + n fills the table where P_b + T would pass it; only the bound has to leave room for T tokens."""
    size, most, hkv = 16, 9, 2
    counts = torch.tensor([4, 1, t, 0])
    pasts = [size * most - 4, size * most - 1, size * most - t, size * most]
    cache, _ = sequences(cp, format, [size * most - 1] * 4, 1, hkv, size, d, 23)
    g = torch.Generator().manual_seed(7)
    table = torch.randperm(cache.pages, generator=g)[:4 * most].int().view(4, most).cuda()
    q = randn((4, t, 4 * hkv, d), 3).cuda()
    got = call(cp, q, cache, table, pasts, counts=counts.cuda(), bound=size * most - t)
    check(got, *attention(q, cache, table, pasts, None, counts))


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("d,t", [(128, 300), (64, 517), (96, 131), (256, 70)])
def test_masks_over_many_tokens(cp, format, d, t):
    """Trees of some hundred tokens, a mask a sequence and one for all, tiles that hold several tokens' keys."""
    pasts, size = [0, 45, 700], 48
    cache, table = sequences(cp, format, pasts, t, 1, size, d, 27)
    q = randn((3, t, 4, d), 3).cuda()
    mask = draft_reference.random_tree(3, t, 31)[0].cuda()
    mask[1, ::7] = False  # rows that see committed positions alone
    for m in (mask, mask[2].contiguous()):
        check(call(cp, q, cache, table.cuda(), pasts, tree_mask=m), *attention(q, cache, table.cuda(), pasts, m))


def test_two_captured_calls_and_an_eager_one_at_once(cp):
    """Two graphs of different calls, replayed in turn and on two streams, beside an eager call: each its own result."""
    pasts = [900, 31, 4000]
    cache, table = sequences(cp, "fp8", pasts, 5, 2, 16, 128, 33)
    table, past = table.cuda(), torch.tensor(pasts).cuda()
    qs = [randn((3, t, 8, 128), t).cuda() for t in (1, 5, 3)]

    def attend(q):
        return cp.cuda_paged_attention(q, cache, table, past_lengths=past, max_past_length=4000)

    want = [attend(q) for q in qs]
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph, q in zip(graphs, qs):
        with torch.cuda.graph(graph):
            outs.append(attend(q))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for x in outs:
            x.fill_(float("nan"))
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        eager = attend(qs[2])
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip([*outs, eager], want))
