"""GPU parity of the drafted-token operators against their 64-bit definitions.

Tolerances, from the arithmetic:
* rotary: two FP32 products and a sum of FP32-accurate factors, one rounding to
  BF16: 2^-8 |y| for the rounding, 2^-20 A (|x_e| + |x_o|) for the rest;
* quantised rows: codes and scales bit-exact with the FP32 definition; values
  read back bit-exact with BF16((code * beta) * gamma);
* attention: the rounding of the result to BF16, 2^-8 |o|; the probabilities,
  each kept to 11 significant bits at least (2^-11), and scores to 2^-11
  absolute: 2^-10 sum_j p_j |v_j|.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import draft_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cp():
    import cuda_primitives

    return cuda_primitives


def randn(shape, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(shape, generator=g)).to(torch.bfloat16)


def rows_of_all_sizes(shape, seed):
    """Rows whose sizes span 2^-20 .. 2^20, a few channels larger than the rest."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp2(40 * torch.rand(shape[:-1] + (1,), generator=g) - 20)
    return (x * (1 + 15 * (torch.rand(shape[-1:], generator=g) < 0.05))).to(torch.bfloat16)


def check_context(got, exact, size):
    err = (got.cpu().double() - exact).abs()
    tol = 2.0 ** -8 * (1 + 2.0 ** -6) * exact.abs() + 2.0 ** -10 * size
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), float((err - tol).max())


# ------------------------------------------------------------------ rotary positions
@pytest.mark.parametrize("b,t,hq,hkv,d,r,interleaved", [
    (1, 1, 24, 6, 128, 128, True),
    (1, 1, 1, 1, 2, 2, True),
    (3, 5, 8, 2, 128, 128, False),
    (2, 7, 12, 3, 256, 64, False),
    (5, 3, 4, 4, 96, 24, True),    # 8-byte and 16-byte pieces that do not line up with the halves
    (5, 3, 4, 4, 96, 24, False),
    (1, 33, 3, 1, 80, 22, False),  # halves of odd length: element by element
    (1, 33, 3, 1, 82, 22, True),
    (4, 130, 2, 1, 64, 32, True),
    (2, 3, 200, 8, 64, 64, False),
])
def test_rope_qk(cp, b, t, hq, hkv, d, r, interleaved):
    q, k = randn((b, t, hq, d), 1), randn((b, t, hkv, d), 2)
    g = torch.Generator().manual_seed(3)
    pos = torch.randint(0, 200_000, (b, t), generator=g)
    pos[0, 0] = 0
    freq = torch.tensor([1e4 ** (-2 * m / r) for m in range(r // 2)], dtype=torch.float32)
    for factor in (1.0, 1.2079):
        out = cp.cuda_apply_rope_qk(q.cuda(), k.cuda(), pos.cuda(), freq.cuda(), interleaved=interleaved,
                                    attention_factor=factor)
        for x, y in zip((q, k), out):
            exact = ref.rope(x, pos, freq, interleaved, factor)
            pair = ref.rope(x.abs(), torch.zeros_like(pos), freq, interleaved, 1.0)  # |x|, shape only
            tol = 2.0 ** -8 * (1 + 2.0 ** -6) * exact.abs() + 2.0 ** -20 * factor * 2 * pair.amax()
            assert ((y.cpu().double() - exact).abs() <= tol).all()
            assert torch.equal(y[..., r:].cpu(), x[..., r:])
        if factor == 1.0:
            assert torch.equal(out[0][0, 0].cpu(), q[0, 0])  # position 0: an exact copy


def test_rope_takes_strided_views_and_shared_positions(cp):
    """q and k cut out of one projection's output, at every alignment of the row."""
    b, t, hq, hkv, d = 2, 5, 4, 2, 64
    freq = torch.full((32,), 0.25).cuda()
    pos = torch.arange(7, 7 + t).cuda()
    for extra in (0, 1, 2, 4):
        flat = randn((b, t, (hq + 2 * hkv) * d + extra), 4).cuda()[..., extra:]
        q = flat[..., :hq * d].unflatten(-1, (hq, d))
        k = flat[..., hq * d:(hq + hkv) * d].unflatten(-1, (hkv, d))
        got = cp.cuda_apply_rope_qk(q, k, pos, freq, interleaved=True)
        want = cp.cuda_apply_rope_qk(q.contiguous(), k.contiguous(), pos.expand(b, t).contiguous(), freq)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    q = randn((t, b, hq, d), 5).cuda().transpose(0, 1)  # tokens outermost
    got = cp.cuda_apply_rope_qk(q, q, pos, freq, interleaved=False)[0]
    assert torch.equal(got, cp.cuda_apply_rope_qk(q.contiguous(), q.contiguous(), pos, freq, interleaved=False)[0])


def test_rope_agrees_with_the_whole_head_operator(cp):
    """Adjacent pairs of the whole head at past + t: the framework's own RoPE, within the angle's FP32 rounding."""
    q = randn((2, 4, 6, 128), 6).cuda()
    freq, _ = cp.rope_frequencies(128)
    got, _ = cp.cuda_apply_rope_qk(q, q, torch.arange(500, 504).cuda(), freq)
    want = cp.cuda_apply_rope(q, 500, 1e4)
    assert (got.float() - want.float()).abs().max() <= 2.0 ** -8 * float(q.abs().max())


def test_rope_keeps_infinities_to_their_pair(cp):
    q = randn((1, 2, 1, 64), 7).cuda()
    q[0, 0, 0, 3] = float("inf")
    freq = torch.full((32,), 0.5).cuda()
    y, _ = cp.cuda_apply_rope_qk(q, q, torch.tensor([0, 1]).cuda(), freq)
    assert torch.equal(y[0, 0], q[0, 0])
    q[0, 1, 0, 3] = float("nan")
    y, _ = cp.cuda_apply_rope_qk(q, q, torch.tensor([0, 1]).cuda(), freq)
    bad = ~torch.isfinite(y[0, 1, 0])
    assert bad.nonzero().flatten().tolist() == [2, 3]


# ------------------------------------------------------------------ the quantised cache
@pytest.mark.parametrize("fmt", ["fp8", "nvfp4"])
@pytest.mark.parametrize("b,t,hkv,d", [(1, 1, 1, 16), (2, 3, 2, 64), (3, 65, 5, 128), (1, 7, 3, 256), (2, 5, 1, 80),
                                       (1, 4, 2, 112)])
def test_append_writes_the_definition_and_nothing_else(cp, fmt, b, t, hkv, d):
    cache = cp.QuantizedKVCache.allocate(b, hkv, 150, d, fmt)
    fields = [getattr(cache, f"{n}_{f}") for n in "kv" for f in ("codes", "row_scales", "block_scales")]
    for x in fields:
        if x is not None:
            x.copy_(torch.full_like(x, 37))
    k, v = rows_of_all_sizes((b, t, hkv, d), 11), rows_of_all_sizes((b, t, hkv, d), 12)
    k[0, 0, 0] = 0
    v[0, 0, 0, 1:] = 0
    k[-1, -1, -1, 3:] = 2.0 ** -130  # a subnormal row scale
    g = torch.Generator().manual_seed(5)
    past = torch.randint(0, 150 - t, (b,), generator=g)
    counts = torch.randint(0, t + 1, (b,), generator=g)
    counts[0] = t
    cp.cuda_quantized_kv_append_(cache, k.cuda(), v.cuda(), past_lengths=past.cuda(), counts=counts.cuda())
    for n, x in (("k", k), ("v", v)):
        stored = [getattr(cache, f"{n}_{f}") for f in ("codes", "row_scales", "block_scales")]
        want = ref.quantize_rows(fmt, x.transpose(1, 2))
        for got, exp in zip(stored, want):
            if exp is None:
                continue
            full = torch.full_like(got.cpu(), 37)
            for i in range(b):
                c = int(counts[i])
                full[i, :, int(past[i]):int(past[i]) + c] = torch.from_numpy(exp)[i, :, :c]
            assert torch.equal(got.cpu(), full)


@pytest.mark.parametrize("fmt", ["fp8", "nvfp4"])
def test_rows_are_as_near_as_their_format_allows(cp, fmt):
    """Half a step of the code times its scale, relative to each row's own size."""
    b, t, hkv, d = 2, 40, 3, 128
    x = rows_of_all_sizes((b, t, hkv, d), 21)
    cache = cp.QuantizedKVCache.allocate(b, hkv, t, d, fmt)
    cp.cuda_quantized_kv_append_(cache, x.cuda(), x.cuda(), 0)
    value = ref.cache_values(cache)[0][:, :, :t]
    x = x.double().transpose(1, 2)
    amax = x.abs().amax(-1, keepdim=True)
    if fmt == "fp8":  # half an E4M3 step: 2^-4 relative, 2^-10 of the unit below 2^-6
        tol = torch.maximum(2.0 ** -4 * x.abs(), 2.0 ** -10 * amax / 448)
    else:  # half an E2M1 step (1 between 4 and 6) of the block's unit, at most 1/6 block amax * (1 + 2^-4)
        block = x.unflatten(-1, (-1, 16)).abs().amax(-1, keepdim=True).expand(*x.shape[:-1], -1, 16).flatten(-2)
        unit = torch.maximum(block / 6 * (1 + 2.0 ** -4), 2.0 ** -9 * amax / 2688)
        tol = unit * 1.0
        tol = torch.where(block < 2.0 ** -10 * 6 * amax / 2688, x.abs(), tol)  # a block scale that rounds to 0
    assert ((value - x).abs() <= tol * (1 + 2.0 ** -20)).all()


@pytest.mark.parametrize("fmt", ["fp8", "nvfp4"])
@pytest.mark.parametrize("d,start,length", [(16, 0, 1), (64, 3, 130), (128, 100, 92), (256, 0, 192), (48, 191, 1)])
def test_read_returns_the_values_rounded_once(cp, fmt, d, start, length):
    cache = cp.QuantizedKVCache.allocate(2, 3, 192, d, fmt)
    x = rows_of_all_sizes((2, 192, 3, d), 31).cuda()
    cp.cuda_quantized_kv_append_(cache, x, -x, 0)
    got = cp.cuda_quantized_kv_read(cache, start, length)
    starts = torch.tensor([start - 5, 192 - length + 3])
    ragged = cp.cuda_quantized_kv_read(cache, length=length, starts=starts.cuda())
    for n, y, z in zip("kv", got, ragged):
        f32 = getattr(cache, n + "_row_scales").cpu()[..., None]
        one = torch.ones((2, 3, 192))
        stored = [getattr(cache, f"{n}_{f}") for f in ("codes", "block_scales")]
        unit = ref.stored_values(fmt, stored[0].cpu().numpy(), one.numpy(),
                                 None if stored[1] is None else stored[1].cpu().numpy())
        want = (unit.float() * f32).to(torch.bfloat16)  # code * beta is exact in FP32
        assert torch.equal(y.cpu(), want[:, :, start:start + length])
        for i in range(2):
            s = int(starts[i])
            lo, hi = max(s, 0), min(s + length, 192)
            exp = torch.zeros((3, length, d), dtype=torch.bfloat16)
            if hi > lo:
                exp[:, lo - s:hi - s] = want[i, :, lo:hi]
            assert torch.equal(z[i].cpu(), exp)


@pytest.mark.parametrize("fmt", ["fp8", "nvfp4"])
def test_rows_with_infinities_or_nan_read_back_as_nan(cp, fmt):
    x = randn((1, 4, 2, 64), 41)
    x[0, 1, 0, 5] = float("inf")
    x[0, 2, 1, 9] = float("nan")
    cache = cp.QuantizedKVCache.allocate(1, 2, 64, 64, fmt)
    cp.cuda_quantized_kv_append_(cache, x.cuda(), x.cuda(), 10)
    k, _ = cp.cuda_quantized_kv_read(cache, 10, 4)
    bad = torch.isnan(k.float()).cpu()
    want = torch.zeros((1, 2, 4, 64), dtype=torch.bool)
    want[0, 0, 1] = want[0, 1, 2] = True
    assert torch.equal(bad, want)
    assert (cache.k_codes[0, 0, 11] == 0).all()


@pytest.mark.parametrize("fmt", ["fp8", "nvfp4"])
def test_append_takes_strided_views_and_skips_slots_outside(cp, fmt):
    flat = randn((2, 6, 4 * 64 + 1), 43).cuda()
    for view in (flat[..., 1:], flat[..., :-1], flat.transpose(0, 1)[:2, :2, 1:]):
        k = view.unflatten(-1, (4, 64))
        a, b = (cp.QuantizedKVCache.allocate(k.shape[0], 4, 64, 64, fmt) for _ in range(2))
        cp.cuda_quantized_kv_append_(a, k, k, 3)
        cp.cuda_quantized_kv_append_(b, k.contiguous(), k.contiguous(), 3)
        assert torch.equal(a.k_codes, b.k_codes) and torch.equal(a.v_row_scales, b.v_row_scales)
    c = cp.QuantizedKVCache.allocate(2, 4, 64, 64, fmt)
    k = randn((2, 6, 4, 64), 44).cuda()
    cp.cuda_quantized_kv_append_(c, k, k, past_lengths=torch.tensor([-1, 61]).cuda())
    assert (c.k_row_scales[0] == 0).all() and (c.k_row_scales[1, :, 61:] != 0).all()
    assert (c.k_row_scales[1, :, :61] == 0).all()


# ------------------------------------------------------------------ tree attention
def filled(cp, fmt, b, hkv, c, d, seed):
    """A cache of random rows, V rows of different sizes; BF16 as a pair."""
    k = randn((b, c, hkv, d), seed)
    g = torch.Generator().manual_seed(seed + 1)
    v = (torch.randn((b, c, hkv, d), generator=g) * torch.exp(torch.randn((b, c, hkv, 1), generator=g))).to(torch.bfloat16)
    if fmt == "bf16":
        return k.transpose(1, 2).contiguous().cuda(), v.transpose(1, 2).contiguous().cuda()
    cache = cp.QuantizedKVCache.allocate(b, hkv, c, d, fmt)
    cp.cuda_quantized_kv_append_(cache, k.cuda(), v.cuda(), 0)
    return cache


def check_tree(cp, fmt, b, t, hq, hkv, d, pasts, cap, seed, mask="tree", q_scale=1.0):
    cache = filled(cp, fmt, b, hkv, cap, d, seed)
    q = randn((b, t, hq, d), seed + 7, q_scale)
    if mask == "tree":
        mask = ref.random_tree(b, t, seed)[0]
    got = cp.cuda_tree_attention_cached(q.cuda(), cache, tree_mask=None if mask is None else mask.cuda(),
                                        past_lengths=torch.tensor(pasts).cuda(), max_past_length=max(pasts))
    exact, size = ref.tree_attention(q, *ref.cache_values(cache), pasts, mask)
    check_context(got, exact, size)
    return cache, q, got


FORMATS = ["bf16", "fp8", "nvfp4"]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("b,t,hq,hkv,d,pasts,cap", [
    (1, 1, 1, 1, 64, [0], 64),               # one key: the drafted token itself
    (1, 1, 24, 6, 128, [511], 512),
    (2, 8, 8, 2, 128, [0, 63], 128),         # 32 rows; drafted tokens across a tile's end
    (3, 5, 6, 6, 64, [64, 1, 130], 192),     # a head group of one, odd counts
    (1, 3, 16, 2, 256, [200], 256),
    (2, 17, 7, 1, 128, [33, 400], 448),      # 119 rows, a group of seven
    (1, 40, 8, 2, 128, [100], 192),          # 160 rows
    (1, 64, 8, 1, 64, [65], 192),            # 512 rows
    (2, 2, 4, 2, 96, [5, 77], 128),          # head dimensions of the general kernel
    (1, 6, 3, 3, 16, [12], 64),
    (1, 2, 2, 1, 240, [31], 64),
])
def test_tree_attention(cp, fmt, b, t, hq, hkv, d, pasts, cap):
    check_tree(cp, fmt, b, t, hq, hkv, d, pasts, cap, seed=b + t + d)


@pytest.mark.parametrize("fmt", FORMATS)
def test_ragged_lengths_share_one_launch(cp, fmt):
    pasts = [0, 1, 15, 16, 63, 64, 65, 127, 1000, 1023]
    check_tree(cp, fmt, len(pasts), 2, 4, 1, 128, pasts, 1088, seed=9)


@pytest.mark.parametrize("fmt", FORMATS)
def test_long_cache_one_sequence_on_every_sm(cp, fmt):
    check_tree(cp, fmt, 1, 2, 8, 2, 128, [20_001], 20_032, seed=2)


@pytest.mark.parametrize("fmt", FORMATS)
def test_sharp_scores(cp, fmt):
    """Large queries: one key takes nearly all of the weight, others underflow."""
    check_tree(cp, fmt, 1, 4, 8, 2, 128, [700], 704, seed=4, q_scale=8.0)


@pytest.mark.parametrize("fmt", FORMATS)
def test_without_a_mask_the_drafted_tokens_form_a_chain(cp, fmt):
    cache, q, got = check_tree(cp, fmt, 2, 7, 8, 2, 128, [50, 0], 64, seed=6, mask=None)
    chain = torch.ones((7, 7), dtype=torch.bool).tril().cuda()
    again = cp.cuda_tree_attention_cached(q.cuda(), cache, tree_mask=chain,
                                          past_lengths=torch.tensor([50, 0]).cuda(), max_past_length=50)
    assert torch.equal(got, again)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d", [64, 96, 128])
def test_queries_that_see_nothing_get_zeros(cp, fmt, d):
    mask = torch.zeros((2, 5, 5), dtype=torch.bool)
    mask[0, 3, 1] = mask[1, 0, 4] = True
    cache = filled(cp, fmt, 2, 2, 64, d, 8)
    q = randn((2, 5, 4, d), 3)
    got = cp.cuda_tree_attention_cached(q.cuda(), cache, tree_mask=mask.cuda(),
                                        past_lengths=torch.tensor([0, 0]).cuda(), max_past_length=0)
    exact, size = ref.tree_attention(q, *ref.cache_values(cache), [0, 0], mask)
    check_context(got, exact, size)
    assert (got[0, 0] == 0).all() and (got[0, 3] != 0).any()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d", [64, 80, 128, 256])
@pytest.mark.parametrize("group", [1, 8])
def test_unseen_slots_may_hold_anything(cp, fmt, d, group):
    """NaN and infinities past P_b + T and in drafted rows that a query does not see."""
    t, p, cap = 20, 53, 192  # the drafted slots span two tiles and end inside a slice of 16
    cache = filled(cp, fmt, 1, 2, cap, d, 14)
    exact_kv = ref.cache_values(cache)
    q = randn((1, t, 2 * group, d), 15)
    mask, _ = ref.random_tree(1, t, 3)
    mask[0, :, 4] = mask[0, :, 11] = False  # nobody sees 4 and 11 ...
    mask[0, 6, 11] = True                   # ... but 6 sees 11
    if fmt == "bf16":
        for x in cache:
            x[0, :, p + t:] = float("nan")
            x[0, :, p + 4] = float("inf")
            x[0, :, p + 11, : d // 2] = float("nan")
    else:
        for n in "kv":
            codes, scales = getattr(cache, n + "_codes"), getattr(cache, n + "_row_scales")
            codes[0, :, p + t:] = 0x7F  # NaN as E4M3
            scales[0, :, p + t:] = float("nan")
            scales[0, :, p + 4] = float("inf")
            scales[0, :, p + 11] = float("nan")
            if fmt == "fp8":
                codes[0, :, p + 4] = 0xFF
            else:
                getattr(cache, n + "_block_scales")[0, :, p + 4] = 0x7F
    got = cp.cuda_tree_attention_cached(q.cuda(), cache, p, tree_mask=mask.cuda())
    assert torch.isnan(got[0, 6].float()).any(-1).all()
    keep = [i for i in range(t) if i != 6]
    mask[0, 6, 11] = False
    exact, size = ref.tree_attention(q, *exact_kv, [p], mask)
    check_context(got[:, keep], exact[:, keep], size[:, keep])


@pytest.mark.parametrize("fmt", FORMATS)
def test_v_rows_of_every_size_and_zero_rows(cp, fmt):
    """V rows from 2^-20 to 2^20, the heaviest-weighted ones small, and rows of zeros."""
    b, t, hq, hkv, d, p, cap = 1, 2, 4, 1, 128, 300, 320
    k, v = randn((b, cap, hkv, d), 50), rows_of_all_sizes((b, cap, hkv, d), 51)
    v[:, ::3] = 0
    q = randn((b, t, hq, d), 52)
    if fmt == "bf16":
        cache = (k.transpose(1, 2).contiguous().cuda(), v.transpose(1, 2).contiguous().cuda())
    else:
        cache = cp.QuantizedKVCache.allocate(b, hkv, cap, d, fmt)
        cp.cuda_quantized_kv_append_(cache, k.cuda(), v.cuda(), 0)
    got = cp.cuda_tree_attention_cached(q.cuda(), cache, p)
    check_context(got, *ref.tree_attention(q, *ref.cache_values(cache), [p]))
    zero = tuple(torch.zeros_like(x) for x in cache) if fmt == "bf16" else cp.QuantizedKVCache.allocate(b, hkv, cap, d, fmt)
    assert (cp.cuda_tree_attention_cached(q.cuda(), zero, p) == 0).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_repeated_calls_and_other_streams_give_the_same_bits(cp, fmt):
    cache = filled(cp, fmt, 3, 2, 1024, 128, 60)
    q = randn((3, 6, 8, 128), 61).cuda()
    past = torch.tensor([1000, 17, 512]).cuda()
    first = cp.cuda_tree_attention_cached(q, cache, past_lengths=past, max_past_length=1000)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [cp.cuda_tree_attention_cached(q, cache, past_lengths=past, max_past_length=1000) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(first, x) for x in again)
    loose = cp.cuda_tree_attention_cached(q, cache, past_lengths=past, max_past_length=1018)
    assert (loose.float() - first.float()).abs().max() <= 2.0 ** -6 * float(first.abs().max())


@pytest.mark.parametrize("fmt", FORMATS)
def test_graph_capture_follows_device_lengths(cp, fmt):
    """A captured call replays with the lengths the device tensor then holds."""
    cache = filled(cp, fmt, 2, 2, 512, 128, 70)
    q = randn((2, 3, 4, 128), 71).cuda()
    past = torch.tensor([10, 400]).cuda()
    call = lambda: cp.cuda_tree_attention_cached(q, cache, past_lengths=past, max_past_length=500)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    past.copy_(torch.tensor([333, 7]))
    graph.replay()
    torch.cuda.synchronize()
    exact, size = ref.tree_attention(q, *ref.cache_values(cache), [333, 7])
    check_context(out, exact, size)


def test_c_interface_agrees_with_the_operator(cp):
    import nvfp4da_capi

    for fmt in FORMATS:
        cache = filled(cp, fmt, 2, 2, 192, 64, 80)
        q = randn((2, 4, 4, 64), 81).cuda()
        mask = ref.random_tree(2, 4, 8)[0].cuda()
        assert torch.equal(nvfp4da_capi.tree_attention(q, cache, 150, tree_mask=mask),
                           cp.cuda_tree_attention_cached(q, cache, 150, tree_mask=mask))


# ------------------------------------------------------------------ refusals
def test_refusals(cp):
    c = cp.QuantizedKVCache.allocate(2, 2, 64, 64, "nvfp4")
    x = randn((2, 3, 2, 64), 90).cuda()
    n = torch.zeros((2,), dtype=torch.int64).cuda()
    for call, text in (
        (lambda: cp.cuda_quantized_kv_append_(c, x, x, 62), "exceeds cache capacity"),
        (lambda: cp.cuda_quantized_kv_append_(c, x, x, -1), "nonnegative"),
        (lambda: cp.cuda_quantized_kv_append_(c, x[:1], x[:1], 0), "matching the cache"),
        (lambda: cp.cuda_quantized_kv_append_(c, x.float(), x.float(), 0), "dtype"),
        (lambda: cp.cuda_quantized_kv_append_(c, x.mT.contiguous().mT, x, 0), "contiguous in its last dimension"),
        (lambda: cp.cuda_quantized_kv_append_(c, x, x, past_lengths=n[:1]), "past_lengths must have shape"),
        (lambda: cp.cuda_quantized_kv_append_(c, x, x, counts=n.int()), "counts must have dtype"),
        (lambda: cp.cuda_quantized_kv_read(c, 0, 65), "length must be in"),
        (lambda: cp.cuda_quantized_kv_read(c, 60, 5), "not inside the cache capacity"),
        (lambda: cp.cuda_tree_attention_cached(x, c, 62), "exceeds cache capacity"),
        (lambda: cp.cuda_tree_attention_cached(x[:, :, :1].contiguous(), c, 0), "divisible by number of KV heads"),
        (lambda: cp.cuda_tree_attention_cached(x.transpose(0, 1), c, 0), "contiguous"),
        (lambda: cp.cuda_tree_attention_cached(x, c, 0, tree_mask=torch.ones(3, 4).bool().cuda()), "tree_mask must have"),
        (lambda: cp.cuda_tree_attention_cached(x, c, 0, tree_mask=torch.ones(3, 3).cuda()), "tree_mask must have dtype"),
        (lambda: cp.cuda_tree_attention_cached(x, c, past_lengths=n, max_past_length=-1), "nonnegative"),
        (lambda: cp.cuda_tree_attention_cached(x, (c.k_codes, c.v_codes), 0), "k_cache must have dtype"),
        (lambda: cp.cuda_apply_rope_qk(x, x, n, torch.ones(32).cuda()), "positions must have shape"),
        (lambda: cp.cuda_apply_rope_qk(x, x, n[:1].expand(3).contiguous(), torch.ones(33).cuda()), "rotary_dim"),
        (lambda: cp.cuda_apply_rope_qk(x, x[:, :2], n, torch.ones(32).cuda()), "must agree"),
        (lambda: cp.cuda_apply_rope_qk(x, x, n[:1].expand(3).contiguous(), torch.ones(32).cuda(),
                                       attention_factor=float("inf")), "finite"),
    ):
        with pytest.raises(RuntimeError, match=text):
            call()


# ------------------------------------------------------------------ the step that runs them together
def step_inputs(cp, b, t, h, hkv, d, seed):
    from nvfp4_tensor import quantize_nvfp4

    g = torch.Generator().manual_seed(seed)
    w = [quantize_nvfp4((0.05 * torch.randn((n, h), generator=g)).cuda()) for n in (h, hkv * d, hkv * d, h)]
    x = torch.randn((b, t, h), generator=g).to(torch.bfloat16).cuda()
    norms = [(1 + 0.05 * torch.randn((n,), generator=g)).to(torch.bfloat16).cuda() for n in (h, d, d)]
    return x, norms, w


def test_chain_step_over_bf16_caches_matches_the_forward(cp):
    """A causal chain over BF16 caches: the decoder-attention forward, end-to-end tolerance."""
    from bf16_metrics import assert_e2e_policy
    from decoder_attention_cuda import cuda_decoder_attention_forward_
    from gpu_util import host_bits
    from tree_decoding import cuda_decoder_attention_tree_forward_

    b, t, h, hkv, d, p = 2, 4, 512, 2, 64, 37
    x, (g_in, g_q, g_k), (wq, wk, wv, wo) = step_inputs(cp, b, t, h, hkv, d, 5)
    caches = [randn((b, hkv, 64, d), s).cuda() for s in (1, 2)]
    other = [c.clone() for c in caches]
    want = cuda_decoder_attention_forward_(x, g_in, wq, wk, wv, g_q, g_k, wo, *caches, p)
    got, k, v = cuda_decoder_attention_tree_forward_(
        x, g_in, wq, wk, wv, g_q, g_k, wo, other, p, depths=torch.arange(t).cuda(),
        inv_freq=cp.rope_frequencies(d)[0])
    assert_e2e_policy(host_bits(got), host_bits(want))
    assert_e2e_policy(host_bits(other[0]), host_bits(caches[0]))
    assert torch.equal(other[1][:, :, p:p + t], v.transpose(1, 2))


@pytest.mark.parametrize("fmt", ["fp8", "nvfp4"])
def test_tree_step_and_acceptance(cp, fmt):
    """Each path of the tree gives what its tokens alone would give as a chain, and
    an accepted path leaves the cache as if only its tokens had been appended."""
    from tree_decoding import accept_drafted_, cuda_decoder_attention_tree_forward_

    b, t, h, hkv, d = 2, 6, 512, 2, 64
    x, (g_in, g_q, g_k), (wq, wk, wv, wo) = step_inputs(cp, b, t, h, hkv, d, 6)
    inv_freq, factor = cp.rope_frequencies(32, scaling="yarn", factor=4.0, original_length=64)
    mask, depths = ref.random_tree(b, t, 12)
    past = torch.tensor([40, 9])
    start = filled(cp, fmt, b, hkv, 64, d, 33)
    args = dict(inv_freq=inv_freq, attention_factor=factor, interleaved=False, max_past_length=58)

    def copy():
        fields = {f: getattr(start, f) for f in ("k_codes", "v_codes", "k_row_scales", "v_row_scales",
                                                 "k_block_scales", "v_block_scales")}
        return cp.QuantizedKVCache(fmt, d, **{f: None if x is None else x.clone() for f, x in fields.items()})

    tree = copy()
    y, k, v = cuda_decoder_attention_tree_forward_(x, g_in, wq, wk, wv, g_q, g_k, wo, tree, depths=depths.cuda(),
                                                   tree_mask=mask.cuda(), past_lengths=past.cuda(), **args)
    path = torch.zeros((b, t), dtype=torch.int64)
    counts = torch.zeros((b,), dtype=torch.int64)
    for i in range(b):  # the path to the last node
        nodes = mask[i, t - 1].nonzero().flatten()
        path[i, :len(nodes)], counts[i] = nodes, len(nodes)
    accept_drafted_(tree, k, v, path.cuda(), past_lengths=past.cuda(), counts=counts.cuda())
    for i in range(b):
        n, nodes = int(counts[i]), path[i, :int(counts[i])]
        chain = copy()
        alone, _, _ = cuda_decoder_attention_tree_forward_(
            x[:, nodes].contiguous(), g_in, wq, wk, wv, g_q, g_k, wo, chain, depths=torch.arange(n).cuda(),
            past_lengths=past.cuda(), **args)
        # the same rows through projections of another batch size: the end-to-end tolerance
        from bf16_metrics import E2E_MAX_REL

        assert (alone[i].float() - y[i, nodes].float()).abs().max() <= E2E_MAX_REL * float(y.abs().max())
        s = slice(int(past[i]), int(past[i]) + n)
        a, c = (cp.cuda_quantized_kv_read(z)[0][i, :, s].float() for z in (tree, chain))
        assert (a - c).abs().mean() <= 2.0 ** -6 * float(c.abs().mean())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("t", [2, 6, 16, 40])  # 8, 24, 64 and 160 query rows a KV head
def test_repeated_calls_agree_and_no_wait_gives_up(cp, fmt, t):
    """Nothing depends on which warp or CTA comes first, across uneven units that many CTAs share."""
    from tree_decoding import check_tree_wait_status

    b, hkv, group, cap, d = 3, 3, 4, 6144, 128
    cache = filled(cp, fmt, b, hkv, cap, d, 41)
    q = randn((b, t, hkv * group, d), 42).cuda()
    mask, _ = ref.random_tree(b, t, 43)
    past = torch.tensor([cap - t, 1717, 70]).cuda() if fmt != "bf16" else None

    def call():
        return cp.cuda_tree_attention_cached(q, cache, 0 if past is not None else cap - t, tree_mask=mask.cuda(),
                                             past_lengths=past, max_past_length=cap - t)

    check_tree_wait_status()
    first = call()
    for _ in range(200):
        again = call()
    assert torch.equal(first, again) and torch.isfinite(first.float()).all()
    check_tree_wait_status()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [8, 9, 12, 13, 16, 17, 32, 33, 64, 65, 128, 129, 257])
def test_rows_on_both_sides_of_every_kernel_rule(cp, fmt, d, rows):
    """Twenty units of uneven length whose parts several CTAs share, joined one or four rows a warp."""
    check_tree(cp, fmt, 5, rows, 4, 4, d, [700, 130, 0, 701, 333], 1024, 51 + rows)
