"""GPU checks of the paged cache at every head dimension: rows byte for byte, and the attention against FP64."""

from __future__ import annotations

import pytest
import torch

import draft_reference
from test_gpu_draft_ops import randn, rows_of_all_sizes
from test_gpu_paged_long import attention, call, check, sequences

pytestmark = pytest.mark.gpu

DIMS = range(16, 257, 16)


@pytest.fixture(scope="module")
def cp():
    import cuda_primitives

    return cuda_primitives


@pytest.mark.parametrize("format", ["bf16", "fp8", "nvfp4"])
@pytest.mark.parametrize("d", DIMS)
def test_rows(cp, format, d):
    b, t, hkv, size = 2, 21, 3, 16
    cache = cp.PagedKVCache.allocate(4, hkv, size, d, format)
    slots = torch.randperm(4 * size, generator=torch.Generator().manual_seed(d))[:b * t].view(b, t)
    page, at = slots // size, slots % size
    rows = [rows_of_all_sizes((b, t, hkv, d), s) for s in (1, 2)]
    cp.cuda_paged_kv_append_(cache, *(x.cuda() for x in rows), slots.cuda())
    read = cp.cuda_paged_kv_read(cache, slots.cuda())
    for n, x, y in zip("kv", rows, read):
        parts = (x, None, None) if format == "bf16" else draft_reference.quantize_rows(format, x)
        for field, part in zip(("codes", "row_scales", "block_scales"), parts):
            if part is not None:
                got = getattr(cache, f"{n}_{field}").cpu()[page, :, at]
                assert torch.equal(got, torch.as_tensor(part))
        values = x if format == "bf16" else draft_reference.stored_values(format, *parts).to(torch.bfloat16)
        assert torch.equal(y.cpu(), values.transpose(1, 2))


@pytest.mark.parametrize("format", ["bf16", "fp8", "nvfp4"])
@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize("t", [1, 9])
def test_attention(cp, format, d, t):
    pasts = [0, 700, 63, 129]
    counts = torch.tensor([t, max(1, t - 2), 0, t])
    cache, table = sequences(cp, format, pasts, t, 2, 48, d, d)
    table[1, 3] = -1
    mask = draft_reference.random_tree(4, t, d)[0].cuda()
    q = randn((4, t, 6, d), 3).cuda()
    got = call(cp, q, cache, table.cuda(), pasts, tree_mask=mask, counts=counts.cuda())
    check(got, *attention(q, cache, table.cuda(), pasts, mask, counts))


@pytest.mark.parametrize("format", ["bf16", "fp8", "nvfp4"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_more_sequences_than_the_streaming_kernel_takes(cp, format, d):
    pasts = torch.randint(0, 80, (1025,), generator=torch.Generator().manual_seed(d)).tolist()
    cache, table = sequences(cp, format, pasts, 2, 1, 16, d, 7)
    q = randn((1025, 2, 5, d), 3).cuda()
    check(call(cp, q, cache, table.cuda(), pasts), *attention(q, cache, table.cuda(), pasts))
