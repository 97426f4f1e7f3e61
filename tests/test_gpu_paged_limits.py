"""GPU checks of the paged operators where their documented limits are."""

from __future__ import annotations

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cp():
    import cuda_primitives

    return cuda_primitives


def test_release_of_the_largest_table_that_names_one_page_everywhere(cp):
    """Almost 2^31 entries name page 0 and the stack is full: their places pass 2^31, and nothing is written."""
    batch, most, pool = 32, (1 << 26) - 1, (1 << 27) - 1
    t = cp.PageTable.allocate(batch, most, pool, 16)
    t.pages.zero_()
    t.held.fill_(most)
    assert int(t.free_count) + batch * most > 1 << 31
    cp.cuda_release_pages_(t, torch.zeros((batch,), dtype=torch.int64).cuda())
    assert int(t.free_count) == pool and (t.held == 0).all()
    assert all((row == -1).all() for row in t.pages)
    assert torch.equal(t.free_pages, torch.arange(pool - 1, -1, -1, dtype=torch.int32, device="cuda"))


# ------------------------------------------------------------------ nothing beside the buffers
def inside(values, margin, fill):
    """A tensor of these values in the middle of a larger one, and the larger one."""
    whole = torch.full((values.numel() + 2 * margin,), fill, dtype=values.dtype, device="cuda")
    part = whole[margin:margin + values.numel()].view(values.shape)
    part.copy_(values)
    return part, whole


def margins(whole, part):
    n = (whole.numel() - part.numel()) // 2
    return whole[:n], whole[n + part.numel():]


@pytest.mark.parametrize("batch,most,pool,tokens", [(3, 4, 6, 4), (37, 5, 40, 33), (1030, 2, 900, 3)])
def test_nothing_is_written_beside_the_table(cp, batch, most, pool, tokens):
    """Tables with values no call would leave, every buffer between margins: reserve and release through the C ABI."""
    import nvfp4da_capi as capi

    lib, size, margin, fill = capi.load(), 16, 300, 0x3b3b3b3b
    g = torch.Generator().manual_seed(batch)

    def wild(shape, near, dtype):
        x = torch.randint(-2, near + 3, shape, generator=g)
        odd = torch.rand(shape, generator=g) < 0.1
        big = torch.tensor([-(1 << 31), (1 << 31) - 1] if dtype == torch.int32 else [-(1 << 62), 1 << 62, 1 << 33])
        return torch.where(odd, big[torch.randint(0, len(big), shape, generator=g)], x).to(dtype)

    for _ in range(6):
        buffers = {}
        for name, values in dict(pages=wild((batch, most), pool, torch.int32), held=wild((batch,), most, torch.int64),
                                 free_pages=wild((pool,), pool, torch.int32), free_count=wild((1,), pool, torch.int64),
                                 slots=torch.zeros((batch, tokens), dtype=torch.int64),
                                 granted=torch.zeros((batch,), dtype=torch.int64)).items():
            buffers[name] = inside(values, margin, fill)
        x = {n: part for n, (part, _) in buffers.items()}
        table = capi.PageTable(*(x[n].data_ptr() for n in ("pages", "held", "free_pages", "free_count")), batch, most,
                               pool, size)
        past = wild((batch,), most * size, torch.int64).cuda()
        counts = wild((batch,), tokens, torch.int64).cuda()
        kept = wild((batch,), most * size, torch.int64).cuda()
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        assert lib.nvfp4da_reserve_pages(ctypes.byref(table), past.data_ptr(), counts.data_ptr(), tokens,
                                         x["slots"].data_ptr(), x["granted"].data_ptr(), stream) == 0
        assert lib.nvfp4da_release_pages(ctypes.byref(table), kept.data_ptr(), stream) == 0
        for part, whole in buffers.values():
            assert all((m == fill).all() for m in margins(whole, part))
        assert ((x["slots"] >= -1) & (x["slots"] < pool * size)).all()
        assert 0 <= int(x["free_count"]) <= pool
