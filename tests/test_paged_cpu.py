"""CPU checks of the paged cache: its classes, refusals before any launch, and the tests' own oracle."""

from __future__ import annotations

import ctypes
from dataclasses import replace

import pytest
import torch

import paged_reference as ref


def pool(format="fp8", **kw):
    from paged_kv_cache import PagedKVCache

    return PagedKVCache.allocate(5, 3, 48, 64, format, device="cpu", **kw)


def table(**kw):
    from paged_kv_cache import PageTable

    return PageTable.allocate(**{**dict(batch=2, max_pages=4, pages=5, page_size=16, device="cpu"), **kw})


@pytest.mark.parametrize("format,row", [("bf16", 128), ("fp8", 64 + 4), ("nvfp4", 32 + 4 + 4)])
def test_a_pool_holds_whole_pages(format, row):
    c = pool(format)
    assert c.pages == 5 and c.page_size == 48 and c.nbytes == 2 * 5 * 3 * 48 * row


@pytest.mark.parametrize("change,error,text", [
    (dict(format="int8"), ValueError, "format must be one of"),
    (dict(head_dim=72), ValueError, "multiple of 16"),
    (dict(head_dim=64.0), TypeError, "head_dim must be an integer"),
    (dict(k_codes=torch.zeros((5, 3, 40, 64), dtype=torch.uint8)), ValueError, "page_size must be a multiple of 16"),
    (dict(k_codes=torch.zeros((5, 3, 48, 32), dtype=torch.uint8)), ValueError, "k_codes must have shape"),
    (dict(v_codes=torch.zeros((5, 3, 48, 64))), TypeError, "v_codes must have dtype"),
    (dict(k_row_scales=None), TypeError, "k_row_scales must be a torch.Tensor"),
    (dict(k_block_scales=torch.zeros((5, 3, 48, 4), dtype=torch.uint8)), ValueError, "no block scales"),
])
def test_pool_fields_are_checked(change, error, text):
    with pytest.raises(error, match=text):
        replace(pool(), **change)


@pytest.mark.parametrize("change,error,text", [
    (dict(page_size=24), ValueError, "multiple of 16"),
    (dict(page_size=True), TypeError, "page_size must be an integer"),
    (dict(held=torch.zeros((3,), dtype=torch.int64)), ValueError, "held must have shape"),
    (dict(free_count=torch.zeros((1,), dtype=torch.int32)), TypeError, "free_count must have dtype"),
    (dict(pages=torch.zeros((2, 0), dtype=torch.int32)), ValueError, "positive"),
    (dict(free_pages=torch.zeros((2, 2), dtype=torch.int32)), TypeError, "rank-1"),
])
def test_table_fields_are_checked(change, error, text):
    with pytest.raises(error, match=text):
        replace(table(), **change)


def test_an_empty_table_has_every_page_free():
    t = table()
    assert t.free_pages.tolist() == [4, 3, 2, 1, 0] and t.free_count.tolist() == [5]
    assert t.held.tolist() == [0, 0] and (t.pages == -1).all()
    with pytest.raises(ValueError, match="batch must be at least 1"):
        table(batch=0)


def test_operators_refuse_cpu_tensors_and_bad_numbers():
    import cuda_primitives as cp

    x, n = torch.zeros((2, 1, 3, 64), dtype=torch.bfloat16), torch.zeros((2,), dtype=torch.int64)
    slots = torch.zeros((2, 1), dtype=torch.int64)
    for call in (lambda: cp.cuda_reserve_pages_(table(), n, 1), lambda: cp.cuda_release_pages_(table(), n),
                 lambda: cp.cuda_paged_kv_append_(pool(), x, x, slots), lambda: cp.cuda_paged_kv_read(pool(), slots),
                 lambda: cp.cuda_paged_attention(x, pool(), table().pages, past_lengths=n, max_past_length=0),
                 lambda: cp.cuda_verify_drafted(torch.ones((2, 1, 7)), slots, torch.zeros((2, 1)))):
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            call()
    with pytest.raises(TypeError, match="tokens must be an integer"):
        cp.cuda_reserve_pages_(table(), n, 1.0)
    with pytest.raises(TypeError, match="max_past_length must be an integer"):
        cp.cuda_paged_attention(x, pool(), table().pages, past_lengths=n, max_past_length=None)


def capi_pool(**change):
    import nvfp4da_capi as capi

    c = capi.KvCache(capi.KV_NVFP4, 256, 256, 256, 256, 256, 256, 70000, 3, 48, 64)
    for k, v in change.items():
        setattr(c, k, v)
    return c


@pytest.mark.parametrize("change,status,text", [
    (dict(format=7), 1, b"unknown cache format"), (dict(head_dim=72), 2, b"multiple of 16"),
    (dict(capacity=40), 1, b"page size must be a multiple of 16"), (dict(v_block_scales=None), 1, b"NULL"),
    (dict(k_row_scales=260), 1, b"16-byte aligned"), (dict(batch=0), 1, b"positive"),
    (dict(batch=1 << 28), 2, b"2^31"), (dict(batch=1 << 62, kv_heads=8), 2, b"2^31"),
])
def test_c_entry_points_refuse_bad_pools(change, status, text):
    import nvfp4da_capi as capi

    lib, c = capi.load(), capi_pool(**change)
    st = (ctypes.c_int64 * 3)(0, 0, 0)
    p, c = ctypes.c_void_p(256), ctypes.byref(c)
    for got in (lib.nvfp4da_paged_kv_append(c, p, st, p, st, 1, 1, p, 1, None, 1, None, None),
                lib.nvfp4da_paged_kv_read(c, p, 1, 1, p, p, None),
                lib.nvfp4da_paged_attention(p, c, p, 1, 4, None, 0, p, 1, 6, p, 0, None, p, 0, None)):
        assert got == status and text in lib.nvfp4da_last_error()
    assert lib.nvfp4da_paged_attention_workspace_size(c, 1, 4, 1, 6, 0) == 0


def test_c_entry_points_refuse_bad_arguments():
    import nvfp4da_capi as capi

    lib, c = capi.load(), ctypes.byref(capi_pool())
    st, st2 = (ctypes.c_int64 * 3)(0, 0, 0), (ctypes.c_int64 * 2)(0, 0)
    p, q = ctypes.c_void_p(256), ctypes.c_void_p(264)
    bad, no = capi.ERR_INVALID_ARGUMENT, capi.ERR_UNSUPPORTED
    append, read = lib.nvfp4da_paged_kv_append, lib.nvfp4da_paged_kv_read
    assert append(c, None, st, p, st, 1, 1, p, 1, None, 1, None, None) == bad
    assert append(c, p, st, p, st, 1, 1, None, 1, None, 1, None, None) == bad
    assert append(c, p, st, p, st, 1, 2, p, 1, None, 2, None, None) == bad  # fewer slots than rows
    assert append(c, p, st, p, st, 1, 2, p, 2, None, 1, None, None) == bad  # rows other than tokens without source
    assert append(c, p, st, p, st, 30000, 1, p, 1, None, 1, None, None) == no
    assert read(c, p, 1, 0, p, p, None) == bad and read(c, p, 1, 1, q, p, None) == bad
    assert read(c, p, 30000, 1, p, p, None) == no

    def attend(q_=p, table_=p, batch=1, most=4, out=p, tokens=1, heads=6, past=p, bound=0, ws=p, size=1 << 40):
        return lib.nvfp4da_paged_attention(q_, c, table_, batch, most, None, 0, out, tokens, heads, past, bound, None, ws,
                                           size, None)

    assert attend(q_=None) == bad and attend(table_=None) == bad and attend(past=None) == bad and attend(q_=q) == bad
    assert attend(heads=7) == bad and attend(tokens=0) == bad and attend(bound=-1) == bad and attend(most=0) == bad
    assert attend(bound=4 * 48, tokens=1) == bad and attend(batch=30000) == no and attend(most=1 << 40) == no
    assert attend(tokens=70000, most=1 << 20) == no
    t = capi.PageTable(256, 256, 256, 256, 2, 4, 5, 16)
    for change, status in ((dict(held=None), bad), (dict(batch=0), bad), (dict(page_size=24), bad),
                           (dict(max_pages=1 << 28), no), (dict(batch=1 << 30), no), (dict(pool=1 << 28), no)):
        u = capi.PageTable(256, 256, 256, 256, 2, 4, 5, 16)
        for k, v in change.items():
            setattr(u, k, v)
        assert lib.nvfp4da_reserve_pages(ctypes.byref(u), p, None, 1, p, p, None) == status
        assert lib.nvfp4da_release_pages(ctypes.byref(u), p, None) == status
    t = ctypes.byref(t)
    assert lib.nvfp4da_reserve_pages(t, None, None, 1, p, p, None) == bad
    assert lib.nvfp4da_reserve_pages(t, p, None, 0, p, p, None) == bad
    assert lib.nvfp4da_reserve_pages(t, p, None, 1 << 21, p, p, None) == no
    assert lib.nvfp4da_release_pages(t, None, None) == bad
    verify = lib.nvfp4da_verify_drafted
    assert verify(None, st2, None, st2, p, None, 0, p, None, 1, 1, 5, p, p, p, None) == bad
    assert verify(p, st2, p, None, p, None, 0, p, None, 1, 1, 5, p, p, p, None) == bad
    assert verify(p, st2, None, st2, p, None, 0, p, None, 1, 0, 5, p, p, p, None) == bad
    assert verify(p, st2, None, st2, p, None, 0, p, None, 1, 1025, 5, p, p, p, None) == no
    assert verify(p, st2, None, st2, p, None, 0, p, None, 1, 1, 1 << 31, p, p, p, None) == no


# ------------------------------------------------------------------ the oracle itself
def test_oracle_release_undoes_reserve():
    pages = [[3, -1, -1], [1, 0, -1], [-1, -1, -1]]
    held, stack = [1, 2, 0], [7, 6, 2, 5, 4]
    a = ref.reserve(pages, held, stack, 16, 8, [5, 30, 0], None, 14)
    assert a[0] == [[3, 4, -1], [1, 0, 5], [2, -1, -1]] and a[1] == [2, 3, 1] and a[2] == [7, 6]
    assert a[3][0][:12] == [53, 54, 55, 56, 57, 58, 59, 60, 61, 62, 63, 64] and a[4] == [14, 14, 14]
    assert ref.release(*a[:3], 16, 8, [5, 30, 0]) == (pages, held, stack)


def test_oracle_planted_mistake_is_seen():
    """A residual that is not what a rejection leaves gives another token."""
    p, q = torch.tensor([[[0.5, 0.5, 0.0], [1.0, 0.0, 0.0]]]), torch.tensor([[[0.9, 0.1, 0.0], [1.0, 0.0, 0.0]]])
    tokens, u = torch.tensor([[2, 0]]), torch.tensor([[0.2, 0.7]])
    assert ref.verify(p, tokens, u, q) == ([[0, -1]], [1], [1])  # 0.7 * 0.9 >= 0.5; what is left is token 1 alone
    assert ref.verify(p, tokens, u, None) == ([[0, -1]], [1], [1])
    assert ref.verify(p, tokens, torch.tensor([[0.2, 0.3]]), q) == ([[0, 1]], [2], [0])
    assert ref.verify(q, tokens, u, q) == ([[0, 1]], [2], [0])


def test_oracle_tokens_follow_the_target():
    """The first new token of a two-candidate tree, over 20,000 draws: within 5 standard deviations everywhere."""
    g = torch.Generator().manual_seed(5)
    n = 20000
    p = torch.tensor([0.1, 0.2, 0.3, 0.4]).expand(n, 3, 4)
    q = torch.tensor([0.4, 0.3, 0.2, 0.1]).expand(n, 3, 4)
    tokens = torch.multinomial(q[0, 0], 3 * n, replacement=True, generator=g).view(n, 3)
    path, count, nexts = ref.verify(p, tokens, torch.rand((n, 3), generator=g), q, torch.tensor([-1, 0, 0]))
    first = torch.tensor([nexts[i] if count[i] == 1 else int(tokens[i, path[i][1]]) for i in range(n)])
    share = torch.bincount(first, minlength=4) / n
    assert ((share - p[0, 0]).abs() <= 5 * (p[0, 0] * (1 - p[0, 0]) / n).sqrt()).all()
