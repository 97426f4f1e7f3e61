"""CPU checks of the drafted-token operators: the cache class, the rotary
frequencies, refusals before any launch, and the tests' own oracle."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

import draft_reference as ref
import oracle


def make(format="fp8", **kw):
    from quantized_kv_cache import QuantizedKVCache

    return QuantizedKVCache.allocate(2, 3, 70, 64, format, device="cpu", **kw)


@pytest.mark.parametrize("format,row", [("fp8", 64 + 4), ("nvfp4", 32 + 4 + 4)])
def test_allocate_rounds_the_capacity_up(format, row):
    c = make(format)
    assert c.capacity == 128 and c.k_row_scales.shape == (2, 3, 128)
    assert c.nbytes == 2 * 2 * 3 * 128 * row


@pytest.mark.parametrize("change,error,text", [
    (dict(format="int8"), ValueError, "format must be one of"),
    (dict(head_dim=72), ValueError, "multiple of 16"),
    (dict(head_dim=64.0), TypeError, "head_dim must be an integer"),
    (dict(k_codes=torch.zeros((2, 3, 128, 32), dtype=torch.uint8)), ValueError, "k_codes must have shape"),
    (dict(v_codes=torch.zeros((2, 3, 128, 64))), TypeError, "v_codes must have dtype"),
    (dict(k_row_scales=torch.zeros((2, 3, 64))), ValueError, "k_row_scales must have shape"),
    (dict(k_block_scales=torch.zeros((2, 3, 128, 4), dtype=torch.uint8)), ValueError, "no block scales"),
])
def test_cache_fields_are_checked(change, error, text):
    from dataclasses import replace

    with pytest.raises(error, match=text):
        replace(make(), **change)


def test_capacity_has_to_be_whole_tiles():
    from quantized_kv_cache import QuantizedKVCache

    z = lambda *s, t=torch.uint8: torch.zeros(s, dtype=t)  # noqa: E731
    with pytest.raises(ValueError, match="capacity must be a multiple of 64"):
        QuantizedKVCache("fp8", 16, z(1, 1, 65, 16), z(1, 1, 65, 16), z(1, 1, 65, t=torch.float32),
                         z(1, 1, 65, t=torch.float32))
    with pytest.raises(ValueError, match="capacity must be positive"):
        QuantizedKVCache.allocate(1, 1, 0, 64, device="cpu")


# ------------------------------------------------------------------ rotary frequencies
def test_unscaled_and_linear_frequencies():
    from quantized_kv_cache import rope_frequencies

    f, a = rope_frequencies(128, 1e4, device="cpu")
    want = np.array([1e4 ** (-2 * m / 128) for m in range(64)])
    assert a == 1.0 and f.dtype == torch.float32
    assert np.array_equal(f.numpy(), want.astype(np.float32))
    f, _ = rope_frequencies(128, 1e4, scaling="linear", factor=8.0, device="cpu")
    assert np.array_equal(f.numpy(), (want / 8).astype(np.float32))


def test_ntk_keeps_the_fastest_pair_and_slows_the_slowest_by_the_factor():
    from quantized_kv_cache import rope_frequencies

    f0, _ = rope_frequencies(64, 1e4, device="cpu")
    f, _ = rope_frequencies(64, 1e4, scaling="ntk", factor=4.0, device="cpu")
    assert f[0] == f0[0]
    assert abs(float(f0[-1] / f[-1]) - 4.0) < 1e-5
    assert torch.all(f[1:] < f0[1:])


def test_yarn_ramp_between_kept_and_slowed_pairs():
    from quantized_kv_cache import rope_frequencies

    f0, _ = rope_frequencies(128, 1e4, device="cpu")
    f, a = rope_frequencies(128, 1e4, scaling="yarn", factor=16.0, original_length=4096, device="cpu")
    assert a == pytest.approx(0.1 * math.log(16.0) + 1.0)
    turns = f0.double() * 4096 / (2 * math.pi)
    ratio = (f0 / f).double()
    assert torch.all(ratio[turns > 40] == 1.0)
    assert torch.allclose(ratio[turns < 0.8], torch.tensor(16.0, dtype=torch.float64), rtol=1e-6)
    assert torch.all(ratio[1:] >= ratio[:-1] - 1e-6)
    assert rope_frequencies(128, scaling="yarn", factor=1.0, device="cpu")[1] == 1.0


@pytest.mark.parametrize("args,kw,error", [
    ((63,), {}, ValueError), ((0,), {}, ValueError), ((64.0,), {}, TypeError), ((64, -1.0), {}, ValueError),
    ((64,), dict(scaling="cubic"), ValueError), ((64,), dict(factor=math.inf), ValueError),
    ((64,), dict(scaling="yarn", beta_fast=1.0, beta_slow=2.0), ValueError),
])
def test_frequency_refusals(args, kw, error):
    from quantized_kv_cache import rope_frequencies

    with pytest.raises(error):
        rope_frequencies(*args, device="cpu", **kw)


# ------------------------------------------------------------------ refusals before any launch
def test_operators_refuse_cpu_tensors():
    import cuda_primitives as cp

    x = torch.zeros((2, 1, 3, 64), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        cp.cuda_apply_rope_qk(x, x, torch.zeros((1,), dtype=torch.int64), torch.ones(32))
    with pytest.raises(RuntimeError, match="k_codes must be a CUDA tensor"):
        cp.cuda_quantized_kv_append_(make(), x, x, 0)
    with pytest.raises(RuntimeError, match="k_codes must be a CUDA tensor"):
        cp.cuda_quantized_kv_read(make(), 0, 1)
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        cp.cuda_tree_attention_cached(x, make(), 0)
    with pytest.raises(TypeError, match="past_length must be an integer"):
        cp.cuda_tree_attention_cached(x, make(), 0.0)
    with pytest.raises(TypeError, match="max_past_length must be an integer"):
        cp.cuda_tree_attention_cached(x, make(), past_lengths=torch.zeros(2, dtype=torch.int64))


def capi_cache(**change):
    import nvfp4da_capi as capi

    c = capi.KvCache(capi.KV_NVFP4, 256, 256, 256, 256, 256, 256, 2, 3, 128, 64)
    for k, v in change.items():
        setattr(c, k, v)
    return c


@pytest.mark.parametrize("change,status,text", [
    (dict(format=7), 1, b"unknown cache format"), (dict(head_dim=72), 2, b"multiple of 16"),
    (dict(head_dim=272), 2, b"at most 256"), (dict(capacity=100), 1, b"multiple of 64"),
    (dict(v_block_scales=None), 1, b"NULL"), (dict(k_row_scales=260), 1, b"16-byte aligned"),
    (dict(batch=0), 1, b"positive"), (dict(batch=40000), 2, b"65535"),
    (dict(batch=2000, kv_heads=8, capacity=1 << 20), 2, b"2^31"),
])
def test_c_entry_points_refuse_bad_caches(change, status, text):
    import nvfp4da_capi as capi

    lib, c = capi.load(), capi_cache(**change)
    st = (ctypes.c_int64 * 3)(0, 0, 0)
    p = ctypes.c_void_p(256)
    for got in (lib.nvfp4da_kv_quant_append(ctypes.byref(c), p, st, p, st, 1, 0, None, None, None),
                lib.nvfp4da_kv_quant_read(ctypes.byref(c), 0, None, 1, p, p, None),
                lib.nvfp4da_tree_attention(p, ctypes.byref(c), None, 0, p, 1, 6, 0, None, 0, p, 0, None)):
        assert got == status and text in lib.nvfp4da_last_error()
    assert lib.nvfp4da_tree_attention_workspace_size(ctypes.byref(c), 1, 6, 0) == 0


def test_c_entry_points_refuse_bad_arguments():
    import nvfp4da_capi as capi

    lib, c = capi.load(), capi_cache()
    st = (ctypes.c_int64 * 3)(0, 0, 0)
    p, q = ctypes.c_void_p(256), ctypes.c_void_p(264)
    bad = capi.ERR_INVALID_ARGUMENT
    ref_c = ctypes.byref(c)
    assert lib.nvfp4da_kv_quant_append(ref_c, None, st, p, st, 1, 0, None, None, None) == bad
    assert lib.nvfp4da_kv_quant_append(ref_c, p, st, p, st, 1, 128, None, None, None) == bad
    assert lib.nvfp4da_kv_quant_append(ref_c, p, st, p, st, 1, -1, None, None, None) == bad
    assert lib.nvfp4da_kv_quant_read(ref_c, 100, None, 29, p, p, None) == bad
    assert lib.nvfp4da_kv_quant_read(ref_c, 0, None, 1, q, p, None) == bad
    assert lib.nvfp4da_tree_attention(p, ref_c, None, 0, p, 1, 7, 0, None, 0, p, 0, None) == bad
    assert lib.nvfp4da_tree_attention(p, ref_c, None, 0, p, 2, 6, 127, None, 0, p, 0, None) == bad
    assert lib.nvfp4da_tree_attention(q, ref_c, None, 0, p, 1, 6, 0, None, 0, p, 1 << 30, None) == bad
    assert lib.nvfp4da_apply_rope_qk(p, st, p, p, st, p, 1, 1, 4, 2, 64, p, 0, p, 65, 1, 1.0, None) == bad
    assert lib.nvfp4da_apply_rope_qk(p, st, p, p, st, p, 1, 1, 4, 2, 64, p, 0, p, 66, 1, 1.0, None) == bad
    assert lib.nvfp4da_apply_rope_qk(p, st, p, p, st, p, 1, 1, 4, 2, 64, p, 0, p, 64, 1, math.nan, None) == bad
    assert lib.nvfp4da_apply_rope_qk(p, st, p, None, st, p, 1, 1, 4, 2, 64, p, 0, p, 64, 1, 1.0, None) == bad


# ------------------------------------------------------------------ the oracle itself
def test_oracle_rows_follow_the_weight_quantiser():
    """A [1, D] matrix of the weight format: the same scales and codes up to
    values on a rounding boundary (the reciprocal of amax is rounded first)."""
    g = torch.Generator().manual_seed(3)
    rows = torch.randn((64, 128), generator=g).to(torch.bfloat16)
    codes, gamma, beta = ref.quantize_rows("nvfp4", rows)
    same = 0
    for i in range(64):
        w = oracle.quantize(rows[i:i + 1].float().numpy())
        assert np.float32(w.global_decode_scale) == gamma[i]
        same += (w.packed_values[0] == codes[i]).mean() + (w.block_scales[0] == beta[i]).mean()
    assert same / 128 > 0.95


def test_oracle_planted_mistake_is_seen():
    """The attention oracle with one wrong mask entry differs from itself."""
    g = torch.Generator().manual_seed(1)
    q = torch.randn((1, 3, 2, 16), generator=g)
    k, v = (torch.randn((1, 1, 9, 16), generator=g).double() for _ in range(2))
    mask, _ = ref.random_tree(1, 3, 5)
    good, _ = ref.tree_attention(q, k, v, [6], mask)
    mask[0, 2, 0] = ~mask[0, 2, 0]
    assert (ref.tree_attention(q, k, v, [6], mask)[0] - good).abs().max() > 1e-3


def test_tree_status_needs_a_place_for_the_flags():
    import nvfp4da_capi as capi

    assert capi.load().nvfp4da_tree_attention_sync_status(None, None, 1) == capi.ERR_INVALID_ARGUMENT


def test_accepted_paths_may_be_padded_with_any_number(monkeypatch):
    """Numbers past a sequence's count are no nodes: they are not looked up (on a device that lookup would stop it)."""
    import tree_decoding

    got = {}
    monkeypatch.setattr(tree_decoding, "cuda_quantized_kv_append_",
                        lambda cache, k, v, past, **kw: got.update(k=k, v=v, past=past, **kw))
    new_k = torch.arange(2 * 3 * 1 * 4, dtype=torch.float32).view(2, 3, 1, 4)
    path = torch.tensor([[0, 2, -1, -1], [1, 7, 1 << 40, -(1 << 62)]])
    counts = torch.tensor([2, 1])
    tree_decoding.accept_drafted_(object(), new_k, -new_k, path, 5, counts=counts)
    assert got["past"] == 5 and got["counts"] is counts and got["k"].shape == (2, 4, 1, 4)
    assert torch.equal(got["k"][0, :2], new_k[0, [0, 2]]) and torch.equal(got["k"][1, :1], new_k[1, [1]])
    assert torch.equal(got["v"], -got["k"])


@pytest.mark.parametrize("flags", [0, 1])
def test_wait_status_is_read_on_the_device_of_the_stream(monkeypatch, flags):
    """The flag is one word per device: the current device's says nothing about another's stream."""
    import contextlib
    import types

    import nvfp4da_capi
    import tree_decoding

    at = []

    @contextlib.contextmanager
    def device(d):
        at.append(d)
        yield
        at.pop()

    def status(stream):
        assert at == [stream.device]
        return flags

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(nvfp4da_capi, "tree_sync_status", status)
    stream = types.SimpleNamespace(device=torch.device("cuda", 3))
    with pytest.raises(RuntimeError, match="timed out") if flags else contextlib.nullcontext():
        tree_decoding.check_tree_wait_status(stream)
    assert at == []
