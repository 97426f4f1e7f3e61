"""The operators of drafted-token verification over a quantised KV cache, as measured cases.

Three groups: rotary positions of q and k, the quantised cache (rows quantised
as they are appended, a window read back) and the attention of a tree of
drafted tokens over a BF16, E4M3 or NVFP4 cache.  ``run`` computes them in
elementary torch operations, or where ``own`` is true through the framework's
entry points; ``exact`` restates the definitions in 64 bits.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path
from types import SimpleNamespace

import torch

own = False

_DEV = "cuda"
_F32_MAX = torch.finfo(torch.float32).max
_PRIMITIVES = None


def _primitives():
    """The framework's operator module (its package directory goes on sys.path, as its users do)."""
    global _PRIMITIVES
    if _PRIMITIVES is None:
        path = str(Path(__file__).resolve().parent.parent / "cuda-nvfp4-decoder-attention_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import cuda_primitives

        _PRIMITIVES = cuda_primitives
    return _PRIMITIVES


# ------------------------------------------------------------------ cases
def listed():
    rope = dict(op="rope", kv_heads=6, q_heads=24, head_dim=128)
    cache = dict(op="cache", kv_heads=6, head_dim=128)
    attn = dict(op="attention", kv_heads=6, q_heads=24, head_dim=128)
    return [
        # One token of one sequence: the launch itself is what counts.
        dict(rope, name="rope_one_token", batch=1, tokens=1, rotary_dim=128, interleaved=True, factor=1.0, first=511),
        # Prefill of four 2,048-token prompts with frequencies scaled for a long context.
        dict(rope, name="rope_prefill_scaled", batch=4, tokens=2048, rotary_dim=128, interleaved=False, factor=8.0,
             first=60000),
        # A quarter of wide heads rotated, an odd number of drafted tokens.
        dict(rope, name="rope_partial_ragged", batch=37, tokens=23, q_heads=12, kv_heads=3, head_dim=256,
             rotary_dim=64, interleaved=False, factor=1.0, first=4097),
        # Odd small call: seven drafted tokens of three sequences, narrow heads.
        dict(cache, name="cache_nvfp4_small_odd", format="nvfp4", batch=3, kv_heads=5, head_dim=64, tokens=7,
             past_lo=90, past_hi=131, window=129),
        # A decode step of 64 ragged sequences: one row each, the last 512 rows looked at.
        dict(cache, name="cache_fp8_decode_64", format="fp8", batch=64, tokens=1, past_lo=1024, past_hi=8190,
             window=512),
        # Four prompts of 2,048 tokens quantised and handed back.
        dict(cache, name="cache_nvfp4_prefill", format="nvfp4", batch=4, tokens=2048, past_lo=0, past_hi=0,
             window=2048),
        # Long caches read back whole, as before a step that wants BF16.
        dict(cache, name="cache_fp8_long_read", format="fp8", batch=4, tokens=8, past_lo=32700, past_hi=32760,
             window=32768),
        # The smallest verification: eight drafted tokens after 511, BF16 cache.
        dict(attn, name="tree_bf16_short", format="bf16", batch=1, tokens=8, past_lo=511, past_hi=511),
        # Batched single-token decode over ragged E4M3 caches.
        dict(attn, name="tree_fp8_decode_64", format="fp8", batch=64, tokens=1, past_lo=1024, past_hi=8191),
        # Single tokens over long NVFP4 caches.
        dict(attn, name="tree_nvfp4_long_decode", format="nvfp4", batch=8, tokens=1, past_lo=32767, past_hi=32767),
        # Sixteen drafted tokens over long NVFP4 caches.
        dict(attn, name="tree_nvfp4_long_16", format="nvfp4", batch=8, tokens=16, past_lo=30001, past_hi=32752),
        # A large tree over BF16 caches: arithmetic counts as well as bytes.
        dict(attn, name="tree_bf16_48", format="bf16", batch=16, tokens=48, past_lo=4000, past_hi=8100),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    op = rng.choice(("rope", "cache", "attention", "attention"))
    group = rng.choice((1, 2, 4, 8))
    hkv = rng.randint(1, 8)
    if op == "rope":
        d = rng.choice((64, 96, 128, 256))
        batch = _log(rng, 1, 48)
        tokens = max(1, min(_log(rng, 1, 2048), 8192 // batch))
        while batch * tokens * hkv * (group + 1) * d > 30_000_000:
            tokens = max(1, tokens // 2)
        return dict(op=op, kv_heads=hkv, q_heads=hkv * group, head_dim=d, batch=batch, tokens=tokens,
                    rotary_dim=d // rng.choice((1, 2, 4)), interleaved=rng.random() < 0.5,
                    factor=rng.choice((1.0, 4.0, 8.0)), first=_log(rng, 1, 100000))
    d = rng.choice((64, 128, 128, 256))
    batch = _log(rng, 1, 64)
    hi = _log(rng, 1, 32700)
    while batch * hkv * hi * d > 200_000_000:
        hi = hi // 2
    lo = hi if rng.random() < 0.3 else rng.randint(hi // 4, hi)
    if op == "cache":
        tokens = max(1, min(_log(rng, 1, 2048), hi))
        while batch * hkv * tokens * d > 8_000_000:
            tokens = max(1, tokens // 2)
        return dict(op=op, format=rng.choice(("fp8", "nvfp4")), kv_heads=hkv, head_dim=d, batch=batch, tokens=tokens,
                    past_lo=lo, past_hi=hi, window=rng.randint(1, hi + tokens))
    tokens = _log(rng, 1, 64)
    while batch * hkv * group * tokens * hi * d > 20_000_000_000 and tokens > 1:
        tokens = tokens // 2
    return dict(op=op, format=rng.choice(("bf16", "fp8", "nvfp4")), kv_heads=hkv, q_heads=hkv * group, head_dim=d,
                batch=batch, tokens=tokens, past_lo=lo, past_hi=hi)


def _pasts(c):
    """Ragged past lengths in [past_lo, past_hi], the same for every seed."""
    span = c["past_hi"] - c["past_lo"] + 1
    return [c["past_lo"] + (b * 7919 + 13) % span for b in range(c["batch"])]


def _capacity(c):
    return -(-(c["past_hi"] + c["tokens"]) // 64) * 64


def _row_bytes(c):
    d = c["head_dim"]
    return {"bf16": 2 * d, "fp8": d + 4, "nvfp4": d // 2 + d // 16 + 4}[c["format"]]


def work(c):
    b, t, d, hkv = c["batch"], c["tokens"], c["head_dim"], c["kv_heads"]
    if c["op"] == "rope":
        n = b * t * (c["q_heads"] + hkv) * d
        rotated = b * t * (c["q_heads"] + hkv) * c["rotary_dim"]
        return {"bytes": 4 * n + 8 * b * t + 2 * c["rotary_dim"], "flops": 3 * rotated}
    if c["op"] == "cache":
        rows = b * hkv * t
        new = 2 * rows * (2 * d + _row_bytes(c))  # read in BF16, written quantised
        old = b * hkv * max(0, c["window"] - t)  # rows of the window that were there before
        read = 2 * old * _row_bytes(c) + 2 * b * hkv * c["window"] * 2 * d
        return {"bytes": new + read + 8 * b, "flops": 4 * rows * d + 4 * b * hkv * c["window"] * d}
    keys = sum(p + t for p in _pasts(c))
    q = b * t * c["q_heads"] * d
    return {"bytes": 2 * keys * hkv * _row_bytes(c) + 4 * q + b * t * t + 8 * b, "flops": 4 * t * c["q_heads"] * d * keys}


# ------------------------------------------------------------------ inputs
def _tree(batch, tokens, g):
    """Ancestor masks [B, T, T] and depths [B, T] of random trees in topological order."""
    parents = (torch.rand((batch, tokens), generator=g) * torch.arange(tokens)).long()
    mask = torch.zeros((batch, tokens, tokens), dtype=torch.bool)
    depth = torch.zeros((batch, tokens), dtype=torch.int64)
    rows = torch.arange(batch)
    for t in range(tokens):
        if t:
            mask[:, t] = mask[rows, parents[:, t]]
            depth[:, t] = depth[rows, parents[:, t]] + 1
        mask[:, t, t] = True
    return mask, depth


def _rows(shape, g, spread):
    """K or V rows as a layer makes them: some channels larger, rows of different size."""
    d = shape[-1]
    x = torch.randn(shape, generator=g, device=_DEV)
    x *= 1.0 + 3.0 * (torch.rand((d,), generator=g, device=_DEV) < 0.06)
    if spread:
        x *= torch.exp(0.7 * torch.randn(shape[:-1] + (1,), generator=g, device=_DEV))
    return x.to(torch.bfloat16)


def _filled_cache(c, g):
    """A cache of _capacity rows, filled; slots at and past P_b hold what an earlier step left there."""
    shape = (c["batch"], c["kv_heads"], _capacity(c), c["head_dim"])
    if c["format"] == "bf16":
        return _rows(shape, g, False), _rows(shape, g, True)
    d, fields = shape[3], {}
    for n in "kv":
        codes = torch.empty(shape[:3] + (d if c["format"] == "fp8" else d // 2,), dtype=torch.uint8, device=_DEV)
        gamma = torch.empty(shape[:3], dtype=torch.float32, device=_DEV)
        beta = torch.empty(shape[:3] + (d // 16,), dtype=torch.uint8, device=_DEV) if c["format"] == "nvfp4" else None
        for b in range(shape[0]):
            parts = _quantize(c["format"], _rows(shape[1:], g, n == "v"))
            for to, x in zip((codes, gamma, beta), parts):
                if to is not None:
                    to[b] = x
        fields.update({n + "_codes": codes, n + "_row_scales": gamma, n + "_block_scales": beta})
    return SimpleNamespace(format=c["format"], head_dim=d, **fields)


def prepare(c, seed):
    g = torch.Generator(device=_DEV).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    b, t, d, hkv = c["batch"], c["tokens"], c["head_dim"], c["kv_heads"]
    s = SimpleNamespace(case=dict(c), op=c["op"])
    if c["op"] == "rope":
        r = c["rotary_dim"]
        s.q = torch.randn((b, t, c["q_heads"], d), generator=g, device=_DEV).to(torch.bfloat16)
        s.k = torch.randn((b, t, hkv, d), generator=g, device=_DEV).to(torch.bfloat16)
        first = c["first"] + torch.randint(0, 64, (b, 1), generator=host)
        s.positions = (first + torch.arange(t)).to(_DEV)
        freq = 10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)
        # the lower half of the frequencies stretched by the factor, as long-context scalings do
        freq[r // 4:] /= c["factor"]
        s.inv_freq = freq.to(torch.float32).to(_DEV)
        s.attention_factor = 1.0 + 0.1 * math.log(c["factor"])
        return s
    pasts = _pasts(c)
    s.past_lengths = torch.tensor(pasts, dtype=torch.int64, device=_DEV)
    s.max_past = max(pasts)
    s.cache = _filled_cache(c, g)
    if c["op"] == "cache":
        s.new_k = _rows((b, t, hkv, d), g, False)
        s.new_v = _rows((b, t, hkv, d), g, True)
        s.starts = (s.past_lengths + t - c["window"]).clamp(min=0)
        return s
    s.q = _rows((b, t, c["q_heads"], d), g, False)
    s.mask = _tree(b, t, host)[0].to(_DEV)
    return s


# ------------------------------------------------------------------ plain forms (32 bits)
def _e4m3_codes(x):
    return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)


def _e4m3_values(codes):
    return codes.view(torch.float8_e4m3fn).to(torch.float32)


def _e2m1_codes(x):
    a = x.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = code + 8 * torch.signbit(x).to(torch.uint8)
    return code[..., 0::2] + 16 * code[..., 1::2]


def _e2m1_values(codes):
    level = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    level = torch.cat((level, -level))
    byte = torch.arange(256, device=codes.device)
    pairs = torch.stack((level[byte % 16], level[byte // 16]), dim=-1)
    return pairs[codes.long()].flatten(-2)


def _quantize(fmt, rows):
    """(codes, row scales, block scales or None) of BF16 rows [..., D]."""
    x = rows.to(torch.float32)
    amax = x.abs().amax(dim=-1)
    top = 448.0 if fmt == "fp8" else 2688.0
    enc = torch.where(amax == 0, torch.ones_like(amax), (top / amax).clamp(max=_F32_MAX))
    gamma = amax * torch.tensor(1.0 / top, dtype=torch.float32, device=x.device)
    if fmt == "fp8":
        return _e4m3_codes(x * enc[..., None]), gamma, None
    blocks = x.unflatten(-1, (-1, 16))
    mult = enc * torch.tensor(1.0 / 6.0, dtype=torch.float32, device=x.device)
    beta = _e4m3_codes(blocks.abs().amax(dim=-1) * mult[..., None])
    value = _e4m3_values(beta)
    factor = (1.0 / (value * (1.0 / enc)[..., None])).clamp(max=_F32_MAX)
    factor = torch.where(value > 0, factor, torch.zeros_like(factor))
    return _e2m1_codes((blocks * factor[..., None]).flatten(-2)), gamma, beta


def _values(fmt, codes, gamma, beta):
    """FP32 rows of quantised storage."""
    if fmt == "fp8":
        return _e4m3_values(codes) * gamma[..., None]
    return (_e2m1_values(codes).unflatten(-1, (-1, 16)) * _e4m3_values(beta)[..., None]).flatten(-2) * gamma[..., None]


def _stored(cache, n):
    return getattr(cache, n + "_codes"), getattr(cache, n + "_row_scales"), getattr(cache, n + "_block_scales")


def _plain_rope(s):
    c = s.case
    r = c["rotary_dim"]
    angle = s.positions.to(torch.float32)[..., None] * s.inv_freq
    cos = (torch.cos(angle) * s.attention_factor)[:, :, None]
    sin = (torch.sin(angle) * s.attention_factor)[:, :, None]

    def rotate(x):
        y = x.to(torch.float32)
        if c["interleaved"]:
            e, o = y[..., 0:r:2], y[..., 1:r:2]
            turned = torch.stack((e * cos - o * sin, e * sin + o * cos), dim=-1).flatten(-2)
        else:
            e, o = y[..., :r // 2], y[..., r // 2:r]
            turned = torch.cat((e * cos - o * sin, e * sin + o * cos), dim=-1)
        return torch.cat((turned.to(x.dtype), x[..., r:]), dim=-1)

    return rotate(s.q), rotate(s.k)


def _plain_cache(s):
    c = s.case
    b, t = c["batch"], c["tokens"]
    seq = torch.arange(b, device=_DEV)[:, None, None]
    head = torch.arange(c["kv_heads"], device=_DEV)[None, :, None]
    slot = s.past_lengths[:, None, None] + torch.arange(t, device=_DEV)
    back = s.starts[:, None, None] + torch.arange(c["window"], device=_DEV)
    out = []
    for n, new in (("k", s.new_k), ("v", s.new_v)):
        stored = _stored(s.cache, n)
        for to, x in zip(stored, _quantize(c["format"], new.transpose(1, 2))):
            if to is not None:
                to[seq, head, slot] = x
        # rows of the window past the capacity do not exist
        inside = (back < stored[0].shape[2])[..., None]
        rows = [None if x is None else x[seq, head, back.clamp(max=x.shape[2] - 1)] for x in stored]
        out.append((_values(c["format"], *rows) * inside).to(torch.bfloat16))
    return tuple(out)


def _plain_attention(s):
    c = s.case
    b, t, d, hkv = c["batch"], c["tokens"], c["head_dim"], c["kv_heads"]
    group, length = c["q_heads"] // hkv, s.max_past + t
    if c["format"] == "bf16":
        k, v = (x[:, :, :length].to(torch.float32) for x in s.cache)
    else:
        k, v = (_values(c["format"], *(None if x is None else x[:, :, :length] for x in _stored(s.cache, n)))
                for n in "kv")
    q = s.q.to(torch.float32).view(b, t, hkv, group, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, t * group, d)
    scores = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(d))
    # key j of sequence b: committed below P_b, the drafted token j - P_b from there on
    u = torch.arange(length, device=_DEV)[None] - s.past_lengths[:, None]
    drafted = torch.gather(s.mask, 2, u.clamp(0, t - 1)[:, None].expand(b, t, length))
    seen = (u < 0)[:, None] | (drafted & (u < t)[:, None])
    scores = scores.view(b, hkv, t, group, length).masked_fill(~seen[:, None, :, None], -math.inf)
    p = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
    p = (p / p.sum(dim=-1, keepdim=True)).view(b, hkv, t * group, length)
    ctx = torch.matmul(p, v * (u < t)[:, None, :, None])
    return ctx.view(b, hkv, t, group, d).permute(0, 2, 1, 3, 4).reshape(b, t, c["q_heads"], d).to(torch.bfloat16)


def run(s):
    if own:
        ops = _primitives()
        if s.op == "rope":
            return ops.cuda_apply_rope_qk(s.q, s.k, s.positions, s.inv_freq, interleaved=s.case["interleaved"],
                                          attention_factor=s.attention_factor)
        if s.op == "cache":
            ops.cuda_quantized_kv_append_(s.cache, s.new_k, s.new_v, past_lengths=s.past_lengths)
            return ops.cuda_quantized_kv_read(s.cache, length=s.case["window"], starts=s.starts)
        return ops.cuda_tree_attention_cached(s.q, s.cache, tree_mask=s.mask, past_lengths=s.past_lengths,
                                              max_past_length=s.max_past)
    return {"rope": _plain_rope, "cache": _plain_cache, "attention": _plain_attention}[s.op](s)


# ------------------------------------------------------------------ the definitions in 64 bits
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_E4M3 = tuple((m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
              for e in range(16) for m in range(8))[:127]


def _nearest(x, levels):
    """The nearest of ascending ``levels`` to x >= 0, an even index where two are as near."""
    table = torch.tensor(levels, dtype=torch.float64, device=x.device)
    hi = torch.searchsorted(table, x.contiguous()).clamp(max=len(levels) - 1)
    lo = (hi - 1).clamp(min=0)
    up, down = (table[hi] - x).abs(), (x - table[lo]).abs()
    return torch.where((up < down) | ((up == down) & (hi % 2 == 0)), table[hi], table[lo])


def _exact_quantized(fmt, rows):
    x = rows.double()
    amax = x.abs().amax(dim=-1, keepdim=True)
    if fmt == "fp8":
        gamma = amax / 448
        return torch.where(amax > 0, x.sign() * _nearest(x.abs() / gamma, _E4M3) * gamma, 0.0)
    blocks, gamma = x.unflatten(-1, (-1, 16)), (amax / 2688)[..., None]
    unit = _nearest(blocks.abs().amax(dim=-1, keepdim=True) / 6 / gamma, _E4M3) * gamma
    return torch.where(unit > 0, blocks.sign() * _nearest(blocks.abs() / unit, _E2M1) * unit, 0.0).flatten(-2)


def _exact_stored(fmt, codes, gamma, beta):
    if fmt == "fp8":
        table = torch.tensor(_E4M3 + (math.nan,), dtype=torch.float64, device=codes.device)
        v = table[(codes & 127).long()] * torch.where(codes > 127, -1.0, 1.0)
    else:
        table = torch.tensor(_E2M1 + tuple(-x for x in _E2M1), dtype=torch.float64, device=codes.device)
        scale = torch.tensor(_E4M3 + (math.nan,), dtype=torch.float64, device=codes.device)[beta.long()]
        v = torch.stack((table[(codes & 15).long()], table[(codes >> 4).long()]), dim=-1).flatten(-2)
        v = (v.unflatten(-1, (-1, 16)) * scale[..., None]).flatten(-2)
    return v * gamma.double()[..., None]


def exact(c, seed):
    s = prepare(c, seed)
    b, t, d, hkv = c["batch"], c["tokens"], c["head_dim"], c["kv_heads"]
    if c["op"] == "rope":
        r = c["rotary_dim"]
        turn = torch.polar(torch.full((), float(s.attention_factor), dtype=torch.float64, device=_DEV),
                           s.positions.double()[..., None] * s.inv_freq.double())[:, :, None]
        out = []
        for x in (s.q.double(), s.k.double()):
            if c["interleaved"]:
                z = torch.view_as_complex(x[..., :r].unflatten(-1, (-1, 2)).contiguous()) * turn
                turned = torch.view_as_real(z).flatten(-2)
            else:
                z = torch.complex(x[..., :r // 2], x[..., r // 2:r]) * turn
                turned = torch.cat((z.real, z.imag), dim=-1)
            out.append(torch.cat((turned, x[..., r:]), dim=-1))
        return tuple(out)
    pasts = _pasts(c)
    if c["op"] == "cache":
        out = []
        for n, new in (("k", s.new_k), ("v", s.new_v)):
            rows = torch.zeros((b, hkv, c["window"], d), dtype=torch.float64, device=_DEV)
            for i, p in enumerate(pasts):
                a = max(0, p + t - c["window"])
                whole = [None if x is None else x[i, :, a:a + c["window"]] for x in _stored(s.cache, n)]
                rows[i, :, :whole[0].shape[1]] = _exact_stored(c["format"], *whole)
                fresh = _exact_quantized(c["format"], new[i].transpose(0, 1))
                from_, to = max(p, a), min(p + t, a + c["window"])
                rows[i, :, from_ - a:to - a] = fresh[:, from_ - p:to - p]
            out.append(rows)
        return tuple(out)
    ctx = torch.zeros((b, t, c["q_heads"], d), dtype=torch.float64, device=_DEV)
    group = c["q_heads"] // hkv
    for i, p in enumerate(pasts):
        seen = torch.cat((torch.ones((t, p), dtype=torch.bool, device=_DEV), s.mask[i]), dim=1)
        for h in range(hkv):
            if c["format"] == "bf16":
                k, v = (x[i, h, :p + t].double() for x in s.cache)
            else:
                k, v = (_exact_stored(c["format"], *(None if x is None else x[i, h, :p + t]
                                                     for x in _stored(s.cache, n))) for n in "kv")
            for j in range(h * group, (h + 1) * group):
                w = (s.q[i, :, j].double() @ k.T / math.sqrt(d)).masked_fill(~seen, -math.inf)
                ctx[i, :, j] = torch.softmax(w, dim=-1) @ v
    return ctx
