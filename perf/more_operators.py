"""The operators of serving drafted tokens from a paged KV cache, as measured cases.

Four groups: block tables and slot maps built from lengths (pages reserved and
given back), rows written and read by slots, attention through the block table
over BF16, E4M3 or NVFP4 pages, and the verification of drafted tokens from
given random numbers.  ``run`` computes them in elementary torch operations, or
where ``own`` is true through the framework's entry points; ``exact`` restates
the definitions in 64 bits.
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
    heads = dict(kv_heads=6, q_heads=24, head_dim=128)
    rows = dict(op="rows", kv_heads=6, head_dim=128)
    return [
        # A decode step of eight sequences asks for its slots: the launches are what counts.
        dict(op="pages", name="pages_decode_8", batch=8, tokens=1, page_size=16, past_lo=500, past_hi=600, short=False),
        # 64 prompts of 2,048 tokens come in while the pool cannot hold them all.
        dict(op="pages", name="pages_prefill_64_short", batch=64, tokens=2048, page_size=16, past_lo=0, past_hi=700,
             short=True),
        # A decode step of 64 sequences: a row each written, the last 512 read, small BF16 pages.
        dict(rows, name="rows_bf16_decode_64", format="bf16", batch=64, tokens=1, page_size=16, past_lo=1024,
             past_hi=8190, window=512),
        # Four prompts quantised into pages and handed back; the last page of each ends early.
        dict(rows, name="rows_nvfp4_prefill", format="nvfp4", batch=4, tokens=2043, page_size=64, past_lo=0, past_hi=0,
             window=2043),
        # The smallest decode: one token after 511, BF16 pages of 16.
        dict(heads, op="attention", name="paged_bf16_short", format="bf16", batch=1, tokens=1, page_size=16,
             past_lo=511, past_hi=511),
        # Batched single-token decode over ragged lengths, BF16 pages of 64.
        dict(heads, op="attention", name="paged_bf16_decode_64", format="bf16", batch=64, tokens=1, page_size=64,
             past_lo=1024, past_hi=8191),
        # The same over E4M3 pages of 16: eight pages in a tile.
        dict(heads, op="attention", name="paged_fp8_decode_64", format="fp8", batch=64, tokens=1, page_size=16,
             past_lo=1024, past_hi=8191),
        # Single tokens over long NVFP4 caches, pages of 32.
        dict(heads, op="attention", name="paged_nvfp4_long_decode", format="nvfp4", batch=8, tokens=1, page_size=32,
             past_lo=32767, past_hi=32767),
        # A tree of five drafted tokens for 37 sequences, narrow heads.
        dict(op="attention", name="paged_fp8_drafts_ragged", format="fp8", batch=37, tokens=5, page_size=32, kv_heads=8,
             q_heads=32, head_dim=64, past_lo=90, past_hi=6003),
        # One sequence, a chain of four drafted tokens, a small vocabulary.
        dict(op="verify", name="verify_chain_1", batch=1, tokens=5, vocab=32000, tree=False, sampled=True),
        # 48 trees whose candidates came without probabilities, an odd vocabulary.
        dict(op="verify", name="verify_given_tree_48", batch=48, tokens=13, vocab=49999, tree=True, sampled=False),
        # 64 trees drawn from a draft model over a large vocabulary.
        dict(op="verify", name="verify_sampled_tree_64", batch=64, tokens=8, vocab=128000, tree=True, sampled=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    op = rng.choice(("pages", "rows", "attention", "attention", "verify"))
    batch = _log(rng, 1, 64)
    if op == "verify":
        vocab = _log(rng, 1000, 128000)
        tokens = rng.randint(1, 16)
        while batch * tokens * vocab > 65_000_000:
            batch = max(1, batch // 2)
        return dict(op=op, batch=batch, tokens=tokens, vocab=vocab, tree=rng.random() < 0.6,
                    sampled=rng.random() < 0.6)
    size = rng.choice((16, 16, 32, 48, 64, 128))
    if op == "pages":
        hi = _log(rng, 1, 8000)
        return dict(op=op, batch=batch, tokens=_log(rng, 1, 2048), page_size=size, past_lo=rng.randint(hi // 4, hi),
                    past_hi=hi, short=rng.random() < 0.3)
    hkv, d = rng.randint(1, 8), rng.choice((64, 96, 128, 128, 256))
    hi = _log(rng, 1, 32700)
    while batch * hkv * hi * d > 200_000_000:
        hi = hi // 2
    lo = hi if rng.random() < 0.3 else rng.randint(hi // 4, hi)
    case = dict(op=op, format=rng.choice(("bf16", "fp8", "nvfp4")), kv_heads=hkv, head_dim=d, batch=batch,
                page_size=size, past_lo=lo, past_hi=hi)
    if op == "rows":
        tokens = max(1, min(_log(rng, 1, 2048), hi))
        while batch * hkv * tokens * d > 8_000_000:
            tokens = max(1, tokens // 2)
        return dict(case, tokens=tokens, window=rng.randint(1, lo + tokens))
    tokens, group = rng.choice((1, 1, rng.randint(2, 8))), rng.choice((1, 2, 4, 8))
    while batch * hkv * group * tokens * hi * d > 1_000_000_000 and tokens * group > 1:
        tokens, group = (tokens // 2, group) if tokens > 1 else (tokens, group // 2)
    return dict(case, tokens=tokens, q_heads=hkv * group)


def _pasts(c):
    """Ragged past lengths in [past_lo, past_hi], the same for every seed."""
    span = c["past_hi"] - c["past_lo"] + 1
    return [c["past_lo"] + (b * 7919 + 13) % span for b in range(c["batch"])]


def _pages_for(c, length):
    return -(-length // c["page_size"])


def _row_bytes(c):
    d = c["head_dim"]
    return {"bf16": 2 * d, "fp8": d + 4, "nvfp4": d // 2 + d // 16 + 4}[c["format"]]


def work(c):
    b, t = c["batch"], c["tokens"]
    if c["op"] == "pages":
        new = sum(_pages_for(c, p + t) - _pages_for(c, p) for p in _pasts(c))
        # lengths and held counts in and out, slots out, the new pages' numbers from the stack to the table and back
        return {"bytes": 8 * b * t + 48 * b + 16 * new, "flops": 2 * b * t}
    if c["op"] == "verify":
        # the row that the next token is drawn from (and the draft's beside it), and the candidates' own probabilities
        rows = 2 if c["sampled"] else 1
        return {"bytes": 4 * b * c["vocab"] * rows + b * t * (4 * rows + 28), "flops": 3 * b * c["vocab"] * rows}
    d, hkv = c["head_dim"], c["kv_heads"]
    if c["op"] == "rows":
        rows = b * hkv * t
        new = 2 * rows * (2 * d + _row_bytes(c))  # read in BF16, written as stored
        old = b * hkv * max(0, c["window"] - t)  # rows of the window that were there before
        read = 2 * old * _row_bytes(c) + 2 * b * hkv * c["window"] * 2 * d
        return {"bytes": new + read + 8 * b * (t + c["window"]), "flops": 4 * rows * d + 4 * b * hkv * c["window"] * d}
    keys = sum(p + t for p in _pasts(c))
    q = b * t * c["q_heads"] * d
    table = 4 * sum(_pages_for(c, p + t) for p in _pasts(c))
    return {"bytes": 2 * keys * hkv * _row_bytes(c) + 4 * q + b * t * t + 8 * b + table,
            "flops": 4 * t * c["q_heads"] * d * keys}


# ------------------------------------------------------------------ inputs
def _parents(batch, tokens, tree, g):
    """Parents [B, T] of random trees (or of chains) in topological order, -1 at the root."""
    t = torch.arange(tokens)
    parents = (torch.rand((batch, tokens), generator=g) * t).long() if tree else (t - 1).expand(batch, tokens).clone()
    parents[:, 0] = -1
    return parents


def _tree_mask(batch, tokens, g):
    """Ancestor masks [B, T, T] of random trees."""
    parents = _parents(batch, tokens, True, g)
    mask = torch.zeros((batch, tokens, tokens), dtype=torch.bool)
    rows = torch.arange(batch)
    for t in range(tokens):
        if t:
            mask[:, t] = mask[rows, parents[:, t]]
        mask[:, t, t] = True
    return mask


def _rows(shape, g, spread):
    """K or V rows as a layer makes them: some channels larger, rows of different size."""
    d = shape[-1]
    x = torch.randn(shape, generator=g, device=_DEV)
    x *= 1.0 + 3.0 * (torch.rand((d,), generator=g, device=_DEV) < 0.06)
    if spread:
        x *= torch.exp(0.7 * torch.randn(shape[:-1] + (1,), generator=g, device=_DEV))
    return x.to(torch.bfloat16)


def _filled_pages(c, pages, g):
    """A pool of pages, all of them holding rows (of these sequences or left by earlier ones)."""
    d, shape = c["head_dim"], (pages, c["kv_heads"], c["page_size"], c["head_dim"])
    width = {"bf16": d, "fp8": d, "nvfp4": d // 2}[c["format"]]
    kind = torch.bfloat16 if c["format"] == "bf16" else torch.uint8
    step, fields = max(1, 2 ** 25 // math.prod(shape[1:])), {}
    for n in "kv":
        codes = torch.empty(shape[:3] + (width,), dtype=kind, device=_DEV)
        gamma = beta = None
        if c["format"] != "bf16":
            gamma = torch.empty(shape[:3], dtype=torch.float32, device=_DEV)
        if c["format"] == "nvfp4":
            beta = torch.empty(shape[:3] + (d // 16,), dtype=torch.uint8, device=_DEV)
        for a in range(0, pages, step):
            some = _rows((min(step, pages - a),) + shape[1:], g, n == "v")
            for to, x in zip((codes, gamma, beta), _stored_form(c["format"], some)):
                if to is not None:
                    to[a:a + step] = x
        fields.update({n + "_codes": codes, n + "_row_scales": gamma, n + "_block_scales": beta})
    return SimpleNamespace(format=c["format"], head_dim=d, page_size=c["page_size"], **fields)


def _block_table(c, lengths, pages, host):
    """A table that gives the sequences' lengths pages of the pool in no order, -1 behind them; and the pages left."""
    order = torch.randperm(pages, generator=host).to(torch.int32)
    table = torch.full((c["batch"], max(1, _pages_for(c, c["past_hi"] + c["tokens"]))), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(_pages_for(c, length) for length in lengths):
        table[b, :n] = order[at:at + n]
        at += n
    return table, order[at:]


def prepare(c, seed):
    g = torch.Generator(device=_DEV).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    b, t = c["batch"], c["tokens"]
    s = SimpleNamespace(case=dict(c), op=c["op"])
    if c["op"] == "verify":
        v = c["vocab"]
        parents = _parents(b, t, c["tree"], host)
        s.parents = parents.to(_DEV)
        logits = 2.5 * torch.randn((b, t, v), generator=g, device=_DEV)
        s.target = torch.softmax(logits, dim=-1)
        draft = torch.softmax(logits.add_(0.7 * torch.randn((b, t, v), generator=g, device=_DEV)), dim=-1)
        del logits
        s.tokens = torch.zeros((b, t), dtype=torch.int64, device=_DEV)
        rows = torch.arange(b, device=_DEV)
        for i in range(1, t):
            q = draft[rows, s.parents[:, i]]
            if c["sampled"]:  # drawn from the draft's row: the least of independent exponential times
                s.tokens[:, i] = torch.empty_like(q).exponential_(generator=g).div_(q).argmin(dim=-1)
            else:  # a parent's children are its most likely candidates
                rank = (parents[:, :i] == parents[:, i:i + 1]).sum(dim=1, keepdim=True).to(_DEV)
                s.tokens[:, i] = q.topk(t, dim=-1).indices.gather(1, rank)[:, 0]
        s.draft = draft if c["sampled"] else None
        s.uniforms = torch.rand((b, t), generator=g, device=_DEV)
        return s
    pasts = _pasts(c)
    s.past_lengths = torch.tensor(pasts, dtype=torch.int64, device=_DEV)
    s.max_past = max(pasts)
    if c["op"] == "pages":
        need = [_pages_for(c, p + t) for p in pasts]
        held = [_pages_for(c, p) for p in pasts]
        left = sum(need) - sum(held)
        pages = sum(held) + (left * 3 // 4 if c["short"] else left + 5)
        table, free = _block_table(c, pasts, pages, host)
        free_pages = torch.zeros((max(1, pages),), dtype=torch.int32)
        free_pages[:free.numel()] = free
        s.table = SimpleNamespace(pages=table.to(_DEV), held=torch.tensor(held, dtype=torch.int64, device=_DEV),
                                  free_pages=free_pages.to(_DEV),
                                  free_count=torch.tensor([free.numel()], dtype=torch.int64, device=_DEV),
                                  page_size=c["page_size"])
        return s
    pages = sum(_pages_for(c, p + t) for p in pasts) + 3
    s.block_table = _block_table(c, [p + t for p in pasts], pages, host)[0].to(_DEV)
    s.cache = _filled_pages(c, pages, g)
    d, hkv = c["head_dim"], c["kv_heads"]
    if c["op"] == "rows":
        s.new_k = _rows((b, t, hkv, d), g, False)
        s.new_v = _rows((b, t, hkv, d), g, True)
        s.slots = _slots(s.block_table, s.past_lengths, t, c["page_size"])
        s.back = _slots(s.block_table, s.past_lengths + t - c["window"], c["window"], c["page_size"])
        return s
    s.q = _rows((b, t, c["q_heads"], d), g, False)
    s.mask = _tree_mask(b, t, host).to(_DEV)
    return s


def _slots(table, first, n, size):
    at = first[:, None] + torch.arange(n, device=table.device)
    return table.gather(1, at // size).to(torch.int64) * size + at % size


# ------------------------------------------------------------------ plain forms (32 bits; probabilities 64)
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


def _stored_form(fmt, rows):
    """(codes, row scales or None, block scales or None) of BF16 rows [..., D]."""
    if fmt == "bf16":
        return rows, None, None
    x = rows.to(torch.float32)
    amax = x.abs().amax(dim=-1)
    top = 448.0 if fmt == "fp8" else 2688.0
    enc = torch.where(amax == 0, torch.ones_like(amax), ((1.0 / amax) * top).clamp(max=_F32_MAX))
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
    """FP32 rows of stored ones."""
    if fmt == "bf16":
        return codes.to(torch.float32)
    if fmt == "fp8":
        return _e4m3_values(codes) * gamma[..., None]
    return (_e2m1_values(codes).unflatten(-1, (-1, 16)) * _e4m3_values(beta)[..., None]).flatten(-2) * gamma[..., None]


def _stored(cache, n):
    return getattr(cache, n + "_codes"), getattr(cache, n + "_row_scales"), getattr(cache, n + "_block_scales")


def _plain_pages(s):
    c, table = s.case, s.table
    t, size = c["tokens"], c["page_size"]
    pages, held, free, count = table.pages, table.held, table.free_pages, table.free_count
    n, most = free.numel(), pages.shape[1]
    column = torch.arange(most, device=_DEV)
    # reserve
    wanted = (s.past_lengths + t + size - 1) // size
    need = (wanted - held).clamp(min=0)
    upto = need.cumsum(0)
    served = (need == 0) | (upto <= count)
    granted = torch.where(served, t, 0)
    new = (column >= held[:, None]) & (column < torch.where(served, wanted, held)[:, None])
    rank = (upto - need)[:, None] + column - held[:, None]
    taken = free[(count - 1 - rank).clamp(0, n - 1)]
    pages.copy_(torch.where(new, taken, pages))
    at = s.past_lengths[:, None] + torch.arange(t, device=_DEV)
    slots = pages.gather(1, at // size).to(torch.int64) * size + at % size
    slots = torch.where(served[:, None], slots, -1)
    held.copy_(torch.where(served, torch.maximum(held, wanted), held))
    count.copy_(count - torch.where(served, need, 0).sum())
    # give back what stands past the committed lengths
    keep = torch.minimum((s.past_lengths + size - 1) // size, held)
    back = (column >= keep[:, None]) & (column < held[:, None])
    order = back.flatten().flip(0).to(torch.int64).cumsum(0).flip(0).view(back.shape)  # last page of the last one first
    to = torch.where(back, count + order - 1, n)
    stack = torch.cat((free, free[:1]))
    stack.scatter_(0, to.flatten(), pages.flatten())
    free.copy_(stack[:n])
    count.copy_(count + back.sum())
    pages.copy_(torch.where(back, -1, pages))
    held.copy_(keep)
    return slots, granted, pages, held, free, count


def _plain_rows(s):
    c = s.case
    size = c["page_size"]
    head = torch.arange(c["kv_heads"], device=_DEV)[None, :, None]
    to, back = s.slots[:, None], s.back[:, None]
    out = []
    for n, new in (("k", s.new_k), ("v", s.new_v)):
        stored = _stored(s.cache, n)
        for store, x in zip(stored, _stored_form(c["format"], new.transpose(1, 2))):
            if store is not None:
                store[to // size, head, to % size] = x
        rows = [None if x is None else x[back // size, head, back % size] for x in stored]
        out.append(_values(c["format"], *rows).to(torch.bfloat16))
    return tuple(out)


def _plain_attention(s):
    c = s.case
    b, t, d, hkv = c["batch"], c["tokens"], c["head_dim"], c["kv_heads"]
    group, length = c["q_heads"] // hkv, s.max_past + t
    table = s.block_table.clamp(min=0).to(torch.int64)
    k, v = (_values(c["format"], *(None if x is None else x[table].transpose(1, 2).flatten(2, 3)[:, :, :length]
                                   for x in _stored(s.cache, n))) for n in "kv")
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


def _plain_verify(s):
    b, t = s.tokens.shape
    rows = torch.arange(b, device=_DEV)
    u = s.uniforms.double()
    path = torch.full((b, t), -1, dtype=torch.int64, device=_DEV)
    path[:, 0] = 0
    count = torch.ones((b,), dtype=torch.int64, device=_DEV)
    node = torch.zeros((b,), dtype=torch.int64, device=_DEV)
    left, total = s.target[:, 0].double(), torch.ones((b,), dtype=torch.float64, device=_DEV)
    some = torch.ones((b,), dtype=torch.bool, device=_DEV)
    column = torch.arange(s.target.shape[2], device=_DEV)
    for i in range(1, t):
        child = (s.parents[:, i] == node) & some
        x = s.tokens[:, i]
        if s.draft is None:
            q = (column == x[:, None]).double()
        else:
            q = s.draft[rows, node].double()
        taken = child & (u[:, i] * q[rows, x] * total < left[rows, x])
        missed = child & ~taken
        path[rows, count] = torch.where(taken, i, path[rows, count.clamp(max=t - 1)])
        count += taken
        node = torch.where(taken, i, node)
        if s.draft is None:
            rest = torch.where(q > 0, 0.0, left)
        else:
            rest = (left - total[:, None] * q).clamp(min=0)
        weight = rest.sum(dim=-1)
        some &= ~(missed & (weight == 0))
        fresh = taken | (missed & (weight == 0))  # the row of the new node, or the old one's again
        left = torch.where(fresh[:, None], s.target[rows, node].double(), torch.where(missed[:, None], rest, left))
        total = torch.where(fresh, 1.0, torch.where(missed, weight, total))
    upto = left.cumsum(dim=-1)
    above = upto > u[:, :1] * upto[:, -1:]
    last = (left > 0).to(torch.int64).mul(column + 1).amax(dim=-1) - 1
    return path, count, torch.where(above.any(dim=-1), above.to(torch.int8).argmax(dim=-1), last)


def run(s):
    if own:
        ops = _primitives()
        if s.op == "pages":
            slots, granted = ops.cuda_reserve_pages_(s.table, s.past_lengths, s.case["tokens"])
            ops.cuda_release_pages_(s.table, s.past_lengths)
            t = s.table
            return slots, granted, t.pages, t.held, t.free_pages, t.free_count
        if s.op == "rows":
            ops.cuda_paged_kv_append_(s.cache, s.new_k, s.new_v, s.slots)
            return ops.cuda_paged_kv_read(s.cache, s.back)
        if s.op == "attention":
            return ops.cuda_paged_attention(s.q, s.cache, s.block_table, tree_mask=s.mask,
                                            past_lengths=s.past_lengths, max_past_length=s.max_past)
        return ops.cuda_verify_drafted(s.target, s.tokens, s.uniforms, draft_probs=s.draft, parents=s.parents)
    return {"pages": _plain_pages, "rows": _plain_rows, "attention": _plain_attention, "verify": _plain_verify}[s.op](s)


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


def _r32(x):
    """Rounded to FP32."""
    return x.to(torch.float32).double()


def _exact_form(fmt, rows):
    """The values that rows are stored as.

    The formats define their scales and scaled elements as single operations,
    each rounded to FP32 (BF16 rows meet the borders of 4 and 8 bits exactly,
    so what a tie becomes depends on them); codes are nearest ones, ties to even.
    """
    x = rows.double()
    if fmt == "bf16":
        return x
    amax = x.abs().amax(dim=-1, keepdim=True)
    top = 448.0 if fmt == "fp8" else 2688.0
    enc = torch.where(amax > 0, _r32(_r32(1.0 / amax) * top).clamp(max=_F32_MAX), 1.0)
    gamma = _r32(amax * _r32(torch.full((), 1.0 / top, dtype=torch.float64, device=_DEV)))
    if fmt == "fp8":
        return x.sign() * _nearest(_r32(x.abs() * enc), _E4M3) * gamma
    blocks, enc, gamma = x.unflatten(-1, (-1, 16)), enc[..., None], gamma[..., None]
    sixth = _r32(torch.full((), 1.0 / 6.0, dtype=torch.float64, device=_DEV))
    beta = _nearest(_r32(blocks.abs().amax(dim=-1, keepdim=True) * _r32(enc * sixth)), _E4M3)
    factor = _r32(1.0 / _r32(beta * _r32(1.0 / enc))).clamp(max=_F32_MAX)
    codes = _nearest(_r32(blocks.abs() * torch.where(beta > 0, factor, 0.0)), _E2M1)
    return (blocks.sign() * codes * beta * gamma).flatten(-2)


def _exact_values(fmt, codes, gamma, beta):
    if fmt == "bf16":
        return codes.double()
    if fmt == "fp8":
        table = torch.tensor(_E4M3 + (math.nan,), dtype=torch.float64, device=codes.device)
        v = table[(codes & 127).long()] * torch.where(codes > 127, -1.0, 1.0)
    else:
        table = torch.tensor(_E2M1 + tuple(-x for x in _E2M1), dtype=torch.float64, device=codes.device)
        scale = torch.tensor(_E4M3 + (math.nan,), dtype=torch.float64, device=codes.device)[beta.long()]
        v = torch.stack((table[(codes & 15).long()], table[(codes >> 4).long()]), dim=-1).flatten(-2)
        v = (v.unflatten(-1, (-1, 16)) * scale[..., None]).flatten(-2)
    return v * gamma.double()[..., None]


def _exact_sequence(s, n, b, first, length):
    """Rows [first, first + length) of sequence b, all heads [Hkv, length, D], as they are stored."""
    size, out = s.case["page_size"], []
    table = s.block_table[b].tolist()
    for x in _stored(s.cache, n):
        if x is None:
            out.append(None)
            continue
        parts = [x[table[i]] for i in range(first // size, (first + length - 1) // size + 1)]
        out.append(torch.cat(parts, dim=1)[:, first % size:first % size + length])
    return _exact_values(s.case["format"], *out)


def _exact_pages(s):
    c, size = s.case, s.case["page_size"]
    pages, held = s.table.pages.tolist(), s.table.held.tolist()
    n = int(s.table.free_count)
    store = s.table.free_pages.tolist()
    stack, slots, granted, out_of_pages = store[:n], [], [], False
    for b, past in enumerate(_pasts(c)):
        wanted = _pages_for(c, past + c["tokens"])
        need = max(0, wanted - held[b])
        out_of_pages |= need > len(stack)
        if need and out_of_pages:
            slots.append([-1] * c["tokens"])
            granted.append(0)
            continue
        for i in range(held[b], wanted):
            pages[b][i] = stack.pop()
        held[b] = max(held[b], wanted)
        granted.append(c["tokens"])
        slots.append([pages[b][p // size] * size + p % size for p in range(past, past + c["tokens"])])
    for b, past in reversed(list(enumerate(_pasts(c)))):
        while held[b] > _pages_for(c, past):
            held[b] -= 1
            stack.append(pages[b][held[b]])
            pages[b][held[b]] = -1
    store[:len(stack)] = stack
    return tuple(torch.tensor(x, dtype=kind, device=_DEV) for x, kind in (
        (slots, torch.int64), (granted, torch.int64), (pages, torch.int32), (held, torch.int64), (store, torch.int32),
        ([len(stack)], torch.int64)))


def _exact_verify(s):
    paths, counts, tokens = [], [], []
    most = s.tokens.shape[1]
    for b in range(s.tokens.shape[0]):
        parents, drafted, u = s.parents[b].tolist(), s.tokens[b].tolist(), s.uniforms[b].double().tolist()
        path = [0]
        while True:
            node, taken = path[-1], None
            p = s.target[b, node].double()
            rest = p.clone()
            for child in (i for i in range(1, most) if parents[i] == node):
                x = drafted[child]
                if s.draft is None:
                    q = torch.zeros_like(p)
                    q[x] = 1.0
                else:
                    q = s.draft[b, node].double()
                if u[child] * float(q[x]) < float(rest[x]):
                    taken = child
                    break
                if s.draft is None:
                    rest[x] = 0.0
                else:
                    rest = (rest - q).clamp(min=0)
                if float(rest.sum()) == 0.0:
                    rest = p
                    break
                rest = rest / rest.sum()
            if taken is None:
                break
            path.append(taken)
        upto = rest.cumsum(0)
        above = torch.nonzero(upto > u[0] * float(upto[-1]))
        tokens.append(int(above[0]) if len(above) else int(torch.nonzero(rest > 0)[-1]))
        counts.append(len(path))
        paths.append(path + [-1] * (most - len(path)))
    return tuple(torch.tensor(x, dtype=torch.int64, device=_DEV) for x in (paths, counts, tokens))


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "pages":
        return _exact_pages(s)
    if c["op"] == "verify":
        return _exact_verify(s)
    b, t, d, hkv = c["batch"], c["tokens"], c["head_dim"], c["kv_heads"]
    pasts = _pasts(c)
    if c["op"] == "rows":
        out = []
        for n, new in (("k", s.new_k), ("v", s.new_v)):
            rows = torch.zeros((b, hkv, c["window"], d), dtype=torch.float64, device=_DEV)
            for i, past in enumerate(pasts):
                a = past + t - c["window"]
                rows[i] = _exact_sequence(s, n, i, a, c["window"])
                fresh = _exact_form(c["format"], new[i].transpose(0, 1))
                from_ = max(past, a)
                rows[i, :, from_ - a:] = fresh[:, from_ - past:]
            out.append(rows)
        return tuple(out)
    ctx = torch.zeros((b, t, c["q_heads"], d), dtype=torch.float64, device=_DEV)
    group = c["q_heads"] // hkv
    for i, past in enumerate(pasts):
        seen = torch.cat((torch.ones((t, past), dtype=torch.bool, device=_DEV), s.mask[i]), dim=1)
        k, v = (_exact_sequence(s, n, i, 0, past + t) for n in "kv")
        for j in range(c["q_heads"]):
            w = (s.q[i, :, j].double() @ k[j // group].T / math.sqrt(d)).masked_fill(~seen, -math.inf)
            ctx[i, :, j] = torch.softmax(w, dim=-1) @ v[j // group]
    return ctx
