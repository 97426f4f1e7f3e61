"""Plain 64-bit restatements of the paged KV cache's operators and of the
verification of drafted tokens, sequence by sequence, on the CPU.  The tests'
oracle; written from the definitions."""

from __future__ import annotations

import math

import numpy as np
import torch

import draft_reference as ref


# ------------------------------------------------------------------ pages
def reserve(pages, held, stack, page_size, pool, pasts, counts, tokens):
    """New (pages, held, stack) as lists, slots [B][T], granted [B]."""
    pages, held, stack = [list(r) for r in pages], list(held), list(stack)
    slots, granted, out = [], [], False
    for b, past in enumerate(pasts):
        n = max(0, min(int(counts[b]), tokens)) if counts is not None else tokens
        if past < 0 or past + n > len(pages[b]) * page_size:
            n = 0
        need = max(0, -(-(past + n) // page_size) - held[b]) if n else 0
        out |= need > len(stack)
        if need and out:
            n = need = 0
        for _ in range(need):
            pages[b][held[b]] = stack.pop()
            held[b] += 1
        granted.append(n)
        row = []
        for t in range(tokens):
            page = pages[b][(past + t) // page_size] if t < n else -1
            row.append(page * page_size + (past + t) % page_size if 0 <= page < pool else -1)
        slots.append(row)
    return pages, held, stack, slots, granted


def release(pages, held, stack, page_size, pool, lengths):
    pages, held, stack = [list(r) for r in pages], list(held), list(stack)
    for b in reversed(range(len(held))):
        while held[b] > max(0, -(-lengths[b] // page_size)):
            held[b] -= 1
            if 0 <= pages[b][held[b]] < pool and len(stack) < pool:
                stack.append(pages[b][held[b]])
            pages[b][held[b]] = -1
    return pages, held, stack


def pool_values(cache):
    """FP64 K and V [N, Hkv, S, D] of a pool."""
    out = []
    for n in "kv":
        fields = [getattr(cache, f"{n}_{f}") for f in ("codes", "row_scales", "block_scales")]
        if cache.format == "bf16":
            out.append(fields[0].cpu().double())
        else:
            out.append(ref.stored_values(cache.format, *(None if x is None else x.cpu().numpy() for x in fields)))
    return tuple(out)


def attention(q, cache, table, pasts, mask=None, counts=None):
    """FP64 context, and sum_j p_j |v_j|; keys a query does not see are left out before any arithmetic."""
    q = q.cpu().double()
    k, v = pool_values(cache)
    b, t, hq, d = q.shape
    n, hkv, size = k.shape[:3]
    table = table.cpu()
    ctx, weight = torch.zeros_like(q), torch.zeros_like(q)
    for i in range(b):
        live = t if counts is None else max(0, min(int(counts[i]), t))
        past = max(0, int(pasts[i]))
        for u in range(live):
            row = torch.arange(t) <= u if mask is None else (mask if mask.ndim == 2 else mask[i])[u].cpu().bool()
            seen = [j for j in list(range(past)) + [past + int(w) for w in row.nonzero().flatten() if w < live]
                    if j // size < table.shape[1] and 0 <= int(table[i, j // size]) < n]
            if not seen:
                continue
            seen = torch.tensor(seen)
            page, at = table[i, seen // size].long(), seen % size
            for h in range(hq):
                kk, vv = (x[page, h // (hq // hkv), at] for x in (k, v))
                w = torch.softmax(kk @ q[i, u, h] / math.sqrt(d), 0)
                ctx[i, u, h], weight[i, u, h] = w @ vv, w @ vv.abs()
    return ctx, weight


# ------------------------------------------------------------------ verification
def clean(x):
    x = np.asarray(x, dtype=np.float64)
    return np.where((x > 0) & np.isfinite(x), x, 0.0)


def verify(target, tokens, uniforms, draft=None, parents=None, counts=None):
    """(path, counts, next tokens) as lists."""
    b, t, v = target.shape
    paths, accepted, nexts = [], [], []
    for i in range(b):
        live = t if counts is None else max(0, min(int(counts[i]), t))
        if live == 0:
            paths.append([-1] * t)
            accepted.append(0)
            nexts.append(-1)
            continue
        up = [n - 1 for n in range(t)] if parents is None else [
            int(x) for x in (parents if parents.ndim == 1 else parents[i])]
        u = [float(x) for x in uniforms[i]]
        path = [0]
        while True:
            node = path[-1]
            p = clean(target[i, node].numpy())
            r, s, taken = p, 1.0, None
            for c in range(node + 1, live):
                x = int(tokens[i, c])
                if up[c] != node or not 0 <= x < v:
                    continue
                if draft is None:
                    q = np.zeros(v)
                    q[x] = 1.0
                else:
                    q = clean(draft[i, node].numpy())
                if u[c] * q[x] * s < r[x]:
                    taken = c
                    break
                r = np.where(q > 0, 0.0, r) if draft is None else np.maximum(r - s * q, 0.0)
                s = math.fsum(r)
                if s == 0.0:
                    r = p
                    break
            if taken is None:
                break
            path.append(taken)
        upto = np.cumsum(r)
        above = np.flatnonzero(upto > u[0] * math.fsum(r))
        some = np.flatnonzero(r > 0)
        above = above[np.isin(above, some)]
        nexts.append(int(above[0]) if len(above) else (int(some[-1]) if len(some) else -1))
        accepted.append(len(path))
        paths.append(path + [-1] * (t - len(path)))
    return paths, accepted, nexts
