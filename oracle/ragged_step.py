"""64-bit definitions of the attention step of a ragged batch: slot maps, head
norms with rotation and cache write, attention (no counterpart in the
reference). Plain loops over sequences and heads; tests only."""

from __future__ import annotations

import math

import torch


def slot_mapping(starts, lens, tables, block, num_tokens, free=None):
    """(positions, slots, tables, number of new blocks) as lists; ``tables`` is a
    list of lists and is not changed."""
    tables = [list(row) for row in tables]
    positions, slots = [-1] * num_tokens, [-1] * num_tokens
    taken = 0
    for s, length in enumerate(lens):
        n = starts[s + 1] - starts[s]
        if n == 0:
            continue
        cached = max(length - n, 0)
        held, need = -(-cached // block), -(-max(length, 0) // block)
        for i in range(n):
            pos = length - n + i
            if pos < 0:
                continue
            positions[starts[s] + i] = pos
            blk = pos // block
            page = -1
            if blk < len(tables[s]):
                if blk < held or free is None:
                    page = tables[s][blk]
                elif taken + blk - held < len(free):
                    page = tables[s][blk] = free[taken + blk - held]
            if page >= 0:
                slots[starts[s] + i] = page * block + pos % block
        taken += max(need - held, 0)
    return positions, slots, tables, taken


def norm_rotate(x, weight, eps, positions, table, neox):
    """x [tokens, heads, head_size]: normed and rotated, float64."""
    x = x.double()
    x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    half = table.shape[1] // 2
    out = x.clone()
    for t, pos in enumerate(positions.tolist()):
        cos, sin = table[pos, :half].double(), table[pos, half:].double()
        for i in range(half):
            a, b = (i, i + half) if neox else (2 * i, 2 * i + 1)
            out[t, :, a] = x[t, :, a] * cos[i] - x[t, :, b] * sin[i]
            out[t, :, b] = x[t, :, b] * cos[i] + x[t, :, a] * sin[i]
    return out


def visible(pos, length, window, prefix):
    """Which of the keys 0 .. length - 1 the token at position pos sees."""
    j = torch.arange(length)
    sees = j <= pos
    if window:
        sees &= j > pos - window
    return sees | (j < prefix)


def attention(q, k_cache, v_cache, tables, lens, starts, scale, window=0, softcap=0.0, slopes=None, prefix=None,
              k_scale=1.0, v_scale=1.0):
    """(out, sum of the weights times |v|), float64 on q's device; rows that no
    sequence owns are zeros. Hidden keys and values are taken out before any
    product."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    block = k_cache.shape[1]
    group = q.shape[1] // k_cache.shape[2]
    for s, length in enumerate(lens):
        n = starts[s + 1] - starts[s]
        pre = min(prefix[s], length) if prefix is not None else 0
        seen = [visible(length - n + i, length, window, pre) for i in range(n)]
        if n == 0 or length == 0:
            continue
        seen = torch.stack(seen).to(q.device)
        used = seen.any(0)
        j = torch.arange(length, device=q.device)[used]
        seen = seen[:, used]
        page = tables[s].long()[j // block]
        kk = k_cache.view(torch.uint8)[page, j % block].view(k_cache.dtype) if k_cache.element_size() == 1 \
            else k_cache[page, j % block]
        vv = v_cache.view(torch.uint8)[page, j % block].view(v_cache.dtype) if v_cache.element_size() == 1 \
            else v_cache[page, j % block]
        kk, vv = kk.double() * k_scale, vv.double() * v_scale
        away = (torch.arange(length - n, length, device=q.device)[:, None] - j[None]).abs()
        for h in range(q.shape[1]):
            x = q[starts[s]:starts[s + 1], h].double() @ kk[:, h // group].t().contiguous() * scale
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            if slopes is not None:
                x = x - slopes[h].double() * away
            x = torch.where(seen, x, torch.tensor(-math.inf, dtype=torch.float64, device=q.device))
            p = torch.softmax(x, -1)
            p = torch.where(seen, p, torch.zeros_like(p))
            v = vv[:, h // group]
            hidden_bad = not bool(torch.isfinite(v).all())
            if hidden_bad:  # a product with a hidden infinity is no product
                y = torch.stack([p[i, seen[i]] @ v[seen[i]] for i in range(n)])
                a = torch.stack([p[i, seen[i]] @ v[seen[i]].abs() for i in range(n)])
            else:
                y, a = p @ v, p @ v.abs()
            any_seen = seen.any(1)
            out[starts[s]:starts[s + 1], h] = torch.where(any_seen[:, None], y, torch.zeros_like(y))
            size[starts[s]:starts[s + 1], h] = torch.where(any_seen[:, None], a, torch.zeros_like(a))
    return out, size
