"""Restatements of the paged-cache operators from their definitions: whole numbers
in plain Python, probabilities in float64."""

from __future__ import annotations

import math

import torch

from . import lm_oracle


def slots(table, held, new, free, count, page, tokens):
    """(slots, positions, q_starts, kv_lens, free_count, table) as lists."""
    table = [list(r) for r in table]
    count = min(max(count, 0), len(free))
    out, positions, starts, lens = [-1] * tokens, [0] * tokens, [0], []
    asked = taken = total = 0
    for b, (h, k) in enumerate(zip(held, new)):
        sane = 0 <= h <= 1 << 30 and 0 <= k <= 1 << 30
        h, k = h if sane else 0, min(max(k, 0), 1 << 30)
        have, want = -(-h // page), -(-(h + k) // page)
        sane = sane and want <= len(table[b])
        at, total = total, total + k
        need = want - have if sane else 0
        asked += need
        ok = sane and total <= tokens and (need == 0 or asked <= count)
        if ok:
            for j in range(need):
                table[b][have + j] = free[count - 1 - (asked - need) - j]
            taken += need
        for i in range(min(k, max(0, tokens - at))):
            positions[at + i] = h + i
            if ok:
                out[at + i] = table[b][(h + i) // page] * page + (h + i) % page
        starts.append(min(tokens, total))
        lens.append(h + k if ok else 0)
    return out, positions, starts, lens, count - taken, table


def release(table, held, kept, free, count, page):
    """(free_count, free_pages)"""
    free = list(free)
    count = min(max(count, 0), len(free))
    for row, h, k in zip(table, held, kept):
        h = h if 0 <= h <= 1 << 30 else 0
        k = min(max(k, 0), h)
        for j in reversed(range(-(-k // page), min(-(-h // page), len(row)))):
            if count < len(free):
                free[count] = row[j]
                count += 1
    return count, free


def gather(cache, row, n):
    """The first n keys of a sequence: (Hk, n, D)."""
    page = cache.shape[2]
    pages = row[: -(-n // page)].long()
    return cache[pages].transpose(0, 1).flatten(1, 2)[:, :n]


def attention(q, k_cache, v_cache, table, kv_lens, q_starts, scale=None):
    """(out, bound, lse, bound) over all rows of ``q`` (N, H, D); lists of whole numbers for lengths and starts."""
    n, h, d = q.shape
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full((n, h), -math.inf, dtype=torch.float64, device=q.device)
    err_o, err_l = torch.zeros_like(out), torch.zeros((n, h), dtype=torch.float64, device=q.device)
    for b, total in enumerate(kv_lens):
        rows = slice(q_starts[b], q_starts[b + 1])
        if rows.start == rows.stop or total == 0:
            continue
        k, v = (gather(c, table[b], total)[None] for c in (k_cache, v_cache))
        res = lm_oracle.attention(q[rows].transpose(0, 1)[None], k, v, scale=scale)
        out[rows], err_o[rows] = (x[0].transpose(0, 1) for x in res["out"])
        lse[rows], err_l[rows] = (x[0].transpose(0, 1) for x in res["lse"])
    return (out, err_o), (lse, err_l)


def verify(logits, ids, q_starts, uniforms, draft_probs=None, temperature=1.0):
    """(tokens, counts) as lists."""
    x, u = logits.double().cpu(), uniforms.double().cpu()
    q = None if draft_probs is None else draft_probs.double().cpu()
    ids = ids.tolist()
    v = x.shape[1]
    tokens, counts = [-1] * len(ids), []
    for lo, hi in zip(q_starts, q_starts[1:]):
        n = 0
        for r in range(lo, hi):
            row = x[r]
            top = row.max()
            if torch.isnan(row).any() or top == math.inf or top == -math.inf:
                p = None
            elif temperature == 0:
                p = torch.zeros(v, dtype=torch.float64)
                p[int((row == top).nonzero()[0])] = 1
            else:
                p = torch.exp((row - top) / temperature)
                p = p / p.sum()
            weight = p
            if r + 1 < hi:
                d = ids[r + 1]
                if temperature == 0 or q is None:
                    qr = torch.zeros(v, dtype=torch.float64)
                    if 0 <= d < v:
                        qr[d] = 1
                else:
                    qr = q[r]
                if p is not None and 0 <= d < v and float(u[r, 0] * qr[d]) < float(p[d]):
                    tokens[r] = d
                    n += 1
                    continue
                if p is not None:
                    weight = (p - qr).clamp(min=0)
                    weight = weight if float(weight.sum()) > 0 else p
            if p is not None:
                upto = weight.cumsum(0)
                over = (upto > u[r, 1] * upto[-1]).nonzero()
                tokens[r] = int(over[0]) if len(over) else int((weight > 0).nonzero()[-1])
                n += 1
            break
        counts.append(n)
    return tokens, counts
