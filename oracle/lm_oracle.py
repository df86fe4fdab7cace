"""Float64 restatements of the language-model operators, with error bounds.

Each function returns the operator's results from its definition, and for
each result the largest error a correct kernel may have, element by element.
The bounds count roundings: ``u`` is half a step of the result's type relative
to the value, ``e`` half a step of fp32; a sum of n terms in fp32 is off by at
most n e times the sum of their magnitudes.
"""

from __future__ import annotations

import math

import torch

E32 = 2.0**-24
HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float32: E32, torch.float64: 0.0}


# ------------------------------------------------------------- attention --


def visible(b, tq, tk, causal, kv_lens, q_start):
    """(B, Tq, Tk) truth values: the keys each query sees."""
    lens = [tk] * b if kv_lens is None else [min(max(int(n), 0), tk) for n in kv_lens]
    seen = torch.zeros(b, tq, tk, dtype=torch.bool)
    for i in range(b):
        start = lens[i] - tq if q_start is None else int(q_start if isinstance(q_start, int) else q_start[i])
        for r in range(tq):
            pos = start + r
            n = lens[i]
            if causal:
                n = pos + 1 if 0 <= pos < lens[i] else 0
            seen[i, r, :n] = True
    return seen


def attention(q, k, v, causal=True, scale=None, kv_lens=None, q_start=None, grad_out=None, grad_lse=None,
              delta_from_p=False):
    """{name: (value, bound)} for out and lse, and dq, dk, dv where ``grad_out`` is given.

    The inputs are taken as they are (bf16 or fp32 tensors, any device); the
    bounds are those of a kernel that computes scores and sums in fp32 and
    rounds the probabilities and score gradients to the inputs' type for the
    products with v, k and q.  Such a kernel may read the row sum of do * o off
    the output, which is rounded; ``delta_from_p``: it forms the sum of p * dp
    instead, in fp32.
    """
    u = HALF_STEP[q.dtype]
    up = u if q.dtype == torch.bfloat16 else 0.0
    b, h, tq, d = q.shape
    hk, tk = k.shape[1], k.shape[2]
    rep = h // hk
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    seen = visible(b, tq, tk, causal, kv_lens, q_start).to(q.device)
    keep = seen.any(1)[:, None, :, None]  # what nothing sees is not used, whatever it holds
    live = seen.any(2)[:, None, :, None]
    q = torch.where(live, q.double(), 0.0)
    k = torch.where(keep, k.double(), 0.0).repeat_interleave(rep, 1)
    v = torch.where(keep, v.double(), 0.0).repeat_interleave(rep, 1)
    mask = seen[:, None]
    s = (q @ k.transpose(-1, -2) * scale).masked_fill(~mask, -math.inf)
    top = s.amax(-1, keepdim=True) if tk else s.new_full((b, h, tq, 1), -math.inf)
    top0 = torch.where(top == -math.inf, 0.0, top)
    w = torch.exp(s - top0)
    total = w.sum(-1, keepdim=True)
    p = w / torch.where(total == 0, 1.0, total)
    out = p @ v
    lse = torch.where(total == 0, -math.inf, top0 + torch.log(torch.where(total == 0, 1.0, total))).squeeze(-1)
    # a score is off by its products' roundings, its scaling's and the exponent's; p relative to itself by
    # twice the worst of them (numerator and sum) and the sum's and the exponential's own
    mags = (q.abs() @ k.abs().transpose(-1, -2)) * abs(scale)
    off = ((d + 4) * E32 * mags + 4 * E32 * torch.where(mask, s.abs(), 0.0)).amax(-1, keepdim=True) if tk else 0.0
    rp = 4 * off + (tk + 32) * E32
    err_o = u * out.abs() + (up + rp) * (p @ v.abs())
    res = {"out": (out, err_o), "lse": (lse, (rp + 4 * E32 * (1 + torch.where(total == 0, 0.0, lse[..., None]).abs()))
                                       .expand(b, h, tq, 1).squeeze(-1))}
    if grad_out is None:
        return res
    g = torch.where(live, grad_out.double(), 0.0)
    delta = (g * out).sum(-1, keepdim=True)
    gl = 0.0 if grad_lse is None else torch.where(live, grad_lse.double()[..., None], 0.0)
    dp = g @ v.transpose(-1, -2)
    ds = p * (dp - delta + gl)
    gv = g.abs() @ v.abs().transpose(-1, -2)
    go = (g.abs() * out.abs()).sum(-1, keepdim=True)
    err_delta = (g.abs() * err_o).sum(-1, keepdim=True) + (d + 4) * E32 * (go + abs(gl))
    if delta_from_p:
        # dp's own error, and the sum's over keys of terms off by p's
        err_delta = (p * ((d + 4) * E32 * gv + (rp + (tk + 4) * E32) * dp.abs())).sum(-1, keepdim=True) + 4 * E32 * abs(gl)
    err_ds = up * ds.abs() + p * (rp * (dp - delta + gl).abs() + (d + 4) * E32 * gv + err_delta)

    def shared(x):
        return x.view(b, hk, rep, tk, d).sum(2)

    dq = ds @ k * scale
    dk = shared(ds.transpose(-1, -2) @ q) * scale
    dv = shared(p.transpose(-1, -2) @ g)
    n = (max(tq * rep, tk) + 4) * E32
    res["dq"] = (dq, u * dq.abs() + abs(scale) * ((err_ds + n * ds.abs()) @ k.abs()))
    res["dk"] = (dk, u * dk.abs() + abs(scale) * shared((err_ds + n * ds.abs()).transpose(-1, -2) @ q.abs()))
    res["dv"] = (dv, u * dv.abs() + shared(((up + rp + n) * p).transpose(-1, -2) @ g.abs()))
    return res


# ---------------------------------------------------------- qk_norm_rope --


def norm_rope(x, w, cos, sin, eps, rows, grad=None):
    """{name: (value, bound)} of one tensor's norm and rotation: y, and dx, dw where ``grad`` is given.

    ``x`` (B, H, T, D); ``rows`` (B, T) the tables' rows (a row outside them gives NaN).
    """
    u = HALF_STEP[x.dtype]
    d = x.shape[-1]
    half = d // 2
    bad = (rows < 0) | (rows >= cos.shape[0])
    at = rows.clamp(0, max(0, cos.shape[0] - 1))
    nan = torch.where(bad, math.nan, 0.0).to(x.device)[:, None, :, None]
    c = cos.double()[at][:, None] + nan
    s = sin.double()[at][:, None] + nan
    x, w = x.double(), w.double()
    r = torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    n = x * r * w
    rot = torch.cat((-n[..., half:], n[..., :half]), -1)
    y = n * c + rot * s
    k = (d + 16) * E32
    res = {"y": (y, u * y.abs() + k * ((n * c).abs() + (rot * s).abs()))}
    if grad is None:
        return res
    g = grad.double()
    gs = g * s
    dn = g * c + torch.cat((gs[..., half:], -gs[..., :half]), -1)
    dn_mag = (g * c).abs() + torch.cat((gs[..., half:], gs[..., :half]), -1).abs()
    m = (w * dn * x).mean(-1, keepdim=True)
    m_mag = (w.abs() * dn_mag * x.abs()).mean(-1, keepdim=True)
    dx = r * (w * dn - x * r.pow(2) * m)
    res["dx"] = (dx, u * dx.abs() + 2 * k * r * (w.abs() * dn_mag + x.abs() * r.pow(2) * m_mag))
    t = dn * x * r
    dw = t.sum((0, 1, 2))
    count = t.numel() // d
    res["dw"] = (dw, u * dw.abs() + (count + d + 16) * E32 * (dn_mag * x.abs() * r).sum((0, 1, 2)))
    return res


# ------------------------------------------------------------- embedding --


def embedding(ids, weight, scale=1.0, padding_idx=None, grad=None):
    """{name: (value, bound)}: out, and dw where ``grad`` is given."""
    u = HALF_STEP[weight.dtype]
    rows, hidden = weight.shape
    flat = ids.reshape(-1).long()
    ok = (flat >= 0) & (flat < rows)
    safe = torch.where(ok, flat, 0)
    w = weight.double()
    out = (w[safe] if rows else w.new_zeros(flat.numel(), hidden)) * scale
    out = torch.where(ok[:, None], out, math.nan).reshape(*ids.shape, hidden)
    res = {"out": (out, (u + 2 * E32) * out.abs())}
    if grad is None:
        return res
    g = grad.reshape(-1, hidden).double()
    use = ok if padding_idx is None else ok & (flat != padding_idx % rows)
    dw = torch.zeros(rows, hidden, dtype=torch.float64, device=weight.device)
    mag = torch.zeros_like(dw)
    dw.index_add_(0, flat[use], g[use] * scale)
    mag.index_add_(0, flat[use], g[use].abs() * abs(scale))
    count = torch.bincount(flat[use], minlength=rows)[:, None].double()
    res["dw"] = (dw, u * dw.abs() + (count + 2) * E32 * mag)
    return res
