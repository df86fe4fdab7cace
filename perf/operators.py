"""The language-model operators beside the routing, and what they are timed and checked on.

``qk_norm_rope``  RMSNorm of every query and key head with the position rotation, forward and backward
``attention``     causal grouped-query attention with its backward, and over a cache for few new tokens
``embedding``     the scaled token lookup and its gradient

Sizes are those of the models this repository names (head size 128; 4, 8 or 32 query
heads over 2, 4 or 8 key heads; vocabulary 49152; 2048 or 4096 tokens) or generic
ones.  With ``own`` false :func:`run` is the operators in plain torch operations in
32 bits, rounded once; with ``own`` true it makes the package's calls.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
EPS = 1e-5
THETA = 500000.0
BF16, FP32 = "bfloat16", "float32"


# ----------------------------------------------------------------- cases --


def listed() -> list:
    return [
        # The 1B model's training step: queries and keys of one layer, forward and backward.
        dict(name="qk_train_1b", kind="qk", batch=4, tokens=2048, heads=8, kv_heads=4, dim=128, train=True, dtype=BF16),
        # A serving batch of 64 sequences that each add one token, at positions of their own.
        dict(name="qk_decode_batch64", kind="qk", batch=64, tokens=1, heads=32, kv_heads=8, dim=128, train=False,
             dtype=BF16),
        # The proxy model's training step: few heads, so few rows to spread over the card.
        dict(name="attn_train_proxy", kind="attn", batch=4, q_len=2048, kv_len=2048, heads=4, kv_heads=2, dim=128,
             causal=True, lens="full", train=True, dtype=BF16),
        # The 8B model's training step: the largest.
        dict(name="attn_train_8b", kind="attn", batch=2, q_len=4096, kv_len=4096, heads=32, kv_heads=8, dim=128,
             causal=True, lens="full", train=True, dtype=BF16),
        # Fine-tuning on a padded batch of ragged sequences, at a smaller head.
        dict(name="attn_train_padded", kind="attn", batch=5, q_len=777, kv_len=777, heads=12, kv_heads=4, dim=64,
             causal=True, lens="padded", train=True, dtype=BF16),
        # A check of gradients in fp32 at sizes that no tile divides.
        dict(name="attn_train_fp32_odd", kind="attn", batch=2, q_len=613, kv_len=613, heads=6, kv_heads=6, dim=80,
             causal=True, lens="full", train=True, dtype=FP32),
        # A long prompt prefilled in pieces: 2048 new tokens behind a cache of 14336.
        dict(name="attn_prefill_chunk", kind="attn", batch=1, q_len=2048, kv_len=16384, heads=32, kv_heads=8, dim=128,
             causal=True, lens="full", train=False, dtype=BF16),
        # One user's next token behind a long cache on the 8B model.
        dict(name="attn_decode_long", kind="attn", batch=1, q_len=1, kv_len=32768, heads=32, kv_heads=8, dim=128,
             causal=True, lens="full", train=False, dtype=BF16),
        # A serving batch on the 1B model: one token each over caches filled to different lengths.
        dict(name="attn_decode_ragged", kind="attn", batch=64, q_len=1, kv_len=4096, heads=8, kv_heads=4, dim=128,
             causal=True, lens="cache", train=False, dtype=BF16),
        # The 8B model's embedding in a training step, and the whole gradient of the table.
        dict(name="embed_train_8b", kind="embed", tokens=16384, vocab=49152, hidden=4096, train=True, padding=0.0,
             dtype=BF16),
        # A padded fp32 batch at sizes that no tile divides; one token (the padding) is most of it.
        dict(name="embed_train_fp32_padded", kind="embed", tokens=5003, vocab=32003, hidden=1000, train=True,
             padding=0.6, dtype=FP32),
        # The tokens of a decode step of a full serving batch.
        dict(name="embed_decode_batch256", kind="embed", tokens=256, vocab=49152, hidden=4096, train=False, padding=0.0,
             dtype=BF16),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    """One more case of the ranges the listed ones stand for."""
    kind = rng.choice(("qk", "attn", "attn", "attn", "embed"))
    case = dict(kind=kind, dtype=FP32 if rng.random() < 0.2 else BF16)
    if kind == "embed":
        case["train"] = rng.random() < 0.7
        case["tokens"] = _log_int(rng, 1, 32768)
        case["vocab"] = _log_int(rng, 200, 65000)
        case["hidden"] = 8 * _log_int(rng, 8, 512)
        case["padding"] = rng.choice((0.0, 0.0, 0.3, 0.9))
    else:
        case["kv_heads"] = rng.choice((1, 2, 4, 8))
        case["heads"] = case["kv_heads"] * rng.choice((1, 2, 3, 4))
        case["train"] = rng.random() < 0.6
    if kind == "qk":
        case["dim"] = rng.choice((32, 64, 72, 96, 128, 256))
        case["batch"] = _log_int(rng, 1, 64)
        case["tokens"] = 1 if rng.random() < 0.3 else _log_int(rng, 1, 8192)
    if kind == "attn":
        case["dim"] = rng.choice((32, 64, 80, 128, 128))
        if case["train"]:
            case["batch"] = rng.randint(1, 6)
            case["q_len"] = case["kv_len"] = _log_int(rng, 1, 4096)
            case["causal"] = rng.random() < 0.8
            case["lens"] = rng.choice(("full", "padded")) if case["causal"] else "full"
        else:
            case["batch"] = _log_int(rng, 1, 128)
            case["kv_len"] = _log_int(rng, 16, 65536)
            case["q_len"] = 1 if rng.random() < 0.5 else min(case["kv_len"], _log_int(rng, 1, 2048))
            case["causal"] = True
            case["lens"] = rng.choice(("full", "cache"))
    most = [work(c) for c in listed()]
    bytes_, flops = max(w["bytes"] for w in most), max(w["flops"] for w in most)

    def too_large() -> bool:
        w = work(case)
        # the plain form holds every score
        scores = case["batch"] * case["heads"] * case["q_len"] * case["kv_len"] if kind == "attn" else 0
        return w["bytes"] > bytes_ or w["flops"] > flops or scores > 1 << 29

    while too_large():
        if kind != "attn":
            case["tokens"] = case["tokens"] * 2 // 3
        elif case["batch"] > 1:
            case["batch"] -= 1
        elif case["train"]:
            case["q_len"] = case["kv_len"] = case["kv_len"] * 2 // 3
        else:
            case["kv_len"] = case["kv_len"] * 2 // 3
            case["q_len"] = min(case["q_len"], case["kv_len"])
    return case


# ---------------------------------------------------------------- inputs --


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _dt(case) -> torch.dtype:
    return getattr(torch, case["dtype"])


def _randn(g, shape, dtype, scale=1.0) -> torch.Tensor:
    return (torch.randn(shape, generator=g, device=DEVICE) * scale).to(dtype)


def _tables(rows: int, dim: int, dtype) -> tuple:
    """cos and sin of every position, full width, in the model's dtype."""
    freqs = 1.0 / THETA ** (torch.arange(0, dim, 2, dtype=torch.float64, device=DEVICE) / dim)
    ang = torch.outer(torch.arange(rows, dtype=torch.float64, device=DEVICE), freqs)
    ang = torch.cat((ang, ang), -1)
    return ang.cos().to(dtype), ang.sin().to(dtype)


def prepare(case, seed) -> dict:
    g = _gen(seed)
    dt = _dt(case)
    s = dict(case=case)
    if case["kind"] == "qk":
        b, t, h, hk, d = (case[k] for k in ("batch", "tokens", "heads", "kv_heads", "dim"))
        # what the projections give: (B, T, heads, D) rows, read as (B, heads, T, D)
        s["q"] = _randn(g, (b, t, h, d), dt, 1.3).transpose(1, 2)
        s["k"] = _randn(g, (b, t, hk, d), dt, 0.8).transpose(1, 2)
        s["wq"] = (1 + 0.1 * torch.randn(d, generator=g, device=DEVICE)).to(dt)
        s["wk"] = (1 + 0.1 * torch.randn(d, generator=g, device=DEVICE)).to(dt)
        s["cos"], s["sin"] = _tables(max(t, 4096), d, dt)
        # one new token per sequence: every sequence at a position of its own
        s["positions"] = torch.randint(0, 4096, (b, 1), generator=g, device=DEVICE) if t == 1 else None
        if case["train"]:
            s["gq"] = _randn(g, (b, t, h, d), dt).transpose(1, 2)
            s["gk"] = _randn(g, (b, t, hk, d), dt).transpose(1, 2)
            for n in ("q", "k", "wq", "wk"):
                s[n].requires_grad_(True)
    elif case["kind"] == "attn":
        b, tq, tk, h, hk, d = (case[k] for k in ("batch", "q_len", "kv_len", "heads", "kv_heads", "dim"))
        # (B, T, heads, D) rows, as projections give them and a cache holds them
        s["q"] = _randn(g, (b, tq, h, d), dt, 1.5).transpose(1, 2)
        s["k"] = _randn(g, (b, tk, hk, d), dt).transpose(1, 2)
        s["v"] = _randn(g, (b, tk, hk, d), dt).transpose(1, 2)
        s["kv_lens"], s["q_start"] = None, None
        if case["lens"] == "padded":  # sequences of their own lengths, padded at the end
            s["kv_lens"] = torch.randint(max(1, tk // 4), tk + 1, (b,), generator=g, device=DEVICE, dtype=torch.int32)
            s["q_start"] = 0
        elif case["lens"] == "cache":  # slots behind a sequence's length are not written yet
            s["kv_lens"] = torch.randint(tq, tk + 1, (b,), generator=g, device=DEVICE, dtype=torch.int32)
        if case["train"]:
            s["g"] = _randn(g, (b, tq, h, d), dt).transpose(1, 2)
            for n in ("q", "k", "v"):
                s[n].requires_grad_(True)
    else:
        n, v, d = case["tokens"], case["vocab"], case["hidden"]
        s["w"] = _randn(g, (v, d), dt, 0.02)
        # token frequencies fall with the rank, as a text's do; ranks spread over the table
        u = torch.rand(n, generator=g, device=DEVICE, dtype=torch.float64)
        rank = (torch.exp(u * math.log(v)) - 1).long().clamp(0, v - 1)
        s["ids"] = torch.randperm(v, generator=g, device=DEVICE)[rank]
        if case["padding"]:
            pad = torch.rand(n, generator=g, device=DEVICE) < case["padding"]
            s["ids"] = torch.where(pad, torch.zeros_like(s["ids"]), s["ids"])
        s["scale"] = math.sqrt(d)
        if case["train"]:
            s["g"] = _randn(g, (n, d), dt)
            s["w"].requires_grad_(True)
    return s


# ------------------------------------------------------------ plain forms --


def _rotate(n, cos, sin):
    half = n.shape[-1] // 2
    return n * cos + torch.cat((-n[..., half:], n[..., :half]), -1) * sin


def _unrotate(g, cos, sin):
    half = g.shape[-1] // 2
    gs = g * sin
    return g * cos + torch.cat((gs[..., half:], -gs[..., :half]), -1)


def _norm_rope(x, w, cos, sin):
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    return _rotate(x * r * w, cos, sin)


def _norm_rope_back(x, w, cos, sin, g):
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    dn = _unrotate(g, cos, sin)
    m = dn * w
    dx = r * (m - x * r.square() * (m * x).mean(-1, keepdim=True))
    return dx, (dn * x * r).sum((0, 1, 2))


def _plain_qk(s) -> list:
    case = s["case"]
    dt = _dt(case)
    q, k, wq, wk, cos, sin = (s[n].detach().float() for n in ("q", "k", "wq", "wk", "cos", "sin"))
    if s["positions"] is None:
        cos, sin = cos[: case["tokens"]], sin[: case["tokens"]]
    else:
        cos, sin = cos[s["positions"]].unsqueeze(1), sin[s["positions"]].unsqueeze(1)
    out = [_norm_rope(q, wq, cos, sin), _norm_rope(k, wk, cos, sin)]
    if case["train"]:
        dq, dwq = _norm_rope_back(q, wq, cos, sin, s["gq"].float())
        dk, dwk = _norm_rope_back(k, wk, cos, sin, s["gk"].float())
        out += [dq, dk, dwq, dwk]
    return [t.to(dt) for t in out]


def _visible(s):
    """(B, 1, 1, q_len, kv_len) truth values: the keys each query sees."""
    case = s["case"]
    b, tq, tk = case["batch"], case["q_len"], case["kv_len"]
    lens = torch.full((b,), tk, device=DEVICE) if s["kv_lens"] is None else s["kv_lens"].long()
    start = lens - tq if s["q_start"] is None else torch.full((b,), s["q_start"], device=DEVICE)
    key = torch.arange(tk, device=DEVICE).view(1, 1, tk)
    seen = key < lens.view(b, 1, 1)
    if case["causal"]:
        pos = start.view(b, 1, 1) + torch.arange(tq, device=DEVICE).view(1, tq, 1)
        seen = seen & (key <= pos) & (pos < lens.view(b, 1, 1))
    else:
        seen = seen.expand(b, tq, tk)
    return seen.view(b, 1, 1, tq, tk)


def _plain_attn(s) -> list:
    case = s["case"]
    dt = _dt(case)
    b, tq, h, hk, d = (case[n] for n in ("batch", "q_len", "heads", "kv_heads", "dim"))
    rep = h // hk
    q = s["q"].detach().float().reshape(b, hk, rep, tq, d)
    k, v = (s[n].detach().float().unsqueeze(2) for n in ("k", "v"))
    scale = 1.0 / math.sqrt(d)
    seen = _visible(s)
    sc = (torch.matmul(q, k.transpose(-1, -2)) * scale).masked_fill(~seen, float("-inf"))
    top = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    o = torch.matmul(p, v)
    out = [o.reshape(b, h, tq, d)]
    if case["train"]:
        g = s["g"].float().reshape(b, hk, rep, tq, d)
        dv = torch.matmul(p.transpose(-1, -2), g).sum(2)
        ds = p * (torch.matmul(g, v.transpose(-1, -2)) - (g * o).sum(-1, keepdim=True))
        dq = torch.matmul(ds, k) * scale
        dk = torch.matmul(ds.transpose(-1, -2), q).sum(2) * scale
        out += [dq.reshape(b, h, tq, d), dk, dv]
    return [t.to(dt) for t in out]


def _plain_embed(s) -> list:
    case = s["case"]
    dt = _dt(case)
    w, ids = s["w"].detach(), s["ids"]
    out = [(w[ids].float() * s["scale"]).to(dt)]
    if case["train"]:
        dw = torch.zeros(w.shape, device=DEVICE)
        dw.index_add_(0, ids, s["g"].float())
        out.append((dw * s["scale"]).to(dt))
    return out


# -------------------------------------------------------------------- run --


def _own_qk(s) -> list:
    import kotodama_amd

    out = list(kotodama_amd.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], EPS,
                                         positions=s["positions"]))
    if s["case"]["train"]:
        out += torch.autograd.grad(out, [s[n] for n in ("q", "k", "wq", "wk")], [s["gq"], s["gk"]])
    return out


def _own_attn(s) -> list:
    import kotodama_amd

    out = [kotodama_amd.attention(s["q"], s["k"], s["v"], causal=s["case"]["causal"], kv_lens=s["kv_lens"],
                                  q_start=s["q_start"])]
    if s["case"]["train"]:
        out += torch.autograd.grad(out, [s[n] for n in ("q", "k", "v")], [s["g"]])
    return out


def _own_embed(s) -> list:
    import kotodama_amd

    out = [kotodama_amd.embedding(s["ids"], s["w"], scale=s["scale"])]
    if s["case"]["train"]:
        out += torch.autograd.grad(out, [s["w"]], [s["g"]])
    return out


def run(state) -> list:
    kind = state["case"]["kind"]
    if own:
        return {"qk": _own_qk, "attn": _own_attn, "embed": _own_embed}[kind](state)
    return {"qk": _plain_qk, "attn": _plain_attn, "embed": _plain_embed}[kind](state)


# ------------------------------------------------------------------- work --


def _pairs(case) -> int:
    """Query-key pairs of one head over the batch; ragged lengths count half-way between their bounds."""
    b, tq, tk = case["batch"], case["q_len"], case["kv_len"]
    if case["lens"] == "padded":
        tq = tk = max(1, tk * 5 // 8)
    elif case["lens"] == "cache":
        tk = (tq + tk) // 2
    if not case["causal"]:
        return b * tq * tk
    return b * sum(max(0, tk - tq + i + 1) for i in range(tq))


def work(case) -> dict:
    e = 2 if case["dtype"] == BF16 else 4
    if case["kind"] == "embed":
        n, v, d = case["tokens"], case["vocab"], case["hidden"]
        rows = 2 * n + (n + v if case["train"] else 0)
        return {"bytes": rows * d * e + 8 * n, "flops": n * d * (2 if case["train"] else 1)}
    if case["kind"] == "qk":
        n = case["batch"] * case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": n * e * (5 if case["train"] else 2), "flops": n * (30 if case["train"] else 10)}
    b, tq, tk, h, hk, d = (case[k] for k in ("batch", "q_len", "kv_len", "heads", "kv_heads", "dim"))
    if case["lens"] == "cache":
        tk = (tq + tk) // 2
    q, kv = b * h * tq * d * e, b * hk * tk * d * e
    # forward: q, k, v read, out written; the backward reads its gradient and writes those of q, k, v
    return {"bytes": 2 * q + 2 * kv + (2 * q + 2 * kv if case["train"] else 0),
            "flops": _pairs(case) * h * d * (14 if case["train"] else 4)}


# ------------------------------------------------------------------ exact --


def _exact_qk(s) -> list:
    case = s["case"]
    b, t, d = case["batch"], case["tokens"], case["dim"]
    half = d // 2
    rows = torch.arange(t, device=DEVICE).expand(b, t) if s["positions"] is None else s["positions"]
    cos, sin = s["cos"].double()[rows][:, None], s["sin"].double()[rows][:, None]
    outs, grads, sums = [], [], []
    for x, w, g in (("q", "wq", "gq"), ("k", "wk", "gk")):
        x, w = s[x].detach().double(), s[w].detach().double()
        inv = (x.pow(2).sum(-1, keepdim=True) / d + EPS).pow(-0.5)
        hat = x * inv
        a, c = (hat * w)[..., :half], (hat * w)[..., half:]
        outs.append(torch.cat((a * cos[..., :half] - c * sin[..., :half], c * cos[..., half:] + a * sin[..., half:]), -1))
        if case["train"]:
            ga, gc = s[g].double()[..., :half], s[g].double()[..., half:]
            dn = torch.cat((ga * cos[..., :half] + gc * sin[..., half:], gc * cos[..., half:] - ga * sin[..., :half]), -1)
            sums.append((dn * hat).flatten(0, 2).sum(0))
            dh = dn * w
            grads.append(inv * (dh - hat * (dh * hat).sum(-1, keepdim=True) / d))
    return outs + grads + sums


def _exact_attn(s) -> list:
    case = s["case"]
    b, tq, tk, h, hk, d = (case[n] for n in ("batch", "q_len", "kv_len", "heads", "kv_heads", "dim"))
    rep = h // hk
    q, k, v = (s[n].detach().double() for n in ("q", "k", "v"))
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    lens = [tk] * b if s["kv_lens"] is None else s["kv_lens"].tolist()
    for i in range(b):
        n = lens[i]
        first = n - tq if s["q_start"] is None else s["q_start"]
        live = slice(0, tq)
        if case["causal"]:  # the queries whose position lies in the sequence
            live = slice(max(0, -first), min(tq, n - first))
        pos = first + torch.arange(tq, device=DEVICE)[live]
        hidden = torch.arange(n, device=DEVICE)[None, :] > pos[:, None]
        for j in range(h):
            kk, vv, qq = k[i, j // rep, :n], v[i, j // rep, :n], q[i, j, live]
            x = qq @ kk.T / math.sqrt(d)
            if case["causal"]:
                x = x.masked_fill(hidden, -math.inf)
            p = torch.softmax(x, -1)
            o = p @ vv
            out[i, j, live] = o
            if case["train"]:
                g = s["g"][i, j, live].double()
                dv[i, j // rep, :n] += p.T @ g
                dp = g @ vv.T
                dx = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(d)
                dq[i, j, live] = dx @ kk
                dk[i, j // rep, :n] += dx.T @ qq
    return [out, dq, dk, dv] if case["train"] else [out]


def _exact_embed(s) -> list:
    w, ids, d = s["w"].detach(), s["ids"], s["case"]["hidden"]
    out = [torch.index_select(w, 0, ids).double() * s["scale"]]
    if s["case"]["train"]:
        dw = torch.zeros(w.shape, device=DEVICE, dtype=torch.float64)
        dw.scatter_add_(0, ids[:, None].expand(-1, d), s["g"].double())
        out.append(dw * s["scale"])
    return out


def exact(case, seed):
    """What :func:`run` returns for these inputs, in 64 bits."""
    s = prepare(case, seed)
    return {"qk": _exact_qk, "attn": _exact_attn, "embed": _exact_embed}[case["kind"]](s)
