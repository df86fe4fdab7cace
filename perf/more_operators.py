"""Serving from a paged cache: its operators, and what they are timed and checked on.

``paged_slots`` / ``paged_release``  block tables, slot maps and the free list, from the requests' lengths
``paged_write``                      new keys and values into their slots
``paged_attention``                  grouped-query attention of new tokens (chunks, drafts, single ones) over the pages
``verify_drafts``                    drafted tokens against the target's logits, and the token after the last accepted

Sizes are those of the models this repository names (head size 128; 8, 24 or 32 query
heads over 4 or 8 key heads; vocabulary 49152) or generic ones.  With ``own`` false
:func:`run` is the operators in plain torch operations, in 32 bits (the tokens'
verification in 64: cumulative sums next to a random number); with ``own`` true it
makes the package's calls.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
BF16, FP32 = "bfloat16", "float32"


# ----------------------------------------------------------------- cases --


def listed() -> list:
    return [
        # One decode step of a serving batch: a new token each, a new page for every sixteenth.
        dict(name="slots_decode_batch64", kind="slots", batch=64, kv_len=4096, q_len=1, new="one", page=16),
        # A full server's step with prompts joining: chunks among single tokens, and too few free pages for all.
        dict(name="slots_mixed_batch512", kind="slots", batch=512, kv_len=8192, q_len=1024, new="mixed", page=64),
        # Rejected drafts and ended requests of a batch give their pages back.
        dict(name="release_batch256", kind="release", batch=256, kv_len=4096, q_len=8, new="draft", page=16),
        # The new keys and values of a decode step on the 8B model.
        dict(name="write_decode_batch64", kind="write", batch=64, kv_len=512, q_len=1, new="one", page=16, kv_heads=8,
             dim=128, dtype=BF16),
        # Prompts written in chunks, ragged, with padding behind them.
        dict(name="write_prefill_ragged", kind="write", batch=16, kv_len=4096, q_len=2048, new="draft", page=64,
             kv_heads=8, dim=128, dtype=BF16),
        # One user's next token behind a long cache on the 8B model.
        dict(name="attn_decode_long", kind="attn", batch=1, kv_len=32768, q_len=1, new="one", lens="full", page=16,
             heads=32, kv_heads=8, dim=128, dtype=BF16),
        # A serving batch on the 1B model: one token each over ragged caches.
        dict(name="attn_decode_ragged", kind="attn", batch=64, kv_len=4096, q_len=1, new="one", lens="ragged", page=16,
             heads=8, kv_heads=4, dim=128, dtype=BF16),
        # A long prompt in chunks on the 8B model: 2048 new tokens behind 14336. The largest.
        dict(name="attn_prefill_chunk", kind="attn", batch=1, kv_len=16384, q_len=2048, new="chunk", lens="full",
             page=64, heads=32, kv_heads=8, dim=128, dtype=BF16),
        # Drafts of the 3B model under verification: up to 8 tokens each over ragged caches, padding behind them.
        dict(name="attn_drafts", kind="attn", batch=32, kv_len=3000, q_len=8, new="draft", lens="ragged", page=32,
             heads=24, kv_heads=8, dim=128, dtype=BF16),
        # A check in fp32 at sizes that no tile divides: chunks of prompts among single tokens.
        dict(name="attn_mixed_fp32_odd", kind="attn", batch=11, kv_len=1237, q_len=301, new="mixed", lens="ragged",
             page=16, heads=6, kv_heads=6, dim=80, dtype=FP32),
        # One user's drafts from a lookup in the prompt (no draft distribution).
        dict(name="verify_one_lookup", kind="verify", batch=1, q_len=5, new="chunk", vocab=49152, probs=False,
             temperature=1.0, dtype=BF16),
        # A serving batch's drafts from a small model.
        dict(name="verify_batch64", kind="verify", batch=64, q_len=8, new="draft", vocab=49152, probs=True,
             temperature=0.75, dtype=BF16),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    """One more case of the ranges the listed ones stand for."""
    kind = rng.choice(("slots", "release", "write", "attn", "attn", "attn", "verify", "verify"))
    case = dict(kind=kind, batch=_log_int(rng, 1, 256))
    case["new"] = rng.choice(("one", "chunk", "draft", "mixed"))
    if kind == "verify":
        case["new"] = rng.choice(("chunk", "draft"))
        case.update(q_len=rng.randint(1, 9), vocab=_log_int(rng, 200, 130000), probs=rng.random() < 0.7,
                    temperature=rng.choice((0.0, 0.75, 1.0, 1.25)), dtype=rng.choice((BF16, FP32)))
    else:
        case.update(kv_len=_log_int(rng, 1, 65536 if kind != "write" else 4096), page=rng.choice((16, 32, 64, 128)))
        case["q_len"] = 1 if case["new"] == "one" else min(case["kv_len"], _log_int(rng, 1, 2048))
    if kind in ("write", "attn"):
        case.update(kv_heads=rng.choice((1, 2, 4, 8)), dim=rng.choice((32, 64, 80, 128, 128)),
                    dtype=FP32 if rng.random() < 0.2 else BF16)
    if kind == "attn":
        case.update(heads=case["kv_heads"] * rng.choice((1, 2, 3, 4)), lens=rng.choice(("full", "ragged")))
    if kind == "slots":
        case["batch"] = _log_int(rng, 1, 2000)
    most = [work(c) for c in listed()]
    bytes_, flops = max(w["bytes"] for w in most), max(w["flops"] for w in most)

    def too_large() -> bool:
        w = work(case)
        held = scores = 0
        if kind in ("write", "attn"):
            held = case["batch"] * (case["kv_len"] + case["page"]) * case["kv_heads"] * case["dim"]
        if kind == "attn":  # the plain form holds every score
            scores = case["batch"] * case["heads"] * case["q_len"] * case["kv_len"]
        if kind == "verify":
            held = 3 * _tokens(case) * case["vocab"]
        return w["bytes"] > bytes_ or w["flops"] > flops or scores > 1 << 30 or held > 1 << 28

    while too_large():
        if case["batch"] > 1:
            case["batch"] = case["batch"] * 2 // 3
        else:
            case["kv_len"] = case["kv_len"] * 2 // 3
            case["q_len"] = min(case["q_len"], case["kv_len"])
    return case


# ---------------------------------------------------------------- inputs --


def _tokens(case) -> int:
    """Rows of the packed batch (the requests' new tokens, and with drafts padding behind them)."""
    b, n = case["batch"], case["q_len"]
    if case["new"] == "one":
        return b
    if case["new"] == "mixed":
        return sum(n if i % 8 == 3 % b else 1 for i in range(b))
    return b * n


def _new(case, rng) -> list:
    b, n = case["batch"], case["q_len"]
    if case["new"] == "one":
        return [1] * b
    if case["new"] == "mixed":
        return [n if i % 8 == 3 % b else 1 for i in range(b)]
    return [n if case["new"] == "chunk" else rng.randint(1, n) for _ in range(b)]


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _randn(g, shape, dtype, scale=1.0) -> torch.Tensor:
    return (torch.randn(shape, generator=g, device=DEVICE) * scale).to(dtype)


def _ints(v) -> torch.Tensor:
    return torch.tensor(v, dtype=torch.int32, device=DEVICE)


def _starts(new) -> list:
    at = [0]
    for n in new:
        at.append(at[-1] + n)
    return at


def prepare(case, seed) -> dict:
    g, rng = _gen(seed), random.Random(seed)
    kind, b = case["kind"], case["batch"]
    new = _new(case, rng)
    s = dict(case=case, tokens=_tokens(case), new_host=new)
    if kind == "verify":
        dt, n, v = getattr(torch, case["dtype"]), s["tokens"], case["vocab"]
        s["q_starts"] = _ints(_starts(new))
        s["logits"] = _randn(g, (n, v), dt, 2.5)
        s["uniforms"] = torch.rand((n, 2), generator=g, device=DEVICE)
        s["draft_probs"] = None
        if case["probs"]:  # a draft model near the target: its distributions, and tokens drawn from them
            near = s["logits"].float() + torch.randn((n, v), generator=g, device=DEVICE)
            s["draft_probs"] = torch.softmax(near, -1).to(dt)
            drawn = torch.multinomial(s["draft_probs"].float() + 1e-9, 1, generator=g)[:, 0]
        else:
            drawn = s["logits"].float().argmax(-1)
        s["ids"] = torch.cat((drawn[:1], drawn[:-1]))  # row i's draft is the next row's token
        return s
    page = case["page"]
    m = -(-case["kv_len"] // page)
    if case.get("lens") == "full":
        total = [max(case["kv_len"], n) for n in new]
    else:
        total = [rng.randint(max(n, case["kv_len"] // 8), max(n, case["kv_len"])) for n in new]
    held = [t - n for t, n in zip(total, new)]
    pages = b * m + 7
    order = torch.randperm(pages, generator=g, device=DEVICE).int()
    s["table"] = order[:b * m].reshape(b, m).clone()
    if kind in ("slots", "release"):
        s["held"], s["new"] = _ints(held if kind == "slots" else total), _ints(new)
        if kind == "slots":  # the free list: enough pages for most steps, not for the mixed ones
            need = sum(-(-t // page) - (-(-h // page)) for t, h in zip(total, held))
            s["free"] = torch.randperm(pages, generator=g, device=DEVICE).int()
            s["count"] = _ints([min(pages, need * 3 // 4 if case["new"] == "mixed" else need + 3)])
        else:  # what of the drafts was kept; some requests end
            s["kept"] = _ints([0 if rng.random() < 0.05 else h + rng.randint(0, n) for h, n in zip(held, new)])
            s["free"] = torch.full((pages,), -1, dtype=torch.int32, device=DEVICE)
            s["free"][:7] = order[b * m:]
            s["count"] = _ints([7])
        return s
    dt, hk, d = getattr(torch, case["dtype"]), case["kv_heads"], case["dim"]
    s["k_cache"] = _randn(g, (pages, hk, page, d), dt)
    s["v_cache"] = _randn(g, (pages, hk, page, d), dt)
    if kind == "write":
        s["k"], s["v"] = _randn(g, (s["tokens"], hk, d), dt), _randn(g, (s["tokens"], hk, d), dt)
        slots = torch.full((s["tokens"],), -1, dtype=torch.int32, device=DEVICE)  # padding has no slot
        seq = torch.repeat_interleave(torch.arange(b, device=DEVICE), torch.tensor(new, device=DEVICE))
        at = torch.arange(len(seq), device=DEVICE) - _ints(_starts(new))[seq] + _ints(held)[seq]
        slots[:len(seq)] = s["table"][seq, at // page] * page + (at % page).int()
        s["slots"] = slots
        return s
    s["q"] = _randn(g, (s["tokens"], case["heads"], d), dt, 1.5)
    s["kv_lens"], s["total_host"] = _ints(total), total
    s["q_starts"] = None if case["new"] == "one" else _ints(_starts(new))
    return s


# ------------------------------------------------------------ plain forms --


def _pages(n, page):
    return torch.div(n + page - 1, page, rounding_mode="floor")


def _plain_slots(s) -> list:
    page, n = s["case"]["page"], s["tokens"]
    held, new, table, count = s["held"].long(), s["new"].long(), s["table"], s["count"].long()
    b, m = table.shape
    have, want = _pages(held, page), _pages(held + new, page)
    ends = new.cumsum(0)
    fits = (want <= m) & (ends <= n)
    need = torch.where(fits, want - have, torch.zeros_like(want))
    upto = need.cumsum(0)
    granted = fits & ((need == 0) | (upto <= count))
    first = upto - need
    taken = torch.where(granted, need, torch.zeros_like(need)).sum()
    # pages come from the top of the free list
    j = torch.arange(m, device=DEVICE)
    source = count - 1 - (first[:, None] + j - have[:, None])
    fresh = granted[:, None] & (j >= have[:, None]) & (j < want[:, None])
    table.copy_(torch.where(fresh, s["free"][source.clamp(0, len(s["free"]) - 1)], table))
    q_starts = torch.cat((torch.zeros_like(ends[:1]), ends)).clamp(max=n)
    tok = torch.arange(n, device=DEVICE)
    seq = torch.searchsorted(q_starts[1:], tok, right=True)
    real = seq < b
    seq = seq.clamp(max=b - 1)
    pos = torch.where(real, held[seq] + tok - q_starts[seq], torch.zeros_like(tok))
    slot = table[seq, (pos // page).clamp(max=m - 1)].long() * page + pos % page
    slot = torch.where(real & granted[seq], slot, torch.full_like(slot, -1))
    kv_lens = torch.where(granted, held + new, torch.zeros_like(held))
    return [slot.int(), pos.int(), q_starts.int(), kv_lens.int(), (count - taken).int(), table]


def _plain_release(s) -> list:
    page = s["case"]["page"]
    held, kept, table, count = s["held"].long(), s["kept"].long(), s["table"], s["count"].long()
    have, keep = _pages(held, page), _pages(kept, page)
    back = have - keep
    upto = back.cumsum(0)
    # place p of the free list: the last page of the first sequence that gives any, and so on
    place = torch.arange(len(s["free"]), device=DEVICE) - count
    seq = torch.searchsorted(upto, place, right=True).clamp(max=len(held) - 1)
    page_at = (have[seq] - 1 - (place - (upto - back)[seq])).clamp(0, table.shape[1] - 1)
    given = (place >= 0) & (place < upto[-1])
    s["free"].copy_(torch.where(given, table[seq, page_at], s["free"]))
    return [(count + upto[-1]).int(), s["free"]]


def _plain_write(s) -> list:
    page = s["case"]["page"]
    at = (s["slots"] >= 0).nonzero()[:, 0]
    slot = s["slots"][at].long()
    s["k_cache"][slot // page, :, slot % page] = s["k"][at]
    s["v_cache"][slot // page, :, slot % page] = s["v"][at]
    return [s["k_cache"], s["v_cache"]]


def _plain_attn(s) -> list:
    case = s["case"]
    b, h, hk, d, page = (case[n] for n in ("batch", "heads", "kv_heads", "dim", "page"))
    rep, most, n = h // hk, max(s["new_host"]), s["tokens"]
    lens = s["kv_lens"].long()
    starts = torch.arange(b + 1, device=DEVICE) if s["q_starts"] is None else s["q_starts"].long()
    news = starts[1:] - starts[:-1]
    # queries padded to (B, most); keys gathered to (B, Hk, slots, D)
    i = torch.arange(most, device=DEVICE)
    row = starts[:-1, None] + i
    real = i < news[:, None]
    row = row.clamp(max=n - 1)
    q = s["q"][row].float().reshape(b, most, hk, rep, d).permute(0, 2, 3, 1, 4).reshape(b, hk, rep * most, d)
    table = s["table"].long()
    k, v = (s[c][table].float().transpose(1, 2).reshape(b, hk, -1, d) for c in ("k_cache", "v_cache"))
    key = torch.arange(k.shape[2], device=DEVICE)
    pos = lens[:, None] - news[:, None] + i
    seen = real[..., None] & (key <= pos[..., None]) & (pos[..., None] >= 0)
    v = torch.where((key < lens[:, None])[:, None, :, None], v, torch.zeros_like(v))
    sc = torch.matmul(q, k.transpose(-1, -2)).reshape(b, hk, rep, most, -1) / math.sqrt(d)
    sc = sc.masked_fill(~seen[:, None, None], float("-inf"))
    top = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    o = torch.matmul(p.reshape(b, hk, rep * most, -1), v).reshape(b, hk, rep, most, d)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, most, h, d)
    # each row from its sequence's place; rows behind the last sequence are zero
    tok = torch.arange(n, device=DEVICE)
    seq = torch.searchsorted(starts[1:], tok, right=True)
    inside = seq < b
    seq = seq.clamp(max=b - 1)
    out = o[seq, (tok - starts[seq]).clamp(0, most - 1)]
    return [torch.where(inside[:, None, None], out, torch.zeros_like(out)).to(s["q"].dtype)]


def _plain_verify(s) -> list:
    case = s["case"]
    n, b, most, t = s["tokens"], case["batch"], case["q_len"], case["temperature"]
    starts, ids, u = s["q_starts"].long(), s["ids"], s["uniforms"].double()
    v = case["vocab"]
    tok = torch.arange(n, device=DEVICE)
    draft = torch.cat((ids[1:], ids[:1]))
    x = s["logits"].double()
    if t > 0:
        e = torch.exp((x - x.amax(-1, keepdim=True)) / t)
        p = e / e.sum(-1, keepdim=True)
    else:
        p = torch.nn.functional.one_hot(x.argmax(-1), v).double()
    if s["draft_probs"] is not None and t > 0:
        q = s["draft_probs"].double()
    else:  # the draft itself, for certain
        q = torch.nn.functional.one_hot(draft, v).double()
    passed = u[:, 0] * q[tok, draft] < p[tok, draft]
    # (B, most): is draft i of the sequence there, and has it passed
    i = torch.arange(most, device=DEVICE)
    news = starts[1:] - starts[:-1]
    drafts = i < news[:, None] - 1
    row = (starts[:-1, None] + i).clamp(max=n - 1)
    accepted = (passed[row] & drafts).long().cumprod(1).sum(1)
    last = starts[:-1] + accepted
    rejected = (accepted < news - 1)[:, None]
    rest = torch.where(rejected, (p[last] - q[last]).clamp(min=0), p[last])
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, p[last])
    upto = rest.cumsum(-1)
    token = torch.searchsorted(upto, (u[last, 1] * upto[:, -1])[:, None], right=True)[:, 0].clamp(max=v - 1)
    seq = torch.searchsorted(starts[1:], tok, right=True)
    inside = seq < b
    seq = seq.clamp(max=b - 1)
    at = tok - starts[seq]
    out = torch.where(at < accepted[seq], draft, torch.full_like(draft, -1))
    out = torch.where(at == accepted[seq], token[seq], out)
    return [torch.where(inside, out, torch.full_like(out, -1)), (accepted + 1).int()]


# -------------------------------------------------------------------- run --


def _own(s) -> list:
    import kotodama_amd

    case, kind = s["case"], s["case"]["kind"]
    if kind == "slots":
        return [*kotodama_amd.paged_slots(s["table"], s["held"], s["new"], s["free"], s["count"], case["page"],
                                          s["tokens"]), s["table"]]
    if kind == "release":
        return [kotodama_amd.paged_release(s["table"], s["held"], s["kept"], s["free"], s["count"], case["page"]),
                s["free"]]
    if kind == "write":
        kotodama_amd.paged_write(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"])
        return [s["k_cache"], s["v_cache"]]
    if kind == "attn":
        return [kotodama_amd.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["kv_lens"],
                                             s["q_starts"])]
    return list(kotodama_amd.verify_drafts(s["logits"], s["ids"], s["q_starts"], s["uniforms"], s["draft_probs"],
                                           temperature=case["temperature"]))


def run(state) -> list:
    if own:
        return _own(state)
    return {"slots": _plain_slots, "release": _plain_release, "write": _plain_write, "attn": _plain_attn,
            "verify": _plain_verify}[state["case"]["kind"]](state)


# ------------------------------------------------------------------- work --


def work(case) -> dict:
    kind, b, n = case["kind"], case["batch"], _tokens(case)
    e = 2 if case.get("dtype") == BF16 else 4
    real = n if case["new"] != "draft" else b * (case["q_len"] + 1) / 2  # tokens of the requests, on average
    if kind == "slots":  # lengths in and out, slots and positions out, table entries of what is new
        return {"bytes": 16 * b + 8 * n + 8 * (real / case["page"] + b), "flops": 10 * (n + b)}
    if kind == "release":
        return {"bytes": 8 * b + 8 * b, "flops": 10 * b}
    if kind == "write":
        return {"bytes": 4 * n + 4 * real * case["kv_heads"] * case["dim"] * e, "flops": n}
    if kind == "verify":  # every row of logits that a draft or the last token asks for; two rows of draft probabilities
        rows = real
        return {"bytes": rows * case["vocab"] * e + (b * case["vocab"] * e if case["probs"] else 0) + 24 * n,
                "flops": rows * case["vocab"] * 4}
    h, hk, d, kv = (case[k] for k in ("heads", "kv_heads", "dim", "kv_len"))
    mean = kv if case["lens"] == "full" else max(case["q_len"], kv * 9 // 16)
    pairs = real * max(1, mean - real / b / 2)
    return {"bytes": 2 * real * h * d * e + 2 * b * mean * hk * d * e + 4 * b * mean / case["page"],
            "flops": 4 * pairs * h * d}


# ------------------------------------------------------------------ exact --


def _exact_slots(s) -> list:
    page, n = s["case"]["page"], s["tokens"]
    held, new, free = s["held"].tolist(), s["new"].tolist(), s["free"].tolist()
    table, left = s["table"].tolist(), int(s["count"])
    top, asked = left, 0
    slots, positions, starts, lens = [-1] * n, [0] * n, [0], []
    for b, (h, k) in enumerate(zip(held, new)):
        have, want, at = -(-h // page), -(-(h + k) // page), starts[-1]
        ok = want <= len(table[b]) and at + k <= n
        need = want - have if ok else 0
        ok = ok and (need == 0 or asked + need <= top)
        for j in range(need if ok else 0):
            table[b][have + j] = free[top - 1 - asked - j]
        left -= need if ok else 0
        asked += need
        for i in range(min(k, n - at)):
            positions[at + i] = h + i
            slots[at + i] = table[b][(h + i) // page] * page + (h + i) % page if ok else -1
        starts.append(min(n, at + k))
        lens.append(h + k if ok else 0)
    return [_ints(v) for v in (slots, positions, starts, lens, [left], table)]


def _exact_release(s) -> list:
    page, free, count = s["case"]["page"], s["free"].tolist(), int(s["count"])
    table = s["table"].tolist()
    for b, (h, k) in enumerate(zip(s["held"].tolist(), s["kept"].tolist())):
        for j in reversed(range(-(-k // page), -(-h // page))):
            free[count] = table[b][j]
            count += 1
    return [_ints([count]), _ints(free)]


def _exact_write(s) -> list:
    page = s["case"]["page"]
    slots = s["slots"].long()
    at = torch.arange(len(slots), device=DEVICE)[slots >= 0]
    out = []
    for rows, cache in (("k", "k_cache"), ("v", "v_cache")):
        flat = s[cache].double().transpose(1, 2).flatten(0, 1)
        flat.index_copy_(0, slots[at], s[rows][at].double())
        out.append(flat.unflatten(0, (-1, page)).transpose(1, 2).contiguous())
    return out


def _exact_attn(s) -> list:
    case = s["case"]
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    at = 0
    for b, (n, total) in enumerate(zip(s["new_host"], s["total_host"])):
        rows = s["table"][b].long()
        pos = total - n + torch.arange(n, device=DEVICE)
        hidden = torch.arange(total, device=DEVICE)[None, :] > pos[:, None]
        for g in range(hk):
            k, v = (s[c][rows, g].double().flatten(0, 1)[:total] for c in ("k_cache", "v_cache"))
            q = s["q"][at:at + n, g * h // hk:(g + 1) * h // hk].double().transpose(0, 1)
            x = torch.matmul(q, k.T) * d ** -0.5
            p = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
            out[at:at + n, g * h // hk:(g + 1) * h // hk] = torch.matmul(p, v).transpose(0, 1)
        at += n
    return [out]


def _exact_verify(s) -> list:
    t = s["case"]["temperature"]
    ids, u = s["ids"].tolist(), s["uniforms"].double().tolist()
    out, counts, at = [-1] * s["tokens"], [], 0
    for n in s["new_host"]:
        for i in range(n):
            x = s["logits"][at + i].double()
            p = torch.softmax(x / t, -1) if t > 0 else (torch.arange(len(x), device=DEVICE) == x.argmax()).double()
            rest = p
            if i < n - 1:
                d = ids[at + i + 1]
                if s["draft_probs"] is not None and t > 0:
                    q = s["draft_probs"][at + i].double()
                else:
                    q = torch.zeros_like(p)
                    q[d] = 1
                if u[at + i][0] * float(q[d]) < float(p[d]):
                    out[at + i] = d
                    continue
                rest = torch.relu(p - q)
                rest = rest if float(rest.sum()) > 0 else p
            upto = torch.cumsum(rest, 0)
            out[at + i] = min(len(p) - 1, int((upto <= u[at + i][1] * upto[-1]).sum()))
            counts.append(i + 1)
            break
        at += n
    return [torch.tensor(out, device=DEVICE), _ints(counts)]


def exact(case, seed):
    """What :func:`run` returns for these inputs, in 64 bits."""
    s = prepare(case, seed)
    return {"slots": _exact_slots, "release": _exact_release, "write": _exact_write, "attn": _exact_attn,
            "verify": _exact_verify}[case["kind"]](s)
