"""The language-model operators on the GPU against their float64 oracle
(oracle/lm_oracle.py), element by element within its bounds, which count the
roundings a correct kernel makes."""

import math

import pytest
import torch

import kotodama_amd
from kotodama_amd import lmops
from oracle import lm_oracle as LO

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
BF, FP = torch.bfloat16, torch.float32


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, dtype=BF, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _within(name, got, want):
    value, bound = want
    assert got.shape == value.shape, name
    got = got.double()
    same = (got == value) | (got.isnan() & value.isnan())  # infinities and NaN as they are
    over = torch.where(same, 0.0, (got - value).abs() / bound.clamp_min(1e-300))
    worst = over.max().item() if over.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3g} times its bound"  # a NaN fails


# ------------------------------------------------------------- attention --


def _heads(g, b, h, t, d, dtype, scale=1.0):
    return _randn(g, b, t, h, d, dtype=dtype, scale=scale).transpose(1, 2)


def _attention_case(b, h, hk, tq, tk, d, dtype, seed=0, causal=True, lens=None, start=None, scale=None,
                    with_lse=False):
    g = _gen(seed)
    print(f"attention b={b} h={h}/{hk} q={tq} k={tk} d={d} {dtype} causal={causal} lens={lens} start={start}", flush=True)
    q, k, v = _heads(g, b, h, tq, d, dtype, 1.5), _heads(g, b, hk, tk, d, dtype), _heads(g, b, hk, tk, d, dtype)
    go = _heads(g, b, h, tq, d, dtype)
    gl = torch.randn((b, h, tq), generator=g, device=DEV) if with_lse else None
    for t in (q, k, v):
        t.requires_grad_(True)
    kv_lens = None if lens is None else torch.tensor(lens, device=DEV, dtype=torch.int32)
    q_start = torch.tensor(start, device=DEV, dtype=torch.int32) if isinstance(start, list) else start
    out, lse = kotodama_amd.attention(q, k, v, causal=causal, scale=scale, kv_lens=kv_lens, q_start=q_start,
                                      want_lse=True)
    outs, grads = ([out, lse], [go, gl]) if with_lse else ([out], [go])
    dq, dk, dv = torch.autograd.grad(outs, (q, k, v), grads)
    res = LO.attention(q.detach(), k.detach(), v.detach(), causal, scale, lens, start, go, gl)
    for name, got in (("out", out), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
        _within(name, got.detach(), res[name])
    with torch.no_grad():  # the same numbers without autograd
        again = kotodama_amd.attention(q, k, v, causal=causal, scale=scale, kv_lens=kv_lens, q_start=q_start)
    assert torch.equal(again, out)


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
@pytest.mark.parametrize("b,h,hk,tq,tk,d", [
    (1, 1, 1, 1, 1, 8), (2, 4, 2, 64, 64, 128), (1, 2, 1, 129, 129, 64), (1, 3, 3, 200, 200, 80),
    (2, 6, 2, 33, 95, 72), (1, 4, 1, 1, 300, 128), (1, 8, 2, 5, 1000, 128), (1, 2, 2, 300, 257, 128),
    (3, 2, 1, 31, 31, 16), (1, 1, 1, 513, 513, 128)])
def test_attention_causal(dtype, b, h, hk, tq, tk, d):
    _attention_case(b, h, hk, tq, tk, d, dtype, seed=tq)


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
@pytest.mark.parametrize("b,h,hk,tq,tk,d,causal,lens,start", [
    (2, 2, 2, 70, 130, 64, False, None, None),       # full
    (4, 2, 1, 150, 150, 128, True, [150, 1, 0, 77], 0),  # padded batch, an empty sequence in it
    (3, 2, 1, 40, 150, 128, False, [150, 64, 0], None),
    (3, 4, 2, 1, 150, 128, True, [150, 65, 0], None),    # a cache's fill
    (3, 4, 2, 7, 150, 64, True, [150, 3, 7], None),      # fewer keys than queries: the first see none
    (2, 2, 2, 40, 100, 128, True, None, [-20, 70]),      # positions before and behind the sequence
    (1, 2, 1, 40, 100, 80, True, None, 10),
    (1, 2, 1, 40, 100, 80, True, None, 500),             # all behind
    (2, 2, 1, 40, 100, 64, True, [1000, -5], [60, 60]),  # lengths are taken into the slots there are
])
def test_attention_masks(dtype, b, h, hk, tq, tk, d, causal, lens, start):
    _attention_case(b, h, hk, tq, tk, d, dtype, seed=tq + tk, causal=causal, lens=lens, start=start)


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
@pytest.mark.parametrize("b,h,hk,tq,tk,d,causal,lens,start", [
    # enough rows that two waves share theirs, or none do
    (4, 16, 16, 530, 530, 64, True, None, None),
    (8, 16, 16, 530, 530, 64, True, None, None),
    (4, 24, 8, 400, 300, 128, True, [300, 1, 0, 177], 0),
    (8, 32, 16, 300, 500, 128, True, [500, 300, 200, 1, 0, 499, 64, 128], None),
    (3, 21, 7, 700, 700, 72, False, [700, 64, 333], None),
    (2, 40, 4, 515, 515, 128, True, None, 3),
])
def test_attention_of_many_rows(dtype, b, h, hk, tq, tk, d, causal, lens, start):
    _attention_case(b, h, hk, tq, tk, d, dtype, seed=tq + b, causal=causal, lens=lens, start=start)


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
@pytest.mark.parametrize("b,h,hk,tq,tk,d,lens", [
    (1, 1, 1, 1, 70000, 64, None),      # more parts than a workgroup's waves hold at once
    (1, 3, 1, 2, 9000, 128, None),
    (5, 4, 2, 1, 3000, 80, [3000, 1, 0, 129, 2500]),  # parts without keys
    (2, 2, 2, 40, 5000, 128, [5000, 41]),
])
def test_attention_over_a_split_cache(dtype, b, h, hk, tq, tk, d, lens):
    g = _gen(tk)
    print(f"attention over a cache b={b} h={h}/{hk} q={tq} k={tk} d={d} {dtype} lens={lens}", flush=True)
    q, k, v = _heads(g, b, h, tq, d, dtype, 1.5), _heads(g, b, hk, tk, d, dtype), _heads(g, b, hk, tk, d, dtype)
    kv_lens = None if lens is None else torch.tensor(lens, device=DEV)
    if lens is not None:  # what is not written yet
        gone = torch.arange(tk, device=DEV)[None, None, :, None] >= kv_lens[:, None, None, None]
        k, v = k.masked_fill(gone, math.nan), v.masked_fill(gone, math.inf)
    out, lse = kotodama_amd.attention(q, k, v, kv_lens=kv_lens, want_lse=True)
    res = LO.attention(q, k, v, kv_lens=lens)
    _within("out", out, res["out"])
    _within("lse", lse, res["lse"])


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
@pytest.mark.parametrize("tq,tk", [(1, 9000), (1, 100), (70, 70), (300, 5000)])
def test_attention_shows_a_nan(dtype, tq, tk):
    # a row that sees a NaN is one, whether its keys are split over workgroups or not
    g = _gen(tk + 1)
    b, h, hk, d = 2, 4, 2, 64
    q, k, v = _heads(g, b, h, tq, d, dtype), _heads(g, b, hk, tk, d, dtype), _heads(g, b, hk, tk, d, dtype)
    print(f"attention of a NaN q={tq} k={tk} {dtype}", flush=True)
    out, lse = kotodama_amd.attention(q, k, v, causal=False, want_lse=True)
    for which in range(3):
        bad = [q.clone(), k.clone(), v.clone()]
        at = (1, 2, tq - 1) if which == 0 else (1, 1, tk // 2)
        bad[which][at][3] = math.nan
        got, got_lse = kotodama_amd.attention(*bad, causal=False, want_lse=True)
        hit = torch.zeros((b, h, tq), dtype=torch.bool, device=DEV)
        if which == 0:
            hit[at] = True
        else:
            hit[1, 2:] = True  # both query heads of the key head
        if which == 2:
            assert got[..., 3][hit].isnan().all() and torch.equal(got_lse, lse)
        else:
            assert got[hit].isnan().all() and got_lse[hit].isnan().all()
            assert torch.equal(got_lse[~hit], lse[~hit])
        assert torch.equal(got[~hit], out[~hit])


def test_attention_gradient_shows_a_nan():
    g = _gen(2)
    q, k, v, go = (_heads(g, 1, 2, 40, 64, BF) for _ in range(4))
    q[0, 1, 7, 0] = math.nan
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    dq, dk, dv = torch.autograd.grad(kotodama_amd.attention(*leaves), leaves, go)
    seen = torch.arange(40, device=DEV) <= 7
    assert dq[0, 1, 7].isnan().all() and not dq[0, 1, 8:].isnan().any() and not dq[0, 0].isnan().any()
    assert dk[0, 1, seen].isnan().all() and dv[0, 1, seen].isnan().all()
    assert not dk[0, 0].isnan().any() and not dv[0, 0].isnan().any()


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
def test_attention_of_wide_groups(dtype):
    _attention_case(1, 33, 1, 5, 70, 64, dtype, seed=5)
    _attention_case(1, 200, 2, 3, 40, 128, dtype, seed=6, lens=[30])
    _attention_case(2, 14, 2, 45, 45, 64, dtype, seed=7, lens=[45, 9], start=0)


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
def test_attention_gradient_through_lse(dtype):
    _attention_case(2, 4, 2, 90, 90, 64, dtype, seed=3, with_lse=True, scale=0.3)
    _attention_case(2, 2, 1, 50, 90, 128, dtype, seed=4, with_lse=True, lens=[90, 0], causal=False)


def test_attention_lse_alone():
    g = _gen(8)
    q, k, v = (_heads(g, 1, 2, 40, 64, FP).requires_grad_(True) for _ in range(3))
    _, lse = kotodama_amd.attention(q, k, v, want_lse=True)
    gl = torch.randn(lse.shape, generator=g, device=DEV)
    got = torch.autograd.grad(lse, (q, k, v), gl)
    res = LO.attention(q.detach(), k.detach(), v.detach(), grad_out=torch.zeros_like(q), grad_lse=gl)
    for name, t in zip(("dq", "dk", "dv"), got):
        _within(name, t, res[name])


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
def test_attention_ignores_what_does_not_exist(dtype):
    # NaN and infinities in unwritten cache slots and in the padding's queries and gradients
    g = _gen(9)
    b, h, hk, t, d = 3, 4, 2, 150, 128
    lens = torch.tensor([150, 70, 0], device=DEV)
    q, k, v, go = (_heads(g, b, n, t, d, dtype) for n in (h, hk, hk, h))
    clean = kotodama_amd.attention(*(x.requires_grad_(True) for x in (q, k, v)), kv_lens=lens, q_start=0)
    want = [clean.detach(), *torch.autograd.grad(clean, (q, k, v), go)]
    gone = torch.arange(t, device=DEV)[None, None, :, None] >= lens[:, None, None, None]
    bad = [torch.where(gone, torch.tensor(x, dtype=dtype, device=DEV), y.detach()).requires_grad_(True)
           for x, y in ((math.nan, q), (math.nan, k), (math.inf, v))]
    out = kotodama_amd.attention(*bad, kv_lens=lens, q_start=0)
    got = [out.detach(), *torch.autograd.grad(out, bad, torch.where(gone, math.nan, go))]
    for a, w in zip(got, want):
        assert torch.equal(a, w)
    assert not out[2].any() and not out[1, :, 70:].any()


def test_attention_strides_and_broadcast():
    g = _gen(10)
    b, h, hk, t, d = 2, 4, 2, 100, 64
    fused = _randn(g, b, t, (h + 2 * hk) * d + 8)  # q, k and v as slices of one projection, rows of odd width
    q = fused[..., :h * d].unflatten(-1, (h, d)).transpose(1, 2)
    k = fused[..., h * d:(h + hk) * d].unflatten(-1, (hk, d)).transpose(1, 2)
    v = fused[..., (h + hk) * d:(h + 2 * hk) * d].unflatten(-1, (hk, d)).transpose(1, 2)
    want = kotodama_amd.attention(q.contiguous(), k.contiguous(), v.contiguous())
    assert torch.equal(kotodama_amd.attention(q, k, v), want)
    # unaligned rows, a column-major last dimension, and one element off 16 bytes are copied
    odd = _randn(g, b, h, t, d + 3)[..., 1:d + 1]
    assert torch.equal(kotodama_amd.attention(odd, k, v), kotodama_amd.attention(odd.contiguous(), k, v))
    turned = _randn(g, b, hk, d, t).transpose(-1, -2)
    assert torch.equal(kotodama_amd.attention(q, turned, v), kotodama_amd.attention(q, turned.contiguous(), v))
    # one sequence's keys for the whole batch: the gradient is the sum over it
    k1 = k[:1].detach().requires_grad_(True)
    out = kotodama_amd.attention(q, k1.expand(b, -1, -1, -1), v)
    go = torch.ones((), device=DEV, dtype=BF).expand_as(out)
    (dk1,) = torch.autograd.grad(out, k1, go)
    kb = k[:1].repeat(b, 1, 1, 1).requires_grad_(True)
    (dkb,) = torch.autograd.grad(kotodama_amd.attention(q, kb, v), kb, go.contiguous())
    assert torch.equal(dk1, dkb.sum(0, keepdim=True))


def test_attention_repeats_bit_for_bit():
    g = _gen(11)
    q, k, v, go = (_heads(g, 2, n, 700, 128, BF) for n in (4, 2, 2, 4))
    for t in (q, k, v):
        t.requires_grad_(True)
    first = torch.autograd.grad(kotodama_amd.attention(q, k, v), (q, k, v), go)
    for _ in range(3):
        again = torch.autograd.grad(kotodama_amd.attention(q, k, v), (q, k, v), go)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_attention_peaked_and_equal_scores():
    g = _gen(12)
    for dtype in (BF, FP):
        q, k, v = _heads(g, 1, 1, 96, 64, dtype, 20.0), _heads(g, 1, 1, 96, 64, dtype, 20.0), _heads(g, 1, 1, 96, 64, dtype)
        _within("out", kotodama_amd.attention(q, k, v), LO.attention(q, k, v)["out"])
        zero = torch.zeros_like(q)
        _within("out", kotodama_amd.attention(zero, k, v), LO.attention(zero, k, v)["out"])


def test_attention_tokens_far_apart():
    # rows 40 MiB apart (a view of every 20th million elements) are copied; 20 MiB apart they are read in place
    g = _gen(13)
    for step in (20 << 20, 10 << 20):
        store = torch.zeros(5 * step + 64, device=DEV, dtype=BF)
        k = store[:5 * step].view(5, step)[:, :64].view(1, 1, 5, 64)
        k.copy_(_randn(g, 1, 1, 5, 64))
        q = _heads(g, 1, 2, 5, 64, BF)
        assert torch.equal(kotodama_amd.attention(q, k, k), kotodama_amd.attention(q, k.contiguous(), k.contiguous()))


def test_no_gradients_of_gradients():
    g = _gen(14)
    q = _heads(g, 1, 2, 9, 64, FP).requires_grad_(True)
    out = kotodama_amd.attention(q, q, q)
    (d,) = torch.autograd.grad(out.sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), q)


def test_attention_index_forms():
    # starts and lengths of any whole-number type and stride, together and apart, give the same rows
    g = _gen(15)
    q, k, v = _heads(g, 3, 4, 6, 64, BF), _heads(g, 3, 2, 90, 64, BF), _heads(g, 3, 2, 90, 64, BF)
    lens, start = torch.tensor([90, 40, 7], device=DEV), torch.tensor([80, 34, 1], device=DEV)
    want = kotodama_amd.attention(q, k, v, kv_lens=lens, q_start=start)
    for a in (lens, lens.int(), lens.repeat_interleave(2)[::2]):
        for b in (start, start.int(), start.repeat_interleave(3)[::3]):
            assert torch.equal(kotodama_amd.attention(q, k, v, kv_lens=a, q_start=b), want)
    far = torch.tensor([1 << 45, -(1 << 45), 1 << 62], device=DEV)
    assert not kotodama_amd.attention(q, k, v, q_start=far).any()
    assert torch.equal(kotodama_amd.attention(q, k, v, kv_lens=far),
                       kotodama_amd.attention(q, k, v, kv_lens=torch.tensor([90, 0, 90], device=DEV)))
    one = lens[:1].expand(3)
    assert torch.equal(kotodama_amd.attention(q, k, v, kv_lens=one), kotodama_amd.attention(q, k, v))


@pytest.mark.parametrize("b,h,hk,tq,tk,d", [(0, 2, 1, 4, 4, 64), (2, 2, 1, 0, 4, 64), (2, 2, 1, 4, 0, 64)])
def test_attention_of_nothing(b, h, hk, tq, tk, d):
    q, k, v = (torch.ones((b, n, t, d), device=DEV, dtype=BF, requires_grad=True)
               for n, t in ((h, tq), (hk, tk), (hk, tk)))
    out = kotodama_amd.attention(q, k, v)
    assert out.shape == q.shape and not out.any()
    for grad, t in zip(torch.autograd.grad(out, (q, k, v), torch.ones_like(out)), (q, k, v)):
        assert grad.shape == t.shape and not grad.any()


# ---------------------------------------------------------- qk_norm_rope --


def _tables(rows, d, dtype):
    ang = torch.outer(torch.arange(rows, dtype=torch.float64, device=DEV),
                      10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device=DEV) / d))
    ang = torch.cat((ang, ang), -1)
    return ang.cos().to(dtype), ang.sin().to(dtype)


def _qk_case(b, h, hk, t, d, dtype, positions=None, table=None, rows=None, seed=0):
    g = _gen(seed)
    print(f"qk_norm_rope b={b} h={h}/{hk} t={t} d={d} {dtype} table={table}", flush=True)
    q, k = _heads(g, b, h, t, d, dtype, 1.5), _heads(g, b, hk, t, d, dtype, 0.3)
    wq, wk = (1 + 0.2 * torch.randn((2, d), generator=g, device=DEV)).to(dtype)
    wq, wk = wq.clone(), wk.clone()
    cos, sin = _tables(rows or t + 3, d, table or dtype)
    gq, gk = _heads(g, b, h, t, d, dtype), _heads(g, b, hk, t, d, dtype)
    leaves = [x.requires_grad_(True) for x in (q, k, wq, wk)]
    yq, yk = kotodama_amd.qk_norm_rope(*leaves, cos, sin, 1e-5, positions=positions)
    dq, dk, dwq, dwk = torch.autograd.grad((yq, yk), leaves, (gq, gk))
    at = torch.arange(t, device=DEV).expand(b, t) if positions is None else positions.long().expand(b, t)
    for x, w, y, go, dx, dw in ((q, wq, yq, gq, dq, dwq), (k, wk, yk, gk, dk, dwk)):
        res = LO.norm_rope(x.detach(), w.detach(), cos, sin, 1e-5, at, go)
        for name, got in (("y", y), ("dx", dx), ("dw", dw)):
            _within(name, got.detach(), res[name])
    with torch.no_grad():
        again = kotodama_amd.qk_norm_rope(*leaves, cos, sin, 1e-5, positions=positions)
    assert all(torch.equal(a.nan_to_num(7.0), y.nan_to_num(7.0)) for a, y in zip(again, (yq, yk)))


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
@pytest.mark.parametrize("b,h,hk,t,d", [(1, 1, 1, 1, 2), (2, 4, 2, 37, 128), (1, 3, 1, 65, 64), (2, 5, 5, 9, 96),
                                        (1, 2, 1, 130, 256), (3, 4, 2, 11, 72), (1, 7, 3, 5, 36), (2, 8, 4, 1500, 128),
                                        (1, 2, 2, 33, 254)])
def test_qk_norm_rope(dtype, b, h, hk, t, d):
    _qk_case(b, h, hk, t, d, dtype, seed=d + t)


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_qk_norm_rope_positions(dtype, index):
    g = _gen(20)
    for shape in ((5, 1), (5, 3), (1, 3), (3,)):
        t = shape[-1]
        pos = torch.randint(0, 1000, shape, generator=g, device=DEV).to(index)
        _qk_case(5, 4, 2, t, 128, dtype, positions=pos, rows=1000, seed=t)
    wide = torch.randint(0, 50, (5, 6), generator=g, device=DEV).to(index)
    _qk_case(5, 4, 2, 3, 64, dtype, positions=wide[:, ::2], rows=50)  # every second
    _qk_case(5, 4, 2, 3, 64, dtype, positions=wide[:, :1].expand(5, 3), rows=50)


def test_qk_norm_rope_positions_outside_the_tables_give_nan():
    pos = torch.tensor([[0, -1, 4], [5, 2, 1 << 40]], device=DEV)
    _qk_case(2, 2, 1, 3, 64, BF, positions=pos, rows=5)
    q = torch.ones((2, 2, 3, 64), device=DEV, dtype=BF)
    cos, sin = _tables(5, 64, BF)
    y, _ = kotodama_amd.qk_norm_rope(q, q, q[0, 0, 0], q[0, 0, 0], cos, sin, 1e-5, positions=pos)
    assert y.isnan().all(-1).tolist() == [[[False, True, False]] * 2, [[True, False, True]] * 2]


def test_qk_norm_rope_fp32_tables_and_odd_strides():
    _qk_case(2, 4, 2, 40, 128, BF, table=FP)
    g = _gen(21)
    fused = _randn(g, 2, 40, 6 * 64 + 2)
    q = fused[..., 1:4 * 64 + 1].unflatten(-1, (4, 64)).transpose(1, 2)  # one element off every alignment
    k = fused[..., 4 * 64 + 1:6 * 64 + 1].unflatten(-1, (2, 64)).transpose(1, 2)
    w = _randn(g, 64)
    cos, sin = _tables(64, 64, BF)
    got = kotodama_amd.qk_norm_rope(q, k, w, w, cos, sin, 1e-5)
    for a, x in zip(got, (q, k)):
        at = torch.arange(40, device=DEV).expand(2, 40)
        _within("y", a, LO.norm_rope(x, w, cos, sin, 1e-5, at)["y"])
    # gradients that are broadcast (a sum's)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, w, w.clone())]
    yq, yk = kotodama_amd.qk_norm_rope(*leaves, cos, sin, 1e-5)
    one = torch.autograd.grad(yq.sum() + yk.sum(), leaves)
    yq, yk = kotodama_amd.qk_norm_rope(*leaves, cos, sin, 1e-5)
    two = torch.autograd.grad((yq, yk), leaves, (torch.ones_like(yq), torch.ones_like(yk)))
    assert all(torch.equal(a, b) for a, b in zip(one, two))


def test_qk_norm_rope_one_result_used():
    g = _gen(22)
    leaves = [x.requires_grad_(True) for x in (_heads(g, 2, 4, 9, 64, FP), _heads(g, 2, 2, 9, 64, FP),
                                               _randn(g, 64, dtype=FP), _randn(g, 64, dtype=FP))]
    cos, sin = _tables(9, 64, FP)
    yq, yk = kotodama_amd.qk_norm_rope(*leaves, cos, sin, 1e-5)
    go = _heads(g, 2, 2, 9, 64, FP)
    dq, dk, dwq, dwk = torch.autograd.grad(yk, leaves, go)
    assert not dq.any() and not dwq.any()
    res = LO.norm_rope(leaves[1].detach(), leaves[3].detach(), cos, sin, 1e-5,
                       torch.arange(9, device=DEV).expand(2, 9), go)
    _within("dx", dk, res["dx"])
    _within("dw", dwk, res["dw"])


def test_qk_norm_rope_without_keys():
    g = _gen(23)
    cos, sin = _tables(9, 64, BF)
    q = _heads(g, 2, 4, 9, 64, BF).requires_grad_(True)
    none = torch.empty((2, 0, 9, 64), device=DEV, dtype=BF, requires_grad=True)
    w = [_randn(g, 64).requires_grad_(True) for _ in range(2)]
    yq, yk = kotodama_amd.qk_norm_rope(q, none, *w, cos, sin, 1e-5)
    want, _ = kotodama_amd.qk_norm_rope(q, q[:, :2], *w, cos, sin, 1e-5)
    assert torch.equal(yq, want) and yk.shape == none.shape
    dq, dk, dwq, dwk = torch.autograd.grad((yq, yk), (q, none, *w), (torch.ones_like(yq), torch.ones_like(yk)))
    assert dk.shape == none.shape and not dwk.any() and dq.any() and dwq.any()


def test_qk_norm_rope_of_many_heads():
    _qk_case(1, 300, 130, 3, 64, BF, seed=9)  # more head rows than the backward's grid has
    _qk_case(40, 6, 2, 1, 128, BF, seed=10)


@pytest.mark.parametrize("b,t", [(0, 4), (2, 0)])
def test_qk_norm_rope_of_nothing(b, t):
    leaves = [torch.ones(s, device=DEV, dtype=BF, requires_grad=True) for s in ((b, 2, t, 64), (b, 1, t, 64), (64,), (64,))]
    cos, sin = _tables(8, 64, BF)
    ys = kotodama_amd.qk_norm_rope(*leaves, cos, sin, 1e-5)
    for grad, x in zip(torch.autograd.grad(ys, leaves, [torch.ones_like(y) for y in ys]), leaves):
        assert grad.shape == x.shape and not grad.any()


# ------------------------------------------------------------- embedding --


def _embed_case(ids, rows, hidden, dtype, scale=1.0, padding_idx=None, seed=0):
    g = _gen(seed)
    print(f"embedding n={ids.numel()} rows={rows} hidden={hidden} {dtype} scale={scale} pad={padding_idx}", flush=True)
    w = _randn(g, rows, hidden, dtype=dtype).requires_grad_(True)
    out = kotodama_amd.embedding(ids, w, scale=scale, padding_idx=padding_idx)
    go = _randn(g, *ids.shape, hidden, dtype=dtype)
    (dw,) = torch.autograd.grad(out, w, go)
    res = LO.embedding(ids, w.detach(), scale, padding_idx, go)
    _within("out", out.detach(), res["out"])
    _within("dw", dw, res["dw"])
    with torch.no_grad():
        assert torch.equal(kotodama_amd.embedding(ids, w, scale=scale, padding_idx=padding_idx).nan_to_num(7.0),
                           out.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
@pytest.mark.parametrize("n,rows,hidden", [(1, 1, 1), (1, 300, 64), (7, 50, 100), (64, 5, 513), (65, 70000, 8),
                                           (1000, 97, 1000), (4099, 2000, 96), (9000, 1, 64), (3000, 200000, 40),
                                           (40000, 500, 24)])
def test_embedding(dtype, n, rows, hidden):
    ids = torch.randint(0, rows, (n,), generator=_gen(n), device=DEV)
    _embed_case(ids, rows, hidden, dtype, scale=1.5)


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
@pytest.mark.parametrize("hidden", [257, 260, 520, 1031])
def test_embedding_of_long_stretches_by_few_lanes(dtype, hidden):
    # stretches of 64 tokens, rows whose last columns a few lanes of a wave hold
    ids = torch.randint(0, 700, (20000,), generator=_gen(hidden), device=DEV)
    _embed_case(ids, 700, hidden, dtype, scale=0.5, padding_idx=3)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_embedding_skewed_and_padded(index):
    g = _gen(30)
    ids = torch.randint(0, 3000, (6, 1500), generator=g, device=DEV)
    ids = torch.where(torch.rand(ids.shape, generator=g, device=DEV) < 0.7, 17, ids).to(index)
    _embed_case(ids, 3000, 128, BF)
    _embed_case(ids, 3000, 130, FP, padding_idx=17)
    _embed_case(ids[:, ::3], 3000, 64, BF, padding_idx=-1)
    _embed_case(torch.full((5000,), 2999, device=DEV, dtype=index), 3000, 72, BF, scale=-0.5)
    runs = torch.arange(4096, device=DEV).div(64, rounding_mode="floor").to(index)  # runs that end on every stretch's end
    _embed_case(runs, 64, 64, FP)
    _embed_case(runs.flip(0), 64, 64, BF)


def test_embedding_ids_outside_the_table():
    ids = torch.tensor([[0, -1, 5], [4, 1 << 40, -(1 << 40)]], device=DEV)
    _embed_case(ids, 5, 64, BF)
    _embed_case(torch.full((100,), -1, device=DEV), 5, 64, FP)


def test_embedding_strides():
    g = _gen(31)
    wide = _randn(g, 100, 3 * 64 + 4, dtype=BF)
    ids = torch.randint(0, 100, (50, 4), generator=g, device=DEV)[:, 1]
    for w in (wide[:, 64:128], wide[:, 1:65], wide[::2, :64].repeat_interleave(2, 0), wide[:64, :100].t(),
              wide[:1, :64].expand(100, 64)):
        assert torch.equal(kotodama_amd.embedding(ids, w), w[ids])
    w = wide[:, :64].detach().clone().requires_grad_(True)
    out = kotodama_amd.embedding(ids, w)
    (one,) = torch.autograd.grad(out.sum(), w)  # a broadcast gradient
    (two,) = torch.autograd.grad(kotodama_amd.embedding(ids, w), w, torch.ones_like(out))
    assert torch.equal(one, two)


def test_embedding_of_one_id_without_dimensions():
    _embed_case(torch.tensor(3, device=DEV), 7, 64, BF, scale=2.0)


def test_embedding_in_an_empty_table():
    w = torch.empty((0, 8), device=DEV, requires_grad=True)
    out = kotodama_amd.embedding(torch.tensor([0, 1], device=DEV), w)
    assert out.isnan().all() and out.shape == (2, 8)
    (dw,) = torch.autograd.grad(out, w, torch.ones_like(out))
    assert dw.shape == (0, 8)


def test_embedding_of_nothing():
    w = torch.ones((10, 64), device=DEV, dtype=BF, requires_grad=True)
    out = kotodama_amd.embedding(torch.zeros((0, 3), device=DEV, dtype=torch.int64), w)
    assert out.shape == (0, 3, 64)
    (dw,) = torch.autograd.grad(out, w, torch.ones_like(out))
    assert dw.shape == w.shape and not dw.any()


def test_embedding_gradient_repeats_bit_for_bit():
    g = _gen(32)
    ids = torch.randint(0, 300, (20000,), generator=g, device=DEV)
    go = _randn(g, 20000, 256, dtype=FP)
    first = lmops.embedding_bwd_op(ids, go, 300, 1.0, -1)
    for _ in range(3):
        assert torch.equal(lmops.embedding_bwd_op(ids, go, 300, 1.0, -1), first)


# ------------------------------------------------ streams, graphs, tracing --


def _layer(x, ids, table, w, norm, cos, sin, lens):
    """Embedding, projections, norms with rotation, attention: one sublayer as a model runs it."""
    x = x + kotodama_amd.embedding(ids, table, scale=2.0)
    b, t, _ = x.shape
    q, k, v = (torch.nn.functional.linear(x, m).unflatten(-1, (-1, 64)).transpose(1, 2) for m in w)
    q, k = kotodama_amd.qk_norm_rope(q, k, norm[0], norm[1], cos, sin, 1e-5)
    o = kotodama_amd.attention(q, k, v, kv_lens=lens, q_start=0)
    return o.transpose(1, 2).reshape(b, t, -1)


def _layer_inputs(seed, dtype=BF):
    g = _gen(seed)
    x = _randn(g, 2, 70, 128, dtype=dtype).requires_grad_(True)
    ids = torch.randint(0, 90, (2, 70), generator=g, device=DEV)
    table = _randn(g, 90, 128, dtype=dtype).requires_grad_(True)
    w = [_randn(g, n * 64, 128, dtype=dtype, scale=0.1).requires_grad_(True) for n in (4, 2, 2)]
    norm = [_randn(g, 64, dtype=dtype).requires_grad_(True) for _ in range(2)]
    cos, sin = _tables(100, 64, dtype)
    lens = torch.tensor([70, 33], device=DEV)
    go = _randn(g, 2, 70, 256, dtype=dtype)
    return (x, ids, table, w, norm, cos, sin, lens), [x, table, *w, *norm], go


def test_operators_together_match_torch_ops():
    # fp32: the same sublayer in plain float64 torch ops; its error there is fp32's over ~1000-term sums
    args, leaves, go = _layer_inputs(40, FP)
    got = [_layer(*args)]
    got += torch.autograd.grad(got[0], leaves, go)
    x, ids, table, w, norm, cos, sin, lens = args
    ref = [t.detach().double().requires_grad_(True) for t in leaves]
    e = ref[0] + torch.nn.functional.embedding(ids, ref[1]) * 2.0
    q, k, v = ((e @ m.t()).unflatten(-1, (-1, 64)).transpose(1, 2) for m in ref[2:5])

    def turn(y, wn):
        y = y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + 1e-5) * wn
        return y * cos[:70].double() + torch.cat((-y[..., 32:], y[..., :32]), -1) * sin[:70].double()

    q, k = turn(q, ref[5]), turn(k, ref[6])
    seen = LO.visible(2, 70, 70, True, lens.tolist(), 0).to(DEV)[:, None]
    s = (q @ k.repeat_interleave(2, 1).transpose(-1, -2) / 8).masked_fill(~seen, -1e300)
    o = (torch.softmax(s, -1) * seen.any(-1, keepdim=True)) @ v.repeat_interleave(2, 1)
    want = [o.transpose(1, 2).reshape(2, 70, -1)]
    want += torch.autograd.grad(want[0], ref, go.double())
    for a, b in zip(got, want):
        assert (a.double() - b).abs().max() <= 1e-4 * b.abs().max()


def test_another_stream():
    args, leaves, go = _layer_inputs(41)
    out = _layer(*args)
    want = [out.detach(), *torch.autograd.grad(out, leaves, go)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = _layer(*args)
        got = [out.detach(), *torch.autograd.grad(out, leaves, go)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_threads_at_once():
    import threading

    cases = [_layer_inputs(50 + i) for i in range(2)]
    want = []
    for args, leaves, go in cases:
        out = _layer(*args)
        want.append([out.detach(), *torch.autograd.grad(out, leaves, go)])
    torch.cuda.synchronize()
    got, errors = [[], []], []

    def work(i):
        try:
            args, leaves, go = cases[i]
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    out = _layer(*args)
                    got[i] = [out.detach(), *torch.autograd.grad(out, leaves, go)]
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001 - reported below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_graphs_that_replay_in_turn():
    # two graphs captured apart, each with its own workspaces, replayed in turn with eager work between
    graphs = []
    for seed in (42, 43):
        args, leaves, go = _layer_inputs(seed)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(_layer(*args), leaves, go)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _layer(*args)
            res = [out.detach(), *torch.autograd.grad(out, leaves, go)]
        del out
        graphs.append((graph, args, leaves, go, res))
    for turn in range(3):
        for graph, args, leaves, go, res in graphs:
            with torch.no_grad():  # new inputs at the same places, other lengths too
                args[0].mul_(0.5 if turn else 1.0)
                args[1].copy_((args[1] * 7 + turn) % 90)
                args[7].copy_(torch.tensor([70 - turn, 20 * turn], device=DEV))
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in res]
            out = _layer(*args)
            want = [out.detach(), *torch.autograd.grad(out, leaves, go)]
            assert all(torch.equal(a, b) for a, b in zip(got, want)), turn


def test_compiled_whole():
    args, leaves, go = _layer_inputs(44)
    out = _layer(*args)
    want = [out.detach(), *torch.autograd.grad(out, leaves, go)]
    fn = torch.compile(_layer, fullgraph=True, dynamic=False)
    out = fn(*args)
    got = [out.detach(), *torch.autograd.grad(out, leaves, go)]
    for a, b in zip(got, want):  # inductor fuses the adds and scalings around the calls: bf16 roundings differ
        assert (a.float() - b.float()).abs().max() <= 2.0**-5 * b.float().abs().max()


class _Native:
    """The native functions: ``taken`` counts the calls they took; with ``off`` they take none."""

    def __init__(self, off):
        self.off, self.taken = off, []

    def __getattr__(self, name):
        from kotodama_amd._native import native

        def call(*args):
            res = None if self.off else getattr(native, name)(*args)
            if res is not None:
                self.taken.append(name)
            return res

        return call


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
def test_native_calls_equal_the_ops(monkeypatch, dtype):
    # bit for bit, recorded and not, and the native path is the one that plain calls take
    results = {}
    for off in (False, True):
        stub = _Native(off)
        monkeypatch.setattr(lmops, "native", stub)
        args, leaves, go = _layer_inputs(46, dtype)
        out = _layer(*args)
        res = [out.detach(), *torch.autograd.grad(out, leaves, go)]
        q = _heads(_gen(47), 2, 4, 30, 64, dtype)
        o, lse = kotodama_amd.attention(q, q[:, :2], q[:, 2:], want_lse=True, scale=0.2, q_start=-3)
        results[off] = [*res, o, lse]
        assert stub.taken == ([] if off else ["embedding", "qk_norm_rope", "attention", "attention"])
    assert all(torch.equal(a, b) for a, b in zip(results[False], results[True]))


def test_calls_left_to_the_ops(monkeypatch):
    stub = _Native(False)
    monkeypatch.setattr(lmops, "native", stub)
    g = _gen(48)
    q = _heads(g, 1, 2, 9, 64, BF)
    odd = _randn(g, 1, 2, 9, 65)[..., 1:]
    kotodama_amd.attention(odd, q, q)  # unaligned rows
    kotodama_amd.embedding(torch.zeros((4, 4), device=DEV, dtype=torch.int64).t()[::2], _randn(g, 5, 8))
    w = _randn(g, 64)
    cos, sin = _tables(9, 64, BF)
    kotodama_amd.qk_norm_rope(q.transpose(-1, -2).contiguous().transpose(-1, -2), q, w, w, cos, sin, 1e-5)
    with torch.overrides.BaseTorchFunctionMode():
        kotodama_amd.attention(q, q, q)
    assert stub.taken == []


@pytest.mark.parametrize("op", ["attention", "qk_norm_rope", "embedding"])
def test_backward_under_compiled_autograd(op):
    # the whole backward of a recorded native call is traced, without a graph break
    def compiler(graph):
        return torch.compile(graph, backend="aot_eager", fullgraph=True)

    g = _gen(49)
    q, k = _heads(g, 2, 4, 9, 64, FP).requires_grad_(True), _heads(g, 2, 2, 9, 64, FP).requires_grad_(True)
    w = [_randn(g, 64, dtype=FP).requires_grad_(True) for _ in range(2)]
    cos, sin = _tables(9, 64, FP)
    ids = torch.randint(0, 64, (5, 7), generator=g, device=DEV)
    lens = torch.tensor([9, 4], device=DEV)
    calls = {
        "attention": ((q, k), lambda: kotodama_amd.attention(q, k, k, kv_lens=lens, q_start=0)),
        "qk_norm_rope": ((q, k, *w), lambda: sum(y.sum(1) for y in kotodama_amd.qk_norm_rope(q, k, *w, cos, sin, 1e-5))),
        "embedding": ((q,), lambda: kotodama_amd.embedding(ids, q[0, 0].reshape(9, 64), scale=0.5)),
    }
    leaves, call = calls[op]
    if op == "embedding":
        ids.remainder_(9)
    torch._dynamo.reset()
    want = torch.autograd.grad(call().square().sum(), leaves)
    for _ in range(2):
        for t in leaves:
            t.grad = None
        loss = call().square().sum()
        with torch._dynamo.compiled_autograd._enable(compiler):
            loss.backward()
        for t, x in zip(leaves, want):
            torch.testing.assert_close(t.grad, x, rtol=1e-6, atol=1e-6)


def test_recorded_calls_appear_in_a_profile():
    args, leaves, go = _layer_inputs(51)
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        torch.autograd.grad(_layer(*args), leaves, go)
    seen = {e.key for e in prof.key_averages() if e.key.startswith("attnres_hip::")}
    assert seen == {f"attnres_hip::{n}{d}" for n in ("attention", "qk_norm_rope", "embedding") for d in ("", "_bwd")}


def test_op_registrations():
    args, _, _ = _layer_inputs(45)
    x, ids, table, w, norm, cos, sin, lens = args
    q = _heads(_gen(1), 2, 4, 9, 64, BF).requires_grad_(True)
    k = _heads(_gen(2), 2, 2, 9, 64, BF).requires_grad_(True)
    torch.library.opcheck(lmops.attention_op, (q, k, k, True, 0.1, lens, None, -(1 << 63)),
                          test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))
    torch.library.opcheck(lmops.qk_norm_rope_op, (q, k, norm[0], norm[1], cos, sin, None, 1e-5),
                          test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))
    torch.library.opcheck(lmops.embedding_op, (ids, table, 1.0, -1),
                          test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))
