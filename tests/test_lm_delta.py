"""The row sums of the attention backward where a row sees few keys.

ds = p (dp - delta), delta = sum_j p_j dp_j = sum_d do_d o_d.  Where every row of
a tile sees at most 256 keys the bf16 kernels take the first form, as the second
reads an output that was rounded to bf16.  Here the values lie on 64 and 64.5
with a mean near 64.2, which bf16 rounds to 64: read off that output, delta is
off by about 0.2 a column, 13 in 64 columns, where dp - delta is about 2.  The
bound of the first form (oracle, ``delta_from_p``) counts fp32 roundings of dp
and delta and the bf16 one of ds; on the CPU both forms are computed and the
second one is shown to break it."""

import math

import pytest
import torch

from oracle import lm_oracle as LO

BF = torch.bfloat16


def _inputs(b, h, hk, tq, tk, d, device, seed):
    g = torch.Generator().manual_seed(seed)

    def rows(n, t, x):
        return x(torch.randn((b, t, n, d), generator=g)).to(BF).to(device).transpose(1, 2)

    q = rows(h, tq, lambda x: 0.3 * x)
    k = rows(hk, tk, lambda x: 1 + 0.2 * x)
    v = rows(hk, tk, lambda x: 64 + 0.5 * (x > 0.2533))  # 0.4 of them
    go = rows(h, tq, lambda x: 1 + 0.3 * x)
    return q, k, v, go


def _worst(got, want):
    value, bound = want
    return ((got.double() - value).abs() / bound.clamp_min(1e-300)).max().item()


def _emulated(q, k, v, go, from_p):
    """dq and dk of whole causal sequences in fp32 with the kernel's roundings."""
    b, h, t, d = q.shape
    rep = h // k.shape[1]
    qf, gf = q.float(), go.float()
    kf, vf = (x.float().repeat_interleave(rep, 1) for x in (k, v))
    seen = torch.ones(t, t, dtype=torch.bool).tril()
    s = (qf @ kf.transpose(-1, -2) / math.sqrt(d)).masked_fill(~seen, -math.inf)
    p = torch.exp(s - torch.logsumexp(s, -1, keepdim=True))
    out = (p.to(BF).float() @ vf).to(BF).float()
    dp = gf @ vf.transpose(-1, -2)
    delta = (p * dp).sum(-1, keepdim=True) if from_p else (gf * out).sum(-1, keepdim=True)
    ds = (p * (dp - delta)).to(BF).float()
    dq = ds @ kf / math.sqrt(d)
    dk = (ds.transpose(-1, -2) @ qf / math.sqrt(d)).view(b, -1, rep, t, d).sum(2)
    return {"dq": dq.to(BF), "dk": dk.to(BF)}


@pytest.mark.parametrize("t,d", [(150, 64), (256, 128)])
def test_the_bound_tells_the_two_forms_apart(t, d):
    q, k, v, go = _inputs(1, 4, 2, t, t, d, "cpu", t)
    want = LO.attention(q, k, v, grad_out=go, delta_from_p=True)
    for from_p in (True, False):
        for name, got in _emulated(q, k, v, go, from_p).items():
            if from_p:
                assert _worst(got, want[name]) <= 1.0, name
            else:
                assert _worst(got, want[name]) > 3.0, name


@pytest.mark.gpu
@pytest.mark.parametrize("b,h,hk,tq,tk,d,causal", [
    (1, 4, 2, 150, 150, 64, True),      # four waves share their rows
    (1, 4, 2, 256, 256, 128, True),     # as many keys as this form is taken for
    (1, 4, 2, 40, 256, 128, False),
    (2, 6, 2, 33, 200, 96, True),       # behind a cache
    (6, 32, 16, 200, 200, 64, True),    # two do
    (12, 32, 16, 190, 190, 128, True),  # none do
    (1, 2, 1, 1, 129, 32, True),
])
def test_rows_of_few_keys(b, h, hk, tq, tk, d, causal):
    import kotodama_amd

    print(f"delta b={b} h={h}/{hk} q={tq} k={tk} d={d} causal={causal}", flush=True)
    q, k, v, go = _inputs(b, h, hk, tq, tk, d, "cuda", tq + tk)
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    dq, dk, dv = torch.autograd.grad(kotodama_amd.attention(*leaves, causal=causal), leaves, go)
    want = LO.attention(q, k, v, causal, grad_out=go, delta_from_p=True)
    for name, got in (("dq", dq), ("dk", dk), ("dv", dv)):
        assert _worst(got, want[name]) <= 1.0, f"{name}: {_worst(got, want[name]):.3g} times its bound"
