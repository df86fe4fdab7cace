"""The oracle of the language-model operators against torch's float64 autograd,
central differences and closed forms, on the CPU."""

import math

import pytest
import torch

from oracle import lm_oracle as LO


def _leaf(g, *shape):
    return torch.randn(shape, generator=g, dtype=torch.float64).requires_grad_(True)


@pytest.mark.parametrize("causal,lens,start", [(True, None, None), (False, None, None), (True, [5, 0], 0),
                                               (False, [3, 7], None), (True, [7, 4], None), (True, None, -2),
                                               (True, [7, 7], [3, 9])])
def test_attention_gradients_are_autograds(causal, lens, start):
    g = torch.Generator().manual_seed(1)
    b, h, hk, tq, tk, d = 2, 4, 2, 6, 7, 8
    q, k, v = _leaf(g, b, h, tq, d), _leaf(g, b, hk, tk, d), _leaf(g, b, hk, tk, d)
    go, gl = torch.randn((b, h, tq, d), generator=g).double(), torch.randn((b, h, tq), generator=g).double()
    seen = LO.visible(b, tq, tk, causal, lens, start)[:, None]
    live = seen.any(-1)
    s = (q @ k.repeat_interleave(2, 1).transpose(-1, -2) / math.sqrt(d)).masked_fill(~seen, -1e300)
    p = torch.softmax(s, -1) * live[..., None]
    out = p @ v.repeat_interleave(2, 1)
    lse = torch.logsumexp(s, -1)
    ((out * go).sum() + (torch.where(live, lse, 0.0) * gl).sum()).backward()
    res = LO.attention(q.detach(), k.detach(), v.detach(), causal, None, lens, start, go, gl)
    torch.testing.assert_close(res["out"][0], out.detach(), rtol=1e-12, atol=1e-13)
    assert torch.equal(res["lse"][0] == -math.inf, ~live.expand(b, h, tq))
    for name, t in (("dq", q), ("dk", k), ("dv", v)):
        torch.testing.assert_close(res[name][0], t.grad, rtol=1e-11, atol=1e-12)


def test_attention_gradients_are_differences():
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn((1, 2, 5, 8), generator=g).double() for _ in range(3))
    go = torch.randn((1, 2, 5, 8), generator=g).double()
    res = LO.attention(q, k, v, grad_out=go)
    step = 1e-6  # central differences: an error of step^2 and of 1e-16 / step
    for name, i in (("dq", 0), ("dk", 1), ("dv", 2)):
        way = torch.randn((1, 2, 5, 8), generator=g).double()
        hi, lo = [q, k, v], [q, k, v]
        hi[i], lo[i] = hi[i] + step * way, lo[i] - step * way
        diff = ((LO.attention(*hi)["out"][0] - LO.attention(*lo)["out"][0]) * go).sum() / (2 * step)
        assert abs(diff.item() - (res[name][0] * way).sum().item()) < 1e-8


def test_attention_of_one_key_is_its_value():
    v = torch.randn(2, 1, 1, 8).double()
    res = LO.attention(torch.randn(2, 3, 1, 8).double(), torch.randn(2, 1, 1, 8).double(), v)
    torch.testing.assert_close(res["out"][0], v.expand(2, 3, 1, 8))


def test_norm_rope_is_autograds_and_keeps_lengths():
    g = torch.Generator().manual_seed(3)
    x, w = _leaf(g, 2, 3, 5, 8), _leaf(g, 8)
    ang = torch.randn((9, 4), generator=g).double()
    cos, sin = torch.cat((ang.cos(), ang.cos()), -1), torch.cat((ang.sin(), ang.sin()), -1)
    rows = torch.randint(0, 9, (2, 5), generator=g)
    go = torch.randn((2, 3, 5, 8), generator=g).double()
    n = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-5) * w
    c, s = cos[rows][:, None], sin[rows][:, None]
    y = n * c + torch.cat((-n[..., 4:], n[..., :4]), -1) * s
    (y * go).sum().backward()
    res = LO.norm_rope(x.detach(), w.detach(), cos, sin, 1e-5, rows, go)
    for name, want in (("y", y.detach()), ("dx", x.grad), ("dw", w.grad)):
        torch.testing.assert_close(res[name][0], want, rtol=1e-11, atol=1e-12)
    torch.testing.assert_close(res["y"][0].norm(dim=-1), n.detach().norm(dim=-1))  # a rotation
    step, way = 1e-6, torch.randn((2, 3, 5, 8), generator=g).double()
    hi, lo = (LO.norm_rope(x.detach() + t * way, w.detach(), cos, sin, 1e-5, rows)["y"][0] for t in (step, -step))
    assert abs((((hi - lo) * go).sum() / (2 * step) - (res["dx"][0] * way).sum()).item()) < 1e-8


def test_embedding_is_autograds():
    g = torch.Generator().manual_seed(4)
    w = _leaf(g, 7, 3)
    ids = torch.tensor([[1, 6, 1], [0, 2, 1]])
    go = torch.randn((2, 3, 3), generator=g).double()
    (torch.nn.functional.embedding(ids, w, padding_idx=2) * 1.5 * go).sum().backward()
    res = LO.embedding(ids, w.detach(), 1.5, 2, go)
    torch.testing.assert_close(res["out"][0], w.detach()[ids] * 1.5)
    torch.testing.assert_close(res["dw"][0], w.grad)
    out = LO.embedding(torch.tensor([-1, 7, 3]), w.detach(), 1.0, None, go[0])
    assert out["out"][0].isnan().all(1).tolist() == [True, True, False]
    assert out["dw"][0].abs().sum(1).nonzero().flatten().tolist() == [3]
