"""The bf16 training step of kotodama_amd.lmstep on this package's embedding, norms
with rotation and attention, against the same model in float64.

Bar: the error of the same step on torch ops.  Both round weights, activations
and gradients to bf16 at the same places; between those the torch ops round
more often (after the norm, each product of the rotation and their sum) and
the kernels once, and both round the probabilities for the product with the
values.  So the kernels' error, as a norm over each gradient, is at most about
the torch ops'; it may be twice that, plus the one rounding that every gradient
ends with."""

import copy

import pytest
import torch

from kotodama_amd import lmstep, workloads

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


@pytest.fixture(autouse=True)
def _eager():
    yield
    lmstep.compile_sublayers(False)


def _step(model, ids, labels, residual):
    model.zero_grad(set_to_none=True)
    loss = model(ids, labels, residual)
    loss.backward()
    return loss.item(), {n: p.grad.double() for n, p in model.named_parameters() if p.grad is not None}


def _route(buf, query, norm, mask, num_active):
    rsqrt = torch.rsqrt(buf.pow(2).mean(-1) + norm.eps)
    logits = ((buf * (query * norm.weight)).sum(-1) * rsqrt).masked_fill(~mask.view(-1, 1, 1), float("-inf"))
    return (torch.softmax(logits, dim=0).unsqueeze(-1) * buf).sum(0)


@pytest.mark.parametrize("residual", ["standard", "attnres"])
@pytest.mark.parametrize("compiled", [False, True])
def test_training_step_bf16(compiled, residual):
    c = lmstep.LMConfig("t", 512, 3, 4, 2, 128, 384, vocab_size=1000, attn_res_n_blocks=2, batch=2, seq=320)
    model = lmstep.LanguageModel(c, DEV, seed=21)
    g = torch.Generator(device=DEV).manual_seed(22)
    with torch.no_grad():  # norms away from one, routing away from uniform
        for name, p in model.named_parameters():
            if "res_query" in name:
                p.copy_(torch.randn(p.shape, generator=g, device=DEV) * 0.2)
            elif "norm" in name:
                p.add_(torch.randn(p.shape, generator=g, device=DEV) * 0.1)
    ids, labels = lmstep.make_batch(c, DEV, seed=23)
    lmstep.compile_sublayers(False)
    ref_loss, ref = _step(model, ids, labels, residual)
    exact = copy.deepcopy(model).double()
    loop = residual if residual == "standard" else (lambda m, x: workloads.stacked_training_forward(m, x, _route))
    exact_loss, want = _step(exact, ids, labels, loop)
    lmstep.compile_sublayers(compiled, kernels=True)
    loss, got = _step(model, ids, labels, residual)
    assert abs(loss - exact_loss) <= 2 * abs(ref_loss - exact_loss) + 2.0**-8 * abs(exact_loss)
    assert got.keys() == want.keys()
    over = {}
    for name, w in want.items():
        err, bar = (got[name] - w).norm().item(), 2 * (ref[name] - w).norm().item() + 2.0**-8 * w.norm().item()
        size = max(w.norm().item(), 1e-300)  # a routing point of one source has a zero gradient
        print(f"{name}: {err / size:.3g} of its norm, bar {bar / size:.3g}")
        if not err <= bar:
            over[name] = err / bar
    assert not over
