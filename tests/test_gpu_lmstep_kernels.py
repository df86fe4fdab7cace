"""The language model of kotodama_amd.lmstep with its embedding and attention on
this package's kernels, and behind a KV cache.

Bars: the fp32 step's loss and gradients against the same model in float64
torch ops, within five times the error of the fp32 torch-ops step plus 2e-4 of
each gradient's largest element (the bar of the routing's own whole-step test:
either fp32 path's roundings grow alike through the layers).  Decoding token by
token against the whole sequence at once computes the same sums in other
tilings: fp32, within 2e-4 of the largest logit."""

import copy

import pytest
import torch

from kotodama_amd import lmstep

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


@pytest.fixture(autouse=True)
def _eager():
    yield
    lmstep.compile_sublayers(False)


def _model(dtype, layers=3, seq=96, seed=5, hidden=512):
    c = lmstep.LMConfig("t", hidden, layers, 4, 2, 128, 384, vocab_size=1000, attn_res_n_blocks=2, batch=2, seq=seq)
    model = lmstep.LanguageModel(c, DEV, dtype=dtype, seed=seed)
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    with torch.no_grad():  # routing away from uniform, norms away from one
        for name, p in model.named_parameters():
            if "res_query" in name:
                p.copy_((torch.randn(p.shape, generator=g, device=DEV) * 0.2).to(dtype))
            elif "norm" in name:
                p.add_((torch.randn(p.shape, generator=g, device=DEV) * 0.1).to(dtype))
    return c, model


def _step(model, ids, labels, residual):
    model.zero_grad(set_to_none=True)
    loss = model(ids, labels, residual)
    loss.backward()
    return loss.item(), {n: p.grad.detach().clone() for n, p in model.named_parameters() if p.grad is not None}


@pytest.mark.parametrize("residual", ["standard", "attnres"])
def test_training_step_fp32(residual):
    c, model = _model(torch.float32)
    ids, labels = lmstep.make_batch(c, DEV, seed=7)
    lmstep.compile_sublayers(False)
    ref_loss, ref = _step(model, ids, labels, residual)
    lmstep.compile_sublayers(False, kernels=True)
    loss, got = _step(model, ids, labels, residual)
    lmstep.compile_sublayers(False)
    exact = copy.deepcopy(model).double()
    if residual == "attnres":  # the routing kernels take no float64: the reference loop
        from kotodama_amd import workloads

        def route(buf, query, norm, mask, num_active):
            qw = query * norm.weight
            rsqrt = torch.rsqrt(buf.pow(2).mean(-1) + norm.eps)
            logits = ((buf * qw).sum(-1) * rsqrt).masked_fill(~mask.view(-1, 1, 1), float("-inf"))
            return (torch.softmax(logits, dim=0).unsqueeze(-1) * buf).sum(0)

        residual = lambda m, x: workloads.stacked_training_forward(m, x, route)  # noqa: E731
    exact_loss, want = _step(exact, ids, labels, residual)
    assert abs(loss - exact_loss) <= 5 * abs(ref_loss - exact_loss) + 1e-6
    assert got.keys() == want.keys()
    for name, w in want.items():
        bar = 5 * (ref[name].double() - w).abs().max().item() + 2e-4 * w.abs().max().item()
        assert (got[name].double() - w).abs().max().item() <= bar, name


@pytest.mark.parametrize("compiled", [False, True])
def test_training_steps_bf16(compiled):
    c, model = _model(torch.bfloat16, seq=128)
    opt = lmstep.optimizer(model)
    ids, labels = lmstep.make_batch(c, DEV, seed=9)
    lmstep.compile_sublayers(compiled, kernels=True)
    for residual in ("standard", "attnres"):
        for _ in range(2):
            loss, grads = _step(model, ids, labels, residual)
            assert loss == loss and all(torch.isfinite(g).all().item() for g in grads.values())
            opt.step()


@pytest.mark.parametrize("prompt", [1, 40])
def test_decoding_behind_a_cache(prompt):
    c, model = _model(torch.float32, seq=64)
    ids, _ = lmstep.make_batch(c, DEV, seed=11)
    whole, past = model.logits(ids)
    assert whole.shape == (2, 64, 1000) and past[0][0].shape == (2, 2, 64, 128)
    scale = whole.abs().max().item()
    got, past = model.logits(ids[:, :prompt])
    rows = [got]
    for t in range(prompt, 64):
        got, past = model.logits(ids[:, t:t + 1], past)
        rows.append(got)
    assert (torch.cat(rows, 1) - whole).abs().max().item() <= 2e-4 * scale
    with pytest.raises(ValueError, match="rope tables"):
        model.logits(ids[:, :1], past)
    # and the uncached forward's hidden states give the same logits
    with torch.no_grad():
        lmstep.compile_sublayers(False, kernels=True)
        x = model.hidden_states(ids, "attnres")
        x = torch.nn.functional.linear(lmstep._rms(x, model.norm.weight, c.norm_eps), model.embed)
    assert (x - whole).abs().max().item() <= 2e-4 * scale
