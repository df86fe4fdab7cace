"""Forward-mode derivatives of the language-model operators are refused, whichever
input has the tangent and whether the call is recorded or not."""

import pytest
import torch
from torch.autograd import forward_ad

import kotodama_amd


def _inputs(op, device):
    def t(*s):
        return torch.ones(s, dtype=torch.bfloat16, device=device)

    if op == "attention":
        return [t(1, 2, 4, 64), t(1, 2, 4, 64), t(1, 2, 4, 64)], lambda q, k, v: kotodama_amd.attention(q, k, v)
    if op == "qk_norm_rope":
        return ([t(1, 2, 4, 64), t(1, 2, 4, 64), t(64), t(64), t(4, 64), t(4, 64)],
                lambda *a: kotodama_amd.qk_norm_rope(*a, 1e-5))
    return [t(5, 64)], lambda w: kotodama_amd.embedding(torch.zeros(3, dtype=torch.int64, device=device), w)


OPS = ["attention", "qk_norm_rope", "embedding"]


def _refused(op, device):
    args, call = _inputs(op, device)
    for grad in (False, True):
        for i in range(len(args)):
            with forward_ad.dual_level():
                leaves = [a.clone() for a in args]
                if grad:
                    leaves[0].requires_grad_(True)
                leaves[i] = forward_ad.make_dual(leaves[i], torch.ones_like(args[i]))
                with pytest.raises(NotImplementedError, match="forward"):
                    call(*leaves)
                with torch.no_grad(), pytest.raises(NotImplementedError, match="forward"):
                    call(*leaves)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(call, tuple(args), tuple(torch.ones_like(a) for a in args))


@pytest.mark.parametrize("op", OPS)
def test_tangents_are_refused(op):
    _refused(op, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("op", OPS)
def test_tangents_are_refused_on_the_gpu(op):
    _refused(op, "cuda")
    args, call = _inputs(op, "cuda")
    with forward_ad.dual_level():  # a level without tangents changes nothing
        got = call(*args)
    want = call(*args)
    for a, b in zip(*((x if isinstance(x, tuple) else (x,)) for x in (got, want))):
        assert torch.equal(a, b)
