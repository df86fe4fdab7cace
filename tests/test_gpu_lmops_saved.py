"""The recorded language-model operators under saved-tensor hooks: what comes back
unchanged gives the same gradients, and what comes back in another shape or
type is refused before anything is launched."""

import pytest
import torch

import kotodama_amd

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
BF = torch.bfloat16


def _attention(unpack):
    g = torch.Generator(device=DEV).manual_seed(3)
    q, k, v, go = (torch.randn((2, n, 33, 64), generator=g, device=DEV).to(BF) for n in (4, 2, 2, 4))
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        out = kotodama_amd.attention(*leaves)
    return torch.autograd.grad(out, leaves, go)


def _embedding(unpack):
    g = torch.Generator(device=DEV).manual_seed(4)
    w = torch.randn((50, 64), generator=g, device=DEV).requires_grad_(True)
    ids = torch.randint(0, 50, (6, 7), generator=g, device=DEV)
    go = torch.randn((6, 7, 64), generator=g, device=DEV)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        out = kotodama_amd.embedding(ids, w)
    return torch.autograd.grad(out, w, go)


@pytest.mark.parametrize("call", [_attention, _embedding])
def test_saved_tensors_through_hooks(call):
    assert all(torch.equal(a, b) for a, b in zip(call(lambda t: t.clone()), call(lambda t: t)))


@pytest.mark.parametrize("call,change,error", [
    (_attention, lambda t: t[:1] if t.dim() == 3 else t, ValueError),                # lse
    (_attention, lambda t: t.to(BF) if t.dim() == 3 else t, TypeError),
    (_attention, lambda t: t[..., :32] if t.shape[1] == 4 and t.dim() == 4 else t, ValueError),  # q and out
    (_embedding, lambda t: t[:2], ValueError),
    (_embedding, lambda t: t.repeat(2, 1), ValueError),
])
def test_saved_tensors_that_do_not_fit(call, change, error):
    with pytest.raises(error):
        call(change)
