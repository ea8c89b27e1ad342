"""Derivatives that the operators at the two ends of the vocabulary do not have, on a B200: forward mode and second derivatives are refused
by name, never dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from speedup_thingy_b200 import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def inputs():
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(4, 40, device=DEV, generator=g)
    tokens = torch.tensor([1, 2, 3, 39], device=DEV)
    top, ids = torch.log_softmax(x * 0.5, -1).topk(5)
    return x, tokens, top, ids


CALLS = {
    "scores": lambda x: K.k_token_logprobs(x, inputs()[1], top_k=2).logprob,
    "distillation": lambda x: K.k_distill_topk(x, *inputs()[2:], tail=True),
    "embedding": lambda x: K.k_embedding(inputs()[1] % 4, x, scale=2.0),
}


@pytest.mark.parametrize("needs_grad", [False, True])
@pytest.mark.parametrize("grad_mode", [False, True])
@pytest.mark.parametrize("name", CALLS)
def test_forward_mode_is_refused(name, grad_mode, needs_grad):
    x = inputs()[0].requires_grad_(needs_grad)
    with fwd.dual_level(), torch.set_grad_enabled(grad_mode):
        dual = fwd.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="jvp"):
            CALLS[name](dual)
        CALLS[name](x)                                           # (no tangent: as ever)


def test_a_teachers_tangent_is_refused():
    x, _, top, ids = inputs()
    with fwd.dual_level(), pytest.raises(RuntimeError, match="jvp"):
        K.k_distill_topk(x, fwd.make_dual(top, torch.ones_like(top)), ids)


@pytest.mark.parametrize("name", CALLS)
def test_second_derivatives_are_refused(name):
    x = inputs()[0].requires_grad_()
    y = CALLS[name](x)
    g = torch.ones_like(y).requires_grad_()
    dx, = torch.autograd.grad([y], [x], [g], create_graph=True)
    plain, = torch.autograd.grad([CALLS[name](x)], [x], [g])
    assert torch.equal(dx.detach(), plain) and not plain.requires_grad       # the first derivative is as ever
    for of in (g,) if name == "embedding" else (x, g):           # (a table's gradient does not depend on the table)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            torch.autograd.grad([(dx * dx).sum() + (x * x).sum() + (g * g).sum()], [of], retain_graph=True)


@pytest.mark.parametrize("name", CALLS)
def test_a_gradient_with_a_graph_can_be_changed_in_place(name):
    x = inputs()[0].requires_grad_()
    want, = torch.autograd.grad([CALLS[name](x).sum()], [x])
    for how in ("grad", "backward"):
        if how == "grad":
            dx, = torch.autograd.grad([CALLS[name](x).sum()], [x], create_graph=True)
        else:
            CALLS[name](x).sum().backward(create_graph=True)
            dx = x.grad
        with torch.no_grad():
            dx.mul_(0.5)
        dx.detach_()
        assert torch.equal(dx, 0.5 * want) and not dx.requires_grad
        x.grad = None
