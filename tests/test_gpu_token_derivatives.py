"""Derivatives that the operators at the two ends of the vocabulary do not have, on a B200: forward mode is refused
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
