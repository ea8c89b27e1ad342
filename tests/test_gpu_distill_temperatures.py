"""Distillation at high temperatures on a B200, where the loss is the square of the temperature times a divergence that falls with it: against
64 bits, relative to the loss.

Tolerances.  The divergence is a sum of terms in 64 bits, each off by a few dozen 2^-53 of numbers below 16, in the operator and in the definition
alike: T^2 2^-43.  The result is rounded to fp32, and the definition's terms with it: 2 2^-24.  A gradient is T times a difference of
probabilities in 64 bits, on the list T 2^-45; outside it is rounded like any other."""
import math

import pytest
import torch

from speedup_thingy_b200 import kernels as K
from tests import test_gpu_token_scores as S

pytestmark = pytest.mark.gpu
DEV, E = S.DEV, S.E


@pytest.mark.parametrize("dtype", S.TYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("T", [8.5, 20.0, 100.0, 1e3, 1e4])
@pytest.mark.parametrize("rows, V, k", [(3, 5, 5), (5, 200, 200), (4, 256, 100), (3000, 2100, 20), (9, 3000, 12), (300, 9001, 30), (5, 40001, 9)])
def test_the_loss_keeps_its_digits(rows, V, k, T, tail, dtype):
    x = S.made(rows, V, dtype)
    x[0, 1] = -math.inf
    x[1, V // 2] = -1e4
    t, ids = S.a_teacher(x, k, T)
    ids = ids.clone()
    if k < V:
        ids[2, 1], ids[2, 3] = ids[2, 0], -1                     # twice, and an unused slot
    leaf = x.detach().requires_grad_()
    loss = K.k_distill_topk(leaf, t, ids, temperature=T, tail=tail)
    want, dz, r = S.distill64(x, t, ids, T, tail)
    S.close(loss, want, 2 * E * want.abs().nan_to_num(0, 0, 0) + T * T * 2.0 ** -43, "loss")
    dx, = torch.autograd.grad([loss], [leaf], [torch.ones_like(loss)])
    # outside the list: the exponential's argument and its own half steps (as in S.check_distill), relative to the gradient
    outside = dz.abs() * (16 + 4 * r["logp"].abs().nan_to_num(0, 0, 0) + 2 * math.log2(V)) * E
    S.close(dx, dz, torch.finfo(dtype).eps / 2 * dz.abs() + outside + T * 2.0 ** -45 + S.smallest(dtype), "dlogits")
