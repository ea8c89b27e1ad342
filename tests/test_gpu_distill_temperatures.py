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
    check(x, t, ids, T, tail)


@pytest.mark.parametrize("dtype", S.TYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("copies, V", [(1, 40), (300, 2100), (1, 3000), (40, 9001), (1, 40001)])
def test_lists_and_rows_in_every_state(copies, V, tail, dtype):
    k, T = 12, 20.0
    x = S.made(12, V, dtype)
    t, ids = S.a_teacher(x, k, T)
    t, ids = t.clone(), ids.clone()
    ids[0, 5:] = -1                                              # a short list
    t[0, 5:] = float("nan")                                      # (what an unused slot holds is not looked at)
    ids[1] = -1                                                  # none
    x[1] = float("nan")
    ids[2, 3] = ids[2, 0]                                        # a token named twice
    ids[3] = ids[3, 0]                                           # a token named by every slot
    t[3] = math.log(0.05)
    t[4, 2:] = -math.inf                                         # slots without probability
    x[5, ids[5, 1]] = -math.inf                                  # the student cannot say it: infinite loss
    x[6].masked_fill_(torch.arange(V, device=DEV) % 2 == 0, -math.inf)
    t[6].masked_fill_(ids[6] % 2 == 0, -math.inf)
    x[7] = -math.inf                                             # a student without a distribution
    keep = torch.zeros(V, dtype=torch.bool, device=DEV)
    keep[ids[9]] = True
    x[9].masked_fill_(~keep, -math.inf)                          # nothing left outside the list
    x[10].masked_fill_(~keep, -3e4)                              # next to nothing
    ids[11, 1::2] = -5
    x, t, ids = x.repeat(copies, 1), t.repeat(copies, 1), ids.repeat(copies, 1)
    loss = check(x, t, ids, T, tail)
    assert loss[1] == 0 and loss[5] == math.inf and loss[7] == math.inf
    assert torch.equal(loss, K.k_distill_topk(x, t, ids, temperature=T, tail=tail))       # without a gradient: the same bits
    for row in (8, 11):                                          # what is not a number stays in its row
        y = x.clone()
        y[row, 3] = float("nan") if row == 8 else math.inf
        leaf = y.requires_grad_()
        bad = K.k_distill_topk(leaf, t, ids, temperature=T, tail=tail)
        dx, = torch.autograd.grad([bad.sum()], [leaf])
        assert bad[row].isnan() and dx[row].isnan().any()
        others = torch.arange(len(x), device=DEV) != row
        assert torch.equal(bad[others], loss[others]) and not dx[others].isnan().any()


def check(x, t, ids, T, tail):
    V, dtype = x.shape[-1], x.dtype
    leaf = x.detach().requires_grad_()
    loss = K.k_distill_topk(leaf, t, ids, temperature=T, tail=tail)
    want, dz, r = S.distill64(x, t, ids, T, tail)
    S.close(loss, want, 2 * E * want.abs().nan_to_num(0, 0, 0) + T * T * 2.0 ** -43, "loss")
    dx, = torch.autograd.grad([loss], [leaf], [torch.ones_like(loss)])
    # outside the list: the exponential's argument and its own half steps (as in S.check_distill), relative to the gradient
    outside = dz.abs() * (16 + 4 * r["logp"].abs().nan_to_num(0, 0, 0) + 2 * math.log2(V)) * E
    S.close(dx, dz, torch.finfo(dtype).eps / 2 * dz.abs() + outside + T * 2.0 ** -45 + S.smallest(dtype), "dlogits")
    return loss.detach()
