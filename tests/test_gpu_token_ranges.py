"""Scores and distillation where a row's logits are far from zero on a B200: masks of a finite constant and logits whose exponents relative
to zero leave fp32's digits, against the definitions in 64 bits and the tolerances of test_gpu_token_scores.py (temperatures are
fp32 numbers, so that they bring no error of their own).

The distillation's definition is written out once more: with log probabilities of -1e13 and beyond, 64 bits do not hold what is added to them, and
the rest's share is formed among the rest itself.  Its gradient's tolerance counts one thing more: probabilities below 2^-126 are flushed
to zero before they are multiplied by T g and at most M + 1."""
import math

import pytest
import torch

from speedup_thingy_b200 import kernels as K
from tests import test_gpu_token_scores as S

pytestmark = pytest.mark.gpu
DEV = S.DEV
INF = math.inf


def fp32(x):
    return torch.tensor(x, dtype=torch.float32).item()


def check_distill(x, teacher, ids, T, tail, seed=0):
    V, dtype = x.shape[-1], x.dtype
    leaf = x.detach().requires_grad_()
    loss = K.k_distill_topk(leaf, teacher, ids, temperature=T, tail=tail)
    t = teacher.double()
    if not tail:
        t = t - t.logsumexp(-1, keepdim=True)
    q = t.exp()
    M = q.sum(-1)
    xd = x.double()
    z = (xd - xd.amax(-1, keepdim=True)) / T
    logp = z - z.logsumexp(-1, keepdim=True)
    p, lp = logp.exp(), logp.gather(-1, ids)
    want = torch.where(q == 0, 0.0, q * (t - lp)).sum(-1)
    qd = torch.zeros_like(p).scatter_add_(-1, ids, q)
    dz = T * (M[..., None] * p - qd)
    if tail:
        outside = torch.zeros_like(p, dtype=torch.bool).scatter_(-1, ids, True)
        high = xd.masked_fill(outside, -INF).amax(-1, keepdim=True)
        r = (1 - M).clamp(min=0.0).masked_fill(high[..., 0] == -INF, 0.0)
        share = ((xd - high.clamp(min=-1e300)) / T).masked_fill(outside, -INF).softmax(-1).nan_to_num(0.0)
        lnP = logp.masked_fill(outside, -INF).logsumexp(-1).masked_fill(high[..., 0] == -INF, 0.0)
        want = want + torch.where(r > 0, r * (r.clamp(min=1e-300).log() - lnP), 0.0)
        M = M + r
        dz = T * (M[..., None] * p - qd - r[..., None] * share)
    want = T * T * want
    err, lnv = S.lse_error(V), math.log(V)
    size = torch.where(q == 0, 0.0, q * (teacher.double().abs() + lp.abs() + lnv + 2)).sum(-1) + lnv + 20
    S.close(loss, want, T * T * ((M + 1) * 3 * err + 8 * S.E * size) + S.E * want.abs(), "loss")
    g = torch.randn(want.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed + 9)) * (64.0 if dtype == torch.float16 else 1.0)
    dx, = torch.autograd.grad([loss], [leaf], [g])
    scale = T * g.abs().double()[..., None]
    dz = dz * g.double()[..., None]
    part = p * (M[..., None] + 1) * (4 * err + torch.where(p > 0, 16 + 4 * logp.abs(), 0.0) * S.E) + qd * 64 * S.E
    rest = (dz.abs() + scale * p * M[..., None]) * 8 * err if tail else 0.0
    S.close(dx, dz, torch.finfo(dtype).eps / 2 * dz.abs() + 8 * S.E * dz.abs() + part * scale + rest + scale * (M[..., None] + 1) * 2.0 ** -126 + S.smallest(dtype), "dlogits")


def masked_rows(V, dtype, mask, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    n = torch.arange(V, device=DEV)
    x = S.made(9, V, dtype, seed=seed)
    x[0].masked_fill_(torch.rand(V, device=DEV, generator=g) < 0.99, mask)
    x[1, : V // 2] = mask
    x[2, V // 2:] = mask
    x[3] = mask
    x[3, V // 3] = 1.5                                           # one token left
    x[4] = mask                                                  # none left: all alike
    x[5] = torch.where(n % 2 == 0, mask, max(2 * mask, torch.finfo(dtype).min))
    x[6].masked_fill_((n // 512) % 2 == 0, mask)                 # whole tiles of a warp
    x[7, 1:] = torch.where(n[1:] % 3 == 0, -INF, mask)
    x[8].masked_fill_((n // 8) % 16 != 3, mask)
    return x


@pytest.mark.parametrize("dtype", S.TYPES)
@pytest.mark.parametrize("T", [1.0, 0.125, 2.0, 2.0 ** -17])
# rows by who walks them: a warp, several tiles of a warp, 128 threads, a cluster of 256
@pytest.mark.parametrize("copies, V", [(1, 50), (330, 2100), (1, 3000), (40, 20011), (1, 40001)])
def test_masks_of_a_finite_constant(copies, V, T, dtype):
    masks = [-1e4, -3e4] if dtype == torch.float16 else [-1e4, -1e9, -1e10, -1e11, -1e12, -1e15, -1e18, -1e20, -1e25, -9e28, -2e29, -1e30]
    for i, mask in enumerate(masks):
        x = masked_rows(V, dtype, mask, seed=i).repeat(copies, 1)
        tokens = torch.randint(0, V, (x.shape[0],), device=DEV, generator=torch.Generator(device=DEV).manual_seed(i))
        tokens[3] = V // 3
        out = S.check_scores(x, tokens, 7, T)
        # one term, 2^(the reference's rounding): the exponential is off by 2^-22.5 = 2.9 half steps, its logarithm by that and the rest's rounding
        assert -4 * S.E <= out.logprob[3] <= 0 and 0 <= out.entropy[3] <= 4 * S.E
        assert abs(out.entropy[4].item() - math.log(V)) < 1e-5 * math.log(V)
        teacher, ids = S.a_teacher(x, 6, T)
        for tail in (False, True):
            check_distill(x, teacher, ids, T, tail)


@pytest.mark.parametrize("dtype", S.TYPES)
@pytest.mark.parametrize("V", [50, 3000, 40001])
@pytest.mark.parametrize("T", [1.0000001e-6, 1e-5, 1e-4, 0.03, 1.0, 128.0])      # (the first of them: the least fp32 number that is not below 1e-6)
def test_logits_far_from_zero(V, T, dtype):
    T = fp32(T)
    tops = [5e3, 3e4, 6.5e4, -5e3, -6.5e4]
    if dtype != torch.float16:
        tops += [1e7, 1e9, 1e10, 1e12, 1e20, 1e28, -1e9, -1e10, -1e12, -1e20, -1e28]
    g = torch.Generator(device=DEV).manual_seed(V)
    steps = torch.randint(0, 30, (len(tops), V), device=DEV, generator=g)      # neighbouring values of the type, below the largest
    x = (torch.tensor(tops, device=DEV, dtype=torch.float64)[:, None] * (1 - torch.finfo(dtype).eps * steps)).to(dtype)
    tokens = torch.randint(0, V, (len(tops),), device=DEV, generator=g)
    S.check_scores(x, tokens, 5, T)
    for tail in (False, True):
        check_distill(x, *S.a_teacher(x, 6, T), T, tail)
