"""Every column is counted once: rows whose logits are 0 or masked, on a B200, where sums of exponentials are whole numbers below 2^24 and exact
whatever their order, so that one column too few or too many (1 / V of the sum) shows.

Tolerances.  ln of an exact count: CUDA's logf and log2f are off by at most one unit in the last place, 2^-23 of the result, products of it by half
of one more; distillation's logarithms are in 64 bits and its loss is rounded once, 2^-24.  A gradient's exponential has the argument -log2(count),
off by one unit of a number below 32 (2^-19), so that it is off by 2^-19 ln 2 = 22 * 2^-24, and by 8 half steps of its own and its products."""
import math

import pytest
import torch

from speedup_thingy_b200 import kernels as K
from tests import test_gpu_token_scores as S

pytestmark = pytest.mark.gpu
DEV, E, INF = S.DEV, S.E, math.inf

# rows by who walks them: a warp, several tiles of a warp, 128 threads, several tiles of 128, clusters of 2 to 8 CTAs
SHAPES = [(3, 1), (3, 7), (3, 50), (5, 300), (3000, 2100), (3000, 4601), (5, 2049), (400, 4099), (300, 20011), (740, 9001), (370, 17000), (150, 33000), (70, 70001), (3, 131075), (1, 300001)]


def rows_of(rows, V, dtype, mask):
    g = torch.Generator(device=DEV).manual_seed(V)
    out = torch.rand(rows, V, device=DEV, generator=g) < torch.rand(rows, 1, device=DEV, generator=g) * 0.5
    out[0] = False                                               # all columns count
    at = torch.randint(0, V, (rows,), device=DEV, generator=g)
    out[torch.arange(rows, device=DEV), at] = False
    return torch.zeros(rows, V, device=DEV).masked_fill_(out, mask).to(dtype), ~out, at


@pytest.mark.parametrize("dtype", S.TYPES)
@pytest.mark.parametrize("mask", [-INF, -3e4])
@pytest.mark.parametrize("rows, V", SHAPES)
def test_scores_count_every_column(rows, V, mask, dtype):
    x, counts, tokens = rows_of(rows, V, dtype, mask)
    n = counts.sum(-1).double()
    for k in (0, min(V, 9)):
        leaf = x.detach().requires_grad_()
        out = K.k_token_logprobs(leaf, tokens, top_k=k, temperature=0.5)
        S.close(out.logprob, -n.log(), 2 * E * n.log(), "logprob")
        S.close(out.entropy, n.log(), 4 * E * n.log(), "entropy")
        dx, = torch.autograd.grad([out.logprob.sum()], [leaf])
        want = counts / n[:, None] * -2.0
        want[torch.arange(rows, device=DEV), tokens] += 2.0
        # (at the token 1 - p: the two are off by half a step of one each)
        S.close(dx, want, want.abs() * torch.finfo(dtype).eps / 2 + counts / n[:, None] * 60 * E + (want > 0) * 4 * E + S.smallest(dtype), "dlogits")


@pytest.mark.parametrize("dtype", S.TYPES)
@pytest.mark.parametrize("mask", [-INF, -3e4])
@pytest.mark.parametrize("rows, V", SHAPES[1:])
def test_distillation_counts_every_column(rows, V, mask, dtype):
    x, counts, tokens = rows_of(rows, V, dtype, mask)
    n = counts.sum(-1).double()
    k = min(V - 1, 40)
    ids = torch.rand(rows, V, device=DEV, generator=torch.Generator(device=DEV).manual_seed(V + 1)).topk(k, -1)[1]
    ids[:, -1] = ids[:, 0]                                       # (twice: left out once)
    inside = torch.zeros_like(counts).scatter_(1, ids, True)
    others = (counts & ~inside).sum(-1).double()
    nothing = torch.full((rows, k), -INF, device=DEV)
    loss = K.k_distill_topk(x, nothing, ids, temperature=0.5, tail=True)          # all of the teacher outside the list
    some = others > 0
    want = torch.where(some, 0.25 * (n.log() - others.clamp(min=1).log()), 0.0)
    if mask == -INF:
        S.close(loss, want, E * want + 1e-14, "the rest")
    else:                                                        # (a rest of masked columns alone is not empty: far below the list)
        S.close(loss[some], want[some], E * want[some] + 1e-14, "the rest")
    one = torch.where(torch.arange(k, device=DEV) == 0, 0.0, -INF).expand(rows, k)
    ids[:, 0] = tokens                                           # all of it at one token
    for tail in (False, True):
        loss = K.k_distill_topk(x, one, ids, temperature=0.5, tail=tail)
        S.close(loss, 0.25 * n.log(), E * n.log() + 1e-14, "one token")
