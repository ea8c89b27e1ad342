"""`k_token_logprobs` and `k_distill_topk` on a B200 against their definitions in 64 bits.

Tolerances.  e = 2^-24 is half a step of fp32.  With d = (x - max) / T, an exponential is off by at most (4 + 2 |d|) e relative (two
roundings of its argument, four half steps of the exponential), which is at most (4 + 2 H') e of the sum with H' = sum p |d| <= ln V; a sum
of fp32 terms of one sign by at most (terms one after the other) e: a thread adds no more than V / 32 of them, and fewer than 64
steps join the threads.  So ln s is off by at most LSE = (70 + V / 32 + 2 ln V) e, and what is made of it by that and a few half steps of
its own size."""
import math

import pytest
import torch

from speedup_thingy_b200 import kernels as K
from speedup_thingy_b200._abi import RteError

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float16, torch.float32]
INF = math.inf


def lse_error(V):
    return (70 + V / 32 + 2 * math.log(V)) * E


def smallest(dtype):
    """Half of the type's smallest step (fp32 results that small are flushed to zero)."""
    return {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126}[dtype]


def made(rows, V, dtype, seed=0, spread=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed * 1009 + V)
    return (torch.randn(rows, V, device=DEV, generator=g) * spread).to(dtype)


# --------------------------------------------------------------------------- definitions in 64 bits
def scores64(x, tokens, k, T, ignore=-100):
    """logprob, entropy, top_logprobs, top_ids and what the gradients need."""
    V = x.shape[-1]
    x = x.detach().double()
    skip = (tokens == ignore) | (tokens < 0) | (tokens >= V)
    empty = (x == -INF).all(-1)
    safe = x.masked_fill((empty | skip)[..., None], 0.0)
    logp = torch.log_softmax(safe / T, -1)
    logp = logp.masked_fill(empty[..., None], -INF)
    p = logp.exp()
    plogp = torch.where(p > 0, p * logp, torch.zeros_like(p)) if not logp.isnan().any() else torch.where(p == 0, torch.zeros_like(p), p * logp)
    H = -plogp.sum(-1)
    at = tokens.long().masked_fill(skip, 0)
    lp = logp.gather(-1, at[..., None])[..., 0].masked_fill(skip, 0.0)
    order = x.sort(dim=-1, descending=True, stable=True)[1][..., :k]
    top = logp.gather(-1, order).masked_fill(skip[..., None], 0.0)
    ids = order.masked_fill(skip[..., None], -1)
    return lp, H.masked_fill(skip, 0.0), top, ids, dict(skip=skip, empty=empty, logp=logp, p=p, plogp=plogp, H=H, at=at, order=order, T=T)


def scores_gradient64(r, g, gh, gt):
    up = torch.zeros_like(r["p"])
    up.scatter_add_(-1, r["at"][..., None], g.double()[..., None])
    if gt is not None and gt.shape[-1]:
        up.scatter_add_(-1, r["order"], gt.double())
    dx = up - r["p"] * up.sum(-1, keepdim=True) - gh.double()[..., None] * (r["plogp"] + r["p"] * r["H"][..., None])
    return (dx / r["T"]).masked_fill((r["skip"] | r["empty"])[..., None], 0.0)


def close(got, want, tol, what=""):
    got, want = got.detach().double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = want.isfinite()
    assert torch.equal(got[~fine].nan_to_num(7e77, 8e88, -8e88), want[~fine].nan_to_num(7e77, 8e88, -8e88)), what
    tol = tol.expand(want.shape)[fine] if torch.is_tensor(tol) else tol
    over = ((got[fine] - want[fine]).abs() - tol)
    assert over.numel() == 0 or over.max().item() <= 0, (what, over.max().item(), int(over.argmax()))


def check_scores(x, tokens, k, T, backward=True, seed=0):
    V, dtype = x.shape[-1], x.dtype
    leaf = x.detach().requires_grad_(backward)
    out = K.k_token_logprobs(leaf, tokens, top_k=k, temperature=T)
    lp, H, top, ids, r = scores64(x, tokens, k, T)
    assert torch.equal(out.top_ids, ids)
    err = lse_error(V)
    # the value: d and its two roundings, ln s, their difference
    lnv = math.log(V) + 1
    close(out.logprob, lp, err + 4 * E * (lp.abs().nan_to_num(0, 0, 0) + lnv), "logprob")
    close(out.top_logprobs, top, err + 4 * E * (top.abs().nan_to_num(0, 0, 0) + lnv), "top_logprobs")
    # H = ln s + sum p |d|: both off by err, the second in proportion to itself (at most ln V) and by the roundings of d
    close(out.entropy, H, err * (2 + lnv) + 8 * E * lnv, "entropy")
    if not backward:
        return out
    gen = torch.Generator(device=DEV).manual_seed(seed + 5)
    scale = 64.0 if dtype == torch.float16 else 1.0
    g, gh = (torch.randn(lp.shape, device=DEV, generator=gen) * scale for _ in range(2))
    gt = torch.randn(top.shape, device=DEV, generator=gen) * scale
    dx, = torch.autograd.grad([out.logprob, out.entropy, out.top_logprobs], [leaf], [g, gh, gt])
    assert dx.shape == x.shape and dx.dtype == dtype
    want = scores_gradient64(r, g, gh, gt)
    # (a gradient beyond the type's largest value rounds to infinity: 64 / T at the lowest temperatures in fp16, whose largest is 65504)
    want = torch.where(want.to(dtype).isinf(), want.to(dtype).double(), want)
    # p is off by err and by the roundings of its argument; what it multiplies by a few half steps of its terms
    every = g.abs() + gt.abs().sum(-1)
    inner = (every[..., None] + gh.abs()[..., None] * (2 * lnv + r["logp"].abs().nan_to_num(0, 0, 0))).double()
    tol = torch.finfo(dtype).eps / 2 * want.abs().nan_to_num(0, 0, 0) + smallest(dtype)
    tol = tol + (r["p"].nan_to_num(0) * inner * (2 * err + (16 + k + 4 * r["logp"].abs().nan_to_num(0, 0, 0)) * E) + 4 * E * inner * (want != 0) * 1e-3) / T
    tol = tol + (4 + k) * E * want.abs().nan_to_num(0, 0, 0) + 4 * E / T * torch.zeros_like(want).scatter_add_(-1, r["at"][..., None], g.abs().double()[..., None])
    if k:
        tol = tol + 4 * E / T * torch.zeros_like(want).scatter_add_(-1, r["order"], gt.abs().double())
    close(dx, want, tol, "dlogits")
    return out


# --------------------------------------------------------------------------- scores
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, V, k, T", [(1, 1, 1, 1.0), (3, 2, 2, 0.5), (5, 7, 3, 1.0), (2, 31, 31, 2.0), (4, 32, 4, 1.0), (3, 33, 0, 1.0), (7, 127, 16, 1.7), (2, 256, 256, 1.0),
                                           (9, 257, 5, 1.0), (300, 1000, 8, 1.0), (2, 2049, 64, 0.7), (5, 4095, 100, 1.0), (129, 5000, 20, 2.0), (3, 32768, 256, 1.0),
                                           (2, 50257, 50, 1.3), (1, 131075, 33, 1.0), (1, 300001, 8, 1.0)])
def test_scores_and_their_gradient(rows, V, k, T, dtype):
    x = made(rows, V, dtype)
    tokens = torch.randint(0, V, (rows,), device=DEV, generator=torch.Generator(device=DEV).manual_seed(V))
    check_scores(x, tokens, k, T)


# rows by who walks them: a warp, several tiles of a warp, 128 threads, several tiles of 128, clusters of 2 to 8 CTAs
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, V, k", [(3000, 300, 20), (3000, 2100, 7), (3000, 4601, 40), (2960, 5003, 256), (2961, 9003, 12), (400, 4099, 100), (300, 20011, 30), (740, 9001, 0),
                                        (370, 17000, 0), (150, 33000, 9), (70, 70001, 50), (30, 65537, 256)])
def test_every_way_to_walk_a_row(rows, V, k, dtype):
    x = made(rows, V, dtype)
    n = torch.arange(V, device=DEV, dtype=torch.float32)
    x[0], x[1], x[2], x[3] = n / V * 9 - 4, 3 - n / V * 9, 1.25, torch.where(n % 7 == 3, 5.0, -INF)
    x[4], x[5], x[6] = -INF, torch.finfo(dtype).min, (n / 50).floor() % 23
    x[7] = torch.where(n == V - 1, 1.0, -INF)
    tokens = torch.randint(0, V, (rows,), device=DEV, generator=torch.Generator(device=DEV).manual_seed(rows))
    tokens[9], tokens[3] = -100, 3
    check_scores(x, tokens, k, 1.0)
    t, ids = a_teacher(x, 20, 1.0)
    ids = ids.clone()
    ids[10], ids[11, 4:] = -1, -1
    ids[12, 5] = ids[12, 6]
    for tail in (False, True):
        check_distill(x[8:], t[8:], ids[8:], 1.0, tail)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [40, 1000, 9001, 70000])
@pytest.mark.parametrize("order", ["equal", "two values", "ascending", "descending", "zeros of both signs", "one huge", "steps"])
def test_ties_and_orders_of_the_alternatives(V, order, dtype):
    n = torch.arange(V, device=DEV, dtype=torch.float32)
    row = {"equal": torch.full((V,), -1.5, device=DEV), "two values": (n % 3 == 1).float(), "ascending": n / V * 8 - 4, "descending": 4 - n / V * 8,
           "zeros of both signs": torch.where(n % 2 == 0, -0.0, 0.0), "one huge": torch.where(n == V - 2, 300.0, 0.0), "steps": (n / 64).floor() % 40}[order]
    x = torch.stack([row, row.roll(5), -row]).to(dtype)
    for k in sorted({1, 7, 40, min(V, 256)}):
        check_scores(x, torch.tensor([0, V - 1, V // 2], device=DEV), k, 1.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [50, 3000, 40001])
def test_masked_logits(V, dtype):
    g = torch.Generator(device=DEV).manual_seed(V)
    low = torch.finfo(dtype).min
    x = made(10, V, dtype)
    x[0].masked_fill_(torch.rand(V, device=DEV, generator=g) < 0.7, -INF)
    x[1] = -INF                                                  # nothing left
    x[2] = -INF
    x[2, V // 3] = 2.0                                           # one token left
    x[3].masked_fill_(torch.rand(V, device=DEV, generator=g) < 0.7, low)
    x[4] = low                                                   # all equal, at the type's end
    x[5, : V // 2] = -INF
    x[6, V // 2:] = -INF
    x[7] = -INF
    x[7, -1] = low
    x[8, 0] = torch.finfo(dtype).max
    tokens = torch.randint(0, V, (10,), device=DEV, generator=g)
    tokens[0] = int(x[0].argmin())                               # a masked token: -inf
    tokens[2] = V // 3
    # (lowest values divided by a temperature below one leave the type's range: T = 1 keeps the definition's 64 bits and fp32 alike)
    for k in (0, 1, 40):
        out = check_scores(x, tokens, k, 1.0)
        assert out.logprob[1] == -INF and out.entropy[1] == 0 and out.logprob[0] == -INF
        if k:
            assert out.top_ids[1].tolist() == list(range(k)) and (out.top_logprobs[1] == -INF).all()
    assert out.entropy[2] == 0 and out.logprob[2] == 0
    assert abs(out.entropy[4].item() - math.log(V)) < 1e-5 * math.log(V)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [1e-6, 1e-3, 50.0, 1e6])
@pytest.mark.parametrize("V", [50, 3000, 40001])
def test_temperatures_at_the_ends_of_their_range(V, T, dtype):
    x = made(4, V, dtype)
    x[1] *= 0.01
    x[2] = -3.0                                                  # all equal
    x[3].masked_fill_(torch.arange(V, device=DEV) % 3 == 0, -INF)
    tokens = torch.tensor([1, V - 2, 2, 4], device=DEV)
    out = check_scores(x, tokens, 5, T)
    assert (out.logprob <= 0).all() and (out.entropy >= 0).all() and (out.top_logprobs <= 0).all()


def test_entropies_and_log_probabilities_keep_their_sign():
    x = torch.zeros(4000, 37, device=DEV)
    x[:, 5] = torch.linspace(0, 60, 4000, device=DEV)            # up to a certain token
    for row_type in TYPES:
        out = K.k_token_logprobs(x.to(row_type), torch.full((4000,), 5, device=DEV), top_k=3, temperature=0.37)
        assert (out.logprob <= 0).all() and (out.entropy >= 0).all() and (out.top_logprobs <= 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [50, 3000, 40001])
def test_nan_and_infinity_stay_in_their_rows(V, dtype):
    x = made(6, V, dtype)
    clean = x.clone()
    x[1, V // 2] = float("nan")
    x[2, 3] = INF
    x[4] = float("nan")
    tokens = torch.tensor([0, 1, 2, 3, 4, 5], device=DEV)
    leaf = x.requires_grad_()
    out = K.k_token_logprobs(leaf, tokens, top_k=4)
    dx, = torch.autograd.grad([out.logprob.sum() + out.entropy.sum()], [leaf])
    want = K.k_token_logprobs(clean.requires_grad_(), tokens, top_k=4)
    for bad in (1, 2, 4):
        assert out.logprob[bad].isnan() and out.entropy[bad].isnan() and out.top_logprobs[bad].isnan().all() and dx[bad].isnan().any()
    assert out.top_ids[1, 0] == V // 2 and out.top_ids[2, 0] == 3 and out.top_ids[4].tolist() == [0, 1, 2, 3]
    for good in (0, 3, 5):
        assert torch.equal(out.logprob[good], want.logprob[good]) and torch.equal(out.top_logprobs[good], want.top_logprobs[good])
        assert torch.equal(out.entropy[good], want.entropy[good]) and dx[good].isfinite().all()


@pytest.mark.parametrize("V", [64, 5000, 50257])
def test_ignored_rows_are_not_read(V):
    x = made(8, V, torch.bfloat16)
    x[2], x[5], x[7] = float("nan"), INF, -INF
    tokens = torch.randint(0, V, (8,), device=DEV)
    tokens[[2, 5, 7]] = -100
    out = check_scores(x, tokens, 6, 1.0)
    assert (out.logprob[[2, 5, 7]] == 0).all() and (out.top_ids[[2, 5, 7]] == -1).all()
    leaf = x.detach().requires_grad_()
    out = K.k_token_logprobs(leaf, tokens, top_k=6)
    nan = torch.full_like(out.logprob, float("nan"))
    nan[[0, 1, 3, 4, 6]] = 1.0
    dx, = torch.autograd.grad([out.logprob, out.entropy], [leaf], [nan, nan])      # what comes back for an ignored row is not looked at
    assert (dx[[2, 5, 7]] == 0).all() and dx.isfinite().all()
    inside = K.k_token_logprobs(leaf, tokens.masked_fill(tokens < 0, 7), ignore_index=7, top_k=6)      # a token of the vocabulary marks padding
    skipped = (tokens < 0) | (tokens == 7)
    for a, b in zip(inside, out):
        assert torch.equal(a[~skipped], b[~skipped])
    assert not inside.logprob[skipped].any() and (inside.top_ids[skipped] == -1).all()
    dx, = torch.autograd.grad([inside.logprob, inside.entropy], [leaf], [nan, nan])
    assert (dx[skipped] == 0).all() and dx.isfinite().all()
    everything = K.k_token_logprobs(x, torch.full_like(tokens, -1), ignore_index=-1, top_k=3)
    assert not everything.logprob.any() and not everything.entropy.any() and (everything.top_ids == -1).all()


def test_a_token_outside_the_vocabulary_is_noted():
    x = made(4, 100, torch.float32)
    tokens = torch.tensor([3, 100, -7, 99], device=DEV)
    ops = K._ops_for(x)
    ops.check_status()
    leaf = x.requires_grad_()
    out = K.k_token_logprobs(leaf, tokens, top_k=2)
    with pytest.raises(RteError, match="index out of range"):
        ops.check_status()
    assert not out.logprob[[1, 2]].any() and (out.top_ids[[1, 2]] == -1).all() and (out.logprob[[0, 3]] < 0).all()
    dx, = torch.autograd.grad([out.logprob.sum()], [leaf])
    assert not dx[[1, 2]].any() and dx[[0, 3]].any()
    ops.check_status()


def test_strides_types_of_ids_and_single_gradients():
    base = made(6, 4000, torch.bfloat16).view(2, 3, 4000)
    tokens = torch.randint(0, 900, (2, 3), device=DEV)
    views = [base[..., 5:1005], base[..., 1::4][..., :950], base.transpose(0, 1)[..., :1000].transpose(0, 1), base[:, :1, 7:1007].expand(2, 3, 1000), base[:, :, :1000].flip(0)]
    for v in views:
        assert tuple(v.shape[:2]) == (2, 3)
        check_scores(v, tokens, 9, 1.0)
    plain = K.k_token_logprobs(base[..., :1000], tokens, top_k=4)
    for same in (K.k_token_logprobs(base[..., :1000].contiguous(), tokens.int(), top_k=4), K.k_token_logprobs(base[..., :1000], tokens.t().contiguous().t(), top_k=4)):
        for a, b in zip(plain, same):
            assert torch.equal(a, b)
    x = made(5, 777, torch.float32)
    tok = torch.randint(0, 777, (5,), device=DEV)
    lp, H, top, ids, r = scores64(x, tok, 3, 1.0)
    zero, one = torch.zeros(5, device=DEV), torch.ones(5, device=DEV)
    for which, g in enumerate([(one, zero, torch.zeros(5, 3, device=DEV)), (zero, one, torch.zeros(5, 3, device=DEV)), (zero, zero, torch.ones(5, 3, device=DEV))]):
        leaf = x.requires_grad_()
        out = K.k_token_logprobs(leaf, tok, top_k=3)
        dx, = torch.autograd.grad([out[which].sum()], [leaf])                     # (the others' gradients are absent)
        assert (dx - scores_gradient64(r, *g)).abs().max() < 8 * lse_error(777) * 10
    no_rows = K.k_token_logprobs(x[:0], tok[:0], top_k=3)
    assert no_rows.logprob.shape == (0,) and no_rows.top_ids.shape == (0, 3)
    scalar = K.k_token_logprobs(x[0], tok[0])
    assert scalar.logprob.shape == () and abs(scalar.logprob.item() - lp[0].item()) < 1e-4


def test_rows_further_apart_than_32_bits_reach():
    far = 2 ** 31 + 24
    store = torch.empty(2 * far + 1000, dtype=torch.bfloat16, device=DEV)
    x = store.as_strided((3, 1000), (far, 1))
    x.copy_(made(3, 1000, torch.bfloat16))
    tokens = torch.tensor([1, 500, 999], device=DEV)
    check_scores(x, tokens, 5, 1.0)
    ids = torch.tensor([[4, 2], [9, 998], [0, 1]], device=DEV)
    check_distill(x, torch.log(torch.tensor([[0.5, 0.2]], device=DEV)).expand(3, 2), ids, 1.0, True)


def test_more_elements_than_32_bits_count():
    rows, V = 66000, 32769                                      # 2.16e9 logits
    x = torch.zeros(rows, V, dtype=torch.bfloat16, device=DEV)
    x[-1] = made(1, V, torch.bfloat16)[0]
    tokens = torch.full((rows,), V - 1, device=DEV)
    leaf = x.requires_grad_()
    out = K.k_token_logprobs(leaf, tokens, top_k=2)
    lp, H, top, ids, r = scores64(x[-1:], tokens[-1:], 2, 1.0)
    assert torch.equal(out.top_ids[-1:], ids) and (out.top_ids[:-1] == torch.tensor([0, 1], device=DEV)).all()
    close(out.logprob[-1:], lp, 2 * lse_error(V), "last row")
    assert (out.logprob[:-1] + math.log(V)).abs().max() < 2 * lse_error(V) + 1e-6
    dx, = torch.autograd.grad([out.logprob.sum()], [leaf])
    want = scores_gradient64(r, torch.ones(1, device=DEV), torch.zeros(1, device=DEV), None)
    close(dx[-1:], want, want.abs() * 2 ** -7 + 1e-6, "last row's gradient")
    assert (dx[:-1, -1] > 0.99).all() and dx[70, 5] < 0


# --------------------------------------------------------------------------- distillation
def distill64(x, teacher, ids, T, tail):
    V = x.shape[-1]
    x, t = x.detach().double(), teacher.double()
    used = (ids >= 0) & (ids < V)
    at = ids.long().masked_fill(~used, 0)
    t = t.masked_fill(~used, -INF)
    none = ~used.any(-1)
    if not tail:
        none = none | (t == -INF).all(-1)
        t = t - torch.logsumexp(t.masked_fill(none[..., None], 0.0), -1, keepdim=True)
    t = t.masked_fill(none[..., None], -INF)
    q = t.exp()
    empty = (x == -INF).all(-1)
    logp = torch.log_softmax(x.masked_fill((empty | none)[..., None], 0.0) / T, -1).masked_fill(empty[..., None], -INF)
    p = logp.exp()
    lp = logp.gather(-1, at)
    terms = torch.where(q == 0, torch.zeros_like(q), q * (t - lp))
    loss = terms.sum(-1)
    member = torch.zeros_like(p).scatter_add_(-1, at, used.double()) > 0
    qd = torch.zeros_like(p).scatter_add_(-1, at, q)
    M = q.sum(-1)
    dz = M[..., None] * p - qd
    if tail:
        # (in logarithms: e^-745 is the smallest number of 64 bits)
        outside = logp.masked_fill(member, -INF)
        lnP = torch.logsumexp(outside, -1)
        r = (1 - M).clamp(min=0.0).masked_fill(lnP == -INF, 0.0)
        lnP = lnP.masked_fill(lnP == -INF, 0.0)
        loss = loss + torch.where(r > 0, r * (r.clamp(min=1e-300).log() - lnP), torch.zeros_like(r))
        dz = dz + r[..., None] * (p - (outside - lnP[..., None]).exp())
    loss = (T * T * loss).masked_fill(none, 0.0)
    dz = (T * dz).masked_fill((none | empty)[..., None], 0.0)
    return loss, dz, dict(none=none, p=p, q=q, qd=qd, logp=logp, lp=lp, M=M)


def check_distill(x, teacher, ids, T, tail, seed=0):
    V, dtype = x.shape[-1], x.dtype
    leaf = x.detach().requires_grad_()
    loss = K.k_distill_topk(leaf, teacher, ids, temperature=T, tail=tail)
    want, dz, r = distill64(x, teacher, ids, T, tail)
    err = lse_error(V)
    # a listed term: q times (ln q, d, ln s with their roundings); the rest's like one of them
    size = (r["q"] * (teacher.double().abs().nan_to_num(0, 0, 0) + r["lp"].abs().nan_to_num(0, 0, 0) + math.log(V) + 2)).masked_fill(r["q"] == 0, 0.0).sum(-1) + math.log(V) + 20
    close(loss, want, T * T * ((r["M"] + 1) * 3 * err + 8 * E * size) + E * want.abs().nan_to_num(0, 0, 0), "loss")
    gen = torch.Generator(device=DEV).manual_seed(seed + 9)
    g = torch.randn(want.shape, device=DEV, generator=gen) * (64.0 if dtype == torch.float16 else 1.0)
    dx, = torch.autograd.grad([loss], [leaf], [g])
    assert dx.shape == x.shape and dx.dtype == dtype
    gw = dz * g.double()[..., None]
    # p as above; 1 / P of the rest is off by err too, q by the rounding of its exponent
    part = (r["p"].nan_to_num(0) * (r["M"][..., None] + 1) * (4 * err + (16 + 4 * r["logp"].abs().nan_to_num(0, 0, 0)) * E) + r["qd"] * 64 * E) * T * g.abs().double()[..., None]
    close(dx, gw, torch.finfo(dtype).eps / 2 * gw.abs().nan_to_num(0, 0, 0) + 8 * E * gw.abs().nan_to_num(0, 0, 0) + part + rest_error(r, dz, T, err, tail) * g.abs().double()[..., None]
          + smallest(dtype), "dlogits")
    return loss


def rest_error(r, dz, T, err, tail):
    """Outside the list the gradient is T p (M - r / P): r / P may be many times M, and is off by 4 err of itself."""
    return (dz.abs() + T * r["p"] * r["M"][..., None]).nan_to_num(0, 0, 0) * 8 * err if tail else torch.zeros_like(dz)


def a_teacher(x, k, T, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed + 31)
    full = torch.log_softmax((0.7 * x.float() + torch.randn(x.shape, device=DEV, generator=gen)) / T, -1)
    top, ids = full.topk(min(k, x.shape[-1]), -1)
    return top, ids


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows, V, k, T", [(1, 1, 1, 1.0), (3, 2, 1, 0.5), (5, 7, 7, 1.0), (2, 33, 8, 2.0), (7, 127, 16, 1.7), (2, 300, 256, 1.0), (300, 1000, 8, 1.0),
                                           (2, 2049, 64, 0.7), (129, 5000, 20, 2.0), (3, 32768, 200, 1.0), (2, 50257, 50, 1.3), (1, 131075, 33, 1.0)])
def test_distillation_and_its_gradient(rows, V, k, T, tail, dtype):
    x = made(rows, V, dtype)
    check_distill(x, *a_teacher(x, k, T), T, tail)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("V", [40, 3000, 40001])
def test_distillation_lists_in_every_state(V, tail, dtype):
    k = 12
    x = made(12, V, dtype)
    t, ids = a_teacher(x, k, 1.0)
    t, ids = t.clone(), ids.clone()
    ids[0, 5:] = -1                                              # a short list
    t[0, 5:] = float("nan")                                      # (what an unused slot holds is not looked at)
    ids[1] = -1                                                  # none
    x[1] = float("nan")
    ids[2, 3] = ids[2, 0]                                        # a token named twice
    ids[3] = ids[3, 0]                                           # a token named by every slot
    t[3] = math.log(0.05)
    t[4, 2:] = -INF                                              # slots without probability
    x[5, ids[5, 1]] = -INF                                       # the student cannot say it: infinite loss
    x[6].masked_fill_(torch.arange(V, device=DEV) % 2 == 0, -INF)
    t[6].masked_fill_(ids[6] % 2 == 0, -INF)
    x[7] = -INF                                                  # a student without a distribution
    t[8] = t[8].logsumexp(0).neg() + t[8]                        # a list that sums to one
    keep = torch.zeros(V, dtype=torch.bool, device=DEV)
    keep[ids[9]] = True
    x[9].masked_fill_(~keep, -INF)                               # nothing left outside the list
    x[10, ids[10]] = 60.0                                        # the rest is far below the list
    ids[11, 1::2] = -5
    loss = check_distill(x, t, ids, 1.0, tail)
    assert loss[1] == 0 and loss[5] == INF and loss[7] == INF
    t[:] = -INF
    none = check_distill(x, t, ids, 1.0, tail)
    assert tail or not none.any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [40, 3000, 40001])
def test_the_rest_of_the_vocabulary_far_below_the_list(V, dtype):
    """Its probability is below fp32's range, its logarithm and the gradient that it takes are ordinary numbers."""
    x = made(4, V, dtype)
    t, ids = a_teacher(x, 5, 1.0)
    t = t - t.logsumexp(-1, keepdim=True) - 0.7
    for row, height in enumerate((90.0, 300.0, 900.0, 20000.0)):
        x[row, ids[row]] = height
    x[3, : V // 2] = -INF
    x[3, ids[3]] = 20000.0
    loss = check_distill(x, t, ids, 1.0, True)
    assert loss.isfinite().all() and (loss[1:] > 100).all()


def test_a_listed_id_outside_the_vocabulary_is_noted():
    x = made(3, 100, torch.float32)
    t, ids = a_teacher(x, 4, 1.0)
    ids[1, 2] = 100
    ops = K._ops_for(x)
    ops.check_status()
    check_distill(x, t, ids, 1.0, False)
    with pytest.raises(RteError, match="index out of range"):
        ops.check_status()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("V, T", [(50, 0.02), (3000, 60.0), (40001, 0.1), (3000, 1e3)])
def test_distillation_at_low_and_high_temperatures(V, T, tail, dtype):
    x = made(5, V, dtype)
    check_distill(x, *a_teacher(x, 9, T), T, tail)


@pytest.mark.parametrize("tail", [False, True])
def test_a_teacher_that_is_not_a_number_stays_in_its_row(tail):
    x = made(5, 900, torch.float32)
    t, ids = a_teacher(x, 6, 1.0)
    want = K.k_distill_topk(x, t, ids, tail=tail)
    t = t.clone()
    t[1, 2] = float("nan")
    t[3] = float("nan")
    leaf = x.clone().requires_grad_()
    loss = K.k_distill_topk(leaf, t, ids, tail=tail)
    dx, = torch.autograd.grad([loss.sum()], [leaf])
    assert loss[[1, 3]].isnan().all() and torch.equal(loss[[0, 2, 4]], want[[0, 2, 4]])
    assert dx[[1, 3]].isnan().any(-1).all() and dx[[0, 2, 4]].isfinite().all()


def test_distillation_views_and_types_of_the_list():
    x = made(6, 4000, torch.bfloat16).view(2, 3, 4000)
    t, ids = a_teacher(x[..., :1000], 8, 2.0)
    want = K.k_distill_topk(x[..., :1000].contiguous(), t, ids, temperature=2.0, tail=True)
    assert want.shape == (2, 3)
    t16 = t.bfloat16()
    wide_t, wide_ids = torch.zeros(2, 3, 20, device=DEV), torch.zeros(2, 3, 20, dtype=torch.int32, device=DEV)
    wide_t[..., 2:10], wide_ids[..., 2:10] = t, ids.int()
    assert torch.equal(want, K.k_distill_topk(x[..., :1000], wide_t[..., 2:10], wide_ids[..., 2:10], temperature=2.0, tail=True))
    assert torch.equal(K.k_distill_topk(x[..., :1000], t16, ids), K.k_distill_topk(x[..., :1000], t16.float(), ids))
    shifted = K.k_distill_topk(x[..., :1000], t + 7.0, ids)                       # renormalised: a constant changes nothing but roundings
    assert (shifted - K.k_distill_topk(x[..., :1000], t, ids)).abs().max() < 1e-4
    for v in (x[..., 5:1005], x.transpose(0, 1)[..., :1000].transpose(0, 1), x[:, :1, 7:1007].expand(2, 3, 1000), x[..., 1::4]):
        check_distill(v, *a_teacher(v, 8, 1.0), 1.0, True)
    assert K.k_distill_topk(x[:0], t[:0], ids[:0]).shape == (0, 3)
    teacher = t.clone().requires_grad_()
    leaf = x.detach().clone().requires_grad_()
    K.k_distill_topk(leaf, teacher, ids).sum().backward()
    assert teacher.grad is None and leaf.grad is not None


# --------------------------------------------------------------------------- both
def test_gradients_against_differences():
    V, h = 23, 1e-5
    x = made(4, V, torch.float32, spread=1.5)
    tokens = torch.tensor([1, 22, 7, 0], device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(3)
    g, gh, gt = (torch.randn(s, device=DEV, generator=gen) for s in ((4,), (4,), (4, 5)))
    t, ids = a_teacher(x, 6, 1.5)

    def scores(y):
        lp, H, _, _, r = scores64(y, tokens, 0, 1.5)
        return (lp * g).sum() + (H * gh).sum() + (r["logp"].gather(-1, order) * gt).sum()

    leaf = x.requires_grad_()
    out = K.k_token_logprobs(leaf, tokens, top_k=5, temperature=1.5)
    order = out.top_ids
    calls = [(scores, torch.autograd.grad([out.logprob, out.entropy, out.top_logprobs], [leaf], [g, gh, gt])[0])]
    for tail in (False, True):
        loss = K.k_distill_topk(leaf, t, ids, temperature=1.5, tail=tail)
        calls.append((lambda y, tail=tail: (distill64(y, t, ids, 1.5, tail)[0] * g).sum(), torch.autograd.grad([loss], [leaf], [g])[0]))
    base = x.detach().double()
    for f, dx in calls:
        for i in range(4):
            for j in range(0, V, 3):
                step = torch.zeros_like(base)
                step[i, j] = h
                slope = (f(base + step) - f(base - step)) / (2 * h)           # off by h^2 of the third derivative and 1e-16 / h
                assert abs(slope.item() - dx[i, j].item()) < 2e-6, (i, j, slope.item(), dx[i, j].item())


def _passes(x, tokens, t, ids, g):
    leaf = x.detach().requires_grad_()
    out = K.k_token_logprobs(leaf, tokens, top_k=6, temperature=1.2)
    a, = torch.autograd.grad([out.logprob, out.entropy, out.top_logprobs], [leaf], [g, g, g[:, None].expand(-1, 6)])
    loss = K.k_distill_topk(leaf, t, ids, temperature=1.2, tail=True)
    b, = torch.autograd.grad([loss], [leaf], [g])
    return [out.logprob.detach(), out.entropy.detach(), out.top_logprobs.detach(), out.top_ids, a, loss.detach(), b]


@pytest.mark.parametrize("rows, V", [(1, 50257), (3, 131072), (40, 2000), (700, 9000)])
def test_same_bits_every_time_on_a_side_stream_and_from_a_graph(rows, V):
    x = made(rows, V, torch.bfloat16)
    tokens = torch.randint(0, V, (rows,), device=DEV)
    t, ids = a_teacher(x, 16, 1.2)
    g = torch.randn(rows, device=DEV)
    first = _passes(x, tokens, t, ids, g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = _passes(x, tokens, t, ids, g)
    torch.cuda.current_stream().wait_stream(side)
    held = [v.clone() for v in (x, tokens, t, ids, g)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = _passes(*held)
    other = made(rows, V, torch.bfloat16, seed=4)
    fresh = [other, torch.randint(0, V, (rows,), device=DEV), *a_teacher(other, 16, 1.2), torch.randn(rows, device=DEV)]
    for src in (fresh, (x, tokens, t, ids, g)):
        for a, b in zip(held, src):
            a.copy_(b)
        graph.replay()
        for i, (a, b) in enumerate(zip(third, _passes(*src))):
            assert torch.equal(a, b), i
    for i, (a, b) in enumerate(zip(first, second)):
        assert torch.equal(a, b), i
    K._ops_for(x).check_status()


@pytest.mark.parametrize("rows, V", [(3, 70), (5, 40000), (700, 9000)])
def test_without_a_gradient_the_same_results(rows, V):
    x = made(rows, V, torch.bfloat16)
    tokens = torch.randint(0, V, (rows,), device=DEV)
    tokens[0] = -100
    t, ids = a_teacher(x, 8, 1.0)
    ids[1] = -1
    leaf = x.clone().requires_grad_()
    for a, b in zip(K.k_token_logprobs(x, tokens, top_k=5), K.k_token_logprobs(leaf, tokens, top_k=5)):
        assert torch.equal(a, b) and not a.requires_grad
    for tail in (False, True):
        assert torch.equal(K.k_distill_topk(x, t, ids, tail=tail), K.k_distill_topk(leaf, t, ids, tail=tail))
    with torch.no_grad():
        assert not K.k_token_logprobs(leaf, tokens).logprob.requires_grad and not K.k_distill_topk(leaf, t, ids).requires_grad


def test_two_threads_on_streams_of_their_own():
    import threading

    jobs = [(made(40, 9000, torch.bfloat16, seed=i), torch.randint(0, 9000, (40,), device=DEV)) for i in range(2)]
    want = [_passes(x, tok, *a_teacher(x, 16, 1.2), torch.ones(40, device=DEV)) for x, tok in jobs]
    torch.cuda.synchronize()
    got = [None, None]

    def work(i):
        x, tok = jobs[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i] = _passes(x, tok, *a_teacher(x, 16, 1.2), torch.ones(40, device=DEV))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(want, got):
        for u, v in zip(a, b):
            assert torch.equal(u, v)


def test_logits_changed_in_place_are_refused_by_backward():
    x = made(2, 64, torch.float32).requires_grad_()
    y = x * 1.0
    loss = K.k_distill_topk(y, *a_teacher(x.detach(), 4, 1.0)).sum() + K.k_token_logprobs(y, torch.zeros(2, dtype=torch.int64, device=DEV)).logprob.sum()
    y.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_tensors_on_another_device_than_the_current_one():
    x = made(3, 500, torch.float32)
    tokens = torch.tensor([1, 2, 3], device=DEV)
    want = K.k_token_logprobs(x, tokens, top_k=3)
    got = K.k_token_logprobs(x.to("cuda:1"), tokens.to("cuda:1"), top_k=3)
    for a, b in zip(want, got):
        assert torch.equal(a, b.to(DEV))
