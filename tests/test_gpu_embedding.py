"""`k_embedding` on a B200 against its definition in 64 bits, and the operators at the two ends of the vocabulary together.

Tolerances: the lookup is one product and one rounding, so it is compared bit for bit.  A gradient's row is a sum of n fp32 terms in
some order, off by at most n 2^-24 of the terms' magnitudes, times the scale (one rounding more), and rounded to the type once."""
import pytest
import torch

from speedup_thingy_b200 import kernels as K
from speedup_thingy_b200._abi import RteError

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]
E = 2.0 ** -24


def some_ids(kind, n, V, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed * 7 + n + V)
    if kind == "zipf":
        w = torch.arange(1, V + 1, dtype=torch.float64, device=DEV).pow(-1.1)
        return torch.searchsorted(w.cumsum(0) / w.sum(), torch.rand(n, dtype=torch.float64, device=DEV, generator=g)).clamp_(max=V - 1)
    if kind == "same":
        return torch.full((n,), V // 2, device=DEV)
    if kind == "distinct":
        return torch.randperm(V, device=DEV, generator=g)[:n] if n <= V else torch.arange(n, device=DEV) % V
    if kind == "ascending":
        return torch.arange(n, device=DEV) * V // max(n, 1)
    if kind == "descending":
        return (V - 1 - torch.arange(n, device=DEV) * V // max(n, 1)).clamp(min=0)
    if kind == "ends":
        return torch.where(torch.rand(n, device=DEV, generator=g) < 0.5, 0, V - 1)
    return torch.randint(0, V, (n,), device=DEV, generator=g)


def check(ids, weight, scale, padding=None, dy=None):
    V, d = weight.shape
    dtype = weight.dtype
    leaf = weight.detach().requires_grad_()
    y = K.k_embedding(ids, leaf, scale=scale, padding_idx=padding)
    bad = (ids < 0) | (ids >= V)
    safe = ids.long().masked_fill(bad, 0)
    want = (weight.float()[safe] * torch.tensor(scale, device=DEV)).to(dtype).masked_fill(bad[..., None], 0)
    assert y.shape == want.shape and y.dtype == dtype and torch.equal(y, want)
    g = torch.Generator(device=DEV).manual_seed(d)
    if dy is None:
        dy = torch.randn(y.shape, device=DEV, generator=g).to(dtype)
    dw, = torch.autograd.grad([y], [leaf], [dy])
    assert dw.shape == weight.shape and dw.dtype == dtype
    skip = bad.reshape(-1) | (safe.reshape(-1) == (-1 if padding is None else padding))
    rows = dy.reshape(-1, d).double()[~skip]
    at = safe.reshape(-1)[~skip]
    ref = torch.zeros(V, d, dtype=torch.float64, device=DEV).index_add_(0, at, rows) * scale
    size = torch.zeros(V, d, dtype=torch.float64, device=DEV).index_add_(0, at, rows.abs()) * abs(scale)
    count = torch.bincount(at, minlength=V).double()[:, None]
    tiny = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126}[dtype]
    over = (dw.double() - ref).abs() - (torch.finfo(dtype).eps / 2 * ref.abs() + (count + 2) * E * size + tiny)
    assert over.max().item() <= 0, over.max().item()
    assert not dw[count[:, 0] == 0].any()
    return y, dw


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [1, 2, 3, 4, 8, 10, 64, 130, 770, 1024, 1536])
@pytest.mark.parametrize("n, V", [(1, 1), (2, 5), (31, 100), (33, 7), (700, 5000)])
def test_rows_and_gradient(n, V, d, dtype):
    w = torch.randn(V, d, device=DEV, generator=torch.Generator(device=DEV).manual_seed(d)).to(dtype)
    check(some_ids("random", n, V), w, 1.0)
    check(some_ids("zipf", n, V), w, 27.75, padding=V // 3)


@pytest.mark.parametrize("kind", ["zipf", "same", "distinct", "ascending", "descending", "ends", "random"])
@pytest.mark.parametrize("n, V", [(32, 40), (64, 64), (100, 300), (1000, 50), (4096, 2048), (4097, 2048), (9000, 5000), (20000, 30000)])
def test_patterns_of_ids(kind, n, V):
    w = torch.randn(V, 40, device=DEV).bfloat16()
    check(some_ids(kind, n, V), w, 0.5)
    check(some_ids(kind, n, V, seed=1), w, 1.0, padding=int(some_ids(kind, n, V, seed=1)[n // 2]))


def test_long_batches_and_heavy_ids():
    for n, V, d, kind in ((2200000, 50, 2, "same"), (8192, 100, 16, "zipf"), (8193, 100, 16, "zipf"), (8193, 5000, 16, "same"), (8192, 20000, 16, "same"), (49152, 3000, 8, "zipf"), (49153, 3000, 8, "zipf"), (49152, 70000, 8, "random"), (60000, 70000, 8, "descending"), (48001, 2, 8, "ends"), (700001, 40000, 4, "zipf"), (700001, 3000000, 4, "random"),
                          (640000, 1 << 21, 2, "descending"), (131072, 131072, 72, "zipf"), (100003, 50257, 24, "zipf"), (70000, 9, 136, "random"), (66000, 300, 8, "same"), (300000, 1000, 4, "zipf")):
        check(some_ids(kind, n, V), torch.randn(V, d, device=DEV).bfloat16(), 3.0)


def test_large_ids_and_padding_everywhere():
    V = (1 << 22) + 3
    w = torch.randn(V, 8, device=DEV)
    ids = some_ids("random", 5000, V)
    ids[:3] = torch.tensor([0, V - 1, 1 << 22], device=DEV)
    check(ids, w, 2.0, padding=V - 1)
    _, dw = check(torch.full((100,), 7, device=DEV), w[:50], 1.0, padding=7)
    assert not dw.any()


def test_table_and_rows_beyond_32_bits():
    V, d = 40000, 65536                                          # 2.6e9 elements
    w = torch.zeros(V, d, dtype=torch.bfloat16, device=DEV)
    w[-1], w[-2] = 1.5, -2.0
    leaf = w.requires_grad_()
    ids = torch.tensor([V - 1, V - 2, 0, V - 1], device=DEV)
    y = K.k_embedding(ids, leaf, scale=2.0)
    assert (y[0] == 3.0).all() and (y[1] == -4.0).all() and not y[2].any()
    dw, = torch.autograd.grad([y], [leaf], [torch.ones_like(y)])
    assert (dw[-1] == 4.0).all() and (dw[-2] == 2.0).all() and (dw[0] == 2.0).all() and not dw[1:-2].any()


@pytest.mark.parametrize("n", [100, 9000])
def test_ids_of_31_bits(n):
    V = (1 << 30) + 5
    w = torch.zeros(V, 1, dtype=torch.bfloat16, device=DEV)
    ids = torch.randint(0, V, (n,), device=DEV, generator=torch.Generator(device=DEV).manual_seed(n))
    ids[:4] = torch.tensor([V - 1, 0, V - 1, 1 << 30], device=DEV)
    w[ids] = 2.0
    leaf = w.requires_grad_()
    y = K.k_embedding(ids, leaf, scale=0.5)
    assert (y == 1).all()
    dw, = torch.autograd.grad([y], [leaf], [torch.ones_like(y)])
    assert dw[V - 1].item() == 1.0 and dw[0].item() == 0.5 and dw[1 << 30].item() == 0.5
    assert (dw[ids] >= 0.5).all() and dw.count_nonzero().item() == ids.unique().numel()


def test_ids_outside_the_table_are_noted():
    w = torch.randn(20, 16, device=DEV)
    ops = K._ops_for(w)
    ops.check_status()
    ids = torch.tensor([[3, 20, -1], [2 ** 40, 3, 19]], device=DEV)
    y, dw = check(ids, w, 1.0)
    assert not y[0, 1:].any() and not y[1, 0].any()
    with pytest.raises(RteError, match="index out of range"):
        ops.check_status()


def test_shapes_types_and_layouts():
    w = torch.randn(50, 24, device=DEV)
    ids = some_ids("random", 24, 50).view(2, 3, 4)
    y, dw = check(ids, w, 1.0)
    assert y.shape == (2, 3, 4, 24)
    check(ids.int(), w, 1.0)
    check(ids.transpose(0, 2), w, 1.0)
    check(torch.tensor(7, device=DEV), w, 1.0)
    check(ids, w.t().contiguous().t(), 1.0)                      # a table stored the other way round
    check(ids, torch.randn(50 * 24 + 1, device=DEV)[1:].view(50, 24), 1.0)      # on an odd boundary
    check(ids, torch.randn(50 * 24 + 1, device=DEV).bfloat16()[1:].view(50, 24), 1.0)
    leaf = w.requires_grad_()
    K.k_embedding(ids, leaf).sum().backward()                    # an expanded gradient
    want = torch.bincount(ids.reshape(-1), minlength=50).float()[:, None].expand(50, 24)
    assert torch.equal(leaf.grad, want)
    K.k_embedding(ids, leaf).sum().backward()
    assert torch.equal(leaf.grad, 2 * want)
    dy = torch.randn(2, 3, 24, 4, device=DEV).transpose(2, 3)    # a gradient in another order
    check(ids, w.detach(), 1.0, dy=dy)
    none = K.k_embedding(ids[:0], leaf)
    assert none.shape == (0, 3, 4, 24)
    dw, = torch.autograd.grad([none.sum()], [leaf])
    assert dw.shape == w.shape and not dw.any()
    with torch.no_grad():
        assert not K.k_embedding(ids, leaf).requires_grad


@pytest.mark.parametrize("n, V, d", [(37, 100, 16), (9000, 3000, 130)])
def test_same_bits_every_time_on_a_side_stream_and_from_a_graph(n, V, d):
    def once(ids, w, dy):
        leaf = w.detach().requires_grad_()
        y = K.k_embedding(ids, leaf, scale=1.5)
        return y.detach(), torch.autograd.grad([y], [leaf], [dy])[0]

    def inputs(seed):
        g = torch.Generator(device=DEV).manual_seed(seed)
        return some_ids("zipf", n, V, seed), torch.randn(V, d, device=DEV, generator=g), torch.randn(n, d, device=DEV, generator=g)

    a, b = inputs(1), inputs(2)
    first = once(*a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once(*a)
    torch.cuda.current_stream().wait_stream(side)
    held = [v.clone() for v in a]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = once(*held)
    for src in (b, a):
        for h, v in zip(held, src):
            h.copy_(v)
        graph.replay()
        for u, v in zip(third, once(*src)):
            assert torch.equal(u, v)
    for u, v in zip(first, second):
        assert torch.equal(u, v)


def test_scores_of_a_teacher_train_a_student_with_a_tied_table():
    """Embedding -> tied logits -> scores: the teacher's alternatives are the student's lists, and the student's one table gets the
    gradient of both of its uses.  The products round to bf16, the operators' own arithmetic does not: against the same run in
    fp32 the gradients agree as the products' two bf16 operands allow, 2^-8 each of the terms' size."""
    torch.manual_seed(0)
    V, d, B, S, k, T = 1000, 64, 4, 32, 16, 2.0
    ids = some_ids("zipf", B * S, V).view(B, S)
    targets = torch.roll(ids, -1, 1).masked_fill(torch.arange(S, device=DEV) == S - 1, -100)
    table = {"teacher": torch.randn(V, d, device=DEV) * 0.2, "student": torch.randn(V, d, device=DEV) * 0.2}
    with torch.no_grad():
        said = K.k_token_logprobs(K.k_logits_full(K.k_embedding(ids, table["teacher"], scale=d ** 0.5), table["teacher"]), targets, top_k=k, temperature=T)
    assert (said.top_ids[:, -1] == -1).all()                     # rows without a target have no list ...

    def loss_of(table, lookup, logits_of, distill, scores):
        h = lookup(table)
        x = logits_of(h, table)
        kd = distill(x)
        lp, entropy = scores(x)
        return (kd.sum() - lp.sum() - 0.1 * entropy.sum()) / (B * S)

    mine = table["student"].clone().requires_grad_()
    loss = loss_of(mine, lambda w: K.k_embedding(ids, w, scale=d ** 0.5), K.k_logits_full,
                   lambda x: K.k_distill_topk(x, said.top_logprobs, said.top_ids, temperature=T, tail=True), lambda x: K.k_token_logprobs(x, targets)[:2])
    loss.backward()

    w = table["student"].clone().requires_grad_()
    keep = targets != -100

    def kd_plain(x):
        logp = torch.log_softmax(x / T, -1)
        at = said.top_ids.clamp(min=0)
        q = said.top_logprobs.exp() * keep[..., None]
        r = (1 - q.sum(-1)).clamp(min=0)
        out = logp.exp().scatter(-1, at, 0.0).sum(-1)
        return T * T * ((q * (said.top_logprobs - logp.gather(-1, at))).sum(-1) + r * (r / out).log()) * keep

    def scores_plain(x):
        logp = torch.log_softmax(x, -1)
        return logp.gather(-1, targets.clamp(min=0)[..., None])[..., 0] * keep, -(logp.exp() * logp).sum(-1) * keep

    ref = loss_of(w, lambda w: w[ids] * d ** 0.5, lambda h, w: h @ w.t(), kd_plain, scores_plain)
    ref.backward()
    assert abs(loss.item() - ref.item()) < 2e-2 * abs(ref.item())
    assert (mine.grad - w.grad).abs().max() < 2e-2 * w.grad.abs().max()
    K._ops_for(mine).check_status()
