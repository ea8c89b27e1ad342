"""The operators at the two ends of the vocabulary at their largest sizes, and two of their graphs at once, on a B200."""
import math

import pytest
import torch

from speedup_thingy_b200 import _abi as A
from speedup_thingy_b200 import kernels as K
from tests.test_gpu_embedding_exact import whole_numbers
from tests.test_gpu_token_scores import E, made

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_the_longest_row_of_logits():
    """Tolerance: a thread adds its tiles' sums one after the other, no more than V / (8 CTAs * 256 threads * 64) of them; then as for other rows."""
    V = 2 ** 31 - 257
    x = torch.zeros(1, V, dtype=torch.bfloat16, device=DEV)
    high = {V // 2: 10.0, 5: 9.0, V - 1: 8.0}
    for at, v in high.items():
        x[0, at] = v
    leaf = x.requires_grad_()
    out = K.k_token_logprobs(leaf, torch.tensor([V - 1], device=DEV), top_k=4)
    s = (V - 3) + sum(math.exp(v) for v in high.values())
    logs = [v - math.log(s) for v in (10.0, 9.0, 8.0, 0.0)]
    H = -sum(l * math.exp(l) for l in logs[:3]) - (V - 3) * logs[3] * math.exp(logs[3])
    tol = (V / (8 * 256 * 64) + 70 + 2 * math.log(V)) * E
    assert out.top_ids.tolist() == [[V // 2, 5, V - 1, 0]]
    for got, want in zip(out.top_logprobs[0].tolist(), logs):
        assert abs(got - want) < tol + 4 * E * (abs(want) + 22)
    assert abs(out.logprob.item() - logs[2]) < tol + 4 * E * 36
    assert abs(out.entropy.item() - H) < 3 * tol + 8 * E * 22
    dx, = torch.autograd.grad([out.logprob.sum()], [leaf])
    assert abs(dx[0, V - 1].item() - 1) < 2.0 ** -8
    p = math.exp(logs[3])
    rest = dx[0, ::4097].double()
    assert (rest[1:] + p).abs().max().item() < p * (2.0 ** -8 + 2 * tol + 200 * E)
    del out, dx, rest
    ids = torch.tensor([[V // 2, V - 1, 5, 7]], device=DEV)
    teacher = torch.tensor([[0.5, 0.2, 0.1, 0.1]], device=DEV).log()
    loss = K.k_distill_topk(leaf, teacher, ids, tail=True)
    q = teacher.double().exp()[0].tolist()
    r = 1 - sum(q)
    want = sum(a * (math.log(a) - l) for a, l in zip(q, (logs[0], logs[2], logs[1], logs[3]))) + r * (math.log(r) - math.log((V - 4) / s))
    assert abs(loss.item() - want) < 2 * tol + 8 * E * 40


@pytest.mark.parametrize("n", [77, 60000])
def test_the_largest_table(n):
    V = 2 ** 31 - 2
    ids = torch.randint(0, V, (n,), device=DEV, generator=torch.Generator(device=DEV).manual_seed(n))
    ids[:3] = torch.tensor([V - 1, 0, V - 1], device=DEV)
    leaf = torch.zeros(V, 1, dtype=torch.bfloat16, device=DEV)
    leaf[ids] = 3.0
    leaf.requires_grad_()
    y = K.k_embedding(ids, leaf)
    assert (y == 3).all()
    dw, = torch.autograd.grad([y], [leaf], [torch.ones_like(y)])
    where, count = ids.unique(return_counts=True)
    assert torch.equal(dw[where, 0].long(), count) and dw.count_nonzero().item() == where.numel()


def test_the_longest_batch():
    n, V, d = A.EMBEDDING_MAX_TOKENS, 5000, 1
    ids = torch.randint(0, V, (n,), device=DEV, generator=torch.Generator(device=DEV).manual_seed(2))
    dy = whole_numbers(n, d, 3)
    leaf = torch.arange(V, dtype=torch.float32, device=DEV)[:, None].requires_grad_()
    y = K.k_embedding(ids, leaf, padding_idx=11)
    assert torch.equal(y[:, 0].detach(), ids.float())
    dw, = torch.autograd.grad([y], [leaf], [dy.float()])
    want = torch.zeros(V, d, dtype=torch.int64, device=DEV).index_add_(0, ids, dy)
    want[11] = 0
    assert torch.equal(dw, want.float())                         # (27 thousand rows an id: whole numbers below 2^24)


def test_two_graphs_at_once():
    """Each graph has its own workspaces: replayed on two streams, they do not disturb one another."""
    g = torch.Generator(device=DEV).manual_seed(5)
    jobs = []
    for i in range(2):
        ids = torch.randint(0, 3000, (60000 if i else 9000,), device=DEV, generator=g)
        dy = torch.randn(ids.numel(), 48, device=DEV, generator=g)
        x, tokens = made(500, 9000, torch.bfloat16, seed=i), torch.randint(0, 9000, (500,), device=DEV, generator=g)

        def passes(ids=ids, dy=dy, x=x, tokens=tokens):
            w, leaf = torch.ones(3000, 48, device=DEV, requires_grad=True), x.detach().requires_grad_()
            dw, = torch.autograd.grad([K.k_embedding(ids, w)], [w], [dy])
            out = K.k_token_logprobs(leaf, tokens, top_k=9)
            dx, = torch.autograd.grad([out.logprob, out.entropy], [leaf], [torch.ones(500, device=DEV)] * 2)
            return dw, dx, out.logprob.detach(), out.top_ids

        want = passes()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = passes()
        jobs.append((graph, got, want, torch.cuda.Stream(), passes))         # (whose inputs have to live on)
    for _ in range(20):
        for graph, _, _, stream, _ in jobs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, got, want, _, _ in jobs:
        for a, b in zip(got, want):
            assert torch.equal(a, b)
