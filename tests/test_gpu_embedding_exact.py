"""`k_embedding`'s gradient over long and heavily repeated ids on a B200, from whole numbers: every sum is exact in fp32 (below 2^24), so that a
row that is dropped, doubled or in the wrong place shows however many others there are."""
import pytest
import torch

from speedup_thingy_b200 import kernels as K
from tests.test_gpu_embedding import some_ids

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def whole_numbers(n, d, seed):
    return torch.randint(-3, 4, (n, d), device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed))


def check(ids, V, d, seed, padding=None):
    n = ids.numel()
    dy = whole_numbers(n, d, seed)
    keep = torch.ones(n, dtype=torch.bool, device=DEV) if padding is None else ids != padding
    want = torch.zeros(V, d, dtype=torch.int64, device=DEV).index_add_(0, ids[keep], dy[keep])
    most = torch.zeros(V, d, dtype=torch.int64, device=DEV).index_add_(0, ids[keep], dy[keep].abs()).max().item()
    assert most < 2 ** 24                                        # (every partial sum is a whole number below it)
    leaf = torch.zeros(V, d, device=DEV, requires_grad=True)
    dw, = torch.autograd.grad([K.k_embedding(ids, leaf, padding_idx=padding)], [leaf], [dy.float()])
    assert torch.equal(dw, want.float()), (ids.shape, V, d, (dw != want).nonzero()[:5].tolist())


@pytest.mark.parametrize("n, V, d, kind", [
    (2200000, 50, 2, "same"), (4100000, 3, 1, "same"), (8192, 100, 16, "zipf"), (8193, 100, 16, "zipf"), (8193, 5000, 16, "same"), (8192, 20000, 16, "same"),
    (49152, 3000, 8, "zipf"), (49153, 3000, 8, "zipf"), (49152, 70000, 8, "random"), (60000, 70000, 8, "descending"), (48001, 2, 8, "ends"), (700001, 40000, 4, "zipf"),
    (700001, 3000000, 4, "random"), (640000, 1 << 21, 2, "descending"), (131072, 131072, 72, "zipf"), (100003, 50257, 24, "zipf"), (70000, 9, 136, "random"),
    (66000, 300, 8, "same"), (300000, 1000, 4, "zipf"), (65, 3, 130, "ends"), (4097, 7, 33, "random")])
def test_every_row_is_added_once(n, V, d, kind):
    ids = some_ids(kind, n, V)
    check(ids, V, d, seed=n)
    check(ids, V, d, seed=n + 1, padding=int(ids[n // 2]))


@pytest.mark.parametrize("n", [7, 8, 9, 16, 17, 31, 33, 64, 100, 8191, 8192, 32767, 32768, 65535, 65536])
def test_runs_that_end_about_a_range(n):
    """Runs of one id as long as one, two and three ranges of 8 to 64 rows, one more and one less."""
    lengths = [8 * r + e for r in (1, 2, 3, 4, 8, 16, 24) for e in (-1, 0, 1)]
    runs, total = [], 0
    while total < n:
        runs.append(min(lengths[len(runs) * 5 % len(lengths)], n - total))
        total += runs[-1]
    ids = torch.repeat_interleave(torch.arange(len(runs), device=DEV), torch.tensor(runs, device=DEV))
    order = torch.randperm(n, device=DEV, generator=torch.Generator(device=DEV).manual_seed(n))
    for v in (ids, ids[order]):
        check(v, len(runs) + 2, 9, seed=n)


@pytest.mark.parametrize("kind", ["zipf", "same", "distinct", "ascending", "ends", "random"])
# few tokens are added in one launch: its limits of tokens, columns and rows, and rows that share 16 bytes
@pytest.mark.parametrize("n, V, d", [(1, 1, 1), (2, 3, 5), (16, 300, 33), (17, 40, 2048), (64, 64 * 2368, 3), (64, 64 * 2368 + 1, 3), (128, 5000, 512), (136, 5000, 512), (2047, 2000, 8),
                                     (2048, 100000, 7), (2049, 100000, 7), (2048, 9, 32), (1000, 151000, 31), (8, 30000, 770), (300, 4097, 130)])
def test_few_tokens(n, V, d, kind):
    ids = some_ids(kind, n, V)
    check(ids, V, d, seed=n)
    check(ids, V, d, seed=n + 1, padding=int(ids[0]))
    check(ids, V, d, seed=n + 2, padding=V - 1)
