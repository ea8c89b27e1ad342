"""`k_embedding` on rows of as many columns as it takes (2^30, whose bytes do not fit into 32 bits), and its refusal of longer ones."""
import pytest
import torch

from speedup_thingy_b200 import _abi as A
from speedup_thingy_b200 import kernels as K
from tests.test_token_operator_refusals import BAD, EMBED, EMBED_BWD

MOST = 1 << 30


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d", [MOST + 1, 2 ** 31 - 3, 2 ** 31])
def test_longer_rows_are_refused(d, dtype):
    with pytest.raises(ValueError, match=f"d <= {MOST}"):
        K.k_embedding(torch.zeros(2, dtype=torch.int64, device="meta"), torch.empty(1, d, dtype=dtype, device="meta"))


@pytest.mark.parametrize("d", [MOST + 1, 2 ** 31 - 1])
def test_the_c_abi_refuses_longer_rows(d):
    assert A.load().rte_embedding_fwd(*{**EMBED, "d": d}.values()) == BAD
    assert A.load().rte_embedding_bwd(*{**EMBED_BWD, "d": d, "bytes": 1 << 50}.values()) == BAD
    assert A.load().rte_embedding_bwd_scratch(4, d) == 0
    assert A.load().rte_embedding_bwd_scratch(4, MOST) >= 8 * MOST


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, d", [(torch.bfloat16, MOST), (torch.float16, MOST - 1), (torch.bfloat16, MOST - 4), (torch.float32, MOST // 2), (torch.float32, MOST // 2 + 3)])
def test_the_longest_rows(dtype, d):
    leaf = torch.empty(2, d, dtype=dtype, device="cuda:0")
    leaf[0], leaf[1] = torch.arange(d, dtype=torch.int32, device="cuda:0") % 253, 3.0
    leaf.requires_grad_()
    ids = torch.tensor([0, 1, 0], device="cuda:0")
    y = K.k_embedding(ids, leaf, scale=0.5)
    for i in range(3):
        assert torch.equal(y[i].detach(), leaf[ids[i]].detach() * 0.5), i       # (half of a whole number below 256: exact)
    dy = torch.ones_like(y)
    dy[1] = leaf[0].detach()
    dw, = torch.autograd.grad([y], [leaf], [dy])
    assert (dw[0] == 1.0).all() and torch.equal(dw[1], leaf[0].detach() * 0.5)
