"""`k_embedding` at scales that are not finite, on a B200."""
import pytest
import torch

from speedup_thingy_b200 import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("scale", [float("inf"), float("nan"), -float("inf")])
def test_ids_outside_the_table_give_zeros_whatever_the_scale(scale):
    w = torch.ones(5, 8, device=DEV)
    ops = K._ops_for(w)
    y = K.k_embedding(torch.tensor([1, -1, 7], device=DEV), w, scale=scale)
    assert not y[1:].any() and not y[0].isfinite().any()
    ops.status.zero_()
