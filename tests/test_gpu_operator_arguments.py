"""GPU: arguments of the lookup, fp8 and AdamW front ends that contradict each other or lie at the ends of their ranges."""
import pytest
import torch

from ddgani_amd import ops
from ddgani_amd._lib import DdgError

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def test_embedding_grad_refuses_an_out_of_another_type(dev):
    ids, dy = torch.zeros(3, dtype=torch.int64, device=dev), torch.ones(3, 8, device=dev)
    out = torch.full((4, 8), 5.0, device=dev)
    for accumulate in (False, True):
        with pytest.raises(DdgError):
            ops.embedding_grad(ids, dy, 4, out_dtype=BF16, out=out, accumulate=accumulate)
    assert (out == 5).all()
    assert ops.embedding_grad(ids, dy, 4).dtype == F32
    assert ops.embedding_grad(ids, dy.to(BF16), 4).dtype == F32
    assert ops.embedding_grad(ids, dy, 4, out=out.to(BF16)).dtype == BF16
    assert ops.embedding_grad(ids, dy, 4, out_dtype=F32, out=out) is out
