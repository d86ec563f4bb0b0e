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


@pytest.mark.parametrize("n", [500, 1_100_003])
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_clips_to_a_norm_below_the_smallest_float(dev, n, bits):
    """max_norm = 1e-50: the clip factor is 1e-50 / |g|, below every fp32 number, for small and for large nets; so the gradients
    count as zeros (g' < 1e-38 where |g| >= 1: an update of lr g' / eps < 1e-32) and the weights stay but for their decay"""
    w = torch.ones(n, device=dev)
    opt = ops.AdamW([w], [torch.full((n,), 0.5, device=dev)], lr=1e-2, weight_decay=0.5, max_norm=1e-50, state_bits=bits)
    norm = opt.step()
    assert abs(float(norm) - 0.5 * n ** 0.5) <= 1e-6 * float(norm)
    assert torch.equal(w, torch.full((n,), 1 - 1e-2 * 0.5, device=dev)) and int(opt.step_count) == 1
    assert float(opt.exp_avg.float().abs().max()) <= 1e-38


def test_adamw_refuses_gradients_inside_parameters(dev):
    """a step writes the parameters while it reads the gradients"""
    buf = torch.zeros(1000, device=dev)
    params = [buf[600:700], buf[100:300], torch.zeros(0, device=dev)]
    fine = [torch.zeros(100, device=dev), torch.zeros(200, device=dev), torch.zeros(0, device=dev)]
    for bad in ([buf[600:700], fine[1]], [buf[650:750], fine[1]], [buf[501:601], fine[1]], [fine[0], buf[299:499]],
                [buf[200:300], fine[1]], [fine[0], buf[50:250]]):
        with pytest.raises(DdgError):
            ops.AdamW(params, bad + fine[2:])
    beside = [buf[500:600], buf[300:500], buf[150:150]]
    opt = ops.AdamW(params, beside)
    opt.step()
    with pytest.raises(DdgError):
        opt.set_grads([buf[699:799]] + beside[1:])
    assert opt.grads[0] is beside[0]
