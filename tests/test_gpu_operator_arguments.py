"""GPU: arguments of the lookup, fp8 and AdamW front ends that contradict each other or lie at the ends of their ranges."""
import pytest
import torch

from ddgani_amd import _lib, ops
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


def test_a_workspace_for_the_largest_call_serves_smaller_ones(dev):
    """the last batch of an epoch: fewer tokens or rows than the workspace was sized for, which take other chunks and splits"""
    L, gen = _lib.lib(), torch.Generator(device=dev).manual_seed(1)
    stream = torch.cuda.current_stream().cuda_stream
    D, V = 64, 100
    ws = torch.empty(L.ddg_embedding_grad_workspace_bytes(70000, D), dtype=torch.uint8, device=dev)
    for n in (70000, 65537, 65536, 1024, 1023, 3):
        ids, dy = torch.randint(0, V, (n,), generator=gen, device=dev), torch.randn(n, D, generator=gen, device=dev)
        out = torch.empty(V, D, device=dev)
        assert L.ddg_embedding_grad(ids.data_ptr(), 1, n, dy.data_ptr(), 0, D, V, D, 1.0, -1, 0, out.data_ptr(), 0, D, ws.data_ptr(),
                                    ws.numel(), stream) == 0
        assert torch.equal(out, ops.embedding_grad(ids, dy, V))
    inn = outd = 4096
    W = ops.Fp8Weight(torch.randn(outd, inn, generator=gen, device=dev))
    ws = torch.empty(L.ddg_fp8_linear_workspace_bytes(600, outd, inn), dtype=torch.uint8, device=dev)
    wg = torch.empty(L.ddg_fp8_linear_grads_workspace_bytes(600, outd, inn), dtype=torch.uint8, device=dev)
    for rows in (600, 512, 128, 17, 1):
        for dt, code in ((F32, 0), (BF16, 1)):
            x, dy = (torch.randn(rows, k, generator=gen, device=dev).to(dt) for k in (inn, outd))
            y, dx, dw = (torch.empty(s, dtype=t, device=dev) for s, t in (((rows, outd), dt), ((rows, inn), dt), ((outd, inn), F32)))
            assert L.ddg_fp8_linear(x.data_ptr(), code, inn, rows, W.packed.data_ptr(), outd, inn, None, y.data_ptr(), code, outd,
                                    ws.data_ptr(), ws.numel(), stream) == 0
            assert L.ddg_fp8_linear_grads(dy.data_ptr(), code, outd, x.data_ptr(), code, inn, rows, W.packed_t.data_ptr(), outd, inn,
                                          dx.data_ptr(), code, inn, dw.data_ptr(), None, wg.data_ptr(), wg.numel(), stream) == 0
            assert torch.equal(y, ops.linear_fp8(x, W))
            for a, b in zip((dx, dw), ops.linear_fp8_grads(dy, x, W)):
                assert torch.equal(a, b)
