"""GPU: the three operators as one training step: categories looked up in a table, a dense layer in 8-bit floating point, the
gradients back through both, and one AdamW step over table, weight and bias."""
import pytest
import torch

from ddgani_amd import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


class Net:
    """y = layer(table[ids]); loss 0.5 |y - target|^2, explicit gradients as everywhere in this package"""

    def __init__(self, dev, bits=8, V=500, D=192, N=320, seed=0):
        g = torch.Generator(device=dev).manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g, device=dev)
        self.E, self.W, self.b = (rnd(V, D) * 0.5).bfloat16(), (rnd(N, D) / D ** 0.5).bfloat16(), torch.zeros(N, device=dev)
        self.V = V
        self.dE, self.dW, self.db = torch.zeros(V, D, device=dev), torch.zeros(N, D, device=dev), torch.zeros(N, device=dev)
        self.w8 = ops.Fp8Weight(self.W)
        self.opt = ops.AdamW([self.E, self.W, self.b], [self.dE, self.dW, self.db], lr=1e-2, betas=(0.9, 0.95),
                             weight_decay=[0.0, 0.1, 0.0], max_norm=1.0, state_bits=bits, masters=True)

    def forward(self, ids):
        self.h = ops.embedding(ids, self.E, scale=2.0)
        return ops.linear_fp8(self.h, self.w8, bias=self.b, out_dtype=torch.float32)

    def step(self, ids, target):
        y = self.forward(ids)
        dy = (y - target) * (1.0 / ids.numel())
        dx, dW, db = ops.linear_fp8_grads(dy, self.h, self.w8, want_bias=True)
        self.dW.copy_(dW)
        self.db.copy_(db)
        ops.embedding_grad(ids, dx, self.V, scale=2.0, out=self.dE)
        norm = self.opt.step()
        self.w8.refresh(self.W)
        return y, norm


@pytest.mark.parametrize("n", [1, 11, 300])
def test_gradients_of_a_step(dev, n):
    """table, weight and bias gradients of one step against the unquantised chain in 64 bits.  Every product of the step has
    two operands rounded to e4m3 (at most 2^-4 of an element each, independent between elements): a gradient is off by at
    most 2 x 2^-4 of sum |terms| per product it went through."""
    net = Net(dev)
    g = torch.Generator(device=dev).manual_seed(n)
    ids = torch.randint(0, 500, (n,), generator=g, device=dev)
    target = torch.randn(n, 320, generator=g, device=dev)
    E, W = net.E.double(), net.W.double()
    y, norm = net.step(ids, target)
    h = (E[ids] * 2).bfloat16().double()
    dy = (y - target).double() / n
    bound = lambda a, b: 2.0 ** -3 * 1.05 * torch.mm(a.abs(), b.abs().contiguous())
    assert ((y.double() - torch.mm(h, W.t().contiguous())).abs() <= bound(h, W.t()) + 1e-5).all()
    assert ((net.dW.double() - torch.mm(dy.t().contiguous(), h)).abs() <= bound(dy.t().contiguous(), h) + 1e-7).all()
    assert (net.db.double() - dy.sum(0)).abs().max() <= 300 * 2.0 ** -24 * dy.abs().sum(0).max()
    dx, tol = torch.mm(dy, W), bound(dy, W)
    ref, rtol = torch.zeros_like(E), torch.zeros_like(E)
    ref.index_add_(0, ids, 2 * dx)
    rtol.index_add_(0, ids, 2 * tol)
    assert ((net.dE.double() - ref).abs() <= rtol + 1e-7).all()
    total = sum(float((t.double() ** 2).sum()) for t in (net.dE, net.dW, net.db)) ** 0.5
    assert abs(float(norm) - total) <= 1e-6 * total


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_equal_eager_ones(dev, bits):
    g = torch.Generator(device=dev).manual_seed(1)
    a, b = Net(dev, bits), Net(dev, bits)
    ids, target = torch.randint(0, 500, (96,), generator=g, device=dev), torch.randn(96, 320, generator=g, device=dev)
    a.step(ids, target), b.step(ids, target)
    graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=s):
        yb, _ = b.step(ids, target)
    for _ in range(4):
        ids.copy_(torch.randint(0, 500, (96,), generator=g, device=dev))
        target.normal_(generator=g)
        torch.cuda.synchronize()
        ya, _ = a.step(ids, target)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ya, yb)
        for x, y in zip((a.E, a.W, a.b), (b.E, b.W, b.b)):
            assert torch.equal(x, y)


def test_one_row_at_a_time_equals_the_batch(dev):
    """serving: a row computed alone (one launch, at most 16 rows) and within a batch is the same layer"""
    net = Net(dev)
    ids = torch.arange(40, device=dev)
    batch = net.forward(ids)
    h = net.h.double()
    tol = 400 * 2.0 ** -24 * torch.mm(h.abs(), net.W.double().abs().t().contiguous()) * 1.2 + 1e-7
    for i in (0, 7, 39):
        one = net.forward(ids[i:i + 1])
        assert ((one[0] - batch[i]).abs() <= tol[i]).all()
