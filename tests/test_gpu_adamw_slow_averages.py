"""GPU: what the 8-bit AdamW states make of gradients that stop, or nearly so, over hundreds of steps, beside the 32-bit states.

A weight whose gradient is 0 from step 21 on moves by the sum of lr m / r over its decaying m, and then rests.  In 32 bits m / r
falls by b1 / sqrt(b2) a step.  In 8 bits m's decay is dithered (right on average) or, in e4m3's normal range at b1 = 0.9, goes to
nearest: code by code from 1 to 1/2 in 7 steps where ln 2 / ln(1 / 0.9) = 6.6 are right, which makes the sum larger by 6.4 % at most.
r steps down by one code c (1/8 of it at most) with probability (1 - sqrt(b2)) r / c, a variance of (1 - sqrt(b2)) / 8 a step
relative to r^2: 0.0032 at b2 = 0.95, and over the ten or twenty steps that m lives a mean of 1 / r that is larger by 1.6 % (half of
them count, weighed by m).  So the mean movement of thousands of weights agrees to 10 %.  A stored m of 0 stays 0 without a
gradient, and then the weight stays bit for bit; the largest code needs 15 halvings to the linear range (100 steps at b1 = 0.9, 200 at
0.95, 1 030 at 0.99), and a last code survives a step with probability b1: the Weyl sequence puts at least one of 4 / (1 - b1)
consecutive numbers into an interval of 1 - b1, and the eight linear codes fall no slower than the last."""
import pytest
import torch

from ddgani_amd import ops

pytestmark = pytest.mark.gpu
LR = 1e-3


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def train(dev, bits, betas, n, steps, quiet, max_norm=None, dtype=torch.float32, at=()):
    """every other weight gets ``quiet(m)`` from step 21 on -> weights after step 20, after the steps ``at`` and at the end, handle"""
    gen = torch.Generator(device=dev).manual_seed(1)
    w, g = torch.zeros(n, device=dev, dtype=dtype), torch.zeros(n, device=dev)
    opt = ops.AdamW([w], [g], lr=LR, betas=betas, weight_decay=0.0, state_bits=bits, max_norm=max_norm,
                    masters=dtype != torch.float32)
    silent = torch.arange(n, device=dev) % 2 == 1
    value = lambda: (w if opt.masters is None else opt.masters[:n]).clone()
    kept = []
    for t in range(1, steps + 1):
        x = torch.randn(n, generator=gen, device=dev)
        if t == 21:
            rest = quiet(opt.exp_avg.float()[:n])
        g.copy_(x if t <= 20 else torch.where(silent, rest, x))
        opt.step()
        if t == 20 or t in at:
            kept.append(value())
    return [k[silent] for k in kept] + [value()[silent]], opt, silent


@pytest.mark.parametrize("betas,rest,steps", [((0.9, 0.95), 500, 2000), ((0.95, 0.95), 900, 2000), ((0.9, 0.999), 500, 2000),
                                              ((0.99, 0.999), 4500, 6000)])
def test_weights_without_a_gradient_come_to_rest(dev, betas, rest, steps):
    n = 4096
    (a, end), _, _ = train(dev, 32, betas, n, steps, torch.zeros_like)
    want = float((end - a).abs().mean())
    (a, mid, end), opt, silent = train(dev, 8, betas, n, steps, torch.zeros_like, at=(rest,))
    assert (opt.exp_avg.float()[silent] == 0).all() and (opt.exp_avg.float()[~silent] != 0).float().mean() > 0.9
    assert torch.equal(mid, end)
    assert abs(float((end - a).abs().mean()) - want) <= 0.1 * want


@pytest.mark.parametrize("max_norm", [None, 1e9])
def test_many_weights_without_a_gradient_come_to_rest(dev, max_norm):
    """more than a million: four blocks per wave; 16-bit parameters with masters"""
    n, betas, dt = 1_100_003, (0.9, 0.95), torch.bfloat16
    (a, end), _, _ = train(dev, 32, betas, n, 600, torch.zeros_like, max_norm, dt)
    want = float((end - a).abs().mean())
    (a, mid, end), _, _ = train(dev, 8, betas, n, 600, torch.zeros_like, max_norm, dt, at=(500,))
    assert torch.equal(mid, end)
    assert abs(float((end - a).abs().mean()) - want) <= 0.1 * want


@pytest.mark.parametrize("betas", [(0.9, 0.95), (0.95, 0.95)])
def test_weights_follow_a_gradient_far_below_a_code(dev, betas):
    """a steady gradient of a quarter of m's lowest code, against the sign that m had: once the old m is gone (as above), the
    stored one is 0 or a code of the gradient's sign, so that weights go against the gradient in every step, and not further than
    in 32 bits, where r is the gradient's size and not at least a code"""
    against = lambda m: torch.where(m > 0, -1e-6, 1e-6)
    (_, at500, end), opt, silent = train(dev, 8, betas, 4096, 1500, against, at=(500,))
    way = -torch.sign(opt.grads[0][silent])
    moved = (end - at500) * way
    assert (moved >= 0).all() and moved.mean() > 0
    assert (moved <= 1000 * LR).all()


@pytest.mark.parametrize("b1", [0.9, 0.95])
def test_codes_of_m(dev, b1):
    """b1 = 0.9: nearest, but the dithered code where the old code and the nearest one are linear (below 2^-6); b1 = 0.95:
    dithered everywhere; either only where the block's largest m grew by less than half.  From the stored state in 64 bits; what
    lies within 1e-4 of a border may go either way (a value in units of a code, up to 16 of them, is off by 16 x 60 x 2^-24 =
    6e-5)."""
    n = 5000
    gen = torch.Generator(device=dev).manual_seed(2)
    g = (torch.rand(n, generator=gen, device=dev) * 40 - 31).exp2() * 4e4       # 2^-31 ... 2^9, times 4e4; smaller or larger each step
    opt = ops.AdamW([torch.zeros(n, device=dev)], [g], betas=(b1, 0.95), lr=0.0, state_bits=8)
    dithered = 0
    for t in range(1, 8):
        g.mul_(torch.randn(n, generator=gen, device=dev))
        spread = lambda: opt.exp_avg_scale.double().repeat_interleave(256)[:n]
        m0, s0 = opt.exp_avg.float().double()[:n] * spread(), spread()
        opt.step()
        y, old = (b1 * m0 + (1 - b1) * g.double()) / spread(), m0.abs() / s0.clamp(min=1e-300)
        grid = torch.exp2(torch.frexp(y.abs().clamp(min=2.0 ** -6))[1].double() - 4)
        u = ((torch.arange(n, device=dev) * 3242174889 + t * 2447445413) % 2 ** 32).double() / 2 ** 32
        low = torch.floor(y.abs() / grid)
        frac = y.abs() / grid - low
        grown, nearest = s0 / spread(), torch.round(y.abs() / grid) * grid
        by_dither = (grown > 0.6667) & ((nearest < 2.0 ** -6) & (old < 2.0 ** -6) | torch.tensor(b1 > 0.93, device=dev))
        want = torch.where(by_dither, (low + (frac + u >= 1)) * grid, nearest)
        want = want.clamp(max=448.0) * torch.sign(y)
        border = ((frac - 0.5).abs() < 1e-4) | ((grown / 0.6667 - 1).abs() < 1e-4)
        border |= by_dither & (((frac + u - 1).abs() < 1e-4) | ((frac < 1e-4) & (low > 0)) | (frac > 1 - 1e-4))
        got = opt.exp_avg.float().double()[:n]
        assert torch.equal(got[~border], want[~border]), t
        assert border.float().mean() < 0.02
        dithered += int((by_dither & (want.abs() != nearest) & ~border).sum())
    assert dithered > 100
