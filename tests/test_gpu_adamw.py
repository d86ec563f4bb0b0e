"""GPU: the AdamW step over many tensors, against the formulas in 64 bits.

Tolerances, u = 2^-24.  g' = c g carries the clip factor's error: the norm is summed in fp64 from fp32 sums of eight squares
(8 u), its root, the division and the product round once each: 14 u.  m: 3 roundings of numbers up to |m| + |g'|, v: 4 of
numbers up to v + g'^2.  The update lr/c1 * m / (r / c2 + eps) divides by r, whose relative error is half of v's: relative
error of the update at most that of m in units of |m| + (14 + 8 + 8) u.  A weight adds 3 u of itself, a 16-bit parameter
eps / 2, 8-bit states the code's half step (m, to nearest) or whole step (sqrt(v), by dither)."""
import math

import pytest
import torch

from ddgani_amd import ops
from ddgani_amd._lib import DdgError

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def tensors(shapes, dt, k, seed, dev):
    g = torch.Generator(device=dev).manual_seed(seed)
    dts = dt if isinstance(dt, list) else [dt] * len(shapes)
    return [(torch.randn(s, generator=g, device=dev) * k).to(d) for s, d in zip(shapes, dts)]


SHAPES = [(1,), (3, 5), (255,), (256,), (257,), (0,), (33, 129), (4096,), (4099,), (), (70, 300)]
H = dict(lr=1e-2, betas=(0.9, 0.95), eps=1e-8)


def values(opt, key):
    """a state as fp64 values, one flat tensor for each parameter"""
    buf = getattr(opt, key).to(F32).double()
    if opt.state_bits == 8 and key != "masters":
        buf = buf * getattr(opt, key + "_scale").double().repeat_interleave(ops.ADAMW_BLOCK)
    return [buf[o:o + p.numel()] for o, p in zip(opt.offsets, opt.params)]


def snapshot(opt):
    p = [p.double().reshape(-1) for p in opt.params]
    w = p if opt.masters is None else [a if q.dtype == F32 else b for q, a, b in zip(opt.params, p, values(opt, "masters"))]
    return dict(m=values(opt, "exp_avg"), r=values(opt, "exp_avg_sq"), w=w, p=p, t=int(opt.step_count))


def check_step(opt, before, grads):
    """one step from ``before`` (snapshot) with ``grads`` against the formulas"""
    b1, b2 = opt.betas
    t = before["t"] + 1
    assert int(opt.step_count) == t
    g64 = [g.double().reshape(-1) for g in grads]
    c = 1.0
    if opt.max_norm is not None:
        norm = math.sqrt(sum(float((g * g).sum()) for g in g64))
        assert abs(float(opt.norm) - norm) <= 8 * U * norm + 1e-45
        c = min(1.0, opt.max_norm / (norm + 1e-6))
    after = snapshot(opt)
    c1, c2 = 1 - b1 ** t, 1 - b2 ** t
    for i, g in enumerate(g64):
        g = g * c
        m0, r0 = before["m"][i], before["r"][i]
        v0 = r0 * r0 if opt.state_bits == 8 else r0
        m, v = b1 * m0 + (1 - b1) * g, b2 * v0 + (1 - b2) * g * g
        r = v.sqrt()
        tm = 20 * U * (m0.abs() + g.abs())
        tv = 40 * U * (v0 + g * g) + 1e-44
        w0, wd = before["w"][i], opt.weight_decay[i]
        own16 = opt.params[i].dtype != F32
        up = opt.lr / c1 * m / (r / math.sqrt(c2) + opt.eps)
        w = w0 * (1 - opt.lr * wd) - up
        scale_up = opt.lr / c1 / (r / math.sqrt(c2) + opt.eps)
        tw = 4 * U * (w0.abs() + w.abs()) + 40 * U * up.abs() + tm * scale_up + up.abs() * (0.5 * tv / v.clamp(min=1e-300)).clamp(max=1)
        eps16 = torch.finfo(opt.params[i].dtype).eps / 2 if own16 else 0.0
        tiny16 = float(torch.finfo(opt.params[i].dtype).smallest_normal) * eps16
        if opt.masters is not None and own16:
            assert ((after["w"][i] - w).abs() <= tw).all(), i
            assert torch.equal(after["p"][i].to(opt.params[i].dtype), after["w"][i].to(F32).to(opt.params[i].dtype)), i
        else:
            assert ((after["p"][i] - w).abs() <= tw + eps16 * w.abs() * 1.01 + tiny16).all(), i
        if opt.state_bits == 32:
            assert ((after["m"][i] - m).abs() <= tm + 1e-44).all(), i
            assert ((after["r"][i] - v).abs() <= tv).all(), i
            continue
        n = g.numel()
        for key, want, slack in (("exp_avg", m, tm), ("exp_avg_sq", r, (tv / r.clamp(min=1e-300)).clamp(max=1e-3) + 20 * U * r)):
            nb = -(-n // 256)
            pad = torch.zeros(nb * 256, dtype=torch.float64, device=g.device)
            pad[:n] = want.abs()
            top = pad.view(nb, 256).amax(1)
            s = getattr(opt, key + "_scale")[opt.offsets[i] // 256:opt.offsets[i] // 256 + nb].double()
            assert ((s - top / 448).abs() <= 60 * U * top / 448 + 1e-40).all(), (i, key)
            unit = s.repeat_interleave(256)[:n]
            step = torch.maximum(want.abs() * 2.0 ** -3, unit * 2.0 ** -9)          # one code, at most
            off = (after["m" if key == "exp_avg" else "r"][i] - want).abs()
            assert (off <= (0.5 if key == "exp_avg" else 1.0) * step * 1.001 + slack + 60 * U * want.abs()).all(), (i, key)
            if key == "exp_avg_sq":
                got = after["r"][i]
                assert ((got > 0) | (want == 0) | (unit == 0)).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("pt,gt,masters", [(F32, F32, False), (F32, BF16, False), (BF16, BF16, True), (BF16, BF16, False),
                                           (F16, F32, True), (F16, F16, False)])
@pytest.mark.parametrize("max_norm", [None, 1.0, 1e6])
def test_steps(dev, bits, pt, gt, masters, max_norm):
    params, grads = tensors(SHAPES, pt, 0.5, 1, dev), tensors(SHAPES, gt, 0.1, 2, dev)
    decay = [0.1 if i % 2 else 0.0 for i in range(len(SHAPES))]
    opt = ops.AdamW(params, grads, weight_decay=decay, max_norm=max_norm, state_bits=bits, masters=masters, **H)
    for k in range(4):
        before = snapshot(opt)
        norm = opt.step(lr=1e-2 / (k + 1))
        assert (norm is None) == (max_norm is None)
        check_step(opt, before, grads)
        for i, g in enumerate(grads):
            g.copy_(tensors([g.shape], gt, 0.1, 100 * k + i, dev)[0])


def test_mixed_types_and_many_tensors(dev):
    """150 tensors (three tables) of three parameter and three gradient types in one call"""
    shapes = [((i * 37) % 700 + 1,) for i in range(150)]
    pt, gt = [[F32, BF16, F16][i % 3] for i in range(150)], [[F32, BF16, F16][i // 3 % 3] for i in range(150)]
    for bits in (32, 8):
        params, grads = tensors(shapes, pt, 0.5, 3, dev), tensors(shapes, gt, 0.1, 4, dev)
        opt = ops.AdamW(params, grads, weight_decay=0.05, max_norm=0.7, state_bits=bits, masters=True, **H)
        for _ in range(2):
            before = snapshot(opt)
            opt.step()
            check_step(opt, before, grads)


def test_unaligned_views_and_neighbours(dev):
    """parameters and gradients that begin at odd elements of larger buffers; what lies around them stays"""
    g = torch.Generator(device=dev).manual_seed(5)
    big, bg = torch.randn(3000, generator=g, device=dev), torch.randn(3000, generator=g, device=dev).to(BF16)
    cuts = [(1, 260), (263, 264), (301, 1999)]
    params, grads = [big[a:b] for a, b in cuts], [bg[a + 2:b + 2] for a, b in cuts]
    for bits in (32, 8):
        opt = ops.AdamW(params, grads, state_bits=bits, max_norm=1.0, **H)
        keep, before = big.clone(), snapshot(opt)
        opt.step()
        check_step(opt, before, grads)
        inside = torch.zeros(3000, dtype=torch.bool, device=dev)
        for a, b in cuts:
            inside[a:b] = True
        assert torch.equal(big[~inside], keep[~inside])
        gaps = torch.ones(opt.state_len, dtype=torch.bool, device=dev)
        for o, p in zip(opt.offsets, params):
            gaps[o:o + p.numel()] = False
        assert (opt.exp_avg.view(torch.uint8).view(opt.state_len, -1)[gaps] == 0).all()


def test_dither_moves_slow_averages(dev):
    """b2 = 0.999 and no gradient: r falls by 0.05 % a step, far less than a code.  Rounding to nearest would keep it; the
    dither's mean has to follow.  400 steps: r / r0 = 0.999^200; the mean over 4 096 elements of a walk whose steps are
    independent of the value to 2^-20 stays within a few per mille, checked at 2 %."""
    n = 4096
    p, g = [torch.zeros(n, device=dev)], [torch.zeros(n, device=dev)]
    opt = ops.AdamW(p, g, lr=0.0, betas=(0.0, 0.999), state_bits=8)
    g[0].copy_(torch.rand(n, generator=torch.Generator(device=dev).manual_seed(6), device=dev) + 0.5)
    opt.step()
    start = values(opt, "exp_avg_sq")[0]
    g[0].zero_()
    for _ in range(400):
        opt.step()
    end = values(opt, "exp_avg_sq")[0]
    assert abs(float(end.mean() / start.mean()) - 0.999 ** 200) < 0.02
    assert (end > 0).all()


def test_dither_codes(dev):
    """the stored code of sqrt(v) is the grid value below, or the next one where fraction + dither number >= 1"""
    n = 2000
    g = [torch.rand(n, generator=torch.Generator(device=dev).manual_seed(7), device=dev) ** 4 + 1e-7]
    opt = ops.AdamW([torch.zeros(n, device=dev)], g, betas=(0.0, 0.0), state_bits=8)          # v = g^2: r = g
    for t in (1, 2, 3):
        opt.step()
        y = g[0].double() / opt.exp_avg_sq_scale.double().repeat_interleave(256)[:n]
        grid = torch.exp2(torch.frexp(y.clamp(min=2.0 ** -6))[1].double() - 4)
        low = torch.floor(y / grid)
        u = ((torch.arange(n, device=dev) * 2654435769 + t * 2246822507) % 2 ** 32).double() / 2 ** 32
        want = (low + (y / grid - low + u >= 1)) * grid
        want = torch.where(y > 0, want.clamp(min=2.0 ** -9, max=448.0), want)
        got = opt.exp_avg_sq.to(F32).double()[:n]
        border = ((y / grid - low + u - 1).abs() < 1e-5) | ((y / grid - torch.round(y / grid)).abs() < 1e-5)
        assert torch.equal(got[~border], want[~border]) and border.float().mean() < 0.01


def test_blocks_too_small_to_scale_and_zero_gradients(dev):
    n = 700
    p, g = [torch.ones(n, device=dev)], [torch.zeros(n, device=dev)]
    g[0][256:512] = 1e-38                                   # second block: below 2^-100 in m, and v underflows
    for bits in (8, 32):
        opt = ops.AdamW(p, g, state_bits=bits, weight_decay=0.0, **H)
        opt.step()
        assert torch.isfinite(p[0]).all()
        if bits == 8:
            assert (opt.exp_avg_scale == 0).all() and (opt.exp_avg.view(torch.uint8) == 0).all()
            assert torch.equal(p[0][:256], torch.ones(256, device=dev))


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("bits", [32, 8])
def test_non_finite_norm_skips_the_step(dev, bits, bad):
    params, grads = tensors([(300,), (5,)], BF16, 0.5, 8, dev), tensors([(300,), (5,)], BF16, 0.1, 9, dev)
    opt = ops.AdamW(params, grads, state_bits=bits, max_norm=1.0, masters=True, **H)
    opt.step()
    saved = {k: v.clone() for k, v in opt.state_dict().items()}
    old = [p.clone() for p in params]
    keep = grads[1][2].clone()
    grads[1][2] = bad
    norm = opt.step()
    assert not math.isfinite(float(norm))
    assert all(torch.equal(a, b) for a, b in zip(old, params))
    for k, v in opt.state_dict().items():
        assert torch.equal(v.view(torch.uint8), saved[k].view(torch.uint8)), k
    grads[1][2] = keep
    before = snapshot(opt)
    opt.step()
    check_step(opt, before, grads)


def test_state_dict_resumes(dev):
    shapes = [(300, 3), (77,)]
    for bits in (32, 8):
        make = lambda: ops.AdamW(tensors(shapes, BF16, 0.5, 10, dev), tensors(shapes, BF16, 0.1, 11, dev), state_bits=bits,
                                 masters=True, max_norm=1.0, **H)
        a, b = make(), make()
        for _ in range(3):
            a.step()
        for x, y in zip(a.params, b.params):
            y.copy_(x)
        b.load_state_dict({k: v.cpu() for k, v in a.state_dict().items()})
        a.step(), b.step()
        for x, y in zip(a.params, b.params):
            assert torch.equal(x, y)
        for k, v in a.state_dict().items():
            assert torch.equal(v.view(torch.uint8), b.state_dict()[k].view(torch.uint8)), k
    with pytest.raises(DdgError):
        a.load_state_dict(ops.AdamW(tensors(shapes, F32, 1, 1, dev), tensors(shapes, F32, 1, 1, dev)).state_dict())


def test_captured_step_counts_on(dev):
    """a captured step replayed with new gradients equals eager steps bit for bit"""
    shapes = [(1000,), (64, 64), (7,)]
    for bits in (32, 8):
        make = lambda: ops.AdamW(tensors(shapes, BF16, 0.5, 12, dev), tensors(shapes, BF16, 0.1, 13, dev), state_bits=bits,
                                 masters=True, max_norm=1.0, **H)
        a, b = make(), make()
        a.step(), b.step()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            b.step()
        for k in range(4):
            for i, (x, y) in enumerate(zip(a.grads, b.grads)):
                x.copy_(tensors([x.shape], BF16, 0.1, 50 * k + i, dev)[0])
                y.copy_(x)
            torch.cuda.synchronize()
            a.step()
            graph.replay()
            torch.cuda.synchronize()
            assert int(a.step_count) == int(b.step_count) == 2 + k
            for x, y in zip(a.params, b.params):
                assert torch.equal(x, y), (bits, k)


def test_against_the_launch_of_one_net(dev):
    """without decay, clip and masters the step is that of ddg_adam_step"""
    class Net:
        pass
    net, keys = Net(), ("a", "b")
    net.t = dict(zip(keys, tensors([(50, 17), (33,)], F32, 0.5, 14, dev)))
    old = ops.ParamGrads(net, keys)
    params = [net.t[k].clone() for k in keys]
    for k, g in zip(keys, tensors([(50, 17), (33,)], F32, 0.1, 15, dev)):
        old.g[k].copy_(g)
    new = ops.AdamW(params, [old.g[k].contiguous() for k in keys], lr=1e-3, weight_decay=0.0)
    for _ in range(3):
        old.adam_step(lr=1e-3)
        new.step()
    # the product step_size * (m / denom) associates alike; the scalars of the two launches differ by their rounding only
    for k, p in zip(keys, params):
        assert (p - net.t[k]).abs().max() <= 4 * U * (net.t[k].abs().max() + 3e-3)


def test_refusals(dev):
    p, g = torch.zeros(10, device=dev), torch.zeros(10, device=dev)
    bad = [lambda: ops.AdamW([p], [g, g]), lambda: ops.AdamW([p], [g[:5]]), lambda: ops.AdamW([p.double()], [g]),
           lambda: ops.AdamW([p], [g.double()]), lambda: ops.AdamW([p, p], [g, g]), lambda: ops.AdamW([p, p[3:5]], [g, g[:2]]),
           lambda: ops.AdamW([torch.zeros(4, 4, device=dev).t()[:, :2]], [torch.zeros(4, 2, device=dev)]),
           lambda: ops.AdamW([p], [g.cpu()])]
    for i, call in enumerate(bad):
        with pytest.raises(DdgError):
            call()
            pytest.fail(f"call {i} was not refused")


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("max_norm", [None, 0.5])
def test_large_tensors(dev, bits, max_norm):
    """more than a million elements: four blocks per wave, the clip in a launch of its own"""
    shapes = [(1100, 1001), (3,), (70001,), (1 << 20,)]
    params, grads = tensors(shapes, BF16, 0.5, 20, dev), tensors(shapes, [BF16, F32, BF16, F32], 0.1, 21, dev)
    opt = ops.AdamW(params, grads, weight_decay=[0.1, 0.0, 0.0, 0.1], max_norm=max_norm, state_bits=bits, masters=True, **H)
    for _ in range(2):
        before = snapshot(opt)
        opt.step()
        check_step(opt, before, grads)
    if max_norm is None:
        return
    saved, old = {k: v.clone() for k, v in opt.state_dict().items()}, [p.clone() for p in params]
    grads[2][70000] = float("inf")
    assert not math.isfinite(float(opt.step()))
    assert all(torch.equal(a, b) for a, b in zip(old, params))
    assert all(torch.equal(v.view(torch.uint8), saved[k].view(torch.uint8)) for k, v in opt.state_dict().items())


def test_nothing_but_empty_tensors(dev):
    opt = ops.AdamW([torch.zeros(0, device=dev)], [torch.zeros(0, device=dev)], max_norm=1.0, state_bits=8)
    assert float(opt.step()) == 0 and int(opt.step_count) == 1


def test_steps_on_another_stream(dev):
    """the handle made on one stream, used on another after a wait"""
    make = lambda: ops.AdamW(tensors([(5000,)], F32, 0.5, 22, dev), tensors([(5000,)], F32, 0.1, 23, dev), max_norm=1.0, **H)
    a, b = make(), make()
    a.step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b.step()
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(a.params[0], b.params[0])


def test_refused_rate_leaves_the_handle(dev):
    opt = ops.AdamW(tensors([(50,)], F32, 0.5, 24, dev), tensors([(50,)], F32, 0.1, 25, dev), **H)
    for lr in (-1.0, float("nan")):
        with pytest.raises(DdgError):
            opt.step(lr=lr)
    assert opt.lr == H["lr"] and int(opt.step_count) == 0
    with pytest.raises(DdgError):
        ops.AdamW(opt.params, opt.grads, weight_decay=-0.1, **H)
    opt.step()
    assert int(opt.step_count) == 1
