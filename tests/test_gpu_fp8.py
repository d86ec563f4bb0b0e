"""GPU: the dense layer in 8-bit floating point, against the definition in 64 bits: operands rounded to e4m3 codes times
power-of-two block scales (an exact operation, reproduced here in 64 bits), products and sums in 64 bits.

Tolerances.  fp32 and fp16 results: exact products added in fp32, an error of at most K 2^-24 sum |a b|, one rounding to the
result's type.  bf16 results: the fp8 matrix instructions cut products below 2^-13 of the largest product that a block can hold
(448^2 times its two scales; measured: 10 in 448^2 = 2^-14.3 for a whole block), so 2^-13 448^2 sa sb for each block."""
import pytest
import torch

from ddgani_amd import ops
from ddgani_amd._lib import DdgError

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def quantise(x, a, b):
    """[R, C] -> (values of the codes, scale of each element), fp64; one scale for each a x b block"""
    x = x.double()
    R, C = x.shape
    z = torch.zeros(-(-R // a) * a, -(-C // b) * b, dtype=torch.float64, device=x.device)
    z[:R, :C] = x
    z = z.view(z.shape[0] // a, a, z.shape[1] // b, b)
    top = z.abs().amax((1, 3), keepdim=True)
    live = top >= 2.0 ** -100
    frac, e = torch.frexp(torch.where(live, top, torch.ones_like(top)))          # top = frac 2^e, frac in [1/2, 1)
    s = torch.exp2(e.double() - 9 + (frac > 0.875))                              # smallest power of two with top / s <= 448
    y = z / s
    step = torch.exp2(torch.frexp(y.abs().clamp(min=2.0 ** -6))[1].double() - 4)
    v = torch.where(live, torch.round(y / step) * step * s, torch.zeros_like(z))
    s = torch.where(live, s, torch.zeros_like(s)).expand_as(z)
    back = lambda t: t.reshape(z.shape[0] * a, -1)[:R, :C]
    return back(v), back(s)


def product(qa, sa, qb, sb):
    """rows of a times rows of b -> (result, sum |a b|, bound of the fp8 instructions' cuts)"""
    mm = lambda x, y: torch.mm(x.contiguous(), y.t().contiguous())
    K = qa.shape[1]
    first = torch.arange(0, K, 128, device=qa.device)
    return mm(qa, qb), mm(qa.abs(), qb.abs()), 2.0 ** -13 * 448 ** 2 * mm(sa[:, first], sb[:, first])


def close(got, ref, mass, cut, K):
    eps = torch.finfo(got.dtype).eps / 2
    tiny = float(torch.finfo(got.dtype).smallest_normal) * torch.finfo(got.dtype).eps
    tol = K * 2.0 ** -24 * mass + ref.abs() * (eps * 1.001 + 2.0 ** -23) + tiny
    if got.dtype == BF16:
        tol = tol + cut
    bad = ~((got.double() - ref).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3].tolist(), float((got.double() - ref).abs().max()))
    rel = float((got.double() - ref).norm() / ref.norm().clamp(min=1e-300))
    assert rel <= {F32: 2e-6, F16: 5e-4, BF16: 3e-3}[got.dtype] or float(ref.norm()) < 1e-30, rel


def data(rows, cols, seed, dev, dt=F32, spread=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, device=dev) * (torch.randn(cols, generator=g, device=dev) * spread).exp()
    return x.to(dt)


def check_linear(x, W, bias, y):
    qx, sx = quantise(x, 1, 128)
    qw, sw = quantise(W, 128, 128)
    ref, mass, cut = product(qx, sx, qw, sw)
    if bias is not None:
        ref, mass = ref + bias.double(), mass + bias.double().abs()
    close(y, ref, mass, cut, x.shape[1] + 1)


SIZES = [(1, 1, 1), (1, 127, 3), (2, 128, 16), (7, 129, 17), (15, 300, 100), (16, 1100, 352), (17, 5, 33), (100, 520, 129),
         (128, 176, 352), (129, 384, 600), (300, 1153, 260), (513, 64, 1000)]


@pytest.mark.parametrize("M,K,N", SIZES)
@pytest.mark.parametrize("xt,ot", [(F32, F32), (BF16, BF16), (F16, F16), (F32, BF16), (BF16, F32)])
def test_linear(dev, M, K, N, xt, ot):
    x, W = data(M, K, 1, dev, xt), data(N, K, 2, dev, xt) * 0.1
    for bias in (None, torch.randn(N, generator=torch.Generator(device=dev).manual_seed(3), device=dev)):
        y = ops.linear_fp8(x, ops.Fp8Weight(W, grads=False), bias=bias, out_dtype=ot)
        assert y.dtype == ot
        check_linear(x, W, bias, y)


@pytest.mark.parametrize("M,K,N", [(3200, 256, 3900), (2048, 640, 8192)])
def test_linear_of_many_tiles(dev, M, K, N):
    """enough 256 x 256 tiles for the wide kernel"""
    x, W = data(M, K, 4, dev, BF16), data(N, K, 5, dev, BF16) * 0.1
    check_linear(x, W, None, ops.linear_fp8(x, ops.Fp8Weight(W)))
    check_linear(x, W, None, ops.linear_fp8(x, ops.Fp8Weight(W), out_dtype=F32))


@pytest.mark.parametrize("M", [5, 200])
def test_strides_and_neighbours(dev, M):
    K, N = 150, 70
    wide, Ww = data(M, K + 9, 6, dev, BF16), data(N, K + 5, 7, dev, BF16)
    x, W = wide[:, 3:3 + K], Ww[:, 1:1 + K]
    buf = torch.full((M, N + 11), 5.0, device=dev)
    ops.linear_fp8(x, ops.Fp8Weight(W), out=buf[:, 4:4 + N])
    check_linear(x, W, None, buf[:, 4:4 + N])
    assert (buf[:, :4] == 5).all() and (buf[:, 4 + N:] == 5).all()


@pytest.mark.parametrize("M", [4, 40])
def test_ranges(dev, M):
    """groups of zeros, of very small and of very large numbers, next to ordinary ones; ties and the top of the grid"""
    x, W = data(M, 640, 8, dev), data(50, 640, 9, dev)
    x[:, :128] = 0
    x[0, 128:256] *= 1e-35                                  # below 2^-100: counts as zeros
    x[1, 128:256] *= 1e25
    x[2, 256:384] = torch.linspace(-448, 448, 128, device=dev)
    x[3, 256:384] = 449.0                                   # just above: the next power of two
    W[:, 384:512] = 0
    y = ops.linear_fp8(x, ops.Fp8Weight(W))
    check_linear(x, W, None, y)
    assert (ops.linear_fp8(torch.zeros_like(x), ops.Fp8Weight(W)) == 0).all()


@pytest.mark.parametrize("M", [4, 40])
@pytest.mark.parametrize("ot", [F32, BF16])
def test_infinities_and_nan_stay_in_their_rows(dev, M, ot):
    x, W = data(M, 200, 10, dev), data(33, 200, 11, dev)
    clean = ops.linear_fp8(x, ops.Fp8Weight(W), out_dtype=ot)
    x[1, 5], x[2, 130] = float("inf"), float("nan")
    y = ops.linear_fp8(x, ops.Fp8Weight(W), out_dtype=ot)
    rest = [i for i in range(M) if i not in (1, 2)]
    assert torch.isnan(y[1]).all() and torch.isnan(y[2]).all() and torch.equal(y[rest], clean[rest])


def check_grads(x, W, dy, dx, dw, db):
    M, K = x.shape
    N = W.shape[0]
    qw, sw = quantise(W, 128, 128)
    qd, sd = quantise(dy, 1, 128)
    close(dx, *product(qd, sd, qw.t(), sw.t()), N)
    qdt, sdt = quantise(dy.t(), 1, 128)
    qxt, sxt = quantise(x.t(), 1, 128)
    assert dw.dtype == F32
    close(dw, *product(qdt, sdt, qxt, sxt), M)
    if db is not None:
        ref, mass = dy.double().sum(0), dy.double().abs().sum(0)
        assert ((db.double() - ref).abs() <= (256 + M / 128) * 2.0 ** -24 * mass + 1e-40).all()


@pytest.mark.parametrize("M,K,N", SIZES + [(2000, 1500, 2100)])
@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_grads(dev, M, K, N, dt):
    x, W, dy = data(M, K, 12, dev, dt), data(N, K, 13, dev, dt) * 0.1, data(M, N, 14, dev, dt, spread=0.3)
    w8 = ops.Fp8Weight(W)
    dx, dw, db = ops.linear_fp8_grads(dy, x, w8, want_bias=True)
    assert dx.dtype == dt
    check_grads(x, W, dy, dx, dw, db)
    again = ops.linear_fp8_grads(dy, x, w8, want_bias=True)
    assert all(torch.equal(a, b) for a, b in zip((dx, dw, db), again))
    assert ops.linear_fp8_grads(dy, x, w8)[2] is None


def test_grads_strided_and_mixed_types(dev):
    M, K, N = 210, 140, 90
    x, dy = data(M, K + 6, 15, dev, F32)[:, 2:2 + K], data(M, N + 7, 16, dev, BF16)[:, 5:5 + N]
    W = data(N, K, 17, dev, F16)
    dx, dw, db = ops.linear_fp8_grads(dy, x, ops.Fp8Weight(W), want_bias=True, out_dtype=F32)
    assert dx.dtype == F32
    check_grads(x, W, dy, dx, dw, db)


def test_grads_against_differences(dev):
    """integers of at most four bits are codes: the layer is exact, linear in x and in W, and central differences along
    integer directions equal the gradients' inner products exactly (all sums stay below 2^24)"""
    g = torch.Generator(device=dev).manual_seed(18)
    ints = lambda *s: torch.randint(-4, 5, s, generator=g, device=dev).float()
    M, K, N = 40, 150, 70
    x, W, dy, hx, hw = ints(M, K), ints(N, K), ints(M, N), ints(M, K), ints(N, K)
    f = lambda X, V: (dy.double() * ops.linear_fp8(X, ops.Fp8Weight(V)).double()).sum()
    dx, dw, db = ops.linear_fp8_grads(dy, x, ops.Fp8Weight(W), want_bias=True)
    assert float((f(x + hx, W) - f(x - hx, W)) / 2) == float((dx.double() * hx.double()).sum())
    assert float((f(x, W + hw) - f(x, W - hw)) / 2) == float((dw.double() * hw.double()).sum())
    assert torch.equal(db, dy.sum(0))


def test_no_rows(dev):
    w8 = ops.Fp8Weight(data(5, 9, 19, dev))
    x, dy = torch.zeros(0, 9, device=dev), torch.zeros(0, 5, device=dev)
    assert ops.linear_fp8(x, w8).shape == (0, 5)
    dx, dw, db = ops.linear_fp8_grads(dy, x, w8, want_bias=True)
    assert dx.shape == (0, 9) and (dw == 0).all() and (db == 0).all()


def test_refresh(dev):
    W, V, x = data(40, 200, 20, dev), data(40, 200, 21, dev), data(30, 200, 22, dev)
    w8 = ops.Fp8Weight(W)
    w8.refresh(V)
    assert torch.equal(ops.linear_fp8(x, w8), ops.linear_fp8(x, ops.Fp8Weight(V)))


def test_rows_past_32_bit_offsets(dev):
    """rows x (padded columns) of the packed x beyond 2^32 bytes, and results beyond 2^32 bytes"""
    M, K, N = 4300000, 1000, 300
    W = data(N, K, 23, dev, BF16)
    x = torch.zeros(M, K, dtype=BF16, device=dev)
    rows = [0, 1, 2097151, 2097152, 4194303, 4194304, M - 1]
    x[rows] = data(len(rows), K, 24, dev, BF16)
    y = ops.linear_fp8(x, ops.Fp8Weight(W, grads=False))
    check_linear(x[rows], W, None, y[rows])
    assert (y[3:2097151] == 0).all() and (y[4194305:M - 1] == 0).all()


def test_captured_and_replayed(dev):
    g = torch.Generator(device=dev).manual_seed(25)
    W = data(200, 300, 26, dev, BF16)
    w8 = ops.Fp8Weight(W)
    for M in (3, 150):
        x, dy = data(M, 300, 27, dev, BF16), data(M, 200, 28, dev, BF16)
        graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=s):
            y = ops.linear_fp8(x, w8)
            grads = ops.linear_fp8_grads(dy, x, w8, want_bias=True)
        for _ in range(3):
            x.normal_(generator=g)
            dy.normal_(generator=g)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, ops.linear_fp8(x, w8))
            assert all(torch.equal(a, b) for a, b in zip(grads, ops.linear_fp8_grads(dy, x, w8, want_bias=True)))


def test_refusals(dev):
    w8, x = ops.Fp8Weight(torch.zeros(5, 9, device=dev), grads=False), torch.zeros(4, 9, device=dev)
    bad = [lambda: ops.Fp8Weight(torch.zeros(0, 9, device=dev)), lambda: ops.Fp8Weight(torch.zeros(9, 5, device=dev).t()),
           lambda: ops.Fp8Weight(torch.zeros(9, device=dev)), lambda: ops.Fp8Weight(torch.zeros(5, 9, device=dev).double()),
           lambda: w8.refresh(torch.zeros(9, 5, device=dev)), lambda: ops.linear_fp8(x[:, :8], w8),
           lambda: ops.linear_fp8(x, w8, bias=torch.zeros(4, device=dev)),
           lambda: ops.linear_fp8(x, w8, bias=torch.zeros(5, dtype=BF16, device=dev)),
           lambda: ops.linear_fp8(x, w8, out_dtype=torch.float64), lambda: ops.linear_fp8(x, w8, out=torch.zeros(4, 6, device=dev)),
           lambda: ops.linear_fp8(x.cpu(), w8), lambda: ops.linear_fp8_grads(torch.zeros(4, 5, device=dev), x, w8),
           lambda: ops.linear_fp8_grads(torch.zeros(3, 5, device=dev), x, ops.Fp8Weight(torch.zeros(5, 9, device=dev)))]
    for i, call in enumerate(bad):
        with pytest.raises(DdgError):
            call()
            pytest.fail(f"call {i} was not refused")


@pytest.mark.parametrize("M,K,N", [(17, 8192, 1000), (40, 4200, 300), (300, 9000, 130), (128, 4096, 4096)])
@pytest.mark.parametrize("ot", [F32, BF16, F16])
def test_long_reductions_of_few_tiles(dev, M, K, N, ot):
    """split reductions, whose parts are added in a second launch"""
    x, W = data(M, K, 30, dev, BF16), data(N, K, 31, dev, BF16) * 0.02
    bias = torch.randn(N, generator=torch.Generator(device=dev).manual_seed(32), device=dev)
    w8 = ops.Fp8Weight(W)
    y = ops.linear_fp8(x, w8, bias=bias, out_dtype=ot)
    check_linear(x, W, bias, y)
    assert torch.equal(y, ops.linear_fp8(x, w8, bias=bias, out_dtype=ot))
    buf = torch.full((M, N + 5), 2.0, device=dev, dtype=ot)
    ops.linear_fp8(x, w8, bias=bias, out=buf[:, 3:3 + N])
    assert torch.equal(buf[:, 3:3 + N], y) and (buf[:, :3] == 2).all() and (buf[:, 3 + N:] == 2).all()


@pytest.mark.parametrize("M,K,N", [(20000, 176, 352), (9001, 100, 130), (33, 5000, 40), (33, 40, 5000), (3200, 3900, 520), (3100, 4000, 1600)])
@pytest.mark.parametrize("dt", [F32, BF16])
def test_grads_of_long_batches_and_wide_layers(dev, M, K, N, dt):
    """split reductions over the batch (dW) and over the layer's output (dX); the last case has a dX of bf16 in 256 x 256 tiles"""
    x, W, dy = data(M, K, 33, dev, dt, spread=0.3), data(N, K, 34, dev, dt) * 0.05, data(M, N, 35, dev, dt, spread=0.3)
    w8 = ops.Fp8Weight(W)
    dx, dw, db = ops.linear_fp8_grads(dy, x, w8, want_bias=True)
    check_grads(x, W, dy, dx, dw, db)
    again = ops.linear_fp8_grads(dy, x, w8, want_bias=True)
    assert all(torch.equal(a, b) for a, b in zip((dx, dw, db), again))


@pytest.mark.parametrize("M,K", [(1, 150000), (7, 40000), (16, 9001), (16, 8704), (1, 140001), (3, 46000)])
def test_few_rows_of_long_reductions(dev, M, K):
    """on either side of what fits a workgroup's LDS"""
    x, W = data(M, K, 36, dev, BF16), data(21, K, 37, dev, BF16) * 0.02
    for ot in (F32, BF16):
        check_linear(x, W, None, ops.linear_fp8(x, ops.Fp8Weight(W), out_dtype=ot))


def test_reduction_with_offsets_past_31_bits(dev):
    """rows of 9 million codes: a tile's last row begins beyond 2^31 bytes of its first"""
    M, K, N = 260, 9000000, 3
    x = torch.zeros(M, K, dtype=BF16, device=dev)
    W = torch.zeros(N, K, dtype=BF16, device=dev)
    at = torch.tensor([0, 127, 128, 4500000, K - 1], device=dev)
    rows = torch.tensor([0, 238, 239, 255, 256, 259], device=dev)
    x[rows[:, None], at] = data(6, 5, 38, dev, BF16)
    W[:, at] = data(N, 5, 39, dev, BF16)
    y = ops.linear_fp8(x, ops.Fp8Weight(W, grads=False), out_dtype=F32)
    # (every element named is alone in its block or shares it with one other row's: scales as in the small problem of these columns)
    ref = torch.zeros(M, N, dtype=torch.float64, device=dev)
    for c in at.tolist():
        lo, hi = c // 128 * 128, min(c // 128 * 128 + 128, K)
        mine = [k for k in at.tolist() if lo <= k < hi]
        if c != mine[0]:
            continue
        qx, qw = quantise(x[:, lo:hi], 1, 128)[0], quantise(W[:, lo:hi], 128, 128)[0]
        ref += torch.mm(qx, qw.t().contiguous())
    assert ((y.double() - ref).abs() <= 8 * 2.0 ** -24 * ref.abs() + 1e-6 * ref.abs().max()).all()
    assert (y[1:238] == 0).all()


@pytest.mark.parametrize("N", [3900, 3905])
def test_wide_tiles_strided_with_bias(dev, N):
    """256 x 256 tiles that end inside the matrix, operands and result at odd offsets"""
    M, K = 3201, 333
    wide, Ww = data(M, K + 9, 40, dev, BF16), data(N, K + 5, 41, dev, BF16) * 0.1
    x, W = wide[:, 3:3 + K], Ww[:, 1:1 + K]
    bias = torch.randn(N + 1, generator=torch.Generator(device=dev).manual_seed(42), device=dev)[1:]
    buf = torch.full((M, N + 11), 5.0, device=dev, dtype=BF16)
    ops.linear_fp8(x, ops.Fp8Weight(W), bias=bias, out=buf[:, 3:3 + N])
    check_linear(x, W, bias, buf[:, 3:3 + N])
    assert (buf[:, :3] == 5).all() and (buf[:, 3 + N:] == 5).all()


def test_layers_on_two_streams(dev):
    """two calls at once, each with its own workspace"""
    x, W = data(900, 700, 43, dev, BF16), data(500, 700, 44, dev, BF16) * 0.1
    w8, want = ops.Fp8Weight(W), []
    for k in (1, 2):
        want.append(ops.linear_fp8(x * k, w8, out_dtype=F32).clone())
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(ops.linear_fp8(x * (k + 1), w8, out_dtype=F32))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[k]) for k in (0, 1) for y in got[k])


@pytest.mark.parametrize("M,K,N", [(1, 300, 40000), (5, 300, 20000), (5, 300, 30000), (16, 4096, 5000)])
def test_few_rows_of_wide_layers(dev, M, K, N):
    """on either side of the rule for the launch of few rows, with and without a workspace"""
    x, W = data(M, K, 45, dev, BF16), data(N, K, 46, dev, BF16) * 0.02
    for ot in (F32, BF16):
        check_linear(x, W, None, ops.linear_fp8(x, ops.Fp8Weight(W), out_dtype=ot))


@pytest.mark.parametrize("M,K,N", [(90001, 300, 176), (20001, 176, 352), (40001, 100, 352)])
@pytest.mark.parametrize("ot", [F32, BF16, F16])
def test_tall_layers(dev, M, K, N, ot):
    """many rows of short reductions: every rule for the tiles' size"""
    x, W = data(M, K, 47, dev), data(N, K, 48, dev) * 0.1
    bias = torch.randn(N, generator=torch.Generator(device=dev).manual_seed(49), device=dev)
    check_linear(x, W, bias, ops.linear_fp8(x, ops.Fp8Weight(W), bias=bias, out_dtype=ot))
