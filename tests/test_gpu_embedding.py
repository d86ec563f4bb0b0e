"""GPU: table lookup with a scale and its gradient by sorted tokens, against the definitions in 64 bits.

Tolerances.  Lookup: one fp32 product (2^-24 relative) and one rounding to the result's type (eps / 2).  Gradient: a row's sum of
m terms is added in fp32 through partial sums of a and of a b terms: at most 2 (a - 1) tokens, 2 (b - 1) and m / (a b) partial sums in a
row, and a - 1 + b - 1 steps inside the longest of these.  (a, b) is (16, 64) below 1 024 tokens and (16, 16) up to 65 536, which is 90 + m / 256 <= 346;
(32, 32) up to 2^20, 186 + m / 1024; then (64, 64), 378 + m / 4096.  The error is at most (400 + m / 1024) 2^-24 sum |terms|; scale,
addition and the rounding to the result's type add 2 x 2^-24 and eps / 2 of the result."""
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


def half_step(t):
    return torch.finfo(t).eps / 2


def smallest(t):
    return float(torch.finfo(t).smallest_normal) * torch.finfo(t).eps      # spacing of the subnormals


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def lookup64(ids, table, scale):
    ok = (ids >= 0) & (ids < table.shape[0])
    y = table.double()[torch.where(ok, ids, 0).long()] * scale
    return torch.where(ok[..., None], y, torch.zeros_like(y))


@pytest.mark.parametrize("shape,V,D", [((0,), 5, 8), ((1,), 1, 1), ((3,), 7, 7), ((2, 33), 50, 8), ((257,), 611, 176),
                                       ((5, 13), 100, 1000), ((9,), 40, 4099), ((4, 700), 3000, 33), ((70000,), 90, 24),
                                       ((40000,), 1000, 260)])
@pytest.mark.parametrize("tt,ot,it", [(F32, F32, torch.int64), (BF16, BF16, torch.int32), (F32, BF16, torch.int64),
                                      (F16, F32, torch.int64), (BF16, F16, torch.int32)])
def test_lookup(dev, shape, V, D, tt, ot, it):
    g = gen(1)
    table = torch.randn(V, D, generator=g, device=dev).to(tt)
    ids = torch.randint(-2, V + 2, shape, generator=g, device=dev).to(it)
    y = ops.embedding(ids, table, scale=1.7, out_dtype=ot)
    assert y.shape == (*shape, D) and y.dtype == ot
    ref = lookup64(ids, table, float(torch.tensor(1.7, dtype=F32)))
    assert ((y.double() - ref).abs() <= ref.abs() * (half_step(ot) * 1.0001 + 2.0 ** -24) + smallest(ot)).all()


def test_lookup_strides_and_extreme_ids(dev):
    g = gen(2)
    wide = torch.randn(50, 40, generator=g, device=dev)
    buf = torch.full((6, 30), 9.0, device=dev)
    ids = torch.tensor([0, 49, 50, -1, 2 ** 62, -2 ** 62], device=dev)
    ops.embedding(ids, wide[:, 3:24], out=buf[:, 5:26])
    ref = torch.zeros(6, 21, device=dev)
    ref[0], ref[1] = wide[0, 3:24], wide[49, 3:24]
    assert torch.equal(buf[:, 5:26], ref)
    assert (buf[:, :5] == 9).all() and (buf[:, 26:] == 9).all()


def test_lookup_past_32_bit_offsets(dev):
    V, D = 1100000, 4096                                  # 4.5e9 elements
    table = torch.zeros(V, D, dtype=BF16, device=dev)
    rows = torch.tensor([0, 524287, 524288, 1048576, V - 1], device=dev)
    table[rows] = torch.randn(5, D, generator=gen(3), device=dev).to(BF16)
    assert torch.equal(ops.embedding(rows, table), table[rows])


def grad64(ids, dy, V, scale, pad=None, old=None):
    """on the CPU: thousands of fp64 atomics on one address are very slow on the device"""
    dev = dy.device
    ids = ids.reshape(-1).long().cpu()
    dy = dy.reshape(ids.numel(), -1).double().cpu()
    ok = (ids >= 0) & (ids < V)
    if pad is not None:
        ok &= ids != pad
    z = torch.zeros(V, dy.shape[1], dtype=torch.float64, device=dy.device)
    total, mass, count = z.clone(), z.clone(), torch.zeros(V, dtype=torch.float64, device=dy.device)
    total.index_add_(0, ids[ok], dy[ok])
    mass.index_add_(0, ids[ok], dy[ok].abs())
    count.index_add_(0, ids[ok], torch.ones_like(ids[ok], dtype=torch.float64))
    total, mass, count = total.to(dev), mass.to(dev), count.to(dev)
    return total * scale + (0 if old is None else old.double()), mass * abs(scale), count


def check_grad(out, ids, dy, V, scale, pad=None, old=None):
    ref, mass, count = grad64(ids, dy, V, scale, pad, old)
    tol = (400 + count / 1024)[:, None] * 2.0 ** -24 * mass + ref.abs() * (2.0 ** -23 + half_step(out.dtype)) + smallest(out.dtype)
    if old is not None:
        tol += old.double().abs() * 2.0 ** -24
        named = count > 0
        assert torch.equal(out[~named], old[~named])
    bad = (out.double() - ref).abs() > tol
    assert not bad.any(), (int(bad.sum()), float((out.double() - ref).abs().max()))


def make_ids(kind, n, V, g, dev):
    if kind == "uniform":
        return torch.randint(0, V, (n,), generator=g, device=dev)
    if kind == "one":
        return torch.full((n,), V - 1, dtype=torch.int64, device=dev)
    if kind == "skewed":
        return (torch.rand(n, generator=g, device=dev) ** 6 * V).long().clamp(max=V - 1)
    return torch.randint(-3, V + 3, (n,), generator=g, device=dev)          # "outside"


@pytest.mark.parametrize("n,V,D", [(1, 1, 1), (63, 2, 7), (64, 1, 8), (65, 3, 9), (257, 611, 176), (4096, 511, 24), (4097, 512, 24),
                                   (4097, 513, 5), (20000, 40000, 33), (9000, 3, 2051), (300000, 70000, 8), (65537, 900, 16), (1100003, 900, 8)])
@pytest.mark.parametrize("kind", ["uniform", "one", "skewed", "outside"])
def test_grad(dev, n, V, D, kind):
    g = gen(n + V)
    ids, dy = make_ids(kind, n, V, g, dev), torch.randn(n, D, generator=g, device=dev)
    out = ops.embedding_grad(ids, dy, V, scale=0.37)
    check_grad(out, ids, dy, V, float(torch.tensor(0.37, dtype=F32)))
    assert torch.equal(out, ops.embedding_grad(ids.int(), dy, V, scale=0.37))          # equal bits, from 32-bit ids too


@pytest.mark.parametrize("dt,ot,accumulate", [(BF16, F32, False), (F16, F16, True), (BF16, BF16, True), (F32, BF16, False),
                                              (F32, F32, True)])
@pytest.mark.parametrize("n,V,D", [(100, 13, 40), (6000, 5000, 61), (12000, 7, 130)])
def test_grad_types_padding_accumulate(dev, dt, ot, accumulate, n, V, D):
    g = gen(n)
    ids = make_ids("outside", n, V, g, dev).view(2, n // 2)
    dy = torch.randn(2, n // 2, D, generator=g, device=dev).to(dt)
    old = torch.randn(V, D, generator=g, device=dev).to(ot) if accumulate else None
    out = None if old is None else old.clone()
    got = ops.embedding_grad(ids, dy, V, scale=2.5, padding_idx=4, out_dtype=ot, out=out, accumulate=accumulate)
    assert got.dtype == ot and (out is None or got is out)
    check_grad(got, ids, dy, V, 2.5, pad=4, old=old)
    if not accumulate:
        assert (got[4] == 0).all()


def test_grad_wide_tables(dev):
    """three and four passes of the sort: more than 2^18 and 2^27 rows"""
    g = gen(5)
    for V, n in ((300001, 10000), ((1 << 27) + 5, 5000)):
        ids, dy = make_ids("uniform", n, V, g, dev), torch.randn(n, 1, generator=g, device=dev).to(BF16)
        ids[:4] = torch.tensor([0, V - 1, V, -1], device=dev)
        out = ops.embedding_grad(ids, dy, V, out_dtype=BF16)
        ok = (ids >= 0) & (ids < V)
        u, inv, cnt = ids[ok].unique(return_inverse=True, return_counts=True)
        s = torch.zeros(len(u), dtype=torch.float64, device=dev).index_add_(0, inv, dy[ok, 0].double())
        m = torch.zeros(len(u), dtype=torch.float64, device=dev).index_add_(0, inv, dy[ok, 0].double().abs())
        assert ((out[u, 0].double() - s).abs() <= s.abs() * 2.0 ** -8 + 400 * 2.0 ** -24 * m).all()
        assert int((out != 0).sum()) <= len(u)


def test_grad_strided_and_guarded(dev):
    g = gen(6)
    n, V, D = 500, 37, 21
    ids, wide = make_ids("uniform", n, V, g, dev), torch.randn(n, 50, generator=g, device=dev)
    buf = torch.full((V, 40), 3.0, device=dev)
    ops.embedding_grad(ids, wide[:, 7:7 + D], V, out=buf[:, 9:9 + D])
    check_grad(buf[:, 9:9 + D].contiguous(), ids, wide[:, 7:7 + D], V, 1.0)
    assert (buf[:, :9] == 3).all() and (buf[:, 9 + D:] == 3).all()


def test_grad_without_tokens(dev):
    none, dy = torch.zeros(0, dtype=torch.int64, device=dev), torch.zeros(0, 9, device=dev)
    assert (ops.embedding_grad(none, dy, 11) == 0).all()
    old = torch.randn(11, 9, generator=gen(7), device=dev)
    assert torch.equal(ops.embedding_grad(none, dy, 11, out=old.clone(), accumulate=True), old)


def test_infinite_and_nan_gradients_stay_in_their_rows(dev):
    ids = torch.tensor([0, 1, 2, 1, -1], device=dev)
    dy = torch.ones(5, 16, device=dev)
    dy[1], dy[2, 3], dy[4] = float("inf"), float("nan"), float("nan")
    out = ops.embedding_grad(ids, dy, 4)
    assert (out[0] == 1).all() and torch.isinf(out[1]).all() and torch.isnan(out[2, 3]) and (out[2, :3] == 1).all()
    assert (out[3] == 0).all()


def test_grad_against_differences(dev):
    """sum(dy * lookup(E)) is linear in E: its central difference along H is <dE, H>, up to the roundings of the lookups"""
    g = gen(8)
    n, V, D = 300, 41, 24
    ids, dy = make_ids("skewed", n, V, g, dev), torch.randn(n, D, generator=g, device=dev)
    E, H = (torch.randn(V, D, generator=g, device=dev) for _ in range(2))
    f = lambda T: (dy.double() * ops.embedding(ids, T, scale=3.0).double()).sum()
    diff = (f(E + H) - f(E - H)) / 2
    dE = ops.embedding_grad(ids, dy, V, scale=3.0)
    # each of the two lookups rounds E +- H and the product: 2 x 2^-24 of 3 (|E| + |H|); dE: as above
    tol = 2 * 2.0 ** -23 * (dy.double().abs() * 3 * (E.abs() + H.abs()).double()[ids]).sum() + \
        450 * 2.0 ** -24 * (grad64(ids, dy, V, 3.0)[1] * H.double().abs()).sum()
    assert abs(float(diff - (dE.double() * H.double()).sum())) <= float(tol)


def test_graphs_on_two_streams_do_not_share_scratch(dev):
    """two captured gradients replayed side by side, several times, each with new inputs"""
    g = gen(9)
    n, V, D = 9000, 700, 64
    cases = []
    for _ in range(2):
        ids, dy = make_ids("skewed", n, V, g, dev), torch.randn(n, D, generator=g, device=dev)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(s):
            ops.embedding_grad(ids, dy, V)
            torch.cuda.synchronize()
            with torch.cuda.graph(graph, stream=s):
                out = ops.embedding_grad(ids, dy, V)
        cases.append((ids, dy, s, graph, out))
    for rep in range(4):
        for ids, dy, *_ in cases:
            ids.copy_(make_ids("skewed", n, V, g, dev))
            dy.normal_(generator=g)
        torch.cuda.synchronize()
        for _, _, s, graph, _ in cases:
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for ids, dy, _, _, out in cases:
            assert torch.equal(out, ops.embedding_grad(ids, dy, V)), rep


def test_refusals(dev):
    t, ids = torch.zeros(4, 8, device=dev), torch.zeros(3, dtype=torch.int64, device=dev)
    bad = [lambda: ops.embedding(ids.float(), t), lambda: ops.embedding(ids, t.double()), lambda: ops.embedding(ids, t.t()),
           lambda: ops.embedding(ids, t[0]), lambda: ops.embedding(ids, t, out=torch.zeros(3, 7, device=dev)),
           lambda: ops.embedding(ids, t, out_dtype=BF16, out=torch.zeros(3, 8, device=dev)),
           lambda: ops.embedding(ids.expand(2, 3), t), lambda: ops.embedding(ids.cpu(), t),
           lambda: ops.embedding(ids, t[:1].expand(4, 8)),
           lambda: ops.embedding_grad(ids, torch.zeros(4, 8, device=dev), 4),
           lambda: ops.embedding_grad(ids, torch.zeros(3, 8, device=dev), 0),
           lambda: ops.embedding_grad(ids, torch.zeros(3, 8, device=dev), 4, accumulate=True),
           lambda: ops.embedding_grad(ids, torch.zeros(3, 8, device=dev), 4, out=torch.zeros(5, 8, device=dev)),
           lambda: ops.embedding_grad(ids, torch.zeros(8, 3, device=dev).t(), 4)]
    for i, call in enumerate(bad):
        with pytest.raises(DdgError):
            call()
            pytest.fail(f"call {i} was not refused")


@pytest.mark.parametrize("n", [70, 5000])
@pytest.mark.parametrize("pad", [None, 2])
def test_grad_of_tokens_that_name_no_row(dev, n, pad):
    """a batch of padding only: long runs of positions that belong to no row"""
    g = gen(8)
    ids = torch.full((n,), -1, dtype=torch.int64, device=dev)
    ids[n // 2:] = 9 if pad is None else pad
    dy = torch.randn(n, 19, generator=g, device=dev).to(BF16)
    dy[0] = float("nan")
    assert (ops.embedding_grad(ids, dy, 9, padding_idx=pad) == 0).all()
    old = torch.randn(9, 19, generator=g, device=dev)
    assert torch.equal(ops.embedding_grad(ids, dy, 9, padding_idx=pad, out=old.clone(), accumulate=True), old)
