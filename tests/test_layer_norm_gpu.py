"""Layer norm against its formula in 64 bits: widths around every group size of the kernels, odd pitches, types, empty inputs."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _inputs(M, C, dtype, pad=0, shift=0.0, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(M, C + pad, generator=g) + shift).to(dtype).cuda()[:, :C]
    dy = torch.randn(M, C + pad, generator=g).to(dtype).cuda()[:, :C]
    gamma, beta = (1 + 0.3 * torch.randn(C, generator=g)).cuda(), (0.3 * torch.randn(C, generator=g)).cuda()
    return x, dy, gamma, beta


def _check(x, dy, gamma, beta, eps=1e-5):
    """Forward and backward against 64 bits.  Bounds, all from counting roundings of half a step each: a sum over a row is at most 32
    additions in a lane and 10 over the lanes, so a mean is off by less than 48 U32 max|x|, a variance by less than 64 U32 of itself;
    what follows is a handful of operations per element; and one rounding to the output's type."""
    from avsi_amd import ops
    u = torch.finfo(x.dtype).eps / 2
    y, mean, rstd = ops.layer_norm(x, gamma, beta, eps)
    X = x.double()
    G = torch.ones(x.shape[1], device="cuda", dtype=torch.float64) if gamma is None else gamma.double()
    m = X.mean(1, keepdim=True)
    r = 1 / torch.sqrt(((X - m) ** 2).mean(1, keepdim=True) + eps)
    H = (X - m) * r
    Y = H * G + (0 if beta is None else beta.double())
    top = X.abs().amax(1, keepdim=True)
    tol = 64 * U32 * G.abs() * (top * r + H.abs() + top * r * H.abs()) + 2 * u * Y.abs()
    assert y.dtype == x.dtype and y.shape == x.shape and bool(((y.double() - Y).abs() <= tol).all())
    assert bool(((mean.double() - m[:, 0]).abs() <= 48 * U32 * top[:, 0]).all())
    assert bool(((rstd.double() / r[:, 0] - 1).abs() <= 64 * U32 * (1 + (top * r)[:, 0])).all())

    dx, dgamma, dbeta = ops.layer_norm_bwd(dy, x, mean, rstd, gamma)
    m, r = mean.double()[:, None], rstd.double()[:, None]
    H, D = (X - m) * r, dy.double()
    E = D * G
    DX = r * (E - E.mean(1, keepdim=True) - H * (E * H).mean(1, keepdim=True))
    tol = 64 * U32 * r * (E.abs() + E.abs().mean(1, keepdim=True) + H.abs() * (E * H).abs().mean(1, keepdim=True)) + 2 * u * DX.abs()
    assert bool(((dx.double() - DX).abs() <= tol).all())
    # a column of a weight's gradient: at most ceil(M / 512) rows in a lane, 16 groups, 32 partials and 16 sums of them
    n = -(-x.shape[0] // 64) + 80
    assert bool(((dgamma.double() - (D * H).sum(0)).abs() <= n * U32 * (D * H).abs().sum(0)).all())
    assert bool(((dbeta.double() - D.sum(0)).abs() <= n * U32 * D.abs().sum(0)).all())
    # and without the weights' gradients the input's is the same
    assert torch.equal(ops.layer_norm_bwd(dy, x, mean, rstd, gamma, want_wgrad=False)[0], dx)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("M,C,pad", [(1, 1, 0), (3, 1, 2), (5, 2, 0), (7, 63, 0), (33, 64, 1), (9, 65, 3), (8, 127, 0), (250, 257, 31), (65, 512, 0),
                                     (4, 513, 8), (6, 1024, 0), (5, 1025, 7), (3, 2048, 0), (3, 2049, 1), (2, 4097, 0), (3, 8193, 0),
                                     (2, 16384, 0), (2, 16385, 3), (2, 33000, 0), (1100, 24, 0), (2500, 128, 0)])
def test_layer_norm_matches_the_formula(dtype, M, C, pad):
    _check(*_inputs(M, C, dtype, pad, seed=M + C))


@pytest.mark.parametrize("weights", ["none", "gamma", "beta", "16 bits"])
def test_layer_norm_weights(weights):
    x, dy, gamma, beta = _inputs(37, 300, torch.bfloat16)
    if weights == "16 bits":
        _check(x, dy, gamma.bfloat16(), beta.bfloat16())
    else:
        _check(x, dy, gamma if weights == "gamma" else None, beta if weights == "beta" else None)


def test_layer_norm_large_mean_keeps_the_variance():
    # a mean of 1000 and a spread of 1: a one-pass sum of squares would lose the variance; the mean's own rounding is what remains
    _check(*_inputs(64, 700, torch.float32, shift=1000.0))


def test_layer_norm_shapes_and_outputs():
    from avsi_amd import ops
    x = torch.randn(3, 5, 40, device="cuda")
    y, mean, rstd = ops.layer_norm(x)
    assert y.shape == x.shape and mean.shape == rstd.shape == (15,)
    assert torch.equal(y.view(15, 40), ops.layer_norm(x.view(15, 40))[0])
    buf = torch.full((15, 64), 7.0, device="cuda")
    ops.layer_norm(x.view(15, 40), y=buf[:, 8:48])
    assert torch.equal(buf[:, 8:48], y.view(15, 40)) and bool((buf[:, :8] == 7).all()) and bool((buf[:, 48:] == 7).all())
    y0, m0, r0 = ops.layer_norm(torch.empty(0, 40, device="cuda"))
    assert y0.shape == (0, 40) and m0.shape == (0,) and r0.shape == (0,)
    dx, dg, db = ops.layer_norm_bwd(y0, y0, m0, r0)
    assert dx.shape == (0, 40) and bool((dg == 0).all()) and bool((db == 0).all())


def test_layer_norm_nan_stays_in_its_row():
    from avsi_amd import ops
    x, dy, gamma, beta = _inputs(40, 100, torch.float32)
    want = ops.layer_norm(x, gamma, beta)[0].clone()
    x = x.clone()
    x[3, 50], x[20, 99] = float("nan"), float("inf")
    y = ops.layer_norm(x, gamma, beta)[0]
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[3] = bad[20] = True
    assert bool(y[bad].isnan().all()) and torch.equal(y[~bad], want[~bad])


def test_layer_norm_constant_rows():
    from avsi_amd import ops
    x = torch.full((4, 96), 3.0, device="cuda")
    beta = torch.randn(96, device="cuda")
    y, mean, rstd = ops.layer_norm(x, None, beta, eps=1e-5)
    assert torch.equal(y, beta.expand(4, 96)) and bool((mean == 3).all())
    assert bool((rstd - 1e-5 ** -0.5).abs().max() <= 4 * U32 * 1e-5 ** -0.5)


def test_layer_norm_gradient_by_differences():
    from avsi_amd import ops
    x, dy, gamma, beta = _inputs(6, 50, torch.float32, seed=3)
    y, mean, rstd = ops.layer_norm(x, gamma, beta)
    dx, dgamma, dbeta = ops.layer_norm_bwd(dy, x, mean, rstd, gamma)
    g = torch.Generator().manual_seed(9)
    vx, vg, vb = (torch.randn(s, generator=g).cuda() for s in ((6, 50), (50,), (50,)))
    h = 2.0 ** -6
    up, down = (ops.layer_norm(x + k * vx, gamma + k * vg, beta + k * vb)[0].double() for k in (h, -h))
    slope = float(((up - down) * dy.double()).sum() / (2 * h))
    want = float((dx.double() * vx).sum() + (dgamma.double() * vg).sum() + (dbeta.double() * vb).sum())
    # the quotient is off by the roundings of y (300 values, U32 |y| |dy| / h each at the most) and by h^2 / 6 of the third
    # derivative along (v): the inputs are of order 1 and so is it, per element
    bound = 300 * (4 * U32 * 4 * 3 / h + h * h)
    assert abs(slope - want) <= bound


def test_layer_norm_streams_and_graph():
    from avsi_amd import ops
    x, dy, gamma, beta = _inputs(500, 257, torch.float32, pad=31)
    want = [t.clone() for t in ops.layer_norm(x, gamma, beta)]
    wantb = [t.clone() for t in ops.layer_norm_bwd(dy, x, want[1], want[2], gamma)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.layer_norm(x, gamma, beta)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.layer_norm(x, gamma, beta)
        gotb = ops.layer_norm_bwd(dy, x, got[1], got[2], gamma)
    for k in range(4):
        x.mul_(-1.0)
        dy.mul_(2.0)
        graph.replay()
        eager = ops.layer_norm(x, gamma, beta)
        eagerb = ops.layer_norm_bwd(dy, x, eager[1], eager[2], gamma)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager)) and all(torch.equal(a, b) for a, b in zip(gotb, eagerb))
    assert len(wantb) == 3
