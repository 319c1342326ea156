"""Sizes at which a launch of one workgroup per block of columns, or of one thread per quad of outputs, would have 2^32 threads and
more, which the runtime refuses: the last launches of the backward passes go over them in several turns."""
import pytest
import torch

from oracle import sequence as O

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _need(gib):
    if torch.cuda.mem_get_info()[0] < gib * 2 ** 30:
        pytest.skip("needs %d GiB of free memory" % gib)


def _near(name, got, want, bound):
    u = torch.finfo(got.dtype).eps / 2
    over = (got.double() - want).abs() / (bound + 1.01 * u * (want.abs() + bound) + 1e-30)
    assert bool((over <= 1).all()), "%s: %.2f times its bound" % (name, float(over.nan_to_num(nan=9e9).max()))


@pytest.fixture(autouse=True)
def _free():
    yield
    torch.cuda.empty_cache()


def test_layer_norm_weight_gradients_of_more_than_two_to_the_26_columns():
    _need(20)
    from avsi_amd import ops
    C = (1 << 26) + 9
    x, dy = torch.randn(2, 2, C, device="cuda").unbind(0)
    dx, dgamma, dbeta = ops.layer_norm_bwd(dy, x, torch.zeros(2, device="cuda"), torch.ones(2, device="cuda"))
    # (a mean of 0 and a spread of 1: one product per row, one sum of two, each rounded once)
    assert torch.equal(dgamma, dy[0] * x[0] + dy[1] * x[1])
    assert torch.equal(dbeta, dy[0] + dy[1])
    assert bool(dx[:, -9:].isfinite().all())


def test_convolution_weight_gradients_of_more_than_two_to_the_26_sums():
    _need(20)
    from avsi_amd import ops
    D = 27_000_001
    x, dy = torch.randn(2, 1, 2, D, device="cuda").unbind(0)
    w, bias = torch.randn(D, 4, device="cuda"), torch.randn(D, device="cuda")
    dx, dw, dbias = ops.causal_conv_bwd(dy, x, w, bias, silu=False)
    assert torch.equal(dbias, dy[0, 0] + dy[0, 1])
    assert torch.equal(dw[:, 2], dy[0, 1] * x[0, 0]) and bool((dw[:, :2] == 0).all())
    for k in (slice(0, 64), slice(D - 64, D)):
        val, err = O.conv_backward(dy[..., k].double(), x[..., k].double(), w[k].double(), bias[k].double(), silu=False)
        for name, got in (("dx", dx[..., k]), ("dw", dw[k]), ("dbias", dbias[k])):
            _near(name, got, val[name], err[name])


def test_scan_weight_gradients_of_more_than_two_to_the_26_sums():
    _need(20)
    from avsi_amd import ops
    T, D, N = 2, 7_500_032, 16
    assert D * (N + 2) > 1 << 27
    r = lambda *s, t=torch.float32: torch.randn(*s, device="cuda", dtype=t)                                            # noqa: E731
    c = {"u": r(1, T, D, t=BF16), "dt": r(1, T, D, t=BF16).sub_(2), "A": -torch.exp(r(D, N)), "B": r(1, T, 1, N, t=BF16),
         "C": r(1, T, 1, N, t=BF16), "D": r(D), "z": None, "dt_bias": 0.3 * r(D)}
    dout = r(1, T, D, t=BF16)
    out, _, kept = ops.selective_scan(**c, keep=True)
    du, ddt, dA, _, _, dD, _, dbias = ops.selective_scan_bwd(dout, **c, kept=kept)
    for k in (slice(0, 64), slice(D // 2, D // 2 + 64), slice(D - 64, D)):
        part = {n: None if v is None else (v[..., k] if n in ("u", "dt") else v[k] if n in ("A", "D", "dt_bias") else v).double()
                for n, v in c.items()}
        val, err = O.scan(**part, dout=dout[..., k].double())
        for name, got in (("out", out[..., k]), ("du", du[..., k]), ("ddt", ddt[..., k]), ("dA", dA[k]), ("dD", dD[k]),
                          ("ddt_bias", dbias[k])):
            _near(name, got, val[name], err[name])


def test_scan_of_more_quads_of_dB_than_a_launch_has_threads():
    _need(100)
    from avsi_amd import ops
    T, tail = (1 << 27) + 48, 64                # 32 quads of dB and dC per step of a state in no whole quads
    r = lambda *s: torch.randn(*s, device="cuda").to(BF16)                                                             # noqa: E731
    u, B, C, dout = r(1, T, 1), r(1, T, 1), r(1, T, 1), r(1, T, 1)
    dt, A = torch.ones(1, 1, 1, dtype=BF16, device="cuda").expand(1, T, 1), torch.full((1, 1), -30.0, device="cuda")
    dt = dt.contiguous()
    kept = ops.selective_scan(u, dt, A, B, C, softplus=False, keep=True)[2]
    dB, dC = ops.selective_scan_bwd(dout, u, dt, A, B, C, softplus=False, kept=kept)[3:5]
    # a state of 12 steps before has decayed by e^-360, and so has a gradient of 12 steps behind: a window knows nothing of the rest
    for a, b in (((1 << 26) - 44, (1 << 26) + 44), (T - tail, T)):            # (where one launch ends and the next begins; the end)
        k, inner = slice(a, b), slice(12, None if b == T else -12)
        val, err = O.scan(u[:, k].double(), dt[:, k].double(), A.double(), B[:, k, None].double(), C[:, k, None].double(),
                          softplus=False, dout=dout[:, k].double())
        for name, got in (("dB", dB), ("dC", dC)):
            _near(name, got[:, k, None][:, inner], val[name][:, inner], err[name][:, inner])
