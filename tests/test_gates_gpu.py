"""Gates far in their tails: x sigmoid(x) keeps its relative accuracy in float32 down to where the sigmoid leaves the normal range."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _tail(B, T, D):
    return torch.linspace(-86, -10, B * T * D, device="cuda").reshape(B, T, D)


def test_convolution_gate_in_its_tail():
    """One tap of weight one: the input is the gate's argument, without a rounding."""
    from avsi_amd import ops
    x = _tail(2, 41, 65)
    w = torch.tensor([[0.0, 0, 0, 1]], device="cuda").repeat(65, 1)
    z = x.double()
    s = torch.sigmoid(z)
    y, _ = ops.causal_conv(x, w)
    # the sigmoid 7.1 half-ulps, the product one
    assert bool(((y.double() - z * s).abs() <= 9 * U * (z * s).abs()).all())
    state = torch.zeros(82, 3, 65, device="cuda")
    assert torch.equal(ops.causal_conv_step(x.reshape(82, 65), w, state=state).reshape(x.shape), y)
    dy = torch.randn(x.shape, generator=torch.Generator("cuda").manual_seed(1), device="cuda")
    dx = ops.causal_conv_bwd(dy, x, w)[0]
    want = dy.double() * s * (1 + z * (1 - s))
    # s 7.1, 1 + z (1 - s) 10/9 + 1 (of 1 - s times z, and of the sum), two products
    assert bool(((dx.double() - want).abs() <= 12 * U * want.abs()).all())


def test_scan_gate_in_its_tail():
    """No states come in (B is zero) and D u is the sum: out = u z sigmoid(z)."""
    from avsi_amd import ops
    z = _tail(2, 41, 65)
    g = torch.Generator("cuda").manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")                                                         # noqa: E731
    c = {"u": r(2, 41, 65), "dt": r(2, 41, 65), "A": -torch.exp(r(65, 16)), "B": torch.zeros(2, 41, 16, device="cuda"), "C": r(2, 41, 16),
         "D": torch.ones(65, device="cuda"), "z": z}
    out, _, kept = ops.selective_scan(**c, keep=True)
    gate = z.double() * torch.sigmoid(z.double())
    want = c["u"].double() * gate
    assert bool(((out.double() - want).abs() <= 10 * U * want.abs()).all())
    one = {k: (v[:, 3] if v.dim() == 3 else v) for k, v in c.items()}
    step = ops.selective_scan_step(**one, state=torch.zeros(2, 65, 16, device="cuda"))
    assert bool(((step.double() - want[:, 3]).abs() <= 10 * U * want[:, 3].abs()).all())
    dout = r(2, 41, 65)
    grads = ops.selective_scan_bwd(dout, **c, kept=kept)
    s = torch.sigmoid(z.double())
    for got, want, n in ((grads[0], dout.double() * gate, 11), (grads[6], dout.double() * c["u"].double() * s * (1 + z.double() * (1 - s)), 13)):
        assert bool(((got.double() - want).abs() <= n * U * want.abs() + 1e-38).all())


@pytest.mark.parametrize("x,y", [(float("inf"), float("inf")), (float("-inf"), float("nan")), (float("nan"), float("nan")), (-1e30, 0.0),
                                 (1e30, 1e30), (0.0, 0.0), (-120.5, 0.0), (200.0, 200.0)])
def test_convolution_gate_at_its_ends(x, y):
    from avsi_amd import ops
    w = torch.ones(5, 2, device="cuda")
    w[:, 0] = 0
    got = ops.causal_conv(torch.full((1, 1, 5), x, device="cuda"), w)[0]
    assert torch.equal(got.nan_to_num(nan=7.0, posinf=8.0), torch.full_like(got, y).nan_to_num(nan=7.0, posinf=8.0))
