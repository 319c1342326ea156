"""The join of the scan's chunks of time where the decay (or growth) over a whole chunk leaves the range of a float and the states of the
recurrence do not: the same answers as the uncut recurrence in 64 bits, forward and backward."""
import pytest
import torch

from oracle import sequence as O

pytestmark = pytest.mark.gpu

B, T, D, N = 1, 320, 5, 16          # (one workgroup: cut into chunks of 64 steps)


def _near(name, got, want, bound):
    u = torch.finfo(got.dtype).eps / 2
    over = (got.double() - want).abs() / (bound + 1.01 * u * (want.abs() + bound) + 1e-30)
    assert bool((over <= 1).all()), "%s: %.2f times its bound" % (name, float(over.nan_to_num(nan=9e9).max()))


def _case(seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)                                                                        # noqa: E731
    c = {"u": r(B, T, D), "dt": -0.2 * torch.rand(B, T, D, generator=g), "A": 0.75 + 0.5 * torch.rand(D, N, generator=g),
         "B": r(B, T, 1, N), "C": r(B, T, 1, N), "D": r(D), "z": r(B, T, D)}
    return {k: v.cuda() for k, v in c.items()}, r(B, T, D).cuda()


def _check(names, c, dout, state=None):
    from avsi_amd import ops
    out, new, kept = ops.selective_scan(**c, softplus=False, state=state, want_state=True, keep=True)
    val, err = O.scan(**{k: v.double() for k, v in c.items()}, softplus=False, state=None if state is None else state.double(),
                      dout=dout.double())
    got = dict(zip(("out", "state", "du", "ddt", "dA", "dB", "dC", "dD", "dz"),
                   (out, new, *ops.selective_scan_bwd(dout, **c, softplus=False, kept=kept, state=state))))
    for name in names:
        _near(name, got[name], val[name], err[name])


FORWARD, BACKWARD = ("out", "state", "dC", "dD", "dz"), ("du", "ddt", "dA", "dB", "dC", "dD", "dz")


def test_growth_from_zero():
    """Two chunks without input grow by e^140 and more each, from a state that is zero; then inputs come and the states decay.  (Their
    adjoint states are beyond the largest float: the gradients that do not hold them are compared.)"""
    c, dout = _case(1)
    c["dt"][:, :128] = 3.0
    c["u"][:, :128] = 0
    _check(FORWARD, c, dout)


def test_growth_from_zero_from_behind():
    """The last two chunks grow, and no gradient comes in from them.  The states are zero, the gradient of u is not."""
    c, dout = _case(2)
    c["dt"][:, 192:] = 3.0
    c["u"].zero_()
    dout[:, 192:] = 0
    _check(BACKWARD, c, dout)


def test_growth_of_a_tiny_state():
    """A state of 1e-30 that grows by e^96 over one chunk, more than the largest float, stays well inside the range."""
    c, dout = _case(3)
    c["A"].fill_(1.0)
    c["dt"][:, :64] = 1.5
    c["u"][:, :64] = 0
    _check(FORWARD, c, dout, torch.full((B, D, N), 1e-30, device="cuda"))


def test_growth_of_a_tiny_gradient():
    """The same from behind: gradients of 1e-30 that grow by e^96 on their way to the first steps."""
    c, dout = _case(3)
    c["A"].fill_(1.0)
    c["dt"][:, :64] = 1.5
    c["u"][:, :64] = 0
    dout[:, :64] = 0
    dout *= 1e-30
    _check(BACKWARD, c, dout)


def test_an_infinite_state_stays():
    from avsi_amd import ops
    c, _ = _case(4)
    c["A"], c["dt"] = -c["A"], -20 * c["dt"] + 2           # (each chunk decays by e^-96 and less: zero as one factor)
    state = torch.zeros(B, D, N, device="cuda")
    state[0, 2, 3] = float("inf")
    new = ops.selective_scan(**c, softplus=False, state=state, want_state=True)[1]
    assert float(new[0, 2, 3]) == float("inf")
    new[0, 2, 3] = 0
    assert bool(new.isfinite().all())
