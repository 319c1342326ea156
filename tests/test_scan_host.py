"""Causal convolution and selective scan: what the entry points refuse, on the host (no GPU needed)."""
import ctypes

import pytest
import torch

import avsi_amd  # noqa: F401
from avsi_amd import _lib, ops

F = torch.zeros


def conv(**over):
    a = dict(x=F(2, 5, 6), w=F(6, 4), bias=F(6), state=F(2, 3, 6), lengths=F(2, dtype=torch.int32))
    a.update(over)
    return a


def scan(lead=(2, 5), **over):
    a = dict(u=F(*lead, 6), dt=F(*lead, 6), A=F(6, 4), B=F(*lead, 2, 4), C=F(*lead, 2, 4), D=F(6), z=F(*lead, 6), dt_bias=F(6))
    a.update(over)
    return a


@pytest.mark.parametrize("over,match", [
    (dict(x=F(2, 5, 6, dtype=torch.float64)), "x must be a float32"), (dict(x=F(5, 6)), "3 dimensions"), (dict(w=F(6, 1)), "2 to 8 taps"),
    (dict(w=F(6, 9)), "2 to 8 taps"), (dict(w=F(5, 4)), "w must be contiguous float32"), (dict(w=F(4, 6).t()), "w must be contiguous"),
    (dict(w=F(6, 4, dtype=torch.bfloat16)), "w must be contiguous float32"), (dict(bias=F(5)), "bias must be"),
    (dict(x=F(2, 6, 5).transpose(1, 2)), "unit stride"), (dict(state=F(2, 4, 6)), "state must be"),
    (dict(state=F(2, 3, 6, dtype=torch.bfloat16)), "state must be"), (dict(state=F(1, 3, 6).expand(2, 3, 6)), "state must be contiguous"),
    (dict(lengths=F(2, dtype=torch.int64)), "lengths must be"), (dict(lengths=F(3, dtype=torch.int32)), "lengths must be"),
    (dict(), "no GPU|device tensor")])
def test_causal_conv_refuses(over, match):
    a = conv(**over)
    with pytest.raises(_lib.AvsiError, match=match):
        ops.causal_conv(**a)
    with pytest.raises(_lib.AvsiError, match=match):
        ops.causal_conv_bwd(F(2, 5, 6), **a)


@pytest.mark.parametrize("over,match", [
    (dict(x=F(2, 5, 6)), "2 dimensions"), (dict(state=F(2, 2, 6)), "state must be"), (dict(x=F(6, 2).t()), "unit stride"),
    (dict(state=F(2, 6, 3).transpose(1, 2)), "state must be contiguous"), (dict(), "no GPU|device tensor")])
def test_causal_conv_step_refuses(over, match):
    a = dict(x=F(2, 6), w=F(6, 4), bias=F(6), state=F(2, 3, 6))
    a.update(over)
    with pytest.raises(_lib.AvsiError, match=match):
        ops.causal_conv_step(**a)


def test_causal_conv_step_refuses_its_own_state():
    state = F(2, 3, 6)
    with pytest.raises(_lib.AvsiError, match="part of the state"):
        ops.causal_conv_step(state[:, 0], F(6, 4), state=state)
    with pytest.raises(_lib.AvsiError, match="dy must be"):
        ops.causal_conv_bwd(F(2, 4, 6), F(2, 5, 6), F(6, 4))


SCAN_REFUSALS = [
    (lambda s: dict(u=F(*s, 6, dtype=torch.float64)), "u must be a float32"), (lambda s: dict(u=F(*s, 0)), "u must be"),
    (lambda s: dict(A=F(6, 65)), "1 to 64 states"), (lambda s: dict(A=F(6, 0)), "1 to 64 states"), (lambda s: dict(A=F(5, 4)), "A must be"),
    (lambda s: dict(A=F(6, 4, dtype=torch.float16)), "A must be contiguous float32"), (lambda s: dict(D=F(5)), "D must be"),
    (lambda s: dict(dt_bias=F(6, 1)), "dt_bias must be"), (lambda s: dict(dt=F(*s, 5)), "dt must be"),
    (lambda s: dict(z=F(*s, 6, dtype=torch.bfloat16)), "z must be"), (lambda s: dict(z=F(*s, 12)[..., ::2]), "unit stride"),
    (lambda s: dict(B=F(*s, 2, 5)), "B must be"), (lambda s: dict(C=F(*s, 2, 4, dtype=torch.float16)), "C must be"),
    (lambda s: dict(C=F(*s, 3, 4)), "one number of groups"), (lambda s: dict(B=F(*s, 4, 4), C=F(*s, 4, 4)), "which divides"),
    (lambda s: dict(C=F(*s, 2, 8)[..., ::2]), "unit stride along its states"), (lambda s: dict(), "no GPU|device tensor")]


@pytest.mark.parametrize("make,match", SCAN_REFUSALS)
def test_selective_scan_refuses(make, match):
    with pytest.raises(_lib.AvsiError, match=match):
        ops.selective_scan(**scan(**make((2, 5))))
    a = scan(**make((2, 5)))
    with pytest.raises(_lib.AvsiError, match=match if "GPU" not in match else "kept must be"):
        ops.selective_scan_bwd(torch.zeros_like(a["u"]), **a, kept=F(1))
    with pytest.raises(_lib.AvsiError, match=match):
        ops.selective_scan_step(**scan((2,), **make((2,))), state=F(2, 6, 4))


def test_selective_scan_refuses_states_and_lengths():
    for over, match in ((dict(state=F(2, 6, 5)), "state must be"), (dict(state=F(2, 6, 4, dtype=torch.bfloat16)), "state must be"),
                        (dict(lengths=F(2)), "lengths must be")):
        with pytest.raises(_lib.AvsiError, match=match):
            ops.selective_scan(**scan(), **over)
    with pytest.raises(_lib.AvsiError, match="state must be"):
        ops.selective_scan_step(**scan((2,)), state=F(2, 4, 6).transpose(1, 2))
    with pytest.raises(_lib.AvsiError, match="dout must be"):
        ops.selective_scan_bwd(F(2, 5, 5), **scan(), kept=F(1))


def _args(**over):
    a = _lib.ScanArgs(0, 2, 5, 6, 4, 2, 1)
    for k in ("u", "dt", "z", "B", "C", "A", "out", "state_out", "kept", "dout", "du", "ddt", "dz", "dB", "dC", "dA"):
        setattr(a, k, 16)           # never dereferenced: every call below is refused on the host
    for k, v in over.items():
        setattr(a, k, v)
    return a


def test_scan_c_entries_return_codes():
    L = _lib.lib()
    assert ctypes.sizeof(_lib.ScanArgs) == 336
    for over in (dict(dtype=3), dict(batch=0), dict(time=0), dict(dim=0), dict(state=0), dict(groups=4), dict(groups=0), dict(u=None),
                 dict(A=None), dict(C=None), dict(out=None), dict(batch=65536)):
        assert L.avsi_selective_scan(_args(**over), 16, 1 << 30, None) == _lib.AVSI_ERR_INVALID_ARG, over
    for over in (dict(dout=None), dict(kept=None), dict(dz=None), dict(z=None), dict(dA=None)):
        assert L.avsi_selective_scan_bwd(_args(**over), 16, 1 << 30, None) == _lib.AVSI_ERR_INVALID_ARG, over
    for over in (dict(time=2), dict(state_out=None), dict(dt=None)):
        assert L.avsi_selective_scan_step(_args(**dict(dict(time=1), **over)), None) == _lib.AVSI_ERR_INVALID_ARG, over
    assert L.avsi_selective_scan(_args(state=65), 16, 1 << 30, None) == _lib.AVSI_ERR_UNSUPPORTED
    assert L.avsi_selective_scan_bwd(_args(state=65), 16, 1 << 30, None) == _lib.AVSI_ERR_UNSUPPORTED
    need = L.avsi_selective_scan_bwd_workspace_bytes(_args())
    assert need > 0 and L.avsi_selective_scan_bwd(_args(), 16, need - 1, None) == _lib.AVSI_ERR_WORKSPACE
    long = _args(time=5000)
    need = L.avsi_selective_scan_workspace_bytes(long)
    assert need > 0 and L.avsi_selective_scan(long, None, need, None) == _lib.AVSI_ERR_WORKSPACE
    assert L.avsi_selective_scan(long, 16, need - 1, None) == _lib.AVSI_ERR_WORKSPACE
    assert L.avsi_selective_scan_kept_floats(_args(time=17)) == 2 * 2 * 6 * 4 and L.avsi_selective_scan_kept_floats(_args(state=0)) == 0


def test_conv_c_entries_return_codes():
    L = _lib.lib()
    ok = dict(x=16, xb=30, xt=6, dtype=1, w=16, bias=None, silu=1, state=None, lengths=None, y=16, yb=30, yt=6, out=None, B=2, T=5, D=6, K=4)
    for k, v in (("x", None), ("w", None), ("y", None), ("dtype", 7), ("B", 0), ("T", 0), ("D", 0), ("K", 1), ("K", 9)):
        assert L.avsi_causal_conv(*dict(ok, **{k: v}).values(), None) == _lib.AVSI_ERR_INVALID_ARG, (k, v)
    need = L.avsi_causal_conv_bwd_workspace_bytes(1, 2, 5, 6, 4)
    bwd = dict(dy=16, gb=30, gt=6, x=16, xb=30, xt=6, dtype=1, w=16, bias=None, silu=1, state=None, lengths=None, dx=16, db=30, dt=6, dw=16,
               dbias=16, B=2, T=5, D=6, K=4, ws=16, n=need)
    for k, v in (("dy", None), ("x", None), ("dx", None), ("dw", None), ("K", 0)):
        assert L.avsi_causal_conv_bwd(*dict(bwd, **{k: v}).values(), None) == _lib.AVSI_ERR_INVALID_ARG, (k, v)
    for k, v in (("ws", None), ("n", need - 1)):
        assert L.avsi_causal_conv_bwd(*dict(bwd, **{k: v}).values(), None) == _lib.AVSI_ERR_WORKSPACE, (k, v)
    assert L.avsi_causal_conv_step(16, 6, 1, 16, None, 1, None, 16, 6, 2, 6, 4, None) == _lib.AVSI_ERR_INVALID_ARG
