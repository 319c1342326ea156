"""The limits of the sequence operators' sizes and strides, as the C entry points refuse what is beyond them (no GPU needed: nothing is
launched, and the pointers are never followed)."""
import pytest
import torch

import avsi_amd  # noqa: F401
from avsi_amd import _lib, ops

SOME = 4096          # a pointer that is only checked for being there


def scan_args(**over):
    a = _lib.ScanArgs(1, 2, 100, 64, 16, 1, 1, 0, *([SOME] * 5), 6400, 64, 6400, 64, 6400, 64, 1600, 16, 16, 1600, 16, 16, SOME, SOME, SOME,
                      None, None, SOME, 6400, 64, SOME, SOME, SOME, 6400, 64, *([SOME] * 8))
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,status", [
    ({"time": (1 << 30) + 1}, _lib.AVSI_ERR_INVALID_ARG), ({"dim": (1 << 26) + 1}, _lib.AVSI_ERR_INVALID_ARG),
    ({"batch": 65536}, _lib.AVSI_ERR_INVALID_ARG), ({"time": 0}, _lib.AVSI_ERR_INVALID_ARG), ({"groups": 3}, _lib.AVSI_ERR_INVALID_ARG),
    ({"dtype": 3}, _lib.AVSI_ERR_INVALID_ARG), ({"state": 65}, _lib.AVSI_ERR_UNSUPPORTED)]
    + [({k: v}, _lib.AVSI_ERR_UNSUPPORTED) for k in ("u_t", "dt_t", "z_t", "B_t", "C_t", "out_t") for v in ((1 << 26) + 1, -64)])
def test_scan_refuses_what_is_beyond_its_limits(over, status):
    L = _lib.lib()
    a = scan_args(**over)
    assert L.avsi_selective_scan(a, SOME, 1 << 60, None) == status
    if "out_t" not in over:
        assert L.avsi_selective_scan_bwd(a, SOME, 1 << 60, None) == status
    if "state" in over or status == _lib.AVSI_ERR_INVALID_ARG:
        assert L.avsi_selective_scan_kept_floats(a) == L.avsi_selective_scan_workspace_bytes(a) == 0
        assert L.avsi_selective_scan_bwd_workspace_bytes(a) == 0
    if over.get("time", 1) == 1 and not any(k.endswith("_t") for k in over):
        a.time = 1
        assert L.avsi_selective_scan_step(a, None) == status


def test_scan_refuses_a_small_workspace():
    L = _lib.lib()
    a = scan_args()
    need = L.avsi_selective_scan_bwd_workspace_bytes(a)
    assert need and L.avsi_selective_scan_bwd(a, SOME, need - 1, None) == _lib.AVSI_ERR_WORKSPACE
    a = scan_args(time=4096, u_b=4096 * 64)
    need = L.avsi_selective_scan_workspace_bytes(a)
    assert need and L.avsi_selective_scan(a, SOME, need - 1, None) == _lib.AVSI_ERR_WORKSPACE
    assert L.avsi_selective_scan(a, None, need, None) == _lib.AVSI_ERR_WORKSPACE


def test_convolution_refuses_what_is_beyond_its_limits():
    L = _lib.lib()
    for dtype, batch, time, dim, taps in ((0, 1, (1 << 30) + 1, 1, 4), (0, 1, 4, 1, 9), (0, 1, 4, 1, 1), (3, 1, 4, 1, 4), (0, 0, 4, 1, 4)):
        assert L.avsi_causal_conv(SOME, 0, 1, dtype, SOME, None, 1, None, None, SOME, 0, 1, None, batch, time, dim, taps, None) \
            == _lib.AVSI_ERR_INVALID_ARG
        assert L.avsi_causal_conv_bwd(SOME, 0, 1, SOME, 0, 1, dtype, SOME, None, 1, None, None, SOME, 0, 1, SOME, None, batch, time, dim,
                                      taps, SOME, 1 << 60, None) == _lib.AVSI_ERR_INVALID_ARG


def test_scan_step_refuses_inputs_out_of_its_state():
    state = torch.zeros(2, 6, 4)
    u, B = torch.zeros(2, 6), torch.zeros(2, 4)
    part = state.view(2, 24)[:, :6]
    for bad in (dict(u=part), dict(dt=part), dict(z=part), dict(B=state.view(2, 24)[:, :4]), dict(C=state.view(2, 24)[:, 8:12])):
        a = dict(u=u, dt=u, A=torch.zeros(6, 4), B=B, C=B, z=u) | bad
        with pytest.raises(_lib.AvsiError, match="part of the state"):
            ops.selective_scan_step(**a, state=state)
