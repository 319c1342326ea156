"""Sizes that the 32-bit fields of the C entry points do not hold, or that no launch could take, are refused on the host (no GPU needed:
tensors without memory carry the shapes, and pointers are never followed)."""
import pytest
import torch

import avsi_amd  # noqa: F401
from avsi_amd import _lib, ops

OVER = 1 << 32          # cut to 32 bits, OVER + n is n


def M(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_layer_norm_columns():
    for n in (OVER + 8, (1 << 30) + 1):
        x, stat = M(1, n), M(1)
        with pytest.raises(_lib.AvsiError, match="at most 1073741824 columns"):
            ops.layer_norm(x)
        with pytest.raises(_lib.AvsiError, match="at most 1073741824 columns"):
            ops.layer_norm_bwd(x, x, stat, stat)


@pytest.mark.parametrize("shape,match", [((1, OVER + 100, 1), "at most 1073741824 steps"), ((1, 1, OVER + 8), "at most 2147482624 channels"),
                                         ((OVER + 2, 1, 1), "at most 2147483647 sequences")])
def test_convolution_sizes(shape, match):
    x, w = M(*shape, dtype=torch.bfloat16), M(shape[2], 4)
    with pytest.raises(_lib.AvsiError, match=match):
        ops.causal_conv(x, w)
    with pytest.raises(_lib.AvsiError, match=match):
        ops.causal_conv_bwd(x, x, w)
    if shape[1] == 1:
        with pytest.raises(_lib.AvsiError, match=match):
            ops.causal_conv_step(x[:, 0], w, state=M(shape[0], 3, shape[2], dtype=torch.bfloat16))


@pytest.mark.parametrize("shape,match", [((1, OVER + 100, 1), "at most 1073741824 steps"), ((1, 1, OVER + 64), "at most 67108864 channels"),
                                         ((OVER + 2, 1, 1), "at most 65535 sequences")])
def test_scan_sizes(shape, match):
    u, A, B = M(*shape), M(shape[2], 4), M(*shape[:2], 4)
    with pytest.raises(_lib.AvsiError, match=match):
        ops.selective_scan(u, u, A, B, B, want_state=True, keep=True)
    with pytest.raises(_lib.AvsiError, match=match):
        ops.selective_scan_bwd(u, u, u, A, B, B, kept=M(4))
    if shape[1] == 1:
        with pytest.raises(_lib.AvsiError, match=match):
            ops.selective_scan_step(u[:, 0], u[:, 0], A, B[:, 0], B[:, 0], state=M(shape[0], shape[2], 4))


def test_sizes_at_the_limits_are_not_refused():
    """At the limit the next check speaks: the operands are on no GPU."""
    last = "no GPU|device tensor"
    with pytest.raises(_lib.AvsiError, match=last):
        ops.layer_norm(M(1, 1 << 30))
    with pytest.raises(_lib.AvsiError, match=last):
        ops.causal_conv(M(1, 1 << 30, 1), M(1, 4))
    with pytest.raises(_lib.AvsiError, match=last):
        ops.selective_scan(M(1, 1 << 30, 1), M(1, 1 << 30, 1), M(1, 4), M(1, 1 << 30, 4), M(1, 1 << 30, 4))


def test_convolution_entry_refuses_channels_behind_which_none_has_a_number():
    L, some = _lib.lib(), 4096
    dim = (1 << 31) - 1023
    assert L.avsi_causal_conv(some, dim, dim, 0, some, None, 1, None, None, some, dim, dim, None, 1, 1, dim, 4, None) \
        == _lib.AVSI_ERR_INVALID_ARG
    assert L.avsi_causal_conv_bwd_workspace_bytes(0, 1, 1, dim, 4) == 0
    assert L.avsi_causal_conv_step(some, dim, 0, some, None, 1, some, some, dim, 1, dim, 4, None) == _lib.AVSI_ERR_INVALID_ARG
