"""What one launch cannot hold -- it has fewer than 2^32 threads -- is refused by the entry points in front of it (no GPU needed: pointers
are never followed)."""
import pytest
import torch

import avsi_amd  # noqa: F401
from avsi_amd import _lib, ops

SOME = 4096


def test_convolution():
    L = _lib.lib()
    dim = 1 << 14
    for batch, time in ((1 << 20, 1), (1 << 22, 4)):
        assert L.avsi_causal_conv(SOME, time * dim, dim, 1, SOME, None, 1, None, None, SOME, time * dim, dim, None, batch, time, dim, 4, None) \
            == _lib.AVSI_ERR_UNSUPPORTED
    assert L.avsi_causal_conv_step(SOME, dim, 1, SOME, None, 1, SOME, SOME, dim, 1 << 20, dim, 4, None) == _lib.AVSI_ERR_UNSUPPORTED


@pytest.mark.parametrize("dim,groups", [(1 << 26, 1 << 26), (1 << 26, 1 << 23), ((1 << 22) * 16, 1 << 24)])
def test_scan_of_many_groups(dim, groups):
    L = _lib.lib()
    a = _lib.ScanArgs(1, 1, 1, dim, 16, groups, 1, 0, *([SOME] * 5), *([0] * 12), SOME, SOME, SOME, None, None, SOME, 0, 0, SOME, SOME, SOME,
                      0, 0, *([SOME] * 8))
    assert L.avsi_selective_scan(a, SOME, 1 << 60, None) == _lib.AVSI_ERR_UNSUPPORTED
    assert L.avsi_selective_scan_bwd(a, SOME, 1 << 60, None) == _lib.AVSI_ERR_UNSUPPORTED
    M = lambda *s: torch.empty(*s, device="meta")                                                                      # noqa: E731
    u, A, B = M(1, 1, dim), M(dim, 4), M(1, 1, groups, 4)
    with pytest.raises(_lib.AvsiError, match="below 2\\^23"):
        ops.selective_scan(u, u, A, B, B)
    with pytest.raises(_lib.AvsiError, match="below 2\\^23"):
        ops.selective_scan_bwd(u, u, u, A, B, B, kept=M(4))
    with pytest.raises(_lib.AvsiError, match="no GPU|device tensor"):                 # (a single token has no such launch)
        ops.selective_scan_step(u[:, 0], u[:, 0], A, B[:, 0], B[:, 0], state=M(1, dim, 4))


def test_adamw_values():
    L = _lib.lib()
    for numel in ((1 << 36) - (1 << 12) + 1, 1 << 40):
        t = (_lib.AdamwTensor * 1)(_lib.AdamwTensor(w=SOME, grad=SOME, m=SOME, v=SOME, numel=numel))
        assert L.avsi_adamw(t, 1, 32, 1e-3, 0.9, 0.999, 1e-8, 1, 1.0, None, 0, None) == _lib.AVSI_ERR_INVALID_ARG
