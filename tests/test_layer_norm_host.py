"""Layer norm: what the entry points refuse, on the host (no GPU needed)."""
import pytest
import torch

import avsi_amd  # noqa: F401
from avsi_amd import _lib, ops


def _x(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("call,match", [
    (lambda: ops.layer_norm(_x(4, 8, dtype=torch.float64)), "float32, bfloat16 or float16"),
    (lambda: ops.layer_norm(torch.zeros(())), "float32, bfloat16 or float16"),
    (lambda: ops.layer_norm(_x(4, 0)), "unit stride"),
    (lambda: ops.layer_norm(_x(8, 4).t()), "unit stride"),
    (lambda: ops.layer_norm(_x(1, 8).expand(4, 8)), "do not overlap"),
    (lambda: ops.layer_norm(_x(4, 6, 8)[:, :5]), "one stride"),
    (lambda: ops.layer_norm(_x(4, 8), gamma=_x(7)), "gamma must be"),
    (lambda: ops.layer_norm(_x(4, 8), beta=_x(16)[::2]), "beta must be"),
    (lambda: ops.layer_norm(_x(4, 8), gamma=_x(8, dtype=torch.bfloat16)), "gamma must be"),
    (lambda: ops.layer_norm(_x(4, 8, dtype=torch.bfloat16), gamma=_x(8), beta=_x(8, dtype=torch.bfloat16)), "one type"),
    (lambda: ops.layer_norm(_x(4, 8), eps=-1e-6), "eps"),
    (lambda: ops.layer_norm(_x(4, 8), eps=float("nan")), "eps"),
    (lambda: ops.layer_norm(_x(4, 8), y=_x(4, 9)), "columns"),
    (lambda: ops.layer_norm(_x(4, 8), y=_x(5, 8)), "x's shape"),
    (lambda: (lambda t: ops.layer_norm(t, y=t))(_x(4, 8)), "memory of its own"),
    (lambda: (lambda t: ops.layer_norm(t[:, :8], y=t[:, 4:]))(_x(4, 12)), "memory of its own"),
    (lambda: ops.layer_norm(_x(4, 8)), "no GPU|device tensor"),
    (lambda: ops.layer_norm_bwd(_x(4, 8), _x(5, 8), _x(5), _x(5)), "differ in shape"),
    (lambda: ops.layer_norm_bwd(_x(4, 8), _x(4, 8, dtype=torch.float16), _x(4), _x(4)), "differ in shape or type"),
    (lambda: ops.layer_norm_bwd(_x(4, 8), _x(4, 8), _x(3), _x(4)), "mean must hold 4"),
    (lambda: ops.layer_norm_bwd(_x(4, 8), _x(4, 8), _x(4), _x(4, dtype=torch.float16)), "rstd must hold 4"),
    (lambda: (lambda t: ops.layer_norm_bwd(t, _x(4, 8), _x(4), _x(4), dx=t))(_x(4, 8)), "memory of its own"),
])
def test_layer_norm_refuses(call, match):
    with pytest.raises(_lib.AvsiError, match=match):
        call()


def test_layer_norm_c_entry_returns_codes():
    L = _lib.lib()
    one = 16        # never dereferenced: every call below is refused on the host
    ok = dict(x=one, xs=8, dtype=0, gamma=None, beta=None, wdtype=0, y=one, ys=8, mean=one, rstd=one, rows=4, cols=8, eps=1e-5)
    for k, v in (("x", None), ("xs", 7), ("dtype", 3), ("dtype", -1), ("wdtype", 1), ("y", None), ("ys", 7), ("mean", None), ("rstd", None),
                 ("rows", 0), ("cols", 0), ("eps", -1.0), ("eps", float("nan"))):
        assert L.avsi_layer_norm(*dict(ok, **{k: v}).values(), None) == _lib.AVSI_ERR_INVALID_ARG, (k, v)
    bwd = dict(dy=one, dys=8, x=one, xs=8, dtype=1, mean=one, rstd=one, gamma=None, wdtype=0, dx=one, dxs=8, dg=one, db=one, rows=4, cols=8,
               ws=one, nbytes=1 << 20)
    for k, v in (("dy", None), ("dys", 7), ("dx", None), ("dxs", 1), ("dg", None), ("db", None), ("wdtype", 2), ("rows", -1)):
        assert L.avsi_layer_norm_bwd(*dict(bwd, **{k: v}).values(), None) == _lib.AVSI_ERR_INVALID_ARG, (k, v)
    need = L.avsi_layer_norm_bwd_workspace_bytes(4, 8, 1)
    assert need > 0 and L.avsi_layer_norm_bwd_workspace_bytes(0, 8, 1) == 0 and L.avsi_layer_norm_bwd_workspace_bytes(4, 8, 9) == 0
    for k, v in (("ws", None), ("nbytes", need - 1)):
        assert L.avsi_layer_norm_bwd(*dict(bwd, **{k: v}).values(), None) == _lib.AVSI_ERR_WORKSPACE
