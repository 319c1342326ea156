"""AdamW over many tensors: what the plan and the entry point refuse, on the host (no GPU needed)."""
import ctypes

import pytest
import torch

import avsi_amd  # noqa: F401
from avsi_amd import _lib, ops

F = torch.zeros
H = torch.bfloat16


@pytest.mark.parametrize("args,kw,match", [
    (([], []), {}, "at least one"), (([F(4)], []), {}, "0 gradients for 1"), (([F(4)], [F(5)]), {}, "gradient must be"),
    (([F(4)], [F(4, dtype=torch.float64)]), {}, "gradient must be"), (([F(4, dtype=H)], [F(4)]), {}, "contiguous float32"),
    (([F(4, 4).t()[:3]], [F(3, 4)]), {}, "contiguous float32"), (([F(4)], [F(8)[::2]]), {}, "gradient must be"),
    (([F(4)], [F(4)]), dict(bits=16), "8 or in 32"), (([F(4)], [F(4)]), dict(weight_decay=[0.1, 0.2]), "as many"),
    (([F(4)], [F(4)]), dict(copies=[None, None]), "as many"), (([F(4)], [F(4)]), dict(copies=[F(4)]), "copy must be"),
    (([F(4)], [F(4)]), dict(copies=[F(5, dtype=H)]), "copy must be"), (([F(4)], [F(4)]), {}, "no GPU|device tensor")])
def test_plan_refuses(args, kw, match):
    with pytest.raises(_lib.AvsiError, match=match):
        ops.AdamwPlan(*args, **kw)


def test_c_entry_returns_codes():
    L = _lib.lib()
    assert ctypes.sizeof(_lib.AdamwTensor) == 72

    def call(count=1, bits=32, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, step=1, scale=1.0, skip=None, n_skip=0, table=True, **over):
        t = (_lib.AdamwTensor * 1)(_lib.AdamwTensor(w=16, grad=16, m=16, v=16, m_scale=16, v_scale=16, numel=4))
        for k, v in over.items():
            setattr(t[0], k, v)
        return L.avsi_adamw(t if table else None, count, bits, lr, b1, b2, eps, step, scale, skip, n_skip, None)
    bad = [dict(table=False), dict(count=-1), dict(bits=16), dict(step=0), dict(b1=1.0), dict(b1=-0.1), dict(b2=1.0), dict(b2=float("nan")),
           dict(eps=-1.0), dict(n_skip=9, skip=16), dict(n_skip=1), dict(n_skip=-1), dict(w=None), dict(grad=None), dict(m=None), dict(v=None),
           dict(numel=-1), dict(grad_dtype=3), dict(copy=16, copy_dtype=-1), dict(bits=8, m_scale=None), dict(bits=8, v_scale=None)]
    for kw in bad:
        assert call(**kw) == _lib.AVSI_ERR_INVALID_ARG, kw
