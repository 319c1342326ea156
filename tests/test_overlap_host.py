"""Operands that share memory with what a call writes are refused wherever they begin, also in front of it (no GPU needed)."""
import pytest
import torch

import avsi_amd  # noqa: F401
from avsi_amd import _lib, ops

F = torch.zeros


@pytest.mark.parametrize("name,shape", [("u", (2, 6)), ("dt", (2, 6)), ("z", (2, 6)), ("B", (2, 4)), ("C", (2, 4)), ("B", (2, 2, 4)),
                                        ("C", (2, 2, 4)), ("A", (6, 4)), ("D", (6,)), ("dt_bias", (6,))])
def test_scan_step(name, shape):
    groups = shape[1:-1]
    a = dict(u=F(2, 6), dt=F(2, 6), A=F(6, 4), B=F(2, *groups, 4), C=F(2, *groups, 4), D=F(6), z=F(2, 6), dt_bias=F(6))
    n = a[name].numel()
    buf = F(n + 48 + n)
    state = buf[n:n + 48].view(2, 6, 4)
    for at, inside in ((0, False), (1, True), (n - 1, True), (n, True), (n + 47, True), (n + 48, False)):
        a[name] = buf[at:at + n].view(shape)
        with pytest.raises(_lib.AvsiError, match="part of the state" if inside else "no GPU|device tensor"):
            ops.selective_scan_step(**a, state=state)


@pytest.mark.parametrize("name,shape", [("x", (2, 6)), ("w", (6, 4)), ("bias", (6,))])
def test_convolution_step(name, shape):
    a = dict(x=F(2, 6), w=F(6, 4), bias=F(6))
    n = a[name].numel()
    buf = F(n + 36 + n)
    state = buf[n:n + 36].view(2, 3, 6)
    for at, inside in ((0, False), (1, True), (n + 35, True), (n + 36, False)):
        a[name] = buf[at:at + n].view(shape)
        with pytest.raises(_lib.AvsiError, match="part of the state" if inside else "no GPU|device tensor"):
            ops.causal_conv_step(**a, state=state)


def test_layer_norm_outputs():
    buf = F(100)
    y = buf[8:40].view(4, 8)
    for kw in (dict(gamma=buf[1:9]), dict(beta=buf[39:47]), dict(gamma=y[2])):
        with pytest.raises(_lib.AvsiError, match="memory of its own"):
            ops.layer_norm(F(4, 8), **kw, y=y)
    a = dict(mean=F(4), rstd=F(4))
    for kw in (dict(mean=buf[5:9]), dict(rstd=buf[39:43]), dict(gamma=buf[1:9])):
        with pytest.raises(_lib.AvsiError, match="memory of its own"):
            ops.layer_norm_bwd(F(4, 8), F(4, 8), **(a | kw), dx=y)
    with pytest.raises(_lib.AvsiError, match="no GPU|device tensor"):
        ops.layer_norm(F(4, 8), gamma=buf[:8], beta=buf[40:48], y=y)
