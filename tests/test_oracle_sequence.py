"""The oracle of the causal convolution and the selective scan against torch's autograd in 64 bits (CPU)."""
import pytest
import torch

from oracle import sequence as O


def _case(seed, ragged, B=3, T=9, D=6, N=5, G=2, K=4):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)                                                   # noqa: E731
    c = {"u": r(B, T, D), "dt": r(B, T, D), "A": -torch.rand(D, N, generator=g, dtype=torch.float64) * 3, "B": r(B, T, G, N),
         "C": r(B, T, G, N), "D": r(D), "z": r(B, T, D), "dt_bias": r(D), "x": r(B, T, D), "w": r(D, K), "bias": r(D)}
    return c, r(B, T, D), r(B, K - 1, D), r(B, D, N), torch.tensor([T, 0, 4], dtype=torch.int32) if ragged else None


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("softplus", [True, False])
def test_scan_gradients_are_autograds(ragged, softplus):
    c, dout, _, state, lengths = _case(1, ragged)
    c["dt"] = c["dt"] if softplus else c["dt"].abs() * 0.2
    names = ("u", "dt", "A", "B", "C", "D", "z", "dt_bias")
    t = {k: c[k].clone().requires_grad_() for k in names}
    B, T, D = t["u"].shape
    x = t["dt"] + t["dt_bias"]
    delta = torch.nn.functional.softplus(x) if softplus else x
    h, outs = state.clone(), []
    for i in range(T):
        on = torch.ones(B, dtype=torch.bool) if lengths is None else i < lengths
        Bw, Cw = (t[k][:, i].repeat_interleave(D // 2, dim=1) for k in ("B", "C"))
        n = torch.exp(delta[:, i, :, None] * t["A"]) * h + (delta[:, i] * t["u"][:, i])[..., None] * Bw
        h = torch.where(on[:, None, None], n, h)
        y = (h * Cw).sum(-1) + t["D"] * t["u"][:, i]
        outs.append(torch.where(on[:, None], y * torch.nn.functional.silu(t["z"][:, i]), torch.zeros(())))
    out = torch.stack(outs, 1)
    val, err = O.scan(*(c[k] for k in names), softplus=softplus, state=state, lengths=lengths, dout=dout)
    assert torch.allclose(val["out"], out, atol=1e-12) and torch.allclose(val["state"], h, atol=1e-12)
    for k, g in zip(names, torch.autograd.grad(out, [t[k] for k in names], dout)):
        assert torch.allclose(val["d" + k], g, atol=1e-11, rtol=1e-11), k
    assert set(err) == set(val) and all(bool((v >= 0).all()) for v in err.values())


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("silu", [True, False])
def test_conv_gradients_are_autograds(ragged, silu):
    c, dy, state, _, lengths = _case(2, ragged)
    x, w, bias = (c[k].clone().requires_grad_() for k in ("x", "w", "bias"))
    D, K = w.shape
    pre = torch.nn.functional.conv1d(torch.cat([state, x], 1).transpose(1, 2), w[:, None], bias, groups=D).transpose(1, 2)
    on = O.inside(x.shape[0], x.shape[1], lengths, "cpu")[..., None]
    y = torch.where(on, torch.nn.functional.silu(pre) if silu else pre, torch.zeros(()))
    f = O.conv_forward(c["x"], c["w"], c["bias"], silu, state, lengths)[0]
    assert torch.allclose(f["y"], y, atol=1e-12)
    val, _ = O.conv_backward(dy, c["x"], c["w"], c["bias"], silu, state, lengths)
    for k, g in zip(("dx", "dw", "dbias"), torch.autograd.grad(y, (x, w, bias), dy)):
        assert torch.allclose(val[k], g, atol=1e-11), k
    for b in range(3):
        n = x.shape[1] if lengths is None else int(lengths[b])
        assert torch.equal(f["state"][b], torch.cat([state[b], c["x"][b, :n]])[n:n + K - 1])
