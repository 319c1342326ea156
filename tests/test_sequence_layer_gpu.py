"""The sequence operators as they are used together: a pre-norm residual layer (layer norm, projection, convolution, scan, projection)
with its backward pass and AdamW steps, against the same layer in 64 bits with torch's autograd; then the same layer fed token by token."""
import pytest
import torch

pytestmark = pytest.mark.gpu

B, T, C, D, N, K = 3, 32, 40, 48, 16, 4        # (the projections reduce over B T rows in whole pieces of 16)
U = 2.0 ** -24


def _weights(seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).cuda()                                                                 # noqa: E731
    return {"gamma": 1 + 0.1 * r(C), "beta": 0.1 * r(C), "w_in": r(C, 2 * D) / C ** 0.5, "conv_w": r(D, K) / 2, "conv_b": 0.1 * r(D),
            "w_bc": r(D, 2 * N) / D ** 0.5, "w_dt": r(D, D) / D ** 0.5, "dt_bias": 0.3 * r(D) - 2, "A": -torch.exp(0.5 * r(D, N)),
            "D": 1 + 0.1 * r(D), "w_out": r(D, C) / D ** 0.5}


def _forward(w, x, lengths, states=None, step=False):
    """(y, what the backward pass needs); x [rows..., C].  One token per sequence with ``step``."""
    from avsi_amd import ops
    lead = x.shape[:-1]
    h, mean, rstd = ops.layer_norm(x, w["gamma"], w["beta"])
    xz = ops.gemm(h.reshape(-1, C), w["w_in"]).view(*lead, 2 * D)
    xc, z = xz[..., :D], xz[..., D:]
    if step:
        u = ops.causal_conv_step(xc, w["conv_w"], w["conv_b"], state=states[0])
    else:
        u, conv_state = ops.causal_conv(xc, w["conv_w"], w["conv_b"], lengths=lengths, want_state=True)
    bc = ops.gemm(u.reshape(-1, D), w["w_bc"]).view(*lead, 2 * N)
    dt = ops.gemm(u.reshape(-1, D), w["w_dt"]).view(*lead, D)
    args = (u, dt, w["A"], bc[..., :N], bc[..., N:], w["D"], z, w["dt_bias"])
    if step:
        s = ops.selective_scan_step(*args, state=states[1])
        return x + ops.gemm(s, w["w_out"]).view_as(x)
    s, state, kept = ops.selective_scan(*args, lengths=lengths, want_state=True, keep=True)
    y = x + ops.gemm(s.reshape(-1, D), w["w_out"]).view_as(x)
    return y, (h, mean, rstd, xc, u, args, s, kept), (conv_state, state)


def _backward(w, x, lengths, saved, dy):
    from avsi_amd import ops
    h, mean, rstd, xc, u, args, s, kept = saved
    rows = B * T
    flat = lambda t: t.reshape(rows, -1)                                                                               # noqa: E731
    grad = lambda a, b: ops.gemm(flat(a).contiguous(), flat(b).contiguous(), trans_a=True)                             # noqa: E731
    g = {"w_out": grad(s, dy)}
    ds = ops.gemm(flat(dy), w["w_out"], trans_b=True).view(B, T, D)
    du, ddt, g["A"], dB, dC, g["D"], dz, g["dt_bias"] = ops.selective_scan_bwd(ds, *args, kept=kept, lengths=lengths)
    dbc = torch.cat([dB, dC], -1)
    g["w_bc"], g["w_dt"] = grad(u, dbc), grad(u, ddt)
    du = du + ops.gemm(flat(dbc), w["w_bc"], trans_b=True).view_as(du) + ops.gemm(flat(ddt), w["w_dt"], trans_b=True).view_as(du)
    dxc, g["conv_w"], g["conv_b"] = ops.causal_conv_bwd(du, xc, w["conv_w"], w["conv_b"], lengths=lengths)
    dxz = torch.cat([dxc, dz], -1)
    g["w_in"] = grad(h, dxz)
    dh = ops.gemm(flat(dxz), w["w_in"], trans_b=True).view_as(x)
    dx, g["gamma"], g["beta"] = ops.layer_norm_bwd(dh, x, mean, rstd, w["gamma"])
    return dy + dx, g


def _reference(w, x, lengths):
    on = torch.arange(T, device="cuda")[None] < lengths[:, None]
    h = torch.nn.functional.layer_norm(x, (C,), w["gamma"], w["beta"])
    xz = h @ w["w_in"]
    pre = torch.nn.functional.conv1d(torch.nn.functional.pad(xz[..., :D], (0, 0, K - 1, 0)).transpose(1, 2), w["conv_w"][:, None], w["conv_b"],
                                     groups=D).transpose(1, 2)
    u = torch.where(on[..., None], torch.nn.functional.silu(pre), 0.0)
    bc, delta = u @ w["w_bc"], torch.nn.functional.softplus(u @ w["w_dt"] + w["dt_bias"])
    st, outs = torch.zeros(B, D, N, dtype=x.dtype, device="cuda"), []
    for t in range(T):
        new = torch.exp(delta[:, t, :, None] * w["A"]) * st + (delta[:, t] * u[:, t])[..., None] * bc[:, t, None, :N]
        st = torch.where(on[:, t, None, None], new, st)
        outs.append(torch.where(on[:, t, None], (st * bc[:, t, None, N:]).sum(-1) + w["D"] * u[:, t], 0.0))
    s = torch.stack(outs, 1) * torch.nn.functional.silu(xz[..., D:])
    return x + s @ w["w_out"]


def _close(name, got, want, depth):
    """Within `depth` roundings of the largest value of the tensor: the layer is a chain of sums of at most 96 terms, each of which
    moves its result by a few U of the terms' sizes, and the sizes are of the order of the largest value."""
    assert bool((got.double() - want).abs().max() <= depth * U * want.abs().max()), (name, float((got.double() - want).abs().max() / want.abs().max() / U))


def test_a_layer_forward_backward_and_steps():
    from avsi_amd import ops
    g = torch.Generator().manual_seed(1)
    x, dy = torch.randn(B, T, C, generator=g).cuda(), torch.randn(B, T, C, generator=g).cuda()
    lengths = torch.tensor([T, 17, 0], dtype=torch.int32, device="cuda")
    w = _weights()
    names = sorted(w)
    grads = {k: torch.empty_like(w[k]) for k in names}
    plan = ops.AdamwPlan([w[k] for k in names], [grads[k] for k in names], weight_decay=[0.01 if w[k].dim() > 1 else 0.0 for k in names])
    for step in (1, 2, 3):
        w64 = {k: v.double().requires_grad_() for k, v in w.items()}
        x64 = x.double().requires_grad_()
        want = _reference(w64, x64, lengths)
        wg = dict(zip(names + ["x"], torch.autograd.grad(want, [w64[k] for k in names] + [x64], dy.double())))
        y, saved, _ = _forward(w, x, lengths)
        dx, got = _backward(w, x, lengths, saved, dy)
        _close("y", y, want, 400)
        _close("x", dx, wg["x"], 2000)
        for k in names:
            _close(k, got[k].view_as(wg[k]), wg[k], 4000)
            grads[k].copy_(got[k].view_as(grads[k]))
        before = {k: v.double() for k, v in w.items()}
        ops.adamw(plan, step, 1e-2, beta1=0.0, beta2=0.0)
        for k in names:      # without memory a step is the gradient's sign (but for eps), and the decay
            gk = grads[k].double()
            moved = before[k] - 1e-2 * (gk / (gk.abs() + 1e-8) + (0.01 if w[k].dim() > 1 else 0.0) * before[k])
            assert bool(((w[k].double() - moved).abs() <= 32 * U * (1e-2 + before[k].abs())).all()), k


def test_a_layer_token_by_token():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(B, T, C, generator=g).cuda()
    lengths = torch.full((B,), T, dtype=torch.int32, device="cuda")
    w = _weights(7)
    want = _reference({k: v.double() for k, v in w.items()}, x.double(), lengths)
    head = torch.full((B,), T - 10, dtype=torch.int32, device="cuda")
    y, _, states = _forward(w, x, head)           # the prompt, its padding behind it
    _close("prompt", y[:, :T - 10], want[:, :T - 10], 400)
    for t in range(T - 10, T):
        _close("token %d" % t, _forward(w, x[:, t].contiguous(), None, states, step=True), want[:, t], 400)
