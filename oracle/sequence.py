"""Short causal convolution and selective state-space scan in 64 bits, step by step, with first-order bounds on what 32-bit
arithmetic may add: every function returns (values, bounds), where a bound is the sum of the roundings a float32 evaluation makes on
its way (U = 2^-24 each), propagated through the recurrences.  Types of 16 bits add their own half step where a value is written.

The constants count operations: a gate (sigmoid, softplus) is at most 8 roundings (for 16-bit types a sigmoid of x may be |x| of them,
which stays far inside the half step of what it is rounded to), a decay exp(delta A) 6 plus what the error of
delta A (8 of delta, 2 of the product, and in a joined chunk the sum over its steps) does to the exponential."""
import torch

U = 2.0 ** -24


def _silu(x):
    return x * torch.sigmoid(x)


def _silu_slope(x):
    s = torch.sigmoid(x)
    return s * (1 + x * (1 - s))


def inside(batch, time, lengths, device):
    """[batch, time]: whether a step is inside its sequence."""
    t = torch.arange(time, device=device)[None]
    if lengths is None:
        return (t >= 0).expand(batch, time)
    return t < lengths.to(device).long()[:, None]


def conv_forward(x, w, bias=None, silu=True, state=None, lengths=None):
    """({y, state}, {y}) of float64 inputs."""
    B, T, D = x.shape
    K = w.shape[1]
    on = inside(B, T, lengths, x.device)[..., None]
    head = x.new_zeros(B, K - 1, D) if state is None else state
    whole = torch.cat([head, torch.where(on, x, torch.zeros((), dtype=x.dtype, device=x.device))], 1)
    pre, top = x.new_zeros(B, T, D), x.new_zeros(B, T, D)
    for k in range(K):
        pre = pre + w[:, k] * whole[:, k:k + T]
        top = top + (w[:, k] * whole[:, k:k + T]).abs()
    if bias is not None:
        pre, top = pre + bias, top + bias.abs()
    err = U * (K + 1) * top
    y, ey = (_silu(pre), 1.1 * err + 10 * U * _silu(pre).abs()) if silu else (pre, err)      # (|slope of silu| < 1.1)
    n = on[..., 0].sum(1)
    last = torch.gather(whole, 1, (n[:, None] + torch.arange(K - 1, device=x.device))[..., None].expand(-1, -1, D))
    zero = torch.zeros_like(y)
    return {"y": torch.where(on, y, zero), "state": last, "pre": pre, "whole": whole, "err_pre": err}, {"y": torch.where(on, ey, zero)}


def conv_backward(dy, x, w, bias=None, silu=True, state=None, lengths=None):
    """({dx, dw, dbias}, the bounds of the same)."""
    B, T, D = x.shape
    K = w.shape[1]
    f = conv_forward(x, w, bias, silu, state, lengths)[0]
    on = inside(B, T, lengths, x.device)[..., None]
    zero = torch.zeros_like(dy)
    dy = torch.where(on, dy, zero)
    d = dy * _silu_slope(f["pre"]) if silu else dy
    e = dy.abs() * (0.5 * f["err_pre"] + 12 * U * (1 + f["pre"].abs())) if silu else zero      # (|slope'| <= 1/2)
    pad = x.new_zeros(B, K - 1, D)
    da, ea = torch.cat([d, pad], 1), torch.cat([e, pad], 1)
    dx, ex, dw, ew = zero.clone(), zero.clone(), [], []
    for k in range(K):
        wk = w[:, K - 1 - k]
        dx += wk * da[:, k:k + T]
        ex += wk.abs() * (ea[:, k:k + T] + U * (K + 1) * da[:, k:k + T].abs())
        taps = f["whole"][:, k:k + T]
        dw.append((d * taps).sum((0, 1)))
        ew.append((e * taps.abs() + U * (B * T / 16 + 80) * (d * taps).abs()).sum((0, 1)))
    return ({"dx": dx, "dw": torch.stack(dw, 1), "dbias": d.sum((0, 1))},
            {"dx": ex, "dw": torch.stack(ew, 1), "dbias": (e + U * (B * T / 16 + 80) * d.abs()).sum((0, 1))})


def _spread(x, D):
    """[batch, time, groups, states] for each of the D channels."""
    return x.repeat_interleave(D // x.shape[2], dim=2)


def scan(u, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=True, state=None, lengths=None, dout=None):
    """({out, state, and with dout: du, ddt, dA, dB, dC, dD, dz, ddt_bias}, the bounds of the same) of float64 inputs; B and C are
    [batch, time, groups, states]."""
    bsz, T, dim = u.shape
    N, G = A.shape[1], B.shape[2]
    on = inside(bsz, T, lengths, u.device)[..., None]
    zero = torch.zeros((), dtype=u.dtype, device=u.device)
    u, dt, B, C = (torch.where(m, x, zero) for m, x in ((on, u), (on, dt), (on[..., None], B), (on[..., None], C)))
    x = dt + (0 if dt_bias is None else dt_bias)
    delta = torch.where(on, torch.nn.functional.softplus(x, threshold=60) if softplus else x, zero)
    slope = torch.where(on, torch.sigmoid(x) if softplus else torch.ones_like(x), zero)
    # relative error of delta: of softplus' argument (one rounding of |dt| + |bias|), its own 8, over delta
    ed = 9 * U * delta.abs() + U * (dt.abs() + (0 if dt_bias is None else dt_bias.abs())) * (slope if softplus else 1)
    ed = torch.where(on, ed, zero)
    z = None if z is None else torch.where(on, z, zero)
    a = torch.exp(delta[..., None] * A)
    # relative error of a decay, and of one that joins chunks: the sum of the step sizes of a chunk is off by its length
    ka = 6 * U + ed[..., None] * A.abs() + U * (4 + T) * (delta[..., None] * A).abs()
    Bw, Cw = _spread(B, dim), _spread(C, dim)
    b = (delta * u)[..., None] * Bw
    eb = (ed * u.abs())[..., None] * Bw.abs() + 4 * U * b.abs()
    h = u.new_zeros(bsz, dim, N) if state is None else state.clone()
    H, E = h.abs(), torch.zeros_like(h)
    hs, Hs, Es, prev, Hprev, Eprev = [], [], [], [], [], []
    for t in range(T):
        prev.append(h), Hprev.append(H), Eprev.append(E)
        E = a[:, t] * E + ka[:, t] * a[:, t] * H + eb[:, t] + 2 * U * (a[:, t] * H + b[:, t].abs())
        h, H = a[:, t] * h + b[:, t], a[:, t] * H + b[:, t].abs()
        hs.append(h), Hs.append(H), Es.append(E)
    hs, Hs, Es, prev, Hprev, Eprev = (torch.stack(v, 1) for v in (hs, Hs, Es, prev, Hprev, Eprev))
    skip = 0 * u if D is None else D * u
    y = (hs * Cw).sum(-1) + skip
    ey = ((Es + U * (N + 8) * Hs) * Cw.abs()).sum(-1) + 4 * U * skip.abs()
    gate = torch.ones_like(u) if z is None else _silu(z)
    out = torch.where(on, y * gate, zero)
    val, err = {"out": out, "state": h}, {"out": torch.where(on, ey * gate.abs() + 12 * U * out.abs(), zero), "state": E}
    if dout is None:
        return val, err
    dout = torch.where(on, dout, zero)
    dy = dout * gate
    if z is not None:
        val["dz"] = dout * y * _silu_slope(z)
        err["dz"] = dout.abs() * (_silu_slope(z).abs() * ey + 14 * U * y.abs() * (1 + z.abs()))
    g, F, Gm = (torch.zeros_like(h) for _ in range(3))        # the adjoint state, its bound, its terms' absolute sum
    gs, Fs, Gs = [], [], []
    for t in reversed(range(T)):
        c = Cw[:, t] * dy[:, t, :, None]
        F = F + 14 * U * c.abs() + 2 * U * Gm
        g, Gm = g + c, Gm + c.abs()
        gs.append(g), Fs.append(F), Gs.append(Gm)
        F = a[:, t] * F + (ka[:, t] + 2 * U) * a[:, t] * Gm
        g, Gm = a[:, t] * g, a[:, t] * Gm
    gs, Fs, Gs = (torch.stack(v[::-1], 1) for v in (gs, Fs, Gs))
    per = dim // G
    fold = lambda v: v.reshape(bsz, T, G, per, N).sum(3)                                                               # noqa: E731
    deep = 32 + per / 16                                      # roundings of a sum over a group's channels
    w = (delta * u)[..., None]
    ew = (ed * u.abs())[..., None]
    val["dB"], err["dB"] = fold(gs * w), fold(Fs * w.abs() + Gs * ew + U * (deep + 4) * Gs * w.abs())
    val["dC"], err["dC"] = fold(hs * dy[..., None]), fold((Es + U * (deep + 14) * Hs) * dy[..., None].abs())
    gB, mB = (gs * Bw).sum(-1), (Gs * Bw.abs()).sum(-1)
    eB = (Fs * Bw.abs()).sum(-1) + U * (N + 4) * mB
    x, xm = gs * a * prev, Gs * a * Hprev
    ex = a * (Fs * Hprev + Gs * Eprev) + (ka + 6 * U) * xm
    gA = (x * A).sum(-1)
    eA = ((ex + U * (N + 4) * xm) * A.abs()).sum(-1)
    mA = (xm * A.abs()).sum(-1)
    through = 0 * u if D is None else D * dy
    val["du"] = torch.where(on, through + delta * gB, zero)
    err["du"] = torch.where(on, delta.abs() * eB + ed * mB + 16 * U * (through.abs() + delta.abs() * mB), zero)
    val["ddt"] = (gA + u * gB) * slope
    err["ddt"] = slope * (eA + u.abs() * eB + 16 * U * (mA + u.abs() * mB))
    long = 48 + T / 16 + bsz                                  # roundings of a sum over time and batch
    val["dA"], err["dA"] = (x * delta[..., None]).sum((0, 1)), (ex * delta.abs()[..., None] + xm * ed[..., None]
                                                                + U * long * xm * delta.abs()[..., None]).sum((0, 1))
    if D is not None:
        val["dD"], err["dD"] = (dy * u).sum((0, 1)), U * (long + 14) * (dy * u).abs().sum((0, 1))
    if dt_bias is not None:
        val["ddt_bias"] = val["ddt"].sum((0, 1))
        err["ddt_bias"] = (err["ddt"] + U * long * val["ddt"].abs()).sum((0, 1))
    return val, err
