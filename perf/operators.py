"""The cases on which the sequence and training operators are measured: layer norm, the short causal convolution with the
selective state-space scan, and the AdamW step over many tensors.

``listed()`` names the cases, ``draw()`` gives others of the same ranges, ``prepare()`` makes a case's inputs on the GPU from a
seed, ``run()`` is one pass -- in elementary torch operations, or through the entry points of ``avsi_amd.ops`` where ``own`` is
true -- and ``exact()`` is the same pass from the definitions in 64 bits.

A pass of the scan's cases goes through the convolution and through the scan, each on inputs of its own: u, which a layer takes
from the convolution, is an input here (and so is its gradient), so that what is compared of one operator holds no rounding of
the other's output."""
import math

import torch

own = False

BLOCK = 256           # values of an AdamW state that share one scale; tensors start at multiples of it in the flat buffers
E4M3_MAX = 448.0
F32_MAX = torch.finfo(torch.float32).max


# ---------------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one new frame of 32 streams, as wide as a BLSTM layer's output: the latency of one small call
        {"name": "norm frame f32", "op": "norm", "rows": 32, "cols": 512, "pad": 0, "dtype": "float32", "wdtype": "float32"},
        # the spectrogram frames of a batch of 32 three-second utterances: 257 bins (odd), rows of a wider buffer
        {"name": "norm bins f32", "op": "norm", "rows": 8000, "cols": 257, "pad": 31, "dtype": "float32", "wdtype": "float32"},
        # training: 16384 tokens of a wide layer, forward and backward
        {"name": "norm bf16", "op": "norm", "rows": 16384, "cols": 2048, "pad": 0, "dtype": "bfloat16", "wdtype": "bfloat16"},
        {"name": "norm back bf16", "op": "norm_back", "rows": 16384, "cols": 2048, "pad": 0, "dtype": "bfloat16", "wdtype": "bfloat16"},
        # the backward pass behind the frames of 32 utterances, 512 units
        {"name": "norm back f32", "op": "norm_back", "rows": 8000, "cols": 512, "pad": 0, "dtype": "float32", "wdtype": "float32"},
        # one long recording fed through in one piece, odd length, its states kept for the tokens behind it
        {"name": "scan prompt long bf16", "op": "prompt", "batch": 1, "time": 8191, "dim": 1536, "state": 16, "groups": 1, "taps": 4,
         "dtype": "bfloat16", "ragged": False, "carry": False},
        # the next piece of 32 utterances of different lengths, behind the states of the piece before
        {"name": "scan prompt ragged f32", "op": "prompt", "batch": 32, "time": 250, "dim": 512, "state": 16, "groups": 2, "taps": 4,
         "dtype": "float32", "ragged": True, "carry": True},
        # one token of one stream, and one token of 256 streams at once
        {"name": "scan token 1", "op": "token", "batch": 1, "dim": 2048, "state": 16, "groups": 1, "taps": 4, "dtype": "bfloat16"},
        {"name": "scan token 256", "op": "token", "batch": 256, "dim": 2048, "state": 16, "groups": 1, "taps": 4, "dtype": "bfloat16"},
        # a training step's forward and backward pass
        {"name": "scan train bf16", "op": "train", "batch": 8, "time": 2048, "dim": 2048, "state": 16, "groups": 1, "taps": 4,
         "dtype": "bfloat16", "ragged": False, "carry": False},
        # the optimiser step of the three-layer BLSTM-250 with its projection, states in 32 bits
        {"name": "adamw blstm 32", "op": "adamw", "bits": 32, "layers": 0, "width": 250, "gdtype": "float32", "copies": ""},
        # and of a deep stack: gradients and a copy of the weights in bf16, states in 8 bits
        {"name": "adamw deep 8", "op": "adamw", "bits": 8, "layers": 12, "width": 2048, "gdtype": "bfloat16", "copies": "bfloat16"},
    ]


def _log_int(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm_back", "prompt", "token", "train", "adamw"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if op.startswith("norm"):
        cols = _log_int(rng, 4, 9000)       # (a row of two has a gradient that cancels to nothing)
        rows = _log_int(rng, 1, min(40000, 33_000_000 // cols))
        return {"op": op, "rows": rows, "cols": cols, "pad": rng.choice([0, 0, 1, 8, 31]), "dtype": dtype,
                "wdtype": rng.choice(["float32", dtype])}
    if op == "adamw":
        return {"op": op, "bits": rng.choice([8, 32]), "layers": _log_int(rng, 1, 12), "width": _log_int(rng, 5, 2048),
                "gdtype": dtype, "copies": rng.choice(["", "bfloat16", "float16"])}
    groups = rng.choice([1, 1, 1, 2, 4])
    state = rng.choice([4, 8, 16, 16, 16, 24, 64])
    dim = groups * _log_int(rng, 3, 2048 // groups)
    case = {"op": op, "batch": _log_int(rng, 1, 256 if op == "token" else 64), "dim": dim, "state": state, "groups": groups,
            "taps": rng.choice([2, 3, 4, 4]), "dtype": dtype}
    if op != "token":
        most = 200_000_000 // (case["batch"] * dim * state)
        case |= {"time": _log_int(rng, 1, max(1, min(16384, most))), "ragged": rng.random() < 0.5, "carry": rng.random() < 0.5}
    return case


# --------------------------------------------------------------------------------------------------------------- the inputs
def _sizes(case):
    """(elements, weight decay) of each tensor: matrices decay, vectors do not."""
    w = case["width"]
    if case["layers"] == 0:       # three bidirectional LSTM layers behind 257 bins, and the projection back to them
        sizes = [s for d in (257, 2 * w, 2 * w) for s in 2 * [((d + w) * 4 * w, 0.01), (4 * w, 0.0)]]
        return sizes + [(2 * w * 257, 0.01), (257, 0.0)]
    return case["layers"] * [(2 * w * w, 0.01), (w * w + w, 0.01), (w, 0.0), (w, 0.0), (2 * w + 1, 0.0), (1, 0.0)]


def _offsets(sizes):
    at, out = 0, []
    for n, _ in sizes:
        out.append(at)
        at += (n + BLOCK - 1) // BLOCK * BLOCK
    return out, at


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) + 17)
    randn = lambda *shape: torch.randn(*shape, device="cuda", generator=g)                                          # noqa: E731
    rand = lambda *shape: torch.rand(*shape, device="cuda", generator=g)                                            # noqa: E731
    op = case["op"]
    if op.startswith("norm"):
        dtype, M, C = getattr(torch, case["dtype"]), case["rows"], case["cols"]
        s = {"op": op, "eps": 1e-5}
        # activations with a mean of their own in each row and a few large columns
        s["x"] = (randn(M, C + case["pad"]) * (1 + 4 * (rand(C + case["pad"]) < 0.01)) + 0.5 * randn(M, 1)).to(dtype)[:, :C]
        s["gamma"] = (1 + 0.2 * randn(C)).to(getattr(torch, case["wdtype"]))
        s["beta"] = (0.2 * randn(C)).to(getattr(torch, case["wdtype"]))
        if op == "norm_back":
            s["dy"] = (randn(M, C + case["pad"])).to(dtype)[:, :C]
            x = s["x"].float()
            s["mean"] = x.mean(1)
            s["rstd"] = (x.var(1, unbiased=False) + s["eps"]).rsqrt()
        return s
    if op == "adamw":
        sizes = _sizes(case)
        offsets, total = _offsets(sizes)
        used = torch.zeros(total, device="cuda")
        decay = torch.zeros(total // BLOCK, 1, device="cuda")
        for (n, wd), o in zip(sizes, offsets):
            used[o:o + n] = 1
            decay[o // BLOCK:-(-(o + n) // BLOCK)] = wd
        gd = getattr(torch, case["gdtype"])
        # gradients whose size differs from region to region by orders of magnitude
        size = torch.exp(2 * randn(total // BLOCK, 1)).expand(-1, BLOCK).reshape(-1) * 1e-3
        s = {"op": op, "bits": case["bits"], "step": 37, "lr": 3e-4, "beta1": 0.9, "beta2": 0.999, "eps": 1e-8, "grad_scale": 0.125,
             "decay": decay, "w": 0.02 * randn(total) * used, "g": (randn(total) * size * used * 8).to(gd)}
        m, v = 0.1 * randn(total) * size * used, ((0.5 + rand(total)) * size * 0.2) ** 2 * used
        if case["bits"] == 8:
            s["m"], s["m_scale"] = _to8(m)
            s["v"], s["v_scale"] = _to8(v.sqrt())
        else:
            s["m"], s["v"] = m, v
        s["copy"] = s["w"].to(getattr(torch, case["copies"])) if case["copies"] else None
        if own:
            from avsi_amd import ops
            part = lambda t: [t[o:o + n] for (n, _), o in zip(sizes, offsets)]                                       # noqa: E731
            s["plan"] = ops.AdamwPlan(part(s["w"]), part(s["g"]), weight_decay=[wd for _, wd in sizes], bits=case["bits"],
                                      copies=part(s["copy"]) if case["copies"] else None,
                                      state={k: s[k] for k in ("m", "v", "m_scale", "v_scale") if k in s})
        return s
    dtype, B, D, N, G, K = getattr(torch, case["dtype"]), case["batch"], case["dim"], case["state"], case["groups"], case["taps"]
    T = case.get("time", 1)
    s = {"op": op, "w": randn(D, K) / math.sqrt(K), "bias": 0.1 * randn(D), "D": 1 + 0.1 * randn(D),
         "A": -(1 + torch.arange(N, device="cuda")).float() * (0.8 + 0.4 * rand(D, N))}
    # step sizes spread over 0.001 .. 0.1, as such layers start with; the bias is what softplus turns into them
    delta = torch.exp(math.log(1e-3) + math.log(100.0) * rand(D))
    s["dt_bias"] = delta + torch.log(-torch.expm1(-delta))
    lead = (B,) if op == "token" else (B, T)
    s["x"], s["z"] = randn(*lead, D).to(dtype), randn(*lead, D).to(dtype)
    s["u"] = _silu(randn(*lead, D)).to(dtype)
    s["dt"] = (0.5 * randn(*lead, D)).to(dtype)
    s["B"], s["C"] = randn(*lead, G, N).to(dtype), randn(*lead, G, N).to(dtype)
    s["conv_state"] = s["state"] = s["lengths"] = None
    if op == "token" or case["carry"]:
        s["conv_state"], s["state"] = randn(B, K - 1, D).to(dtype), 0.3 * randn(B, D, N)
    if case.get("ragged"):
        s["lengths"] = torch.randint(0, T + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
        s["lengths"][0] = T
    if op == "train":
        s["dout"], s["du"] = randn(*lead, D).to(dtype), randn(*lead, D).to(dtype)
    return s


# ----------------------------------------------------------------------------------------------------- one pass, either way
def run(s):
    op = s["op"]
    if own:
        from avsi_amd import ops
        if op == "norm":
            return ops.layer_norm(s["x"], s["gamma"], s["beta"], eps=s["eps"])
        if op == "norm_back":
            return ops.layer_norm_bwd(s["dy"], s["x"], s["mean"], s["rstd"], s["gamma"])
        if op == "adamw":
            ops.adamw(s["plan"], s["step"], s["lr"], beta1=s["beta1"], beta2=s["beta2"], eps=s["eps"], grad_scale=s["grad_scale"])
            return _adamw_outputs(s)
        if op == "token":
            y = ops.causal_conv_step(s["x"], s["w"], s["bias"], state=s["conv_state"])
            out = ops.selective_scan_step(s["u"], s["dt"], s["A"], s["B"], s["C"], s["D"], s["z"], s["dt_bias"], state=s["state"])
            return {"y": y, "out": out, "conv_state": s["conv_state"], "state": s["state"]}
        if op == "prompt":
            y, conv_state = ops.causal_conv(s["x"], s["w"], s["bias"], state=s["conv_state"], lengths=s["lengths"], want_state=True)
            out, state, _ = ops.selective_scan(s["u"], s["dt"], s["A"], s["B"], s["C"], s["D"], s["z"], s["dt_bias"],
                                               state=s["state"], lengths=s["lengths"], want_state=True)
            return {"y": y, "out": out, "conv_state": conv_state, "state": state}
        y, _ = ops.causal_conv(s["x"], s["w"], s["bias"], state=s["conv_state"], lengths=s["lengths"])
        out, _, kept = ops.selective_scan(s["u"], s["dt"], s["A"], s["B"], s["C"], s["D"], s["z"], s["dt_bias"], state=s["state"],
                                          lengths=s["lengths"], keep=True)
        du, ddt, dA, dB, dC, dD, dz, ddt_bias = ops.selective_scan_bwd(s["dout"], s["u"], s["dt"], s["A"], s["B"], s["C"], s["D"],
                                                                       s["z"], s["dt_bias"], kept=kept, state=s["state"],
                                                                       lengths=s["lengths"])
        dx, dw, dbias = ops.causal_conv_bwd(s["du"], s["x"], s["w"], s["bias"], state=s["conv_state"], lengths=s["lengths"])
        return {"y": y, "out": out, "dx": dx, "dw": dw, "dbias": dbias, "du": du, "ddt": ddt, "dA": dA, "dB": dB, "dC": dC, "dD": dD,
                "dz": dz, "ddt_bias": ddt_bias}
    return {"norm": _norm, "norm_back": _norm_back, "adamw": _adamw, "token": _token, "prompt": _prompt, "train": _train}[op](s)


# ------------------------------------------------------------------------------------------------------- the plain forms
def _norm(s):
    x = s["x"].float()
    mean = x.mean(1)
    d = x - mean[:, None]
    rstd = 1 / torch.sqrt((d * d).mean(1) + s["eps"])
    return (d * rstd[:, None] * s["gamma"].float() + s["beta"].float()).to(s["x"].dtype), mean, rstd


def _norm_back(s):
    h = (s["x"].float() - s["mean"][:, None]) * s["rstd"][:, None]
    dy = s["dy"].float()
    e = dy * s["gamma"].float()
    dx = (e - e.mean(1, keepdim=True) - h * (e * h).mean(1, keepdim=True)) * s["rstd"][:, None]
    return dx.to(s["x"].dtype), (dy * h).sum(0), dy.sum(0)


def _to8(x):
    """(codes, scales): blocks of 256 values as 8-bit floats of the block's largest / 448; a positive value of a state that is
    held as its square root keeps at least the smallest code, so that no update is divided by a zero that is none."""
    x = x.reshape(-1, BLOCK)
    top = x.abs().amax(1, keepdim=True)
    y = x * torch.where(top > 0, E4M3_MAX / top, torch.zeros_like(top)).clamp(max=F32_MAX)
    return y.to(torch.float8_e4m3fn).reshape(-1), (top * (1 / E4M3_MAX)).reshape(-1)


def _root8(x):
    code, scale = _to8(x)
    least = torch.full((), 2.0 ** -9, device=x.device)
    return torch.where(x > 0, torch.maximum(code.float(), least), code.float()).to(torch.float8_e4m3fn), scale


def _adamw_outputs(s):
    return {k: s[k] for k in ("w", "m", "v", "m_scale", "v_scale", "copy") if s.get(k) is not None}


def _adamw(s):
    b1, b2 = s["beta1"], s["beta2"]
    g = s["g"].float() * s["grad_scale"]
    if s["bits"] == 8:
        m = (s["m"].float().reshape(-1, BLOCK) * s["m_scale"][:, None]).reshape(-1)
        v = (s["v"].float().reshape(-1, BLOCK) * s["v_scale"][:, None]).reshape(-1).square()
    else:
        m, v = s["m"], s["v"]
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    step = (m / (1 - b1 ** s["step"])) / (torch.sqrt(v / (1 - b2 ** s["step"])) + s["eps"])
    w = s["w"].reshape(-1, BLOCK)
    s["w"].copy_((w - s["lr"] * (step.reshape(-1, BLOCK) + s["decay"] * w)).reshape(-1))
    if s["bits"] == 8:
        for key, x, code in (("m", m, _to8), ("v", torch.sqrt(v), _root8)):
            c, scale = code(x)
            s[key].copy_(c)
            s[key + "_scale"].copy_(scale)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    if s["copy"] is not None:
        s["copy"].copy_(s["w"])
    return _adamw_outputs(s)


def _silu(x):
    return x / (1 + torch.exp(-x))


def _silu_slope(x):
    p = 1 / (1 + torch.exp(-x))
    return p * (1 + x * (1 - p))


def _delta(s):
    x = s["dt"].float() + s["dt_bias"]
    return torch.where(x > 20, x, torch.log1p(torch.exp(x.clamp(max=20)))), 1 / (1 + torch.exp(-x))


def _valid(s):
    """[batch, time, 1]: whether a position is inside its sequence."""
    B, T = s["x"].shape[:2]
    if s["lengths"] is None:
        return torch.ones(B, T, 1, dtype=torch.bool, device="cuda")
    return (torch.arange(T, device="cuda")[None] < s["lengths"][:, None])[..., None]


def _taps(s):
    """The convolution's inputs behind its state, and as [taps, batch, time, dim]."""
    x = s["x"].float()
    K = s["w"].shape[1]
    head = x.new_zeros(x.shape[0], K - 1, x.shape[2]) if s["conv_state"] is None else s["conv_state"].float()
    whole = torch.cat([head, x], 1)
    return whole, torch.stack([whole[:, k:k + x.shape[1]] for k in range(K)])


def _conv(s):
    """(u in the inputs' type, what silu was taken of, the taps, the last taps - 1 inputs of each sequence)."""
    whole, taps = _taps(s)
    pre = (taps * s["w"].t()[:, None, None]).sum(0) + s["bias"]
    K, (B, T) = s["w"].shape[1], s["x"].shape[:2]
    ends = torch.full((B,), T, device="cuda") if s["lengths"] is None else s["lengths"].long()
    at = ends[:, None] + torch.arange(K - 1, device="cuda")
    last = torch.gather(whole, 1, at[..., None].expand(-1, -1, whole.shape[2]))
    return torch.where(_valid(s), _silu(pre), 0.0).to(s["x"].dtype), pre, taps, last.to(s["x"].dtype)


def _recur(a, b):
    """h[t] = a[t] h[t - 1] + b[t] along axis 1, by doubling."""
    span = 1
    while span < a.shape[1]:
        b = torch.cat([b[:, :span], b[:, span:] + a[:, span:] * b[:, :-span]], 1)
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], 1)
        span *= 2
    return b


def _wide(x, D):
    """[..., groups, state] for each of the D channels of the groups."""
    return x.float().repeat_interleave(D // x.shape[-2], dim=-2)


def _scan(s):
    u, D = s["u"], s["u"].shape[-1]
    valid = _valid(s)
    delta, slope = _delta(s)
    delta = torch.where(valid, delta, 0.0)
    uf = torch.where(valid, u.float(), 0.0)
    Bw, Cw = _wide(s["B"], D), _wide(s["C"], D)
    a = torch.exp(delta[..., None] * s["A"])
    b = (delta * uf)[..., None] * Bw
    if s["state"] is not None:
        b[:, 0] += a[:, 0] * s["state"]
    h = _recur(a, b)
    y = (h * Cw).sum(-1) + s["D"] * uf
    z = s["z"].float()
    return torch.where(valid, y * _silu(z), 0.0).to(u.dtype), h, (a, delta, slope, uf, Bw, Cw, y, z, valid)


def _prompt(s):
    y, _, _, conv_state = _conv(s)
    out, h, _ = _scan(s)
    return {"y": y, "out": out, "conv_state": conv_state, "state": h[:, -1].contiguous()}


def _token(s):
    x, K = s["x"].float(), s["w"].shape[1]
    taps = torch.cat([s["conv_state"].float(), x[:, None]], 1)
    y = _silu((taps * s["w"].t()).sum(1) + s["bias"]).to(s["x"].dtype)
    s["conv_state"].copy_(taps[:, 1:])
    delta, _ = _delta(s)
    uf, D = s["u"].float(), s["u"].shape[-1]
    h = torch.exp(delta[..., None] * s["A"]) * s["state"] + (delta * uf)[..., None] * _wide(s["B"], D)
    s["state"].copy_(h)
    out = ((h * _wide(s["C"], D)).sum(-1) + s["D"] * uf) * _silu(s["z"].float())
    return {"y": y, "out": out.to(y.dtype), "conv_state": s["conv_state"], "state": s["state"]}


def _train(s):
    dtype, G = s["x"].dtype, s["B"].shape[2]
    conv, pre, taps, _ = _conv(s)
    out, h, (a, delta, slope, uf, Bw, Cw, y, z, valid) = _scan(s)
    dout = torch.where(valid, s["dout"].float(), 0.0)
    dy = dout * _silu(z)
    dz = dout * y * _silu_slope(z)
    after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    dh = _recur(after.flip(1), (dy[..., None] * Cw).flip(1)).flip(1)
    first = torch.zeros_like(h[:, 0]) if s["state"] is None else s["state"]
    carried = dh * a * torch.cat([first[:, None], h[:, :-1]], 1)
    B, T, D, N = h.shape
    dB = (dh * (delta * uf)[..., None]).reshape(B, T, G, D // G, N).sum(3)
    dC = (dy[..., None] * h).reshape(B, T, G, D // G, N).sum(3)
    hB = (dh * Bw).sum(-1)
    ddt = torch.where(valid, ((carried * s["A"]).sum(-1) + uf * hB) * slope, 0.0)
    du = torch.where(valid, s["D"] * dy + delta * hB, 0.0)
    dpre = torch.where(valid, s["du"].float() * _silu_slope(pre), 0.0)
    K = taps.shape[0]
    ahead = torch.cat([dpre, dpre.new_zeros(B, K - 1, D)], 1)
    dx = torch.stack([ahead[:, k:k + T] for k in range(K)])        # dpre[t + k] reads x[t] through tap K - 1 - k
    dx = (dx * s["w"].t().flip(0)[:, None, None]).sum(0)
    live = torch.where(valid, taps, 0.0)
    return {"y": conv, "out": out, "du": du.to(dtype), "dx": dx.to(dtype), "dw": (live * dpre).sum((1, 2)).t().contiguous(), "dbias": dpre.sum((0, 1)),
            "ddt": ddt.to(dtype), "dA": (carried * delta[..., None]).sum((0, 1)), "dB": dB.to(dtype), "dC": dC.to(dtype),
            "dD": (dy * uf).sum((0, 1)), "dz": torch.where(valid, dz, 0.0).to(dtype), "ddt_bias": ddt.sum((0, 1))}


# --------------------------------------------------------------------------------------------------- what a pass has to do
def work(case):
    size = {"float32": 4, "bfloat16": 2, "float16": 2, "": 0}
    op = case["op"]
    if op == "norm":
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * n * size[case["dtype"]] + 8 * case["rows"] + 2 * case["cols"] * size[case["wdtype"]], "flops": 8 * n}
    if op == "norm_back":
        n = case["rows"] * case["cols"]
        return {"bytes": 3 * n * size[case["dtype"]] + 8 * case["rows"] + case["cols"] * (size[case["wdtype"]] + 8), "flops": 15 * n}
    if op == "adamw":
        n = sum(k for k, _ in _sizes(case))
        states = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
        return {"bytes": n * (8 + states + size[case["gdtype"]] + size[case["copies"]]), "flops": 16 * n}
    e, B, D, N, G, K = size[case["dtype"]], case["batch"], case["dim"], case["state"], case["groups"], case["taps"]
    weights = 4 * D * (N + K + 3)
    states = B * D * (4 * N + e * (K - 1))
    if op == "token":
        return {"bytes": B * (D * e * 4 + 2 * G * N * e) + 2 * states + weights, "flops": B * D * (7 * N + 2 * K + 20)}
    tokens = B * case["time"]
    carry = states if case["carry"] else 0
    if op == "prompt":      # x, dt, z in, the gated output out; and the convolution's output
        return {"bytes": tokens * (6 * D + 2 * G * N) * e + carry + states + weights, "flops": tokens * D * (7 * N + 2 * K + 20)}
    # forward as above; backward: dout, u, dt, z, B, C, x in, du out and in, ddt, dz, dB, dC, dx out, and the weights' gradients
    return {"bytes": tokens * (6 * D + 2 * G * N) * e + tokens * (10 * D + 4 * G * N) * e + 2 * carry + 3 * weights,
            "flops": tokens * D * (25 * N + 8 * K + 60)}


# ------------------------------------------------------------------------------------------- the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    d = lambda k: None if s.get(k) is None else s[k].double()                                                          # noqa: E731
    op = case["op"]
    if op == "norm" or op == "norm_back":
        x, gamma, beta = d("x").requires_grad_(), d("gamma").requires_grad_(), d("beta").requires_grad_()
        var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
        y = (x - mean) / torch.sqrt(var + s["eps"]) * gamma + beta
        if op == "norm":
            return y.detach(), mean[:, 0].detach(), (1 / torch.sqrt(var + s["eps"]))[:, 0].detach()
        return torch.autograd.grad(y, (x, gamma, beta), d("dy"))
    if op == "adamw":
        each = lambda k: d(k + "_scale").repeat_interleave(BLOCK)                                                      # noqa: E731
        m, v, w, g = d("m"), d("v"), d("w"), d("g") * s["grad_scale"]
        if s["bits"] == 8:
            m, v = m * each("m"), (v * each("v")) ** 2
        m, v = torch.lerp(g, m, s["beta1"]), torch.lerp(g ** 2, v, s["beta2"])
        w = w * (1 - s["lr"] * s["decay"].double().expand(-1, BLOCK).reshape(-1)) - s["lr"] * (m / (1 - s["beta1"] ** s["step"])) / (
            (v / (1 - s["beta2"] ** s["step"])).sqrt() + s["eps"])
        out = {"w": w, "copy": w if case["copies"] else None}
        if s["bits"] == 8:    # a code is a choice among 256: it has no value in 64 bits
            return out | {"m": None, "v": None, "m_scale": m.abs().view(-1, BLOCK).amax(1) / E4M3_MAX,
                          "v_scale": v.sqrt().view(-1, BLOCK).amax(1) / E4M3_MAX}
        return out | {"m": m, "v": v}
    train, token = op == "train", op == "token"
    lead = ("x", "u", "dt", "z", "B", "C")
    t64 = {k: (d(k)[:, None] if token else d(k)) if k in lead else d(k) for k in lead + ("w", "bias", "D", "A", "dt_bias")}
    if train:
        t64 = {k: v.requires_grad_() for k, v in t64.items()}
    B, T, D = t64["x"].shape
    N, K = t64["A"].shape[1], t64["w"].shape[1]
    ends = torch.full((B,), T, device="cuda") if s["lengths"] is None else s["lengths"].long()
    window = list((torch.zeros(B, K - 1, D, device="cuda", dtype=torch.float64) if s["conv_state"] is None else d("conv_state")).unbind(1))
    h = torch.zeros(B, D, N, device="cuda", dtype=torch.float64) if s["state"] is None else d("state")
    group = torch.arange(D, device="cuda") // (D // t64["B"].shape[2])
    last = torch.stack(window, 1)
    xs, us, dts, zs, Bs, Cs = (t64[k].unbind(1) for k in lead)
    taps = t64["w"].unbind(1)
    ys, outs, zero = [], [], torch.zeros((), device="cuda", dtype=torch.float64)
    for t in range(T):
        inside = (t < ends)[:, None]
        window.append(xs[t])
        pre = t64["bias"] + sum(w * x for w, x in zip(taps, window))
        window = window[1:]
        ys.append(torch.where(inside, pre * torch.sigmoid(pre), zero))
        step = torch.nn.functional.softplus(dts[t] + t64["dt_bias"], threshold=40)
        new = torch.exp(step[..., None] * t64["A"]) * h + (step * us[t])[..., None] * Bs[t][:, group]
        h = torch.where(inside[..., None], new, h)
        y = (h * Cs[t][:, group]).sum(-1) + t64["D"] * us[t]
        outs.append(torch.where(inside, y * zs[t] * torch.sigmoid(zs[t]), zero))
        if not train:
            last = torch.where(inside[..., None], torch.stack(window, 1), last)
    y, out = torch.stack(ys, 1), torch.stack(outs, 1)
    if not train:
        return {"y": y[:, 0] if token else y, "out": out[:, 0] if token else out, "conv_state": last, "state": h}
    names = ("u", "dt", "A", "B", "C", "D", "z", "dt_bias")
    grads = dict(zip(names, torch.autograd.grad(out, [t64[k] for k in names], d("dout"))))
    grads |= dict(zip(("x", "w", "bias"), torch.autograd.grad(y, [t64[k] for k in ("x", "w", "bias")], d("du"))))
    return {"y": y.detach(), "out": out.detach()} | {"d" + k: v for k, v in grads.items()}
