"""Operators of token sequences over the C ABI: layer norm, the short causal convolution and the selective state-space scan,
each with its backward pass and, for serving, its form for single tokens.  Part of the public surface of ``ops``.

float32, bfloat16 and float16 tensors; all sums, states and statistics are float32.  Every call runs on the current stream of the
device its tensors live on (which need not be the current device) and allocates its outputs and workspaces from torch's caching
allocator, so it may be captured into a graph.  No arithmetic happens here."""
import torch

from . import _lib

_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}

# Largest sizes, those that the C entry points state.  They are checked here, before anything is allocated: the entry points take sizes
# in 32 bits, and ctypes cuts a larger number without a word.
_MOST = {"columns": 1 << 30, "steps": 1 << 30, "scan channels": 1 << 26, "channels": (1 << 31) - 1024, "sequences": (1 << 31) - 1}


def _bad(what, *args):
    raise _lib.AvsiError(what % args)


def _fits(what, size, n):
    if n > _MOST[size]:
        _bad("%s: at most %d %s, not %d", what, _MOST[size], size.split()[-1], n)


def _device(what, first, *others):
    """The device of the operands; all of them have to be on it."""
    if not first.is_cuda:
        _lib.require_cuda(first)
    index = first.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            _bad("%s: operands on %s and %s", what, first.device, t.device)
    return first.device


def _p(t):
    return None if t is None else t.data_ptr()


def _overlap(a, b):
    """Whether two tensors share memory (by the span of their elements)."""
    lo, hi = a.data_ptr(), b.data_ptr()
    if lo > hi:
        a, b, lo, hi = b, a, hi, lo
    return bool(a.numel() and b.numel()) and hi < lo + (1 + sum((n - 1) * s for n, s in zip(a.shape, a.stride()))) * a.element_size()


# ------------------------------------------------------------------------------------------------------------- layer norm
def _rows(what, name, t, cols=None):
    """(rows, columns, row stride) of a tensor that is normalised over its last dimension."""
    if t.dtype not in _CODES or t.dim() < 1:
        _bad("%s: %s must be a float32, bfloat16 or float16 tensor", what, name)
    C = t.shape[-1]
    _fits(what, "columns", C)
    if cols is not None and C != cols:
        _bad("%s: %s has %d columns, not %d", what, name, C, cols)
    if t.dim() == 2:
        M, stride = t.shape[0], t.stride(0)
    elif t.is_contiguous():
        M, stride = (t.numel() // C if C else 0), C
    else:
        try:
            t = t.view(-1, C)
        except RuntimeError:
            _bad("%s: the rows of %s do not lie at one stride", what, name)
        M, stride = t.shape[0], t.stride(0)
    if M <= 1:
        stride = C
    if C < 1 or (C > 1 and t.stride(-1) != 1) or stride < C:
        _bad("%s: %s must have unit stride along its last dimension and rows that do not overlap", what, name)
    return M, C, stride


def _norm_weight(what, name, w, cols, dtype):
    if w is not None and (tuple(w.shape) != (cols,) or not w.is_contiguous() or (w.dtype != torch.float32 and w.dtype != dtype)):
        _bad("%s: %s must be a contiguous vector of %d float32 values, or of the input's type", what, name, cols)


def layer_norm(x, gamma=None, beta=None, eps=1e-5, y=None):
    """(y, mean, rstd): y = (x - mean) * rstd * gamma + beta over the last dimension of x (avsi_layer_norm).

    x: any leading shape whose rows lie at one stride (a slice of a wider buffer is fine), unit stride along a row.  gamma, beta:
    float32 or x's type, either may be None.  y: where to write (x's shape and type, in memory of its own), allocated if None.  mean, rstd:
    float32, one per row, flat -- what ``layer_norm_bwd`` takes.  A row that holds a NaN or an infinity comes out NaN."""
    M, C, xs = _rows("layer_norm", "x", x)
    _norm_weight("layer_norm", "gamma", gamma, C, x.dtype)
    _norm_weight("layer_norm", "beta", beta, C, x.dtype)
    if gamma is not None and beta is not None and gamma.dtype != beta.dtype:
        _bad("layer_norm: gamma and beta have to be of one type")
    if not eps >= 0:
        _bad("layer_norm: eps must not be negative")
    ys = C
    if y is not None:
        ys = _rows("layer_norm", "y", y, C)[2]
        if y.shape != x.shape or y.dtype != x.dtype or any(t is not None and _overlap(t, y) for t in (x, gamma, beta)):
            _bad("layer_norm: y must have x's shape and type and memory of its own")
    dev = _device("layer_norm", x, gamma, beta, y)
    if y is None:
        y = x.new_empty(x.shape)
    stats = x.new_empty((2, M), dtype=torch.float32)
    if M:
        w = gamma if gamma is not None else beta
        p = stats.data_ptr()
        _lib.launch_on(dev, "avsi_layer_norm", x.data_ptr(), xs, _CODES[x.dtype], _p(gamma), _p(beta), 0 if w is None else _CODES[w.dtype],
                       y.data_ptr(), ys, p, p + 4 * M, M, C, eps)
    return (y, *stats.unbind(0))


def layer_norm_bwd(dy, x, mean, rstd, gamma=None, want_wgrad=True, dx=None):
    """(dx, dgamma, dbeta) of ``layer_norm`` (avsi_layer_norm_bwd): dy and x of one shape and type, mean and rstd as the forward pass
    returned them.  dgamma, dbeta: float32 (sums over all rows), None with ``want_wgrad=False``.  dx: where to write (memory of its own), allocated
    if None."""
    M, C, xs = _rows("layer_norm_bwd", "x", x)
    dys = _rows("layer_norm_bwd", "dy", dy, C)[2]
    if dy.shape != x.shape or dy.dtype != x.dtype:
        _bad("layer_norm_bwd: dy and x differ in shape or type")
    for name, t in (("mean", mean), ("rstd", rstd)):
        if t.dtype != torch.float32 or t.numel() != M or not t.is_contiguous():
            _bad("layer_norm_bwd: %s must hold %d contiguous float32 values", name, M)
    _norm_weight("layer_norm_bwd", "gamma", gamma, C, x.dtype)
    dxs = C
    if dx is not None:
        dxs = _rows("layer_norm_bwd", "dx", dx, C)[2]
        if dx.shape != x.shape or dx.dtype != x.dtype or any(t is not None and _overlap(t, dx) for t in (x, dy, mean, rstd, gamma)):
            _bad("layer_norm_bwd: dx must have x's shape and type and memory of its own")
    dev = _device("layer_norm_bwd", dy, x, mean, rstd, gamma, dx)
    if dx is None:
        dx = x.new_empty(x.shape)
    code = _CODES[x.dtype]
    grads, ws, nbytes = None, None, 0
    if want_wgrad:
        grads = x.new_empty((2, C), dtype=torch.float32)
        if not M:
            grads.zero_()
    if M:
        if want_wgrad:
            nbytes = _lib.lib().avsi_layer_norm_bwd_workspace_bytes(M, C, code)
            ws = torch.empty(nbytes // 4, dtype=torch.float32, device=dev)
        p = _p(grads)
        _lib.launch_on(dev, "avsi_layer_norm_bwd", dy.data_ptr(), dys, x.data_ptr(), xs, code, mean.data_ptr(), rstd.data_ptr(), _p(gamma),
                       0 if gamma is None else _CODES[gamma.dtype], dx.data_ptr(), dxs, p, None if p is None else p + 4 * C, M, C, _p(ws),
                       nbytes)
    return (dx, *grads.unbind(0)) if want_wgrad else (dx, None, None)


# -------------------------------------------------------------------------------------------------------- causal convolution
def _seq(what, name, t, shape, dtype):
    """(batch stride, time stride) of a [batch, time, dim] tensor; its channels lie next to each other."""
    if t.dtype != dtype or tuple(t.shape) != shape:
        _bad("%s: %s must be %s of shape %s, not %s of %s", what, name, dtype, shape, t.dtype, tuple(t.shape))
    if shape[2] > 1 and t.stride(2) != 1:
        _bad("%s: %s must have unit stride along its channels", what, name)
    return t.stride(0), t.stride(1)


def _vector(what, name, t, *shape):
    """A contiguous float32 weight."""
    if t is not None and (t.dtype is not torch.float32 or t.shape != shape or not t.is_contiguous()):
        _bad("%s: %s must be contiguous float32 of shape %s", what, name, shape)


def _state(what, t, shape, dtype):
    if t is not None and (t.dtype is not dtype or t.shape != shape or not t.is_contiguous()):
        _bad("%s: state must be contiguous %s of shape %s", what, dtype, shape)


def _lengths(what, t, batch):
    if t is not None and (t.dtype != torch.int32 or tuple(t.shape) != (batch,) or not t.is_contiguous()):
        _bad("%s: lengths must be %d contiguous int32 values", what, batch)


def _conv_args(what, x, w, bias, dims):
    if x.dtype not in _CODES or x.dim() != dims:
        _bad("%s: x must be a float32, bfloat16 or float16 tensor of %d dimensions", what, dims)
    B, D = x.shape[0], x.shape[-1]
    if B > _MOST["sequences"] or D > _MOST["channels"] or dims == 3 and x.shape[1] > _MOST["steps"]:
        _fits(what, "sequences", B)
        _fits(what, "channels", D)
        _fits(what, "steps", x.shape[1])
    if w.dim() != 2 or not 2 <= w.shape[1] <= 8 or D < 1:
        _bad("%s: w must be [channels, taps] with 2 to 8 taps", what)
    _vector(what, "w", w, D, w.shape[1])
    _vector(what, "bias", bias, D)
    return B, D, w.shape[1]


def causal_conv(x, w, bias=None, silu=True, state=None, lengths=None, want_state=False):
    """(y, new_state): the short causal convolution along time, one filter per channel (avsi_causal_conv).

    x [batch, time, channels], w [channels, taps] and bias [channels] float32; y = silu(pre) or pre.  state [batch, taps - 1, channels]
    of x's type: the inputs in front of x (None: zeros).  lengths: int32, steps of each sequence (values outside 0 .. time are
    clamped); behind them y is zero and x is not read.  new_state (None unless asked for): the state behind each sequence's end, for
    the next piece or ``causal_conv_step``."""
    B, D, K = _conv_args("causal_conv", x, w, bias, 3)
    T = x.shape[1]
    xb, xt = _seq("causal_conv", "x", x, (B, T, D), x.dtype)
    _state("causal_conv", state, (B, K - 1, D), x.dtype)
    _lengths("causal_conv", lengths, B)
    dev = _device("causal_conv", x, w, bias, state, lengths)
    y = torch.empty((B, T, D), dtype=x.dtype, device=dev)
    new = torch.empty((B, K - 1, D), dtype=x.dtype, device=dev) if want_state else None
    if B and T:
        _lib.launch_on(dev, "avsi_causal_conv", x.data_ptr(), xb, xt, _CODES[x.dtype], w.data_ptr(), _p(bias), int(silu), _p(state),
                       _p(lengths), y.data_ptr(), T * D, D, _p(new), B, T, D, K)
    elif want_state and B:
        new.zero_() if state is None else new.copy_(state)
    return y, new


def causal_conv_bwd(dy, x, w, bias=None, silu=True, state=None, lengths=None, want_wgrad=True):
    """(dx, dw, dbias) of ``causal_conv`` (avsi_causal_conv_bwd): dy of x's shape and type, the other arguments as in the forward
    call.  dw, dbias: float32, None with ``want_wgrad=False`` (dbias also without a bias).  No gradient goes into the state."""
    B, D, K = _conv_args("causal_conv_bwd", x, w, bias, 3)
    T = x.shape[1]
    xb, xt = _seq("causal_conv_bwd", "x", x, (B, T, D), x.dtype)
    gb, gt = _seq("causal_conv_bwd", "dy", dy, (B, T, D), x.dtype)
    _state("causal_conv_bwd", state, (B, K - 1, D), x.dtype)
    _lengths("causal_conv_bwd", lengths, B)
    dev = _device("causal_conv_bwd", x, dy, w, bias, state, lengths)
    dx = torch.empty((B, T, D), dtype=x.dtype, device=dev)
    dw = torch.empty((D, K), dtype=torch.float32, device=dev) if want_wgrad else None
    dbias = torch.empty(D, dtype=torch.float32, device=dev) if want_wgrad and bias is not None else None
    if B and T:
        code = _CODES[x.dtype]
        nbytes = _lib.lib().avsi_causal_conv_bwd_workspace_bytes(code, B, T, D, K) if want_wgrad else 0
        ws = torch.empty(nbytes // 4, dtype=torch.float32, device=dev) if nbytes else None
        _lib.launch_on(dev, "avsi_causal_conv_bwd", dy.data_ptr(), gb, gt, x.data_ptr(), xb, xt, code, w.data_ptr(), _p(bias), int(silu),
                       _p(state), _p(lengths), dx.data_ptr(), T * D, D, _p(dw), _p(dbias), B, T, D, K, _p(ws), nbytes)
    else:
        for t in (dw, dbias):
            if t is not None:
                t.zero_()
    return dx, dw, dbias


def causal_conv_step(x, w, bias=None, silu=True, *, state):
    """y [batch, channels] of one token per sequence (avsi_causal_conv_step): x [batch, channels]; ``state`` [batch, taps - 1, channels]
    of x's type moves on by one input, in place."""
    B, D, K = _conv_args("causal_conv_step", x, w, bias, 2)
    if D > 1 and x.stride(1) != 1:
        _bad("causal_conv_step: x must have unit stride along its channels")
    _state("causal_conv_step", state, (B, K - 1, D), x.dtype)
    lo, size, p = state.data_ptr(), x.element_size(), x.data_ptr()
    hi = lo + size * B * (K - 1) * D
    w_at, bias_at = w.data_ptr(), _p(bias)
    if lo and B and (p < hi and p + size * ((B - 1) * x.stride(0) + D) > lo or w_at < hi and w_at + 4 * D * K > lo
              or bias_at and bias_at < hi and bias_at + 4 * D > lo):
        _bad("causal_conv_step: x, w and bias must not be part of the state")
    dev = _device("causal_conv_step", x, w, bias, state)
    y = x.new_empty((B, D))
    if B:
        _lib.launch_on(dev, "avsi_causal_conv_step", p, x.stride(0), _CODES[x.dtype], w_at, bias_at, int(silu), lo, y.data_ptr(), D, B, D, K)
    return y


# ------------------------------------------------------------------------------------------------------------ selective scan
def _groups(what, name, t, lead, N, dtype):
    """(groups, strides of batch, time and group) of B or C: [..., groups, state], or [..., state] for one group."""
    n, shape, st = len(lead), t.shape, t.stride()
    if t.dtype is not dtype or len(shape) - n not in (1, 2) or shape[:n] != lead or shape[-1] != N:
        _bad("%s: %s must be %s of shape %s + [groups, %d]", what, name, dtype, tuple(lead), N)
    if N > 1 and st[-1] != 1:
        _bad("%s: %s must have unit stride along its states", what, name)
    one = len(shape) == n + 1
    return 1 if one else shape[n], (st[0], st[1] if n == 2 else 0, 0 if one else st[n])


def _scan_operands(what, u, dt, A, B, C, D, z, dt_bias, softplus):
    """The operands that all forms of the scan take, checked, as the leading fields of avsi_scan_args; u is [..., channels]."""
    dtype, shape, su = u.dtype, u.shape, u.stride()
    lead, dim, two = shape[:-1], shape[-1], len(shape) == 3
    if dtype not in _CODES or dim < 1:
        _bad("%s: u must be a float32, bfloat16 or float16 tensor with channels", what)
    _fits(what, "scan channels", dim)
    if two:
        _fits(what, "steps", lead[1])
    if A.dim() != 2 or not 1 <= A.shape[1] <= 64:
        _bad("%s: A must be [channels, states] with 1 to 64 states", what)
    N = A.shape[1]
    _vector(what, "A", A, dim, N)
    _vector(what, "D", D, dim)
    _vector(what, "dt_bias", dt_bias, dim)
    if lead[0] > 65535:
        _bad("%s: at most 65535 sequences", what)
    if dt.dtype is not dtype or dt.shape != shape:
        _bad("%s: dt must be %s of shape %s, not %s of %s", what, dtype, tuple(shape), dt.dtype, tuple(dt.shape))
    sd = dt.stride()
    if z is None:
        sz = (0, 0, 1)
    else:
        if z.dtype is not dtype or z.shape != shape:
            _bad("%s: z must be %s of shape %s, not %s of %s", what, dtype, tuple(shape), z.dtype, tuple(z.shape))
        sz = z.stride()
    if dim > 1 and not su[-1] == sd[-1] == sz[-1] == 1:
        _bad("%s: u, dt and z must have unit stride along their channels", what)
    G, sB = _groups(what, "B", B, lead, N, dtype)
    G2, sC = _groups(what, "C", C, lead, N, dtype)
    if G != G2 or G < 1 or dim % G:
        _bad("%s: B and C must have one number of groups, which divides the %d channels", what, dim)
    if two and G * -(-(dim // G) // 16) >= 1 << 23:
        _bad("%s: groups * ceil(channels / groups / 16) has to be below 2^23", what)
    t = (lambda s: s[1]) if two else (lambda s: 0)
    return N, (_CODES[dtype], lead[0], lead[1] if two else 1, dim, N, G, int(softplus), 0, u.data_ptr(), dt.data_ptr(), _p(z), B.data_ptr(),
               C.data_ptr(), su[0], t(su), sd[0], t(sd), sz[0], t(sz), *sB, *sC, A.data_ptr(), _p(D), _p(dt_bias))


def selective_scan(u, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=True, state=None, lengths=None, want_state=False, keep=False):
    """(out, new_state, kept): the selective state-space scan of whole sequences (avsi_selective_scan).

        delta = softplus(dt + dt_bias),  h[t] = exp(delta A) h[t - 1] + delta u B[t],  y = C[t] . h[t] + D u,  out = y silu(z)

    u, dt, z [batch, time, channels]; B, C [batch, time, groups, states] ([batch, time, states] for one group) of u's type; A
    [channels, states], D, dt_bias [channels] float32; D, z, dt_bias may be None.  ``softplus=False`` takes dt + dt_bias as it is.
    state: float32 [batch, channels, states] in front of the first step (None: zeros).  lengths: int32 steps per sequence (clamped to
    0 .. time); behind them out is zero, the state stands still and nothing is read.  new_state (None unless asked for): float32, the
    state behind each sequence's end.  kept (None unless ``keep``): what ``selective_scan_bwd`` needs, a quarter of a byte per channel,
    step and state.  States count as the next power of two from 4 on; with states in no whole quads, or fewer than four channels, as
    64, here and in the workspace of the backward pass (2 x 4 bytes per state, step and block of 64 channels, of 16 at 64 states)."""
    what = "selective_scan"
    if u.dim() != 3:
        _bad("%s: u must be [batch, time, channels]", what)
    bsz, T, dim = u.shape
    N, operands = _scan_operands(what, u, dt, A, B, C, D, z, dt_bias, softplus)
    _state(what, state, (bsz, dim, N), torch.float32)
    _lengths(what, lengths, bsz)
    dev = _device(what, u, dt, A, B, C, D, z, dt_bias, state, lengths)
    out = u.new_empty((bsz, T, dim))
    new = A.new_empty((bsz, dim, N)) if want_state else None
    kept = None
    if not (bsz and T):
        if want_state and bsz:
            new.zero_() if state is None else new.copy_(state)
        return out, new, torch.empty(0, dtype=torch.float32, device=dev) if keep else None
    L = _lib.lib()
    a = _lib.ScanArgs(*operands, _p(state), _p(lengths), out.data_ptr(), T * dim, dim, _p(new))
    if keep:
        kept = A.new_empty(L.avsi_selective_scan_kept_floats(a))
        a.kept = kept.data_ptr()
    nbytes = L.avsi_selective_scan_workspace_bytes(a)
    ws = A.new_empty(nbytes // 4) if nbytes else None
    _lib.launch_on(dev, "avsi_selective_scan", a, _p(ws), nbytes)
    return out, new, kept


def selective_scan_bwd(dout, u, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=True, *, kept, state=None, lengths=None):
    """(du, ddt, dA, dB, dC, dD, dz, ddt_bias) of ``selective_scan`` (avsi_selective_scan_bwd): dout of u's shape and type, ``kept``
    from the forward call with ``keep=True``, the other arguments as there.  du, ddt, dz, dB, dC have the inputs' type; dA, dD,
    ddt_bias are float32; what belongs to an argument that is None is None.  No gradient goes into the state."""
    what = "selective_scan_bwd"
    if u.dim() != 3:
        _bad("%s: u must be [batch, time, channels]", what)
    bsz, T, dim = u.shape
    N, operands = _scan_operands(what, u, dt, A, B, C, D, z, dt_bias, softplus)
    gb, gt = _seq(what, "dout", dout, (bsz, T, dim), u.dtype)
    _state(what, state, (bsz, dim, N), torch.float32)
    _lengths(what, lengths, bsz)
    L = _lib.lib()
    a = _lib.ScanArgs(*operands)
    if kept.dtype != torch.float32 or not kept.is_contiguous() or kept.numel() != L.avsi_selective_scan_kept_floats(a):
        _bad("%s: kept must be what selective_scan returned with keep=True for these operands", what)
    dev = _device(what, u, dt, A, B, C, D, z, dt_bias, dout, kept, state, lengths)
    du, ddt = torch.empty((2, bsz, T, dim), dtype=u.dtype, device=dev).unbind(0)
    dz = None if z is None else torch.empty((bsz, T, dim), dtype=u.dtype, device=dev)
    dB, dC = torch.empty(B.shape, dtype=u.dtype, device=dev), torch.empty(C.shape, dtype=u.dtype, device=dev)
    dA = torch.empty((dim, N), dtype=torch.float32, device=dev)
    dD = None if D is None else torch.empty(dim, dtype=torch.float32, device=dev)
    ddt_bias = None if dt_bias is None else torch.empty(dim, dtype=torch.float32, device=dev)
    if bsz and T:
        a.lengths, a.kept, a.dout, a.dout_b, a.dout_t = _p(lengths), kept.data_ptr(), dout.data_ptr(), gb, gt
        a.du, a.ddt, a.dz, a.dB, a.dC = du.data_ptr(), ddt.data_ptr(), _p(dz), dB.data_ptr(), dC.data_ptr()
        a.dA, a.dD, a.ddt_bias = dA.data_ptr(), _p(dD), _p(ddt_bias)
        nbytes = L.avsi_selective_scan_bwd_workspace_bytes(a)
        ws = torch.empty(nbytes // 4, dtype=torch.float32, device=dev)
        _lib.launch_on(dev, "avsi_selective_scan_bwd", a, ws.data_ptr(), nbytes)
    else:
        for t in (dA, dD, ddt_bias):
            if t is not None:
                t.zero_()
    return du, ddt, dA, dB, dC, dD, dz, ddt_bias


def selective_scan_step(u, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=True, *, state):
    """out [batch, channels] of one token per sequence (avsi_selective_scan_step): u, dt, z [batch, channels]; B, C [batch, groups,
    states] or [batch, states]; ``state`` float32 [batch, channels, states] moves on by one step, in place: no other operand may share
    memory with it."""
    what = "selective_scan_step"
    if u.dim() != 2:
        _bad("%s: u must be [batch, channels]", what)
    bsz, dim = u.shape
    N, operands = _scan_operands(what, u, dt, A, B, C, D, z, dt_bias, softplus)
    _state(what, state, (bsz, dim, N), torch.float32)
    lo = state.data_ptr()
    hi = lo + 4 * bsz * dim * N
    (G, _, _, u_at, dt_at, z_at, B_at, C_at, ub, _, tb, _, zb, _, Bb, _, Bg, Cb, _, Cg, A_at, D_at, bias_at) = operands[5:]
    last, size, vec = bsz - 1, u.element_size(), 4 * dim
    if lo and bsz and (u_at < hi and u_at + size * (last * ub + dim) > lo or dt_at < hi and dt_at + size * (last * tb + dim) > lo
                or z_at and z_at < hi and z_at + size * (last * zb + dim) > lo
                or B_at < hi and B_at + size * (last * Bb + (G - 1) * Bg + N) > lo
                or C_at < hi and C_at + size * (last * Cb + (G - 1) * Cg + N) > lo
                or A_at < hi and A_at + vec * N > lo or D_at and D_at < hi and D_at + vec > lo
                or bias_at and bias_at < hi and bias_at + vec > lo):
        _bad("%s: the inputs must not be part of the state", what)
    dev = _device(what, u, dt, A, B, C, D, z, dt_bias, state)
    out = u.new_empty((bsz, dim))
    if bsz:
        _lib.launch_on(dev, "avsi_selective_scan_step",
                       _lib.ScanArgs(*operands, None, None, out.data_ptr(), dim, 0, state.data_ptr()))
    return out
