"""Operators of token sequences over the C ABI: layer norm, the short causal convolution and the selective state-space scan,
each with its backward pass and, for serving, its form for single tokens.  Part of the public surface of ``ops``.

float32, bfloat16 and float16 tensors; all sums, states and statistics are float32.  Every call runs on the current stream of the
device its tensors live on (which need not be the current device) and allocates its outputs and workspaces from torch's caching
allocator, so it may be captured into a graph.  No arithmetic happens here."""
import torch

from . import _lib

_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _bad(what, *args):
    raise _lib.AvsiError(what % args)


def _device(what, first, *others):
    """The device of the operands; all of them have to be on it."""
    if not first.is_cuda:
        _lib.require_cuda(first)
    dev = first.device
    for t in others:
        if t is not None and t.device != dev:
            _bad("%s: operands on %s and %s", what, dev, t.device)
    return dev


def _p(t):
    return None if t is None else t.data_ptr()


def _overlap(a, b):
    """Whether two tensors share memory (by the span of their elements)."""
    def span(t):
        if not t.numel():
            return 0, 0
        lo = t.data_ptr()
        return lo, lo + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


# ------------------------------------------------------------------------------------------------------------- layer norm
def _rows(what, name, t, cols=None):
    """(rows, columns, row stride) of a tensor that is normalised over its last dimension."""
    if t.dtype not in _CODES or t.dim() < 1:
        _bad("%s: %s must be a float32, bfloat16 or float16 tensor", what, name)
    C = t.shape[-1]
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
    float32 or x's type, either may be None.  y: where to write (x's shape and type; not x itself), allocated if None.  mean, rstd:
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
        if y.shape != x.shape or y.dtype != x.dtype or _overlap(x, y):
            _bad("layer_norm: y must have x's shape and type and memory of its own")
    dev = _device("layer_norm", x, gamma, beta, y)
    if y is None:
        y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    stats = torch.empty((2, M), dtype=torch.float32, device=dev)
    if M:
        w = gamma if gamma is not None else beta
        p = stats.data_ptr()
        _lib.launch_on(dev, "avsi_layer_norm", x.data_ptr(), xs, _CODES[x.dtype], _p(gamma), _p(beta), 0 if w is None else _CODES[w.dtype],
                       y.data_ptr(), ys, p, p + 4 * M, M, C, eps)
    return y, stats[0], stats[1]


def layer_norm_bwd(dy, x, mean, rstd, gamma=None, want_wgrad=True, dx=None):
    """(dx, dgamma, dbeta) of ``layer_norm`` (avsi_layer_norm_bwd): dy and x of one shape and type, mean and rstd as the forward pass
    returned them.  dgamma, dbeta: float32 (sums over all rows), None with ``want_wgrad=False``.  dx: where to write, allocated if
    None."""
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
        if dx.shape != x.shape or dx.dtype != x.dtype or _overlap(dx, x) or _overlap(dx, dy):
            _bad("layer_norm_bwd: dx must have x's shape and type and memory of its own")
    dev = _device("layer_norm_bwd", dy, x, mean, rstd, gamma, dx)
    if dx is None:
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev)
    code = _CODES[x.dtype]
    grads, ws, nbytes = None, None, 0
    if want_wgrad:
        grads = torch.empty((2, C), dtype=torch.float32, device=dev)
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
    return (dx, grads[0], grads[1]) if want_wgrad else (dx, None, None)
