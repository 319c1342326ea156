"""AdamW over many tensors at once, moments in 32 or in 8 bits (avsi_adamw).  Part of the public surface of ``ops``."""
import torch

from . import _lib
from .sequence_ops import _CODES, _bad, _p

BLOCK = 256            # values that share a scale of the 8-bit moments; tensors start at multiples of it in the flat buffers


def _spans_clash(written, read):
    """Whether two of the written tensors share memory, or a read one shares any with a written one (contiguous tensors)."""
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in written if t.numel())
    if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
        return True
    import bisect
    starts = [a for a, _ in spans]
    for t in read:
        if t.numel():
            lo, hi = t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()
            k = bisect.bisect_left(starts, hi)                  # spans that start in front of its end
            if k and spans[k - 1][1] > lo:
                return True
    return False


class AdamwPlan:
    """The tensors of one optimiser, checked once: ``adamw(plan, step, lr)`` then costs a launch per 48 tensors.

    params: contiguous float32 tensors, updated in place.  grads: one per parameter, of its shape, contiguous float32, bfloat16 or
    float16; the step reads them where they lie (``set_grads`` for others).  weight_decay: one rate, or one per parameter.  copies:
    None, or per parameter None or a bfloat16 / float16 tensor that receives the rounded weights.  bits: 32, or 8 (blocks of 256
    values share a scale; see ``avsi_adamw``).

    state: None (zeros), or a dict of 'm' and 'v' -- for 8 bits also 'm_scale' and 'v_scale' -- to go on from, used in place: each a
    flat tensor of ``numel`` values (``numel / 256`` scales), in which parameter i starts at ``offsets[i]``, or (32 bits) a list of one
    tensor per parameter.  ``plan.state`` is that dict: what a checkpoint holds.  8-bit moments are torch.float8_e4m3fn: m =
    code * m_scale, sqrt(v) = code * v_scale of the block.

    The plan holds on to all of these tensors.  No two of the written ones may share memory."""

    def __init__(self, params, grads, weight_decay=0.01, bits=32, copies=None, state=None):
        params, self.bits = list(params), bits
        if bits not in (8, 32):
            _bad("AdamwPlan: moments are held in 8 or in 32 bits")
        copies = [None] * len(params) if copies is None else list(copies)
        decay = [float(weight_decay)] * len(params) if isinstance(weight_decay, (int, float)) else [float(x) for x in weight_decay]
        if not params or len(copies) != len(params) or len(decay) != len(params):
            _bad("AdamwPlan: parameters, copies and rates of decay have to be as many, and at least one")
        self.offsets, self.numel = [], 0
        for p, c in zip(params, copies):
            if p.dtype != torch.float32 or not p.is_contiguous():
                _bad("AdamwPlan: parameters must be contiguous float32")
            if c is not None and (c.dtype not in (torch.bfloat16, torch.float16) or c.shape != p.shape or not c.is_contiguous()):
                _bad("AdamwPlan: a copy must be contiguous bfloat16 or float16 of its parameter's shape")
            self.offsets.append(self.numel)
            self.numel += (p.numel() + BLOCK - 1) // BLOCK * BLOCK
        self._params, self._copies = params, copies
        self._check_grads(grads)
        self.device = dev = params[0].device
        if not params[0].is_cuda:
            _lib.require_cuda(params[0])
        self.state = self._make_state(state, dev)
        tensors = params + [c for c in copies if c is not None]
        lists = {k: self._split(k, v) for k, v in self.state.items()}
        tensors += [t for v in lists.values() for t in v]
        if any(t.device != dev for t in tensors + self._grads):
            _bad("AdamwPlan: all tensors have to be on %s", dev)
        self._written = tensors
        if _spans_clash(tensors, self._grads):
            _bad("AdamwPlan: parameters, copies and moments must not share memory with each other or with gradients")
        self._table = (_lib.AdamwTensor * len(params))()
        for i, (row, p, c) in enumerate(zip(self._table, params, copies)):
            row.w, row.copy, row.numel, row.weight_decay = p.data_ptr(), _p(c), p.numel(), decay[i]
            row.copy_dtype = 0 if c is None else _CODES[c.dtype]
            for k, v in lists.items():
                setattr(row, k, v[i].data_ptr())
        self._watched = params + [c for c in copies if c is not None]
        self._at = [t.data_ptr() for t in self._watched]
        self._point_at_grads()

    def _make_state(self, state, dev):
        kinds = {"m": torch.float32, "v": torch.float32}
        if self.bits == 8:
            kinds = {"m": torch.float8_e4m3fn, "v": torch.float8_e4m3fn, "m_scale": torch.float32, "v_scale": torch.float32}
        size = {k: self.numel // BLOCK if k.endswith("scale") else self.numel for k in kinds}
        if state is None:
            return {k: torch.zeros(size[k], dtype=torch.uint8, device=dev).view(t) if t.itemsize == 1 else
                    torch.zeros(size[k], dtype=t, device=dev) for k, t in kinds.items()}
        if set(state) != set(kinds):
            _bad("AdamwPlan: the state of %d-bit moments is a dict of %s", self.bits, ", ".join(sorted(kinds)))
        for k, t in kinds.items():
            s = state[k]
            if isinstance(s, (list, tuple)) and self.bits == 32:
                ok = len(s) == len(self._params) and all(x.dtype == t and x.shape == p.shape and x.is_contiguous()
                                                         for x, p in zip(s, self._params))
            else:
                ok = isinstance(s, torch.Tensor) and s.dtype == t and s.dim() == 1 and s.numel() == size[k] and s.is_contiguous()
            if not ok:
                _bad("AdamwPlan: state[%r] must be a flat contiguous %s of %d values%s", k, t, size[k],
                     ", or a list of one tensor per parameter" if self.bits == 32 else "")
        return dict(state)

    def _split(self, k, s):
        if not isinstance(s, torch.Tensor):
            return list(s)
        if k.endswith("scale"):
            return [s[o // BLOCK:o // BLOCK + -(-p.numel() // BLOCK)] for o, p in zip(self.offsets, self._params)]
        return [s[o:o + p.numel()] for o, p in zip(self.offsets, self._params)]

    def _check_grads(self, grads):
        grads = list(grads)
        if len(grads) != len(self._params):
            _bad("AdamwPlan: %d gradients for %d parameters", len(grads), len(self._params))
        for g, p in zip(grads, self._params):
            if g.dtype not in _CODES or g.shape != p.shape or not g.is_contiguous():
                _bad("AdamwPlan: a gradient must be contiguous float32, bfloat16 or float16 of its parameter's shape")
        self._grads = grads

    def _point_at_grads(self):
        self._grads_at = [g.data_ptr() for g in self._grads]
        for row, g, at in zip(self._table, self._grads, self._grads_at):
            row.grad, row.grad_dtype = at, _CODES[g.dtype]

    def set_grads(self, grads):
        """Read other gradient tensors from now on: one per parameter, checked as at the start."""
        old = self._grads
        self._check_grads(grads)
        if any(g.device != self.device for g in self._grads) or _spans_clash(self._written, self._grads):
            self._grads = old
            _bad("AdamwPlan: gradients have to be on %s, in memory of their own", self.device)
        self._point_at_grads()


def adamw(plan, step, lr, beta1=0.9, beta2=0.999, eps=1e-8, grad_scale=1.0, skip=None):
    """Step ``step`` (1-based) of AdamW on all tensors of ``plan``, in place (avsi_adamw):

        g = grad * grad_scale,  m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g^2
        w -= lr * (m / (1 - beta1^step) / (sqrt(v / (1 - beta2^step)) + eps) + weight_decay * w)

    ``skip``: device float32 words (<= 8, the step guard); nothing is written when any of them is not exactly zero.  The numbers are
    arguments of the launch: a captured call repeats the same step at the same rate."""
    if skip is not None and (skip.dtype != torch.float32 or not skip.is_contiguous() or skip.numel() > 8 or skip.device != plan.device):
        _bad("adamw: skip must be at most 8 contiguous float32 words on %s", plan.device)
    if step < 1 or not (0 <= beta1 < 1 and 0 <= beta2 < 1 and eps >= 0):
        _bad("adamw: step counts from 1, beta1 and beta2 are in [0, 1), eps is not negative")
    if [t.data_ptr() for t in plan._watched] != plan._at or [g.data_ptr() for g in plan._grads] != plan._grads_at:
        _bad("adamw: a tensor of the plan has moved since the plan was made")
    _lib.launch_on(plan.device, "avsi_adamw", plan._table, len(plan._table), plan.bits, lr, beta1, beta2, eps, int(step), grad_scale,
                   _p(skip), 0 if skip is None else skip.numel())
