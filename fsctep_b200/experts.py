"""Routed experts: a mixture of linear channel maps in which every row takes a few of many experts.

The sparse sibling of the ``mix_bucket_*`` operators (whose gates are dense over all paths), with what
stands around it, on the sm_100a kernels of ``libfsctep_b200.so``:

* :func:`add_rms_norm` / :func:`add_rms_norm_q8` -- RMS norm of rows with the residual's addition,
  also with e4m3 output and row scales;
* :func:`route_experts` -- softmax or sigmoid scores, balance bias, groups, top-k, renormalised weights;
* :func:`expert_linear` / :func:`expert_linear_q8` -- the experts' products, summed with the weights;
* :class:`RoutedChannelMix` -- the three as one equivariant layer on the models' node features, to be
  given to a model as its ``sync_after_scatter``.

The first three differentiate through autograd (once; a second derivative and forward mode are refused), and
each has its gradient as a function of its own (``*_backward``) for callers that run or capture the reverse
pass themselves.  Inputs must be CUDA tensors (there is no CPU path); wrong shapes, types and devices
raise ``RuntimeError``.  Work is launched on the current stream, nothing waits on the host, outputs
and workspaces come from torch's allocator, so the calls can be captured into CUDA graphs; capture a
reverse pass through the ``*_backward`` functions, which return plain tensors without a graph
(autograd's own engine refuses to capture while an eager graph of the same leaves is alive).  Every wait in a kernel is bounded: one that runs out leaves
NaN in the outputs, and :meth:`ExpertPlan.check` says where.  A plan belongs to the stream that it was built on.  Equal
inputs give equal outputs, bit for bit.
"""

from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad

from fsctep_b200 import _native as N

__all__ = [
    "add_rms_norm", "add_rms_norm_q8", "add_rms_norm_backward", "route_experts", "route_experts_backward",
    "ExpertPlan", "expert_plan", "expert_linear", "expert_linear_q8", "expert_linear_backward", "quantize_experts",
    "RoutedChannelMix",
]

_DTYPES = {torch.float32: N.FSC_F32, torch.bfloat16: N.FSC_BF16, torch.float16: N.FSC_F16}
_SCORES = {"softmax": 0, "sigmoid": 1}
E4M3_MAX = 448.0


def _check(cond, msg):
    if not cond:
        raise RuntimeError(msg)


def _dtype(t, name):
    _check(t.is_cuda, f"{name} must be a CUDA tensor")
    _check(t.dtype in _DTYPES, f"{name} must be float32, bfloat16 or float16")
    return _DTYPES[t.dtype]


def _like(t, ref, name, dtype=None):
    _check(t.device == ref.device, f"{name} must be on {ref.device}")
    _check(t.dtype == (dtype or ref.dtype), f"{name} must be {dtype or ref.dtype}")


_FN = {}
_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _fn(name):
    f = _FN.get(name)
    if f is None:
        f = _FN[name] = getattr(N.lib(), name)
    return f


def _call(name, t, *args):
    """C entry point ``name`` on the current stream of the tensor's device, which is made the current one."""
    i = t.get_device()
    if i == _device():
        status = _fn(name)(*args, _stream(i))
    else:
        with torch.cuda.device(i):
            status = _fn(name)(*args, _stream(i))
    if status:
        N.check(status, name[4:])


def _ptr(t):
    return None if t is None else t.data_ptr()


def _refuse_tangents(*ts):
    """Forward mode (also without grad mode): a tangent would be lost, as the kernels see values alone."""
    if forward_ad._current_level >= 0:
        for t in ts:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("the routed-expert operators have no forward-mode derivative")


def _differentiable(*ts):
    _refuse_tangents(*ts)
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


class _Refuse(torch.autograd.Function):
    """A gradient that depends on ``deps`` in a way that has no derivative here."""

    @staticmethod
    def forward(ctx, grad, *deps):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("the routed-expert operators have no second derivative")


def _first_order(grads, *deps):
    """The gradients; under create_graph marked so that differentiating them again raises."""
    if not torch.is_grad_enabled():
        return grads
    deps = [d for d in deps if d is not None]
    return tuple(g if g is None else _Refuse.apply(g, *deps) for g in grads)


def _empty_like(t):
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _rows(t):
    """(rows, dim) with contiguous columns; a view wherever the strides allow it."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


# ---- RMS norm ------------------------------------------------------------------------------------

def _norm_inputs(x, weight, residual):
    dt, dev = x.dtype, x.get_device()  # the usual call in one condition; what is wrong with another is found below
    if (dev >= 0 and dt in _DTYPES and x.dim() >= 1 and weight.dim() == 1 and weight.shape[0] == x.shape[-1] >= 1
            and weight.get_device() == dev and (weight.dtype == dt or weight.dtype == torch.float32)
            and (residual is None or (residual.dtype == dt and residual.get_device() == dev and residual.shape == x.shape))):
        return
    _dtype(x, "x")
    _check(x.dim() >= 1 and x.shape[-1] >= 1, "x must have a last dimension of at least 1")
    _check(weight.shape == x.shape[-1:], "weight must have x's last dimension")
    _check(weight.dtype in (x.dtype, torch.float32), "weight must have x's dtype or float32")
    _check(weight.device == x.device, "weight must be on x's device")
    if residual is not None:
        _like(residual, x, "residual")
        _check(residual.shape == x.shape, "residual must have x's shape")


def _norm_launch(x, weight, residual, eps, q8):
    xr, w = _rows(x), weight.contiguous()
    n, d = xr.shape
    rr = h = scale = None
    if residual is not None:
        rr, h = _rows(residual), _empty_like(x)
    if q8:
        q, scale = x.new_empty(x.shape, dtype=torch.float8_e4m3fn), x.new_empty(x.shape[:-1], dtype=torch.float32)
        y, py, pq = q, None, q.data_ptr()
    else:
        y = _empty_like(x)
        py, pq = y.data_ptr(), None
    _call("fsc_rms_norm_forward", x, _DTYPES[x.dtype], _DTYPES[w.dtype], xr.data_ptr(), xr.stride(0), _ptr(rr),
          0 if rr is None else rr.stride(0), w.data_ptr(), eps, py, _ptr(h), pq, _ptr(scale), n, d)
    return y, scale, h


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, _, h = _norm_launch(x, weight, residual, eps, False)
        ctx.eps, ctx.with_residual = eps, residual is not None
        ctx.save_for_backward(x if h is None else h, weight)
        ctx.set_materialize_grads(False)
        return (y, h) if ctx.with_residual else y

    @staticmethod
    def backward(ctx, grad_y, grad_h=None):
        h, weight = ctx.saved_tensors
        gx, gw = grad_h, None
        if grad_y is not None:
            gx, gw = add_rms_norm_backward(grad_y, h, weight, grad_h, eps=ctx.eps,
                                           weight_gradient=ctx.needs_input_grad[1])
        gx, gw = _first_order((gx, gw), h, weight, grad_y, grad_h)
        return gx, gw, gx if ctx.with_residual else None, None


def add_rms_norm(x, weight, residual=None, *, eps=1e-6):
    """``y = s / sqrt(mean(s^2) + eps) * weight`` over the last dimension, ``s = x + residual``.

    Returns ``y``, or ``(y, h)`` with a residual, where ``h = s`` is the new residual stream.  ``s``
    is normalised before it is rounded to the type of ``h``; the gradient is taken at the rounded
    ``h``.  ``weight`` has ``x``'s dtype or float32.  The squares are summed in 32 bits: a row's sum of
    squares has to stay below 3.4e38 (beyond it ``y`` is 0)."""
    _norm_inputs(x, weight, residual)
    if _differentiable(x, weight, residual):
        return _RmsNorm.apply(x, weight, residual, float(eps))
    y, _, h = _norm_launch(x, weight, residual, float(eps), False)
    return y if residual is None else (y, h)


def add_rms_norm_q8(x, weight, residual=None, *, eps=1e-6):
    """:func:`add_rms_norm` with e4m3 output: returns ``(q, scale)`` or ``(q, scale, h)`` where ``q *
    scale[..., None]`` stands for ``y`` and ``scale = max|y| / 448`` of each row (0 for a row of
    zeros).  For serving: it is not differentiable and refuses inputs that require gradients."""
    _norm_inputs(x, weight, residual)
    _check(not _differentiable(x, weight, residual), "add_rms_norm_q8 is not differentiable")
    y, scale, h = _norm_launch(x, weight, residual, float(eps), True)
    return (y, scale) if residual is None else (y, scale, h)


def add_rms_norm_backward(grad_y, h, weight, grad_h=None, *, eps=1e-6, weight_gradient=True):
    """``(grad_x, grad_weight)`` at the stored ``h`` (``x`` itself without a residual).  ``grad_x``,
    to which ``grad_h`` (the gradient of ``h``, or None) is added, is the residual's gradient too.
    ``grad_weight`` is None unless asked for."""
    _refuse_tangents(grad_y, h, weight, grad_h)
    _norm_inputs(h, weight, grad_h)
    _like(grad_y, h, "grad_y")
    _check(grad_y.shape == h.shape, "grad_y must have h's shape")
    hr, gy, w = _rows(h), _rows(grad_y), weight.contiguous()
    gh = None if grad_h is None else _rows(grad_h)
    n, d = hr.shape
    gx = h.new_empty(h.shape)
    gw = torch.empty_like(w) if weight_gradient else None
    nbytes = _fn("fsc_rms_norm_backward_workspace_bytes")(n, d) if weight_gradient else 0
    ws = h.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _call("fsc_rms_norm_backward", h, _DTYPES[h.dtype], _DTYPES[w.dtype], gy.data_ptr(), gy.stride(0), _ptr(gh),
          0 if gh is None else gh.stride(0), hr.data_ptr(), hr.stride(0), w.data_ptr(), float(eps), gx.data_ptr(),
          _ptr(gw), n, d, _ptr(ws), nbytes)
    return gx, gw


# ---- router --------------------------------------------------------------------------------------

def _logits_2d(logits):
    return logits if logits.stride(1) == 1 or logits.shape[1] == 1 else logits.contiguous()


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, *args):
        weights, indices = _route_launch(logits, *args)
        ctx.save_for_backward(logits, indices)
        ctx.kw = dict(scores=args[5], renormalize=args[6], scale=args[7])
        ctx.mark_non_differentiable(indices)
        return weights, indices

    @staticmethod
    def backward(ctx, grad_weights, _):
        logits, indices = ctx.saved_tensors
        gl = route_experts_backward(grad_weights, logits, indices, **ctx.kw)
        return _first_order((gl,), logits, grad_weights) + (None,) * 8


def _route_launch(logits, top_k, bias, row_mask, num_groups, groups_kept, scores, renormalize, scale):
    lg = _logits_2d(logits)
    t, x = lg.shape
    weights = lg.new_empty((t, top_k), dtype=torch.float32)
    indices = lg.new_empty((t, top_k), dtype=torch.int32)
    bias = None if bias is None else bias.contiguous()
    mask = None if row_mask is None else row_mask.contiguous()
    _call("fsc_route_experts", lg, _DTYPES[lg.dtype], lg.data_ptr(), lg.stride(0), _ptr(bias), _ptr(mask),
          weights.data_ptr(), indices.data_ptr(), t, x, top_k, num_groups, groups_kept, _SCORES[scores], renormalize,
          scale)
    return weights, indices


def _route_inputs(logits, bias, row_mask, scores):
    _dtype(logits, "logits")
    _check(logits.dim() == 2, "logits must have shape (rows, experts)")
    _check(scores in _SCORES, "scores must be 'softmax' or 'sigmoid'")
    if bias is not None:
        _like(bias, logits, "bias", torch.float32)
        _check(bias.shape == logits.shape[1:], "bias must have shape (experts,)")
        _check(not _differentiable(bias), "bias has no gradient: detach it")
    if row_mask is not None:
        _like(row_mask, logits, "row_mask", torch.bool)
        _check(row_mask.shape == logits.shape[:1], "row_mask must have shape (rows,)")


def route_experts(logits, top_k, *, bias=None, row_mask=None, num_groups=1, groups_kept=None, scores="softmax",
                  renormalize=True, scale=1.0):
    """Chooses ``top_k`` experts for each row of ``logits`` (rows, experts).

    Returns ``weights`` (rows, top_k, float32) and ``indices`` (int32), best first, equal scores in
    the order of their index.  The scores are the row's softmax or the logits' sigmoids; ``bias``
    (float32, no gradient) is added for the choice alone; with groups, the ``groups_kept`` groups
    whose two best biased scores sum highest stay open.  ``weights`` are the chosen scores without
    the bias, divided by their sum (+ 1e-20) if ``renormalize``, times ``scale``.  Without a bias and
    with all groups open the choice goes by the logits, whose order is the scores' also where these
    are equal in floating point (sigmoids of 40 and 50); with them by the scores in 64 bits.

    A logit of -inf or NaN is never chosen (+inf counts as the largest float).  Where ``row_mask``
    (bool) is False, or fewer than ``top_k`` experts are available, the rest has index -1 and weight
    0; :func:`expert_linear` leaves such slots out."""
    if (bias is not None or row_mask is not None or logits.dim() != 2 or logits.dtype not in _DTYPES
            or logits.get_device() < 0 or scores not in _SCORES):
        _route_inputs(logits, bias, row_mask, scores)
    args = (int(top_k), bias, row_mask, int(num_groups), int(num_groups if groups_kept is None else groups_kept), scores,
            bool(renormalize), float(scale))
    _check(1 <= args[0] <= 32, "top_k must be 1 to 32")
    if _differentiable(logits):
        return _Route.apply(logits, *args)
    return _route_launch(logits, *args)


def route_experts_backward(grad_weights, logits, indices, *, scores="softmax", renormalize=True, scale=1.0):
    """Gradient of the weights that :func:`route_experts` returned with ``indices``, in the logits."""
    _refuse_tangents(grad_weights, logits)
    _dtype(logits, "logits")
    _check(logits.dim() == 2 and indices.dim() == 2 and indices.shape[0] == logits.shape[0],
           "logits (rows, experts) and indices (rows, top_k) must have the same rows")
    _like(indices, logits, "indices", torch.int32)
    _like(grad_weights, logits, "grad_weights", torch.float32)
    _check(grad_weights.shape == indices.shape, "grad_weights must have the shape of indices")
    _check(scores in _SCORES, "scores must be 'softmax' or 'sigmoid'")
    lg, idx, g = _logits_2d(logits), indices.contiguous(), grad_weights.contiguous()
    out = lg.new_empty(lg.shape)
    _call("fsc_route_experts_backward", lg, _DTYPES[lg.dtype], g.data_ptr(), lg.data_ptr(), lg.stride(0), idx.data_ptr(),
          out.data_ptr(), lg.shape[0], lg.shape[1], idx.shape[1], _SCORES[scores], bool(renormalize), float(scale))
    return out


# ---- the experts' products -----------------------------------------------------------------------

class ExpertPlan:
    """The slots of ``indices`` (rows, top_k) grouped by expert, for the products of one routing: build
    it once with :func:`expert_plan` and give it to every product (and gradient) of these indices.

    It belongs to the contents that ``indices`` had when it was built; changing them in place
    afterwards makes the products refuse it (inference tensors do not count their changes)."""

    def __init__(self, indices, num_experts):
        _check(indices.is_cuda and indices.dtype == torch.int32, "indices must be an int32 CUDA tensor")
        _check(indices.dim() == 2 and 1 <= indices.shape[1] <= 32, "indices must have shape (rows, top_k), top_k <= 32")
        _check(indices.numel() < 2 ** 31, "too many slots")
        self.num_experts = int(num_experts)
        _check(1 <= self.num_experts <= 1024, "num_experts must be 1 to 1024")
        self.source = indices
        self.indices = indices.contiguous()
        self.version = None if indices.is_inference() else indices._version
        (t, k), x = self.indices.shape, self.num_experts
        nbytes = _fn("fsc_expert_plan_workspace_bytes")(t, k, x)
        bins = _fn("fsc_expert_joint_bins")(t, k, x)
        # [offsets: experts + 1][status][order: slots][joint offsets: bins + 1][joint order: rows]
        self._data = indices.new_empty(x + 2 + t * k + (bins + 1 + t if bins else 0))
        ws = indices.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        base = self._data.data_ptr()
        self._offsets, self._status, self._order = base, base + 4 * (x + 1), base + 4 * (x + 2)
        self._joint_offsets = self._order + 4 * t * k if bins else None
        self._joint_order = self._joint_offsets + 4 * (bins + 1) if bins else None
        _call("fsc_expert_plan", indices, self.indices.data_ptr(), t, k, x, self._offsets, self._order,
              self._joint_offsets, self._joint_order, self._status, _ptr(ws), nbytes)

    @property
    def offsets(self):
        """(experts + 1): expert e's slots are ``order[offsets[e]:offsets[e + 1]]``."""
        return self._data[:self.num_experts + 1]

    @property
    def order(self):
        """Slot numbers (row * top_k + choice) by expert; the tail past ``offsets[-1]`` is undefined."""
        return self._data[self.num_experts + 2:self.num_experts + 2 + self.indices.numel()]

    def check(self):
        """Waits for the products launched with this plan and raises if a bounded wait in one ran out (what that
        product had still to write, and all that this plan's later products write, is NaN)."""
        code = int(self._data[self.num_experts + 1])
        if code:
            raise N.NativeError(f"expert_linear: a pipeline wait ran out (code {code})")

    def _fits(self, indices, num_experts):
        same = indices is self.source or indices is self.indices or (
            indices.data_ptr() == self.source.data_ptr() and indices.shape == self.source.shape
            and indices.stride() == self.source.stride() and indices.device == self.source.device)
        _check(same and num_experts == self.num_experts, "plan was built for other indices or another number of experts")
        _check(self.version is None or self.source._version == self.version,
               "indices were changed in place after the plan was built")


def expert_plan(indices, num_experts) -> ExpertPlan:
    """Groups the slots of ``indices`` (rows, top_k; int32) by expert.  Indices outside [0,
    num_experts) mark slots without an expert."""
    return ExpertPlan(indices, num_experts)


def _linear_dims(x, w, indices, weights, slots):
    dev, lead = x.get_device(), 2 if slots else 1  # the usual call in one condition, as in _norm_inputs
    if (w.dim() == 3 and indices.dim() == 2 and x.dim() == lead + 1 and w.dtype == x.dtype and w.get_device() == dev
            and indices.dtype == torch.int32 and indices.get_device() == dev and 0 not in w.shape
            and x.shape[:lead] == indices.shape[:lead] and x.shape[-1] == w.shape[2]
            and (weights is None or (weights.dtype == torch.float32 and weights.get_device() == dev
                                     and weights.shape == indices.shape))):
        return indices.shape[0], indices.shape[1], (), w.shape[0], w.shape[2], w.shape[1]
    _check(w.dim() == 3 and min(w.shape) >= 1, "w must have shape (experts, outputs, inputs)")
    _check(indices.dim() == 2, "indices must have shape (rows, top_k)")
    _like(indices, x, "indices", torch.int32)
    t, k = indices.shape
    lead = 2 if slots else 1
    _check(x.dim() in (lead + 1, lead + 2),
           "x must have shape (rows, top_k, [components,] inputs)" if slots else "x must have shape (rows, [components,] inputs)")
    _check(tuple(x.shape[:lead]) == ((t, k) if slots else (t,)), "x and indices must have the same rows")
    _check(x.shape[-1] == w.shape[2], "x's last dimension must be w's inputs")
    mid = tuple(x.shape[lead:-1])
    _check(not mid or 1 <= mid[0] <= 1024, "x must have 1 to 1024 components")
    if weights is not None:
        _like(weights, x, "weights", torch.float32)
        _check(weights.shape == indices.shape, "weights must have the shape of indices")
    return t, k, mid, w.shape[0], w.shape[2], w.shape[1]


def _dense(t):
    """Contiguous and starting on 16 bytes, as the products' copies need it."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _plan_for(plan, indices, num_experts):
    if plan is None:
        return ExpertPlan(indices, num_experts)
    plan._fits(indices, num_experts)
    return plan


def _few(t, k, mid, i, slots):
    """Whether the matrix-vector form takes these rows (the limits of fsc_expert_few_fits)."""
    c = mid[0] if mid else 1
    return 0 < t * k <= 32 and c <= 16 and (k if slots else 1) * c * i <= 12288


def _linear_launch(x, w, indices, weights, slots, plan):
    """The product and the plan it was given or made (None for a few rows, which need none)."""
    t, k, mid, e, i, o = _linear_dims(x, w, indices, weights, slots)
    if plan is not None:
        plan._fits(indices, e)
    x, w = _dense(x), _dense(w)
    wt = None if weights is None else weights.contiguous()
    out = x.new_empty((t,) + (() if weights is not None else (k,)) + mid + (o,))
    c = mid[0] if mid else 1
    dt = _DTYPES[x.dtype]
    if _few(t, k, mid, i, slots):
        idx = indices.contiguous()
        _call("fsc_expert_linear_few", x, dt, dt, x.data_ptr(), None, w.data_ptr(), None, idx.data_ptr(), _ptr(wt),
              out.data_ptr(), t, k, c, e, i, o, slots)
        return out, plan
    if plan is None:
        plan = ExpertPlan(indices, e)
    nbytes = _fn("fsc_expert_linear_workspace_bytes")(dt, t, k, c, e, i, o, slots, wt is not None,
                                                      plan._joint_offsets is not None)
    ws = x.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _call("fsc_expert_linear", x, dt, x.data_ptr(), w.data_ptr(), plan.indices.data_ptr(), _ptr(wt), plan._offsets,
          plan._order, plan._joint_offsets, plan._joint_order, plan._status, out.data_ptr(), t, k, c, e, i, o, slots,
          _ptr(ws), nbytes)
    return out, plan


class _ExpertLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, indices, weights, slots, plan):
        out, ctx.plan = _linear_launch(x, w, indices, weights, slots, plan)
        ctx.slots = slots
        ctx.save_for_backward(x, w, indices, weights)
        return out

    @staticmethod
    def backward(ctx, grad_out):
        x, w, indices, weights = ctx.saved_tensors
        need = ctx.needs_input_grad
        gx, gw, gwt = expert_linear_backward(grad_out, x, w, indices, weights, slots=ctx.slots, plan=ctx.plan,
                                             input_gradient=need[0], weight_gradient=need[1],
                                             routing_gradient=need[3])
        gx, gw, gwt = _first_order((gx, gw, gwt), x, w, weights, grad_out)
        return gx, gw, None, gwt, None, None


def expert_linear(x, w, indices, weights=None, *, slots=False, plan=None):
    """Products of rows with their experts' matrices ``w`` (experts, outputs, inputs).

    With ``weights`` (rows, top_k; float32): ``out[t] = sum_j weights[t, j] * x[t] @ w[indices[t, j]].T``
    of shape (rows, [components,] outputs).  Without: the products stay apart, (rows, top_k,
    [components,] outputs).  ``x`` is (rows, [components,] inputs) -- the components of a row, such
    as the 2l + 1 of an irrep, share its experts -- or, with ``slots=True``, holds a row for each slot:
    (rows, top_k, [components,] inputs).  An expert MLP is a product without weights, the
    activation, and a product with ``slots=True`` and the weights.

    Indices outside [0, experts) (:func:`route_experts` gives -1) are slots without an expert: they
    count as zero, whatever the rows of ``x`` that only they name hold.  float32 is multiplied to
    float32 accuracy on the tensor cores (sums of three bfloat16); finite inputs only -- an infinity
    in ``x`` or ``w`` may come out as NaN (in the weights' gradient of float16 too)."""
    _dtype(x, "x")
    _like(w, x, "w")
    if _differentiable(x, w, weights):
        return _ExpertLinear.apply(x, w, indices, weights, bool(slots), plan)
    return _linear_launch(x, w, indices, weights, bool(slots), plan)[0]


def expert_linear_backward(grad_out, x, w, indices, weights=None, *, slots=False, plan=None, input_gradient=True,
                           weight_gradient=True, routing_gradient=True):
    """``(grad_x, grad_w, grad_weights)`` of :func:`expert_linear`; None where not asked for (and
    ``grad_weights`` without ``weights``)."""
    _refuse_tangents(grad_out, x, w, weights)
    _dtype(x, "x")
    _like(w, x, "w")
    _like(grad_out, x, "grad_out")
    t, k, mid, e, i, o = _linear_dims(x, w, indices, weights, slots)
    _check(tuple(grad_out.shape) == (t,) + (() if weights is not None else (k,)) + mid + (o,),
           "grad_out must have the output's shape")
    plan = _plan_for(plan, indices, e)
    x, w, g = _dense(x), _dense(w), _dense(grad_out)
    wt = None if weights is None else weights.contiguous()
    gx = x.new_empty(x.shape) if input_gradient else None
    gw = w.new_empty(w.shape) if weight_gradient else None
    gwt = x.new_empty((t, k), dtype=torch.float32) if routing_gradient and wt is not None else None
    c = mid[0] if mid else 1
    dt, slots = _DTYPES[x.dtype], bool(slots)
    nbytes = _fn("fsc_expert_linear_backward_workspace_bytes")(
        dt, t, k, c, e, i, o, slots, wt is not None, gx is not None or gwt is not None, gw is not None,
        plan._joint_offsets is not None)
    ws = x.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _call("fsc_expert_linear_backward", x, dt, g.data_ptr(), x.data_ptr(), w.data_ptr(), plan.indices.data_ptr(),
          _ptr(wt), plan._offsets, plan._order, plan._joint_offsets, plan._joint_order, plan._status, _ptr(gx), _ptr(gw),
          _ptr(gwt), t, k, c, e, i, o, slots, _ptr(ws), nbytes)
    return gx, gw, gwt


def quantize_experts(w):
    """Experts' matrices as e4m3 with a scale for each output: ``(q, scale)``, once when they are loaded."""
    _check(w.dim() == 3, "w must have shape (experts, outputs, inputs)")
    wf = w.detach().float()
    scale = wf.abs().amax(-1) / E4M3_MAX
    q = wf / torch.where(scale > 0, scale, torch.ones_like(scale)).unsqueeze(-1)
    q = q.clamp(-E4M3_MAX, E4M3_MAX)  # a scale below the normal floats may be too small
    return q.to(torch.float8_e4m3fn), scale.contiguous()


def expert_linear_q8(x, x_scale, w, w_scale, indices, weights=None, *, slots=False, plan=None,
                     out_dtype=torch.bfloat16):
    """:func:`expert_linear` of e4m3 rows (rows, [top_k,] inputs) with a scale each, as
    :func:`add_rms_norm_q8` gives them, and e4m3 experts with a scale for each output
    (:func:`quantize_experts`).  Sums are fp32.  For serving: not differentiable."""
    f8 = torch.float8_e4m3fn
    _check(x.is_cuda and x.dtype == f8, "x must be a float8_e4m3fn CUDA tensor")
    _like(w, x, "w", f8)
    _check(out_dtype in _DTYPES, "out_dtype must be float32, bfloat16 or float16")
    t, k, mid, e, i, o = _linear_dims(x, w, indices, weights, slots)
    _check(not mid, "x must have shape (rows, inputs), or (rows, top_k, inputs) with slots")
    _like(x_scale, x, "x_scale", torch.float32)
    _check(x_scale.shape == x.shape[:-1], "x_scale must have a scale for each row of x")
    _like(w_scale, x, "w_scale", torch.float32)
    _check(w_scale.shape == w.shape[:-1], "w_scale must have shape (experts, outputs)")
    _check(not _differentiable(x_scale, w_scale, weights), "expert_linear_q8 is not differentiable")
    x, w, xs, wsc = _dense(x), _dense(w), x_scale.contiguous(), w_scale.contiguous()
    wt = None if weights is None else weights.contiguous()
    out = x.new_empty((t,) + (() if weights is not None else (k,)) + (o,), dtype=out_dtype)
    dt, slots = _DTYPES[out_dtype], bool(slots)
    if _few(t, k, mid, i, slots):
        if plan is not None:
            plan._fits(indices, e)
        idx = indices.contiguous()
        _call("fsc_expert_linear_few", x, N.FSC_E4M3, dt, x.data_ptr(), xs.data_ptr(), w.data_ptr(), wsc.data_ptr(),
              idx.data_ptr(), _ptr(wt), out.data_ptr(), t, k, 1, e, i, o, slots)
        return out
    plan = _plan_for(plan, indices, e)
    nbytes = _fn("fsc_expert_linear_workspace_bytes")(N.FSC_E4M3, t, k, 1, e, i, o, slots, wt is not None, 0)
    ws = x.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _call("fsc_expert_linear_q8", x, dt, x.data_ptr(), xs.data_ptr(), w.data_ptr(), wsc.data_ptr(),
          plan.indices.data_ptr(), _ptr(wt), plan._offsets, plan._order, plan._status, out.data_ptr(), t, k, 1, e, i, o,
          slots, _ptr(ws), nbytes)
    return out


# ---- a layer for the models' node features --------------------------------------------------------

class RoutedChannelMix(torch.nn.Module):
    """Equivariant residual layers of routed experts on node features in the models' layout.

    ``forward`` takes and returns (N, sum of channels * (2l + 1) over ``degrees``): per irrep block,
    channel-major, the first block the invariant one -- what the drop-in models hand to their
    ``sync_after_scatter``, so ``model(..., sync_after_scatter=RoutedChannelMix(64))`` evaluates the
    layer after every convolution and its gradient in the forces.  Each of ``layers`` steps is

        y, h = add_rms_norm(delta, weight, residual=h)     (all components of an atom together)
        logits = router @ y's invariant channels
        delta = sum over the chosen experts of weight * W_e y  (one matrix for all components)

    and the result is ``h + delta``.  The choice and its weights come from invariants and the matrices
    act on channels, so the layer commutes with rotations.

    As a model's hook it is evaluated with the parameters it has: the models differentiate their energy
    in positions, cell and edge vectors alone, so ``backward`` through a model leaves the ``grad`` of the
    layer's parameters (as of the model's own) as it was.  Called by itself in a program of torch
    modules, it differentiates in its parameters too.  ``degrees`` is (0, 1, 2) for
    pure-cartesian-ictd and (0, 1, 1, 2) for the o3 model's 0e, 1e, 1o, 2e."""

    def __init__(self, channels, num_experts=8, top_k=2, *, degrees=(0, 1, 2), layers=1, scores="softmax", scale=1.0,
                 eps=1e-6):
        super().__init__()
        _check(len(degrees) >= 1 and degrees[0] == 0, "the first irrep block must be the invariant one")
        self.channels, self.top_k, self.degrees, self.layers = int(channels), int(top_k), tuple(degrees), int(layers)
        self.scores, self.scale, self.eps = scores, float(scale), float(eps)
        c, x = self.channels, int(num_experts)
        _check(c >= 1 and self.layers >= 1 and 1 <= x <= 1024, "channels and layers must be at least 1, num_experts 1 to 1024")
        _check(1 <= self.top_k <= min(x, 32), "top_k must be 1 to 32 and at most num_experts")
        _check(scores in _SCORES, "scores must be 'softmax' or 'sigmoid'")
        self.norm = torch.nn.Parameter(torch.ones(self.layers, len(self.degrees), c))
        self.router = torch.nn.Parameter(torch.randn(self.layers, x, c) / math.sqrt(c))
        self.experts = torch.nn.Parameter(torch.randn(self.layers, x, c, c) / math.sqrt(c))
        block = [b for b, l in enumerate(self.degrees) for _ in range(2 * l + 1)]
        self.register_buffer("block", torch.tensor(block), persistent=False)
        self.register_buffer("bias", torch.zeros(self.layers, x))

    def _to_rows(self, f):
        n, c, off, parts = f.shape[0], self.channels, 0, []
        for l in self.degrees:
            m = 2 * l + 1
            parts.append(f[:, off:off + c * m].reshape(n, c, m).transpose(1, 2))
            off += c * m
        return torch.cat(parts, 1)

    def _from_rows(self, x):
        n, c, off, parts = x.shape[0], self.channels, 0, []
        for l in self.degrees:
            m = 2 * l + 1
            parts.append(x[:, off:off + m].transpose(1, 2).reshape(n, c * m))
            off += m
        return torch.cat(parts, 1)

    def forward(self, f):
        c, k = self.channels, self.block.shape[0]
        _check(f.dim() == 2 and f.shape[1] == c * k, f"features must have shape (N, {c * k})")
        h = self._to_rows(f).reshape(-1, k * c)
        delta = None
        for i in range(self.layers):
            weight = self.norm[i][self.block].reshape(-1)
            if delta is None:
                y = add_rms_norm(h, weight, eps=self.eps)
            else:
                y, h = add_rms_norm(delta, weight, residual=h, eps=self.eps)
            logits = torch.nn.functional.linear(y[:, :c], self.router[i])
            bias = self.bias[i].float()  # also of a layer converted to 16 bits
            weights, indices = route_experts(logits, self.top_k, bias=bias, scores=self.scores, scale=self.scale)
            delta = expert_linear(y.view(-1, k, c), self.experts[i], indices, weights).view(-1, k * c)
        return self._from_rows((h + delta).view(-1, k, c))
