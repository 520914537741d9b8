"""What a ray's learned channels are read with: a loss and an answer against a table of labels, and attention to a memory.

The tracer blends up to eight auxiliary channels of the surfels along a ray (`others_precomp` -> `aux`; several traces side by
side make more).  The operators here take such channels, or what a caller's layer makes of them, the last step: the rays x
labels or rays x memory matrix of a softmax that they go through is never stored.  HIP kernels behind the same
library (see DstLabelParams and DstAttendParams in include/dst_api.h); no fallback path.  No counterpart in the reference,
which hands `out_aux` to its caller.
"""
import ctypes as C

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _C

__all__ = ["label_loss", "label_rays", "attend_memory"]

MAX_CHANNELS = 256
_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_FORWARD, _BACKWARD, _BEST = 0, 1, 2


def _fail(rc):
    raise RuntimeError("%s (status %d)" % (_C.load_library().dst_op_error().decode(), rc))


def _rows(t, name):
    if not isinstance(t, torch.Tensor):
        raise RuntimeError("%s must be a tensor" % name)
    if t.dtype not in _DTYPES:
        raise RuntimeError("%s must be float32, bfloat16 or float16 (got %s)" % (name, t.dtype))
    if not t.is_cuda:
        raise RuntimeError("%s must be a CUDA tensor" % name)
    if t.dim() < 1 or not 1 <= t.size(-1) <= MAX_CHANNELS:
        raise RuntimeError("%s must have 1 to %d channels in its last dimension" % (name, MAX_CHANNELS))


def _beside(t, first, name, dtype=None):
    """`t` on the device of `first` (and of a dtype), or an error."""
    if not isinstance(t, torch.Tensor) or t.device != first.device:
        raise RuntimeError("%s must be a tensor on %s" % (name, first.device))
    if dtype is not None and t.dtype != dtype:
        raise RuntimeError("%s must be of %s, as the others are (got %s)" % (name, dtype, t.dtype))


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _transforms_active():
    """Whether more goes on than the call shows: inputs that may carry tangents of forward-mode differentiation or
    functorch's levels (the autograd function refuses what it has no rule for), or a trace being recorded (the autograd
    function is a node of it; its launches alone would leave only the empty output tensors there)."""
    return (forward_ad._current_level >= 0 or torch._C._are_functorch_transforms_active()
            or torch._C._get_tracing_state() is not None)


class _on:
    """The device of a tensor, for the length of a call."""

    def __init__(self, t):
        self.guard = None if t.device.index == torch._C._cuda_getDevice() else torch.cuda.device(t.device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *a):
        if self.guard is not None:
            self.guard.__exit__(*a)


def _workspace(size, like):
    """Scratch memory of the current stream's, given back when the call is done."""
    return torch.empty(size, dtype=torch.uint8, device=like.device) if size else None


# ---- labels --------------------------------------------------------------------------------------------------------
def _matrix(t, width):
    """(rows, width) with consecutive values in a row and rows that do not overlap."""
    t = t.reshape(-1, width)
    return t if t.stride(1) == 1 and (t.size(0) < 2 or t.stride(0) >= width) else t.contiguous()


def _label_params(x, w, bias):
    p = _C.DstLabelParams()
    p.rays, p.channels, p.labels, p.dtype = x.size(0), x.size(1), w.size(0), _DTYPES[x.dtype]
    p.features, p.features_stride = x.data_ptr(), x.stride(0) if x.size(0) > 1 else x.size(1)
    p.weight, p.weight_stride = w.data_ptr(), w.stride(0) if w.size(0) > 1 else w.size(1)
    p.bias = None if bias is None else bias.data_ptr()
    return p


def _run_labels(p, what, launch, like):
    lib = _C.load_library()
    ws = _workspace(lib.dst_label_workspace_bytes(C.byref(p), what), like)
    if ws is not None:
        p.workspace, p.workspace_bytes = ws.data_ptr(), ws.numel()
    rc = launch(C.byref(p), _C._stream())
    if rc != 0:
        _fail(rc)


def _set_stats(p, stats):
    """What the forward pass leaves of every ray for the backward pass: `lse`, and the three values of `stats`."""
    at = stats.data_ptr()
    p.lse, p.stats = at, at + 4 * p.rays


def _loss_forward(x, w, targets, bias, ignore_index, reduction):
    with _on(x):
        p = _label_params(x, w, bias)
        p.reduction, p.targets, p.ignore_index = reduction, targets.data_ptr(), ignore_index
        f32 = dict(dtype=torch.float32, device=x.device)
        loss = torch.empty(x.size(0) if reduction == 0 else (), **f32)
        stats = torch.empty(4 * x.size(0), **f32)
        inverse = None if reduction == 0 else torch.empty((), **f32)
        p.loss, p.inverse = loss.data_ptr(), None if inverse is None else inverse.data_ptr()
        _set_stats(p, stats)
        _run_labels(p, _FORWARD, _C.load_library().dst_label_loss_forward, x)
    return loss, stats, inverse


class _LabelLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, targets, bias, ignore_index, reduction):
        loss, stats, inverse = _loss_forward(x, w, targets, bias, ignore_index, reduction)
        ctx.save_for_backward(x, w, targets, bias, stats, inverse)
        ctx.ignore_index, ctx.reduction = ignore_index, reduction
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, upstream):
        x, w, targets, bias, stats, inverse = ctx.saved_tensors
        with _on(x):
            p = _label_params(x, w, bias)
            p.reduction, p.targets, p.ignore_index = ctx.reduction, targets.data_ptr(), ctx.ignore_index
            p.inverse = None if inverse is None else inverse.data_ptr()
            _set_stats(p, stats)
            upstream = upstream.contiguous()
            p.upstream = upstream.data_ptr()
            want_x, want_w, _, want_bias = ctx.needs_input_grad[:4]
            dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if want_x else None
            dw = torch.empty(w.shape, dtype=w.dtype, device=w.device) if want_w else None
            db = torch.empty(bias.shape, dtype=bias.dtype, device=w.device) if want_bias else None
            p.grad_features = None if dx is None else dx.data_ptr()
            p.grad_weight = None if dw is None else dw.data_ptr()
            p.grad_bias = None if db is None else db.data_ptr()
            _run_labels(p, _BACKWARD, _C.load_library().dst_label_loss_backward, x)
        return dx, dw, None, db, None, None


def _check_labels(features, weight, bias):
    _rows(features, "features")
    _beside(weight, features, "weight", features.dtype)
    if weight.dim() != 2 or weight.size(1) != features.size(-1) or weight.size(0) < 1:
        raise RuntimeError("weight must have dimensions (labels, %d), the channels of features" % features.size(-1))
    if bias is not None:
        _beside(bias, features, "bias")
        if tuple(bias.shape) != (weight.size(0),) or bias.dtype not in (torch.float32, features.dtype):
            raise RuntimeError("bias must have dimensions (labels,), in float32 or the dtype of features")


def label_loss(features, weight, targets, bias=None, *, ignore_index=-100, reduction="mean"):
    """Softmax cross entropy of rays against a table of labels: `log sum_v exp(s_v) - s_target` with
    `s = features @ weight.T + bias`, without the logits ever in memory, forward or backward.

    features: (..., channels), 1 to 256 channels, for instance a trace's `aux` (H, W, channels); weight: (labels, channels);
    both float32, bfloat16 or float16 (gradients in float16 are formed in 32 bits and rounded once); bias: (labels,), -inf switches a
    label off; targets: whole numbers of the leading dimensions of features.  `ignore_index` takes a ray out: no loss, no
    gradient, whatever its channels hold.  Any other target outside 0..labels-1 makes the loss and the gradients it
    reaches NaN.  Returns float32: the mean over the rays not ignored (NaN, without gradients, if there are none), the sum, or with "none" a loss
    for every ray.  Differentiable (once) in features, weight and bias; sums in 32 bits or more in one order: the same bits every time.
    Logits beyond 32 bits count as infinite."""
    _check_labels(features, weight, bias)
    if reduction not in _REDUCTIONS:
        raise RuntimeError("reduction must be one of none, sum, mean (got %r)" % (reduction,))
    _beside(targets, features, "targets")
    if targets.is_floating_point() or targets.is_complex() or targets.dtype == torch.bool or targets.shape != features.shape[:-1]:
        raise RuntimeError("targets must be whole numbers of dimensions %s, those of features without the last"
                           % (tuple(features.shape[:-1]),))
    ignore_index = int(ignore_index)
    if not -2 ** 63 <= ignore_index < 2 ** 63:
        raise RuntimeError("ignore_index must be a whole number of 64 bits (got %d)" % ignore_index)
    shape, d = features.shape[:-1], features.size(-1)
    wants = _wants_grad(features, weight, bias)
    x, w, t = _matrix(features, d), _matrix(weight, d), targets.reshape(-1).to(torch.int64).contiguous()
    b = None if bias is None else bias.to(torch.float32).contiguous()
    args = (x, w, t, b, ignore_index, _REDUCTIONS[reduction])
    loss = _LabelLoss.apply(*args) if wants or _transforms_active() else _loss_forward(*args)[0]
    return loss.reshape(shape) if reduction == "none" else loss


def _best_forward(x, w, bias):
    with _on(x):
        p = _label_params(x, w, bias)
        best = torch.empty(x.size(0), dtype=torch.int64, device=x.device)
        log_prob = torch.empty(x.size(0), dtype=torch.float32, device=x.device)
        p.best, p.log_prob = best.data_ptr(), log_prob.data_ptr()
        _run_labels(p, _BEST, _C.load_library().dst_label_best, x)
    return best, log_prob


class _LabelRays(torch.autograd.Function):
    """Only where a transform or a trace is under way; it has no rule for either derivative."""

    @staticmethod
    def forward(ctx, x, w, bias):
        return _best_forward(x, w, bias)


@torch.no_grad()
def label_rays(features, weight, bias=None):
    """The label of every ray, `argmax_v (features @ weight.T + bias)_v`, and its log probability, without the logits in
    memory: (int64, float32) of the leading dimensions of features.

    The label is the one that 64 bits give: rays whose two best labels 32 bits cannot tell apart are decided again; the lowest
    of equal ones.  A ray with NaN among its logits, or with every label switched off, gets some label and log probability NaN.
    Arguments as in `label_loss`; not differentiable."""
    _check_labels(features, weight, bias)
    shape, d = features.shape[:-1], features.size(-1)
    x, w = _matrix(features, d), _matrix(weight, d)
    b = None if bias is None else bias.to(torch.float32).contiguous()
    best, log_prob = _LabelRays.apply(x, w, b) if _transforms_active() else _best_forward(x, w, b)
    return best.reshape(shape), log_prob.reshape(shape)


# ---- attention -----------------------------------------------------------------------------------------------------
def _consecutive(t):
    return t if t.size(-1) == 1 or t.stride(-1) == 1 else t.contiguous()


def _strides(t):
    """By batch, row and head; 0 for a dimension of one (its stride says nothing)."""
    return (C.c_int64 * 3)(*(t.stride(i) if t.size(i) > 1 else 0 for i in range(3)))


def _attend_params(q, k, v, lengths, scale):
    p = _C.DstAttendParams()
    p.batch, p.queries, p.heads, p.channels = q.shape
    p.memory, p.kv_heads, p.value_channels, p.dtype = k.size(1), k.size(2), v.size(3), _DTYPES[q.dtype]
    p.scale = scale
    p.q, p.k, p.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    p.q_strides, p.k_strides, p.v_strides = _strides(q), _strides(k), _strides(v)
    p.lengths = None if lengths is None else lengths.data_ptr()
    return p


def _run_attend(p, what, launch, like):
    lib = _C.load_library()
    ws = _workspace(lib.dst_attend_workspace_bytes(C.byref(p), what), like)
    if ws is not None:
        p.workspace, p.workspace_bytes = ws.data_ptr(), ws.numel()
    rc = launch(C.byref(p), _C._stream())
    if rc != 0:
        _fail(rc)


def _attend_forward(q, k, v, lengths, scale, for_backward):
    with _on(q):
        p = _attend_params(q, k, v, lengths, scale)
        out = torch.empty(q.shape[:3] + v.shape[3:], dtype=q.dtype, device=q.device)
        lse = low = None
        if for_backward:
            lse = torch.empty(q.size(0) * q.size(1) * q.size(2), dtype=torch.float32, device=q.device)
            p.lse = lse.data_ptr()
            if q.dtype != torch.float32:
                low = torch.empty(out.shape, dtype=out.dtype, device=q.device)
                p.out_low = low.data_ptr()
        p.out = out.data_ptr()
        _run_attend(p, _FORWARD, _C.load_library().dst_attend_forward, q)
    return out, lse, low


class _Attend(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, scale):
        out, lse, low = _attend_forward(q, k, v, lengths, scale, True)
        ctx.save_for_backward(q, k, v, lengths, out, lse, low)
        ctx.scale = scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, upstream):
        q, k, v, lengths, out, lse, low = ctx.saved_tensors
        with _on(q):
            p = _attend_params(q, k, v, lengths, ctx.scale)
            upstream = upstream.contiguous()
            p.out, p.lse, p.upstream = out.data_ptr(), lse.data_ptr(), upstream.data_ptr()
            p.out_low = None if low is None else low.data_ptr()
            dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) if want else None
                          for t, want in zip((q, k, v), ctx.needs_input_grad))
            p.grad_q, p.grad_k, p.grad_v = (None if t is None else t.data_ptr() for t in (dq, dk, dv))
            _run_attend(p, _BACKWARD, _C.load_library().dst_attend_backward, q)
        return dq, dk, dv, None, None


def attend_memory(queries, keys, values, lengths=None, *, scale=None):
    """Attention of rays' queries to a memory of another length (a feature bank, an image encoder's states):
    `softmax(scale * queries . keys) @ values`, without the weights ever in memory, forward or backward.

    queries: (batch, queries, heads, channels); keys: (batch, memory, kv_heads, channels); values: (batch, memory, kv_heads,
    value_channels); 1 to 256 channels; float32, bfloat16 or float16, one dtype for all (gradients in float16 are
    formed in 32 bits and rounded once); any strides.  heads is a multiple of kv_heads: query head h reads kv head h // (heads // kv_heads).
    lengths: (batch,) whole numbers on the same device, how much of its memory each batch has (clamped to 0..memory; None: all).  What lies behind
    it is not used and gets a gradient of zero; a batch without memory gets zeros.  scale: 1 / sqrt(channels) by default.
    Returns (batch, queries, heads, value_channels).  Differentiable (once) in queries, keys and values; the same bits
    every time."""
    for t, name in ((queries, "queries"), (keys, "keys"), (values, "values")):
        _rows(t, name)
        _beside(t, queries, name, queries.dtype)
        if t.dim() != 4:
            raise RuntimeError("%s must have dimensions (batch, %s, heads, channels)" % (name, "queries" if name == "queries" else "memory"))
    if keys.shape[:3] != values.shape[:3] or keys.size(0) != queries.size(0) or keys.size(3) != queries.size(3):
        raise RuntimeError("keys must have dimensions (batch, memory, kv_heads, channels) with the batch and channels of queries, "
                           "and values those of keys but for the channels")
    if keys.size(2) < 1 or queries.size(2) < 1 or queries.size(2) % keys.size(2) != 0:
        raise RuntimeError("the heads of queries must be a multiple of the heads of keys")
    if lengths is not None:
        _beside(lengths, queries, "lengths")
        if tuple(lengths.shape) != (queries.size(0),) or lengths.is_floating_point() or lengths.is_complex() or lengths.dtype == torch.bool:
            raise RuntimeError("lengths must be whole numbers of dimensions (batch,)")
        if lengths.dtype != torch.int32:   # (clamped before 32 bits could wrap them)
            lengths = lengths.to(torch.int64).clamp(0, keys.size(1)).to(torch.int32)
        lengths = lengths.contiguous()
    scale = int(queries.size(3)) ** -0.5 if scale is None else float(scale)   # (a recorded trace gives sizes as tensors)
    wants = _wants_grad(queries, keys, values)
    q, k, v = _consecutive(queries), _consecutive(keys), _consecutive(values)
    if wants or _transforms_active():
        return _Attend.apply(q, k, v, lengths, scale)
    return _attend_forward(q, k, v, lengths, scale, False)[0]
