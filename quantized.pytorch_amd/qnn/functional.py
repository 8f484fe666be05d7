"""Float operators of a student's training step and of its serving, on MI355X (ROCm / gfx950).

Beside the int8 layers of `qnn.quantize` (`QLinear`, `RangeBN`) stand their float counterparts, and
the loss that a quantized student learns from:

* `linear_act` / `LinearAct`: matrix product with bias, residual and activation in its epilogue;
* `layer_norm` / `LayerNorm`: layer norm over the last dimension;
* `topk_distill_loss` / `TopKDistillLoss`: distillation from a teacher's top logits.

All run the HIP kernels of `include/qnn.h` forward and backward, in bfloat16, float16 and float32,
with fp32 sums and statistics and one rounding of each output.  As in the rest of the package there
is no fallback: a CPU tensor raises `RuntimeError`, a missing library `QnnLibraryError`.  Calls run
on the current stream of their tensors' device and allocate their workspaces there through torch, so
they may be captured into a graph (`torch.cuda.graph`), each graph with workspaces of its own.  To
capture a backward pass take `torch.autograd.grad` inside the capture and let no eager autograd graph
of the same leaves live across it (torch ties a leaf's gradient to the stream that met it first).
Results are the same from run to run.  Gradients of gradients are not offered.
"""
import ctypes
import functools

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # QNN_F32, QNN_BF16, QNN_F16
_ACTS = {"none": 0, "relu": 1, "gelu": 2}  # QNN_ACT_*
_MAX_TOP = 1024


# ------------------------------------------------------------------------------- what all share
def _check(op, name, t, dtypes, device=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"qnn: {op} expects a tensor for {name}, got {type(t).__name__}")
    if not t.is_cuda:
        raise RuntimeError(f"qnn: {op} runs on the MI355X path only (ROCm device tensor required for {name}, got "
                           f"{t.device})")
    if t.dtype not in dtypes:
        raise TypeError(f"qnn: {op} expects {name} of {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    if device is not None and t.device != device:
        raise RuntimeError(f"qnn: {op} expects its tensors on one device, got {name} on {t.device} and not {device}")


def _rows(t):
    """t as a matrix of rows along its last dimension, with dense rows that begin on the boundaries the
    kernels read at: t itself, a view, or a copy; and its row stride."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1]) if t.numel() else t.new_empty((0, t.shape[-1]))
    ld, n = t.stride(0), t.shape[1]
    if t.shape[0] <= 1:
        ld = n
    if ((t.stride(1) != 1 and n > 1) or ld < n or t.data_ptr() % 16 != 0
            or (ld != n and ld * t.element_size() % 16 != 0)):
        t, ld = t.clone(memory_format=torch.contiguous_format), n
    return t, ld


def _vector(t):
    if t is None or (t.is_contiguous() and t.data_ptr() % 16 == 0):
        return t
    return t.clone(memory_format=torch.contiguous_format)


class _On:
    """The device of a call's tensors as the current one, where it is not."""

    def __new__(cls, device):
        return torch.cuda.device(device) if device.index != torch.cuda.current_device() else _HERE


class _Here:
    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return False


_HERE = _Here()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


@functools.lru_cache(maxsize=4096)
def _work_bytes(name, *args):
    n = ctypes.c_int64(0)
    _lib.call(name, *args, ctypes.byref(n))
    return n.value


def _work(name, device, *args):
    n = _work_bytes(name, *args)
    return (torch.empty(n, dtype=torch.uint8, device=device) if n else None), n


# ------------------------------------------------------------------------------------ linear_act
def _linear_fwd(x, ldx, w, ldw, b, r, ldr, act, need_slope):
    m, k = x.shape
    n = w.shape[0]
    code = _DTYPES[x.dtype]
    dev = x.device
    y = torch.empty((m, n), dtype=x.dtype, device=dev)
    slope = None
    if need_slope and act == 1:
        slope = torch.empty((m, (n + 7) // 8), dtype=torch.uint8, device=dev)
    elif need_slope and act == 2:
        slope = torch.empty((m, n), dtype=torch.float32 if code == 0 else torch.int16, device=dev)
    with _On(dev):
        work, nwork = _work("qnn_linear_act_fwd_work", dev, m, n, k, code)
        _lib.call("qnn_linear_act_fwd", _ptr(x), ldx, _ptr(w), ldw, _ptr(b), _ptr(r), ldr, _ptr(y), _ptr(slope), m, n,
                  k, code, act, _ptr(work), nwork, _stream(dev))
    return y, slope


class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, r, act):
        x2, ldx = _rows(x)
        w2, ldw = _rows(w)
        r2, ldr = (None, 0) if r is None else _rows(r)
        y, slope = _linear_fwd(x2, ldx, w2, ldw, _vector(b), r2, ldr, act, True)
        ctx.act, ctx.x_shape = act, x.shape
        need = ctx.needs_input_grad
        ctx.save_for_backward(x2 if need[1] else None, w2 if need[0] else None, slope)
        ctx.sizes = (x2.shape[0], w2.shape[0], x2.shape[1])
        ctx.dtype = x.dtype
        return y.view(*x.shape[:-1], w.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, slope = ctx.saved_tensors
        need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
        m, n, k = ctx.sizes
        act, dt, dev = ctx.act, ctx.dtype, dy.device
        code = _DTYPES[dt]
        dy2, ldy = _rows(dy)
        if x is not None:
            x, ldx = _rows(x)
        else:
            ldx = k
        if w is not None:
            w, ldw = _rows(w)
        else:
            ldw = k
        dz = torch.empty((m, n), dtype=dt, device=dev) if act else None
        dx = torch.empty((m, k), dtype=dt, device=dev) if need_x else None
        dw = torch.empty((n, k), dtype=dt, device=dev) if need_w else None
        db = torch.empty((n,), dtype=dt, device=dev) if need_b else None
        if act or need_x or need_w or need_b:
            with _On(dev):
                work, nwork = _work("qnn_linear_act_bwd_work", dev, m, n, k, code)
                _lib.call("qnn_linear_act_bwd", _ptr(dy2), ldy, _ptr(slope), _ptr(x), ldx, _ptr(w), ldw, _ptr(dz),
                          _ptr(dx), _ptr(dw), _ptr(db), m, n, k, code, act, _ptr(work), nwork, _stream(dev))
        dr = None
        if need_r:
            dr = dz.view(dy.shape) if act else dy
        return (dx.view(ctx.x_shape) if need_x else None), dw, db, dr, None


def linear_act(x, weight, bias=None, residual=None, activation="none"):
    """act(x @ weight.T + bias + residual): one launch where the product fills the chip, with the sum,
    the residual and the activation in fp32 and one rounding at the end.

    x [..., in], weight [out, in], bias [out], residual [..., out] (the output's shape; expand it for
    a broadcast one), all of one type; activation "none", "relu" or "gelu" (the erf form), applied
    after the residual as in the int8 layers' epilogue.  Under autograd gradients flow to all four;
    between the passes a bit an element is kept for ReLU, and the slope for GELU (16 bits, 32 in
    float32).  The gradient of z is rounded to the type once, before the two products it enters."""
    _check("linear_act", "x", x, _DTYPES)
    dev, dt = x.device, (x.dtype,)
    _check("linear_act", "weight", weight, dt, dev)
    act = _ACTS.get(activation)
    if act is None:
        raise ValueError(f"qnn: linear_act activation must be one of {sorted(_ACTS)}, got {activation!r}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"qnn: linear_act needs x [..., in] and weight [out, in], got {tuple(x.shape)} and "
                         f"{tuple(weight.shape)}")
    n, k = weight.shape
    if n == 0 or k == 0:
        raise ValueError("qnn: linear_act needs at least one input and one output feature")
    if bias is not None:
        _check("linear_act", "bias", bias, dt, dev)
        if bias.shape != (n,):
            raise ValueError(f"qnn: linear_act needs bias [{n}], got {tuple(bias.shape)}")
    if residual is not None:
        _check("linear_act", "residual", residual, dt, dev)
        if residual.shape[:-1] != x.shape[:-1] or residual.dim() != x.dim() or residual.shape[-1] != n:
            raise ValueError(f"qnn: linear_act needs a residual of the output's shape, got {tuple(residual.shape)} "
                             f"for x {tuple(x.shape)} and weight {tuple(weight.shape)}")
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or
                                    (bias is not None and bias.requires_grad) or
                                    (residual is not None and residual.requires_grad)):
        return _LinearAct.apply(x, weight, bias, residual, act)
    x2, ldx = _rows(x.detach())
    w2, ldw = _rows(weight.detach())
    r2, ldr = (None, 0) if residual is None else _rows(residual.detach())
    y, _ = _linear_fwd(x2, ldx, w2, ldw, _vector(bias), r2, ldr, act, False)
    return y.view(*x.shape[:-1], n)


class LinearAct(nn.Linear):
    """nn.Linear with an activation, and a residual given at the call: `linear_act` as a module."""

    def __init__(self, in_features, out_features, bias=True, activation="none", device=None, dtype=None):
        super().__init__(in_features, out_features, bias, device=device, dtype=dtype)
        if activation not in _ACTS:
            raise ValueError(f"qnn: LinearAct activation must be one of {sorted(_ACTS)}, got {activation!r}")
        self.activation = activation

    def forward(self, input, residual=None):
        return linear_act(input, self.weight, self.bias, residual, self.activation)

    def extra_repr(self):
        return f"{super().extra_repr()}, activation={self.activation}"


# ------------------------------------------------------------------------------------ layer_norm
def _norm_fwd(x, ldx, w, b, eps, wcode, need_stats):
    rows, dim = x.shape
    dev = x.device
    y = torch.empty((rows, dim), dtype=x.dtype, device=dev)
    stats = torch.empty((2, rows), dtype=torch.float32, device=dev) if need_stats else None
    mean = _ptr(stats)
    with _On(dev):
        _lib.call("qnn_layer_norm_fwd", _ptr(x), ldx, _ptr(w), _ptr(b), _ptr(y), mean,
                  None if mean is None else mean + 4 * rows, rows, dim, eps, _DTYPES[x.dtype], wcode, _stream(dev))
    return y, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, eps, wcode):
        x2, ldx = _rows(x)
        w2 = _vector(w)
        y, stats = _norm_fwd(x2, ldx, w2, _vector(b), eps, wcode, True)
        ctx.save_for_backward(x2, w2, stats)
        ctx.shape, ctx.wcode = x.shape, wcode
        ctx.wdtype = w.dtype if w is not None else b.dtype if b is not None else None
        return y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, stats = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        rows, dim = x.shape
        dev, code = dy.device, _DTYPES[x.dtype]
        dy2, ldy = _rows(dy)
        x, ldx = _rows(x)
        dx = torch.empty((rows, dim), dtype=x.dtype, device=dev) if need_x else None
        dw = torch.empty((dim,), dtype=ctx.wdtype, device=dev) if need_w else None
        db = torch.empty((dim,), dtype=ctx.wdtype, device=dev) if need_b else None
        mean = _ptr(stats)
        with _On(dev):
            work, nwork = _work("qnn_layer_norm_bwd_work", dev, rows, dim, code)
            _lib.call("qnn_layer_norm_bwd", _ptr(dy2), ldy, _ptr(x), ldx, _ptr(w), mean, mean + 4 * rows, _ptr(dx),
                      _ptr(dw), _ptr(db), rows, dim, code, ctx.wcode, _ptr(work), nwork, _stream(dev))
        return (dx.view(ctx.shape) if need_x else None), dw, db, None, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension, with the biased variance.

    x [..., dim]; weight and bias [dim] (either may be None), both of x's type or both float32.  Mean
    and variance are fp32, the variance from the deviations; under autograd two floats a row are kept
    beside x."""
    _check("layer_norm", "x", x, _DTYPES)
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"qnn: layer_norm needs x [..., dim] with dim > 0, got {tuple(x.shape)}")
    if not eps >= 0.0:
        raise ValueError(f"qnn: layer_norm needs eps >= 0, got {eps}")
    dim, wcode = x.shape[-1], _DTYPES[x.dtype]
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            _check("layer_norm", name, t, (x.dtype, torch.float32), x.device)
            if t.shape != (dim,):
                raise ValueError(f"qnn: layer_norm needs {name} [{dim}], got {tuple(t.shape)}")
            wcode = _DTYPES[t.dtype]
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"qnn: layer_norm needs weight and bias of one type, got {weight.dtype} and {bias.dtype}")
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or
                                    (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, float(eps), wcode)
    x2, ldx = _rows(x.detach())
    return _norm_fwd(x2, ldx, _vector(weight), _vector(bias), float(eps), wcode, False)[0].view(x.shape)


class LayerNorm(nn.LayerNorm):
    """nn.LayerNorm over one (the last) dimension on `layer_norm`; same parameters and state_dict."""

    def __init__(self, normalized_shape, eps=1e-5, elementwise_affine=True, bias=True, device=None, dtype=None):
        super().__init__(normalized_shape, eps, elementwise_affine, bias, device=device, dtype=dtype)
        if len(self.normalized_shape) != 1:
            raise ValueError(f"qnn: LayerNorm normalizes the last dimension, got {tuple(self.normalized_shape)}")

    def forward(self, input):
        if input.shape[-1:] != tuple(self.normalized_shape):
            raise ValueError(f"qnn: LayerNorm({self.normalized_shape[0]}) got an input {tuple(input.shape)}")
        return layer_norm(input, self.weight, self.bias, self.eps)


# ----------------------------------------------------------------------------- topk_distill_loss
_REDUCTIONS = ("mean", "sum", "none")


def _distill_fwd(s, lds, t, ldt, i, ldi, temp, reduction):
    rows, vocab = s.shape
    top = t.shape[1]
    dev, code = s.device, _DTYPES[s.dtype]
    stats = torch.empty(4 * rows + 4, dtype=torch.float32, device=dev)
    row_loss = torch.empty(rows, dtype=torch.float32, device=dev)
    loss = None if reduction == "none" else torch.empty((), dtype=torch.float32, device=dev)
    with _On(dev):
        work, nwork = _work("qnn_topk_distill_fwd_work", dev, rows, vocab, code)
        _lib.call("qnn_topk_distill_fwd", _ptr(s), lds, _ptr(t), ldt, _ptr(i), ldi, rows, vocab, top, temp,
                  int(reduction == "mean"), code, _DTYPES[t.dtype], i.element_size(), _ptr(row_loss), _ptr(stats),
                  _ptr(loss), _ptr(work), nwork, _stream(dev))
    return (row_loss if loss is None else loss), stats


class _TopKDistill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, s, t, i, temp, reduction):
        s2, lds = _rows(s)
        t2, ldt = _rows(t)
        i2, ldi = _rows(i)
        loss, stats = _distill_fwd(s2, lds, t2, ldt, i2, ldi, temp, reduction)
        ctx.save_for_backward(s2, t2, i2, stats)
        ctx.args = (temp, reduction, s.shape)
        return loss if reduction != "none" else loss.view(s.shape[:-1])

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        s, t, i, stats = ctx.saved_tensors
        temp, reduction, shape = ctx.args
        rows, vocab = s.shape
        s, lds = _rows(s)
        t, ldt = _rows(t)
        i, ldi = _rows(i)
        g = g.contiguous()
        ds = torch.empty((rows, vocab), dtype=s.dtype, device=s.device)
        with _On(s.device):
            _lib.call("qnn_topk_distill_bwd", _ptr(s), lds, _ptr(t), ldt, _ptr(i), ldi, _ptr(stats), _ptr(g),
                      int(reduction == "none"), _ptr(ds), rows, vocab, t.shape[1], temp, int(reduction == "mean"),
                      _DTYPES[s.dtype], _DTYPES[t.dtype], i.element_size(), _stream(s.device))
        return ds.view(shape), None, None, None, None


def topk_distill_loss(logits, teacher_logits, teacher_index, temperature=1.0, reduction="mean"):
    """temperature^2 KL(p || q) between a teacher known by its top logits and a student.

    logits [..., vocab]; teacher_logits [..., top] (any of the three types) at the classes
    teacher_index [..., top] (int64 or int32), top <= 1024.  p is the softmax of teacher_logits /
    temperature over a row's entries, q that of logits / temperature over the vocabulary.  An entry
    with a negative index is absent (padding); a class that is named twice has the sum of its
    entries; an index past the vocabulary makes its row's loss and gradient NaN.  A row without
    entries (or whose teacher logits are all -inf) is not counted: loss 0, gradient 0.

    The loss is float32: the mean over the counted rows (0 if there is none), their sum, or with
    "none" the rows' losses [...].  Gradients flow to logits alone, in their type; the teacher is a
    constant."""
    _check("topk_distill_loss", "logits", logits, _DTYPES)
    dev = logits.device
    _check("topk_distill_loss", "teacher_logits", teacher_logits, _DTYPES, dev)
    _check("topk_distill_loss", "teacher_index", teacher_index, (torch.int64, torch.int32), dev)
    if reduction not in _REDUCTIONS:
        raise ValueError(f"qnn: topk_distill_loss reduction must be one of {_REDUCTIONS}, got {reduction!r}")
    temp = float(temperature)
    if not 0.0 < temp < float("inf"):
        raise ValueError(f"qnn: topk_distill_loss needs a positive, finite temperature, got {temperature}")
    if logits.dim() < 1 or logits.shape[-1] == 0:
        raise ValueError(f"qnn: topk_distill_loss needs logits [..., vocab], got {tuple(logits.shape)}")
    if (teacher_logits.shape != teacher_index.shape or teacher_logits.dim() != logits.dim()
            or teacher_logits.shape[:-1] != logits.shape[:-1]):
        raise ValueError(f"qnn: topk_distill_loss needs teacher_logits and teacher_index [..., top] beside logits "
                         f"{tuple(logits.shape)}, got {tuple(teacher_logits.shape)} and {tuple(teacher_index.shape)}")
    if not 1 <= teacher_logits.shape[-1] <= _MAX_TOP:
        raise ValueError(f"qnn: topk_distill_loss takes 1 to {_MAX_TOP} entries a row, got {teacher_logits.shape[-1]}")
    teacher_logits = teacher_logits.detach()
    if torch.is_grad_enabled() and logits.requires_grad:
        return _TopKDistill.apply(logits, teacher_logits, teacher_index, temp, reduction)
    s, lds = _rows(logits.detach())
    t, ldt = _rows(teacher_logits)
    i, ldi = _rows(teacher_index)
    loss, _ = _distill_fwd(s, lds, t, ldt, i, ldi, temp, reduction)
    return loss if reduction != "none" else loss.view(logits.shape[:-1])


class TopKDistillLoss(nn.Module):
    """`topk_distill_loss` as a module."""

    def __init__(self, temperature=1.0, reduction="mean"):
        super().__init__()
        self.temperature, self.reduction = temperature, reduction

    def forward(self, logits, teacher_logits, teacher_index):
        return topk_distill_loss(logits, teacher_logits, teacher_index, self.temperature, self.reduction)
