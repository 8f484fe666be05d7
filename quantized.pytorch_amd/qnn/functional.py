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
Results are the same from run to run.  Gradients of gradients and forward-mode derivatives are not
offered: a dual tensor with a tangent raises `RuntimeError`, and so does a call under `torch.jit.trace`.
Gradients made under `create_graph` raise it when they are differentiated further by way of the gradient
that came in; if that does not require one they are constants, with a warning.

The checks, allocations and autograd nodes are a CPython extension (`csrc/functional.cpp`, built beside
the library), since the calls are short.
"""
import ctypes
import importlib

import torch
import torch.nn as nn

from . import _lib

_ACTS = {"none": 0, "relu": 1, "gelu": 2}  # QNN_ACT_*
_REDUCTIONS = {"mean": 0, "sum": 1, "none": 2}
_ENTRIES = ("qnn_last_error", "qnn_linear_act_fwd_work", "qnn_linear_act_fwd", "qnn_linear_act_bwd_work",
            "qnn_linear_act_bwd", "qnn_layer_norm_fwd", "qnn_layer_norm_bwd_work", "qnn_layer_norm_bwd",
            "qnn_topk_distill_fwd_work", "qnn_topk_distill_fwd", "qnn_topk_distill_bwd")

_native = None


def load():
    """The extension, bound to the library's entries (cached).  Raises QnnLibraryError if either is absent."""
    global _native
    if _native is None:
        lib = _lib.load()
        try:
            native = importlib.import_module("._float", __package__)
        except ImportError as e:
            raise _lib.QnnLibraryError(f"qnn: the float operators' extension does not load ({e}) - build it with "
                                       "`make -C quantized.pytorch_amd`") from e
        native.bind({n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in _ENTRIES})
        _native = native
    return _native


# ------------------------------------------------------------------------------------ linear_act
def linear_act(x, weight, bias=None, residual=None, activation="none"):
    """act(x @ weight.T + bias + residual): one launch where the product fills the chip, with the sum,
    the residual and the activation in fp32 and one rounding at the end.

    x [..., in], weight [out, in], bias [out], residual [..., out] (the output's shape; expand it for
    a broadcast one), all of one type; activation "none", "relu" or "gelu" (the erf form), applied
    after the residual as in the int8 layers' epilogue.  Under autograd gradients flow to all four;
    between the passes a bit an element is kept for ReLU, and the slope d for GELU: 32 bits in float32,
    in bfloat16 and float16 16 bits that are off by 2^-11 of d, and by 5e-5 |d|^(3/4), an eighth and
    (from |d| = 1e-4 on) at most the whole of the type's half step.  The gradient of z is rounded to the
    type once, before the two products it enters."""
    act = _ACTS.get(activation)
    if act is None:
        raise ValueError(f"qnn: linear_act activation must be one of {sorted(_ACTS)}, got {activation!r}")
    return (_native or load()).linear_act(x, weight, bias, residual, act)


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
def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension, with the biased variance.

    x [..., dim]; weight and bias [dim] (either may be None), both of x's type or both float32.  Mean
    and variance are fp32, the variance from the deviations; under autograd two floats a row are kept
    beside x."""
    return (_native or load()).layer_norm(x, weight, bias, eps)


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
def topk_distill_loss(logits, teacher_logits, teacher_index, temperature=1.0, reduction="mean"):
    """temperature^2 sum_e p_e (log p_e - log q_index[e]) between a teacher known by its top logits
    and a student: temperature^2 KL(p || q) where a row's classes are distinct.

    logits [..., vocab]; teacher_logits [..., top] (any of the three types) at the classes
    teacher_index [..., top] (int64 or int32), top <= 1024.  p is the softmax of teacher_logits /
    temperature over a row's entries, q that of logits / temperature over the vocabulary.  An entry
    with a negative index is absent (padding).  A class that is named twice takes part with each of
    its entries: the gradient is that of the KL whose P at the class is the sum of them, and the
    value is that KL plus temperature^2 sum_e p_e log(p_e / P_index[e]), a constant of the teacher,
    which is 0 without such classes and else negative.  An index past the vocabulary, or a teacher
    logit that is NaN, makes its row's loss and gradient NaN.  A row without entries (or whose
    teacher logits are all -inf) is not counted: loss 0, gradient 0.

    The loss is float32: the mean over the counted rows (0 if there is none), their sum, or with
    "none" the rows' losses [...].  Gradients flow to logits alone, in their type; the teacher is a
    constant."""
    code = _REDUCTIONS.get(reduction)
    if code is None:
        raise ValueError(f"qnn: topk_distill_loss reduction must be one of {tuple(_REDUCTIONS)}, got {reduction!r}")
    return (_native or load()).topk_distill_loss(logits, teacher_logits, teacher_index, temperature, code)


class TopKDistillLoss(nn.Module):
    """`topk_distill_loss` as a module."""

    def __init__(self, temperature=1.0, reduction="mean"):
        super().__init__()
        self.temperature, self.reduction = temperature, reduction

    def forward(self, logits, teacher_logits, teacher_index):
        return topk_distill_loss(logits, teacher_logits, teacher_index, self.temperature, self.reduction)
