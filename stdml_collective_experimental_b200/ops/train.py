"""Operators that the models are trained with, on CUDA tensors: ``group_norm`` with its
activation and the shortcut of a residual block, ``gated_linear``, the gated projection
of a feed-forward block, and ``distill_loss`` against a teacher's top logits.

They run on the current stream of their tensors' GPU, whichever GPU is current, are
differentiable once (backward; tangents are refused), and can be captured into a CUDA graph (after a first call outside of
one; forward and backward together, as autograd allows: no graph of the same leaves may live
that was made on another stream).
Workspaces and whatever is kept for the backward pass come from PyTorch's allocator; the
same inputs give the same bits.  What is wrong with the arguments raises ``ValueError`` /
``TypeError`` before anything is launched.  The reference has no operators of a model: its
users bring them with their framework.
"""
import ctypes

import torch

from .. import _native

_ACTS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
_NORM_ACTS = {k: v for k, v in _ACTS.items() if v < 4}
_GATES = {k: v for k, v in _ACTS.items() if v > 1}
_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def _code(table, name, what):
    try:
        return table[name]
    except (KeyError, TypeError):
        raise ValueError(f"unknown {what} {name!r}") from None


def group_norm(x, groups, weight=None, bias=None, eps=1e-5, activation=None, residual=None):
    """act(group_norm(x) * weight + bias [+ residual]) of (N, C, ...) images.

    x: bf16, f16 or f32, 2 dimensions or more; C is a multiple of `groups`.  Channels-last
    tensors (any row and image stride) are read where they lie, others are copied first; the
    result is channels last.  weight, bias: one value for each channel, of any of the three
    types; residual: as x.  activation: None, "relu", "silu", "gelu".  Statistics are taken
    over the positions and channels of a group: in 32 bits over runs of 16 positions, about a mean
    nearby, and in 64 beyond; values next to the border of "relu" are placed in 64."""
    return _native.fastcall().group_norm(x, residual, weight, bias, groups, eps,
                                         _code(_NORM_ACTS, activation, "activation"))


def distill_loss(logits, teacher_logits, teacher_index, labels=None, temperature=1.0, alpha=0.5,
                 ignore_index=-100, reduction="mean"):
    """alpha * CE(z, label) + (1 - alpha) * t^2 * KL(teacher || softmax(z / t)) of the rows z of
    (..., classes) logits; without labels t^2 * KL, whatever alpha.

    The teacher gives its largest logits, (..., k) `teacher_logits` at the classes
    `teacher_index` (int32 or int64), k <= 4096; its distribution is their softmax at
    temperature t.  An index outside [0, classes) is no entry, so rows may have fewer than k;
    a class named twice counts twice.  A row counts where its label lies in [0, classes) and
    is not `ignore_index`, or without labels where the teacher has an entry of any weight; a row
    that counts but has no entry has no second term.  reduction: "mean" over the rows that count
    (0 where none does), "sum", "none" (0 in rows that do not count).  The loss is f32; the
    gradient goes to the logits alone, in their type.

    With reduction "mean" or "sum", bf16 and f32 logits that want a gradient get it in the
    forward pass already, for a loss of gradient 1; for another the backward pass computes it
    again.  Under torch.no_grad() the loss alone is computed."""
    return _native.fastcall().distill_loss(logits, teacher_logits, teacher_index, labels,
                                           temperature, alpha, ignore_index,
                                           _code(_REDUCTIONS, reduction, "reduction"))


def gated_linear(x, w_gate, w_up, b_gate=None, b_up=None, activation="gelu"):
    """act(x w_gate^T + b_gate) * (x w_up^T + b_up): both projections of a gated feed-forward
    block, the activation and the product.

    x: (..., hidden) of bf16, f16 or f32; weights (ffn, hidden) and biases (ffn,) of the same
    type, rows of any stride (the halves of one fused weight, for instance); both biases or
    none.  activation: "gelu", "gelu_tanh", "silu".  Products are summed in 32 bits; f32
    operands keep their 24 bits (an infinity among them comes out as NaN).  For gradients of
    16-bit types those of the two projections are rounded to the type once (in f16 after
    scaling, so that none leaves its range), and multiplied in it."""
    return _native.fastcall().gated_linear(x, w_gate, w_up, b_gate, b_up,
                                           _code(_GATES, activation, "activation"))


def check(device=None):
    """Waits for all work of a GPU (the current one, if none is named) and raises DeviceTimeoutError if
    a bounded wait inside one of these operators has run out since the last question: its results are
    not complete then.  Not while a graph is being captured."""
    where = torch.device("cuda" if device is None else device)
    if where.type != "cuda":
        raise ValueError(f"check: CUDA device expected, got {where}")
    index = torch.cuda.current_device() if where.index is None else where.index
    status = ctypes.c_int()
    _native.check(_native.lib().stdmlc_train_status(index, ctypes.byref(status)))
    if status.value:
        raise _native.DeviceTimeoutError(4, f"a bounded wait of an operator ran out on GPU {index}")
