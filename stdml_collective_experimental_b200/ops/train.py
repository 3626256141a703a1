"""Operators that the models are trained with, on CUDA tensors: ``group_norm`` with its
activation and the shortcut of a residual block, ``gated_linear``, the gated projection
of a feed-forward block, and ``distill_loss`` against a teacher's top logits.

They run on the current stream of their tensors' GPU, whichever GPU is current, are
differentiable once, and can be captured into a CUDA graph.  Workspaces and whatever is
kept for the backward pass come from PyTorch's allocator.  What is wrong with the
arguments raises ``ValueError`` / ``TypeError`` before anything is launched.  The
reference has no operators of a model: its users bring them with their framework.
"""
import torch

from .. import _native

_ACTS = {None: 0, "none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def _code(table, name, what):
    try:
        return table[name]
    except (KeyError, TypeError):
        raise ValueError(f"unknown {what} {name!r}") from None


def _once(call):
    """Second derivatives would silently lack what goes through this operator."""
    if torch.is_grad_enabled():
        raise RuntimeError(f"{call} is differentiable once: backward with create_graph=True is refused")


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, groups, eps, act):
        y, stats, xr, rr = _native.fastcall().norm_forward(x, residual, weight, bias, groups, eps, act)
        ctx.save_for_backward(xr, rr if act else None, weight, bias, stats)
        ctx.consts = (groups, eps, act)
        return y

    @staticmethod
    def backward(ctx, dy):
        _once("group_norm")
        x, residual, weight, bias, stats = ctx.saved_tensors
        wants = ctx.needs_input_grad
        return (*_native.fastcall().norm_backward(dy, x, residual, weight, bias, stats, *ctx.consts,
                                                  *wants[:4]), None, None, None)


def group_norm(x, groups, weight=None, bias=None, eps=1e-5, activation=None, residual=None):
    """act(group_norm(x) * weight + bias [+ residual]) of (N, C, ...) images.

    x: bf16, f16 or f32, 2 dimensions or more; C is a multiple of `groups`.  Channels-last
    tensors (any row and image stride) are read where they lie, others are copied first; the
    result is channels last.  weight, bias: one value for each channel, of any of the three
    types; residual: as x.  activation: None, "relu", "silu", "gelu".  Statistics are taken
    over the positions and channels of a group, in 64 bits, and values next to the border of
    "relu" are placed in 64."""
    act = _code(_ACTS, activation, "activation")
    if act == 4:
        raise ValueError(f"unknown activation {activation!r}")
    return _GroupNorm.apply(x, residual, weight, bias, groups, eps, act)


class _DistillLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top, index, labels, *consts):
        loss, stats = _native.fastcall().distill_forward(logits, top, index, labels, *consts)
        ctx.save_for_backward(logits, top, index, labels, stats)
        ctx.consts = consts
        return loss

    @staticmethod
    def backward(ctx, dloss):
        _once("distill_loss")
        grad = _native.fastcall().distill_backward(dloss, *ctx.saved_tensors, *ctx.consts)
        return grad, None, None, None, None, None, None, None


def distill_loss(logits, teacher_logits, teacher_index, labels=None, temperature=1.0, alpha=0.5,
                 ignore_index=-100, reduction="mean"):
    """alpha * CE(z, label) + (1 - alpha) * t^2 * KL(teacher || softmax(z / t)) of the rows z of
    (..., classes) logits; without labels t^2 * KL, whatever alpha.

    The teacher gives its largest logits, (..., k) `teacher_logits` at the classes
    `teacher_index` (int32 or int64), k <= 4096; its distribution is their softmax at
    temperature t.  An index outside [0, classes) is no entry, so rows may have fewer than k;
    a class named twice counts twice.  A row counts where its label lies in [0, classes) and
    is not `ignore_index`, or without labels where the teacher has an entry; a row that counts
    but has no entry has no second term.  reduction: "mean" over the rows that count (0 where
    none does), "sum", "none" (0 in rows that do not count).  The loss is f32; the gradient
    goes to the logits alone, in their type."""
    if not isinstance(teacher_logits, torch.Tensor) or teacher_logits.requires_grad:
        raise ValueError("distill_loss: teacher_logits are constants: a tensor without gradient expected")
    return _DistillLoss.apply(logits, teacher_logits, teacher_index, labels, temperature, alpha,
                              ignore_index, _code(_REDUCTIONS, reduction, "reduction"))


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, b_gate, b_up, act):
        follows = any(ctx.needs_input_grad)
        h, saved = _native.fastcall().gated_forward(x, w_gate, w_up, b_gate, b_up, act, follows)
        if follows:
            ctx.save_for_backward(x, w_gate, w_up, b_gate, b_up, saved)
            ctx.act = act
        return h

    @staticmethod
    def backward(ctx, dh):
        _once("gated_linear")
        wants = ctx.needs_input_grad
        return (*_native.fastcall().gated_backward(dh, *ctx.saved_tensors, ctx.act, *wants[:5]), None)


def gated_linear(x, w_gate, w_up, b_gate=None, b_up=None, activation="gelu"):
    """act(x w_gate^T + b_gate) * (x w_up^T + b_up): both projections of a gated feed-forward
    block, the activation and the product.

    x: (..., hidden) of bf16, f16 or f32; weights (ffn, hidden) and biases (ffn,) of the same
    type, rows of any stride (the halves of one fused weight, for instance); both biases or
    none.  activation: "gelu", "gelu_tanh", "silu".  Products are summed in 32 bits; f32
    operands keep their 24 bits."""
    act = _code(_ACTS, activation, "activation")
    if act < 2:
        raise ValueError(f"unknown activation {activation!r}")
    return _GatedLinear.apply(x, w_gate, w_up, b_gate, b_up, act)
