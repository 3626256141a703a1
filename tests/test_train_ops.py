"""The operators that models are trained with (group_norm, distill_loss, gated_linear): refusals
on any machine; on a GPU the results against plain implementations in 64 bits.

Tolerances are bounds, not observations.  U = 2^-24 is half a step of 32 bits, of which each
elementary operation and each exp, erf, tanh costs a few; `half(t)` is half a step of the
result's type.  Sums are bounded by the sum of their terms' sizes."""
import math

import pytest
import torch

from stdml_collective_experimental_b200 import ops

U = 2.0 ** -24
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = [BF16, F16, F32]
gpu = pytest.mark.gpu
cuda = torch.device("cuda", 0)


def half(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    """What a rounding may lose below the normal numbers."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def within(got, want, tol):
    """Every element of `got` within `tol` of `want` plus the rounding to its type."""
    assert got.shape == want.shape
    w = want.double()
    if not torch.is_tensor(tol):
        tol = torch.full_like(w, tol)
    tol = tol.double() * (1 + 2 * half(got.dtype)) + half(got.dtype) * w.abs() + least(got.dtype)
    bad = ~((got.double() - w).abs() <= tol)
    bad &= ~(got.double().isnan() & w.isnan()) & ~(got.double() == w)
    if bad.any():
        i = torch.nonzero(bad)[0].tolist()
        raise AssertionError(f"{int(bad.sum())} of {bad.numel()} values off, first at {i}: got "
                             f"{got[tuple(i)].item()}, want {w[tuple(i)].item()} +- {tol[tuple(i)].item()}")


def rand(shape, seed, dtype=F32, scale=1.0, shift=0.0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    return (torch.randn(shape, device=cuda, generator=g) * scale + shift).to(dtype)


def channels_last(shape, seed, dtype, scale=1.0, shift=0.0):
    n, c, *s = shape
    return rand((n, *s, c), seed, dtype, scale, shift).movedim(-1, 1)


# ------------------------------------------------------------------------- refusals
@pytest.mark.parametrize("change,error", [
    ({}, "CUDA tensor expected"),
    ({"x": torch.zeros(4)}, r"\(N, C, ...\)"),
    ({"groups": 3}, "do not divide"),
    ({"groups": 0}, "do not divide"),
    ({"eps": -1.0}, "eps"),
    ({"eps": math.nan}, "eps"),
    ({"weight": torch.zeros(3)}, "weight and bias"),
    ({"bias": torch.zeros(4, 1)}, "weight and bias"),
    ({"weight": torch.zeros(4), "bias": torch.zeros(4).bfloat16()}, "one dtype"),
    ({"residual": torch.zeros(2, 4, 5)}, "residual of"),
    ({"residual": torch.zeros(2, 4, 6).half()}, "dtype"),
    ({"x": torch.zeros(2, 4, 6).double()}, "float32 expected"),
    ({"x": torch.zeros(2, 4, 6).int()}, "float32 expected"),
    ({"activation": "tanh"}, "unknown activation"),
    ({"activation": "gelu_tanh"}, "unknown activation"),
    ({"x": None}, "tensor expected"),
])
def test_group_norm_refuses(native_lib, change, error):
    args = {"x": torch.zeros(2, 4, 6), "groups": 2, **change}
    with pytest.raises((ValueError, TypeError), match=error):
        ops.group_norm(**args)


@pytest.mark.parametrize("change,error", [
    ({}, "CUDA tensor expected"),
    ({"logits": torch.zeros(3, 0)}, "classes"),
    ({"logits": torch.zeros(())}, "classes"),
    ({"logits": torch.zeros(3, 7).double()}, "float32 expected"),
    ({"teacher_logits": torch.zeros(4, 2)}, "rows expected"),
    ({"teacher_logits": torch.zeros(3, 2, 1)}, "rows expected"),
    ({"teacher_logits": torch.zeros(3, 2).long()}, "float32 expected"),
    ({"teacher_logits": torch.zeros(3, 2, requires_grad=True)}, "constants"),
    ({"teacher_index": torch.zeros(3, 1).long()}, "teacher_index of"),
    ({"teacher_index": torch.zeros(3, 2)}, "int32 or int64"),
    ({"labels": torch.zeros(2).long()}, "label"),
    ({"labels": torch.zeros(3)}, "int32 or int64"),
    ({"temperature": 0.0}, "temperature"),
    ({"temperature": math.nan}, "temperature"),
    ({"temperature": math.inf}, "temperature"),
    ({"alpha": 1.5}, "alpha"),
    ({"alpha": math.nan}, "alpha"),
    ({"reduction": "max"}, "reduction"),
    ({"teacher_logits": torch.zeros(3, 4097), "teacher_index": torch.zeros(3, 4097).long()}, "4096"),
])
def test_distill_loss_refuses(native_lib, change, error):
    args = {"logits": torch.zeros(3, 7), "teacher_logits": torch.zeros(3, 2),
            "teacher_index": torch.zeros(3, 2).long(), **change}
    with pytest.raises((ValueError, TypeError), match=error):
        ops.distill_loss(**args)


@pytest.mark.parametrize("change,error", [
    ({}, "CUDA tensor expected"),
    ({"x": torch.zeros(())}, "hidden"),
    ({"x": torch.zeros(2, 3)}, "weights of"),
    ({"x": torch.zeros(2, 4).double()}, "float32 expected"),
    ({"x": torch.zeros(2, 4).half()}, "dtype"),
    ({"w_up": torch.zeros(5, 4)}, "two weights"),
    ({"w_gate": torch.zeros(6, 4, 1)}, "two weights"),
    ({"w_up": torch.zeros(6, 4).half()}, "dtype"),
    ({"b_gate": torch.zeros(6)}, "both biases"),
    ({"b_up": torch.zeros(6)}, "both biases"),
    ({"b_gate": torch.zeros(5), "b_up": torch.zeros(6)}, "biases of"),
    ({"b_gate": torch.zeros(6), "b_up": torch.zeros(6).half()}, "dtype"),
    ({"x": torch.zeros(2, 0), "w_gate": torch.zeros(6, 0), "w_up": torch.zeros(6, 0)}, "empty"),
    ({"activation": "relu"}, "unknown activation"),
    ({"activation": None}, "unknown activation"),
])
def test_gated_linear_refuses(native_lib, change, error):
    args = {"x": torch.zeros(2, 4), "w_gate": torch.zeros(6, 4), "w_up": torch.zeros(6, 4), **change}
    with pytest.raises((ValueError, TypeError), match=error):
        ops.gated_linear(**args)


# ------------------------------------------------------------------------- group norm
ACTS = {None: lambda v: v, "relu": torch.relu, "silu": torch.nn.functional.silu,
        "gelu": torch.nn.functional.gelu,
        "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}


def check_norm(x, groups, weight, bias, eps, act, residual, dy, call=ops.group_norm):
    """Forward and every gradient of one call against 64 bits."""
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, residual, weight, bias)]
    y = call(leaves[0], groups, leaves[2], leaves[3], eps=eps, activation=act, residual=leaves[1])
    given = [t for t in leaves if t is not None]
    grads = dict(zip([i for i, t in enumerate(leaves) if t is not None], torch.autograd.grad(y, given, dy)))

    n, c = x.shape[:2]
    per = (1, c) + (1,) * (x.dim() - 2)
    x64 = x.double()
    r64 = torch.zeros_like(x64) if residual is None else residual.double()
    w = torch.ones(per, device=x.device).double() if weight is None else weight.double().view(per)
    b = torch.zeros(per, device=x.device).double() if bias is None else bias.double().view(per)
    grouped = x64.reshape(n, groups, -1)
    mean = grouped.mean(2, keepdim=True)
    rstd = (grouped.var(2, unbiased=False, keepdim=True) + eps).rsqrt()

    def over(t):  # group means, back over the group
        return t.reshape(n, groups, -1).mean(2, keepdim=True).expand_as(grouped).reshape(x.shape)

    xh = ((grouped - mean) * rstd).reshape(x.shape)
    rs, mn = (t.expand_as(grouped).reshape(x.shape) for t in (rstd, mean))
    z = (xh * w + b + r64).requires_grad_()
    want = ACTS[act](z)
    dz, = torch.autograd.grad(want, z, dy.double())
    size = (x64.abs() + mn.abs()) * rs * w.abs() + b.abs() + r64.abs()
    # six roundings up to z, then the activation: at most four steps, slope below 1.13
    assert y.dtype == x.dtype and (y.dim() < 3 or y.movedim(1, -1).is_contiguous())
    within(y, want.detach(), 16 * U * size)

    # the derivatives change by at most 1.2 times the error of z, and cost a few steps themselves
    dd = dy.double().abs() * (16 * U * (1 + 2 * size) if act in ("silu", "gelu") else 4 * U)
    dxh, xa = dz * w, xh.abs() + 4 * U * (x64.abs() + mn.abs()) * rs
    dx = rs * (dxh - over(dxh) - xh * over(dxh * xh))
    # sums of a group: terms in 32 bits, at most 64 additions of them before 64 bits take over
    s1, s2 = over(dxh.abs()), over((dxh * xh).abs())
    e1, e2 = over(dd * w.abs()) + 72 * U * s1, over(dd * w.abs() * xa) + 72 * U * s2
    xe = 4 * U * (x64.abs() + mn.abs()) * rs
    e2 = e2 + over(dxh.abs() * xe)
    tol = rs * (dd * w.abs() + e1 + xa * e2 + xe * s2 + 16 * U * (dxh.abs() + s1 + xa * s2))
    within(grads[0], dx, tol)
    if residual is not None:
        within(grads[1], dz, dd)
    dims = [i for i in range(x.dim()) if i != 1]
    if weight is not None:
        within(grads[2], (dz * xh).sum(dims), (dd * xa + dz.abs() * xe + 72 * U * (dz * xh).abs()).sum(dims))
    if bias is not None:
        within(grads[3], dz.sum(dims), (dd + 72 * U * dz.abs()).sum(dims))


NORM_SHAPES = [
    ((1, 2048, 7, 7), 32), ((3, 90, 13, 9), 30), ((2, 64, 56, 56), 32), ((5, 30, 11), 1), ((4, 96), 8),
    ((2, 7, 3, 5), 7), ((1, 32, 1, 17), 32), ((2, 40, 3, 4, 5), 8), ((70, 16, 3, 3), 4), ((1, 8, 301, 307), 2),
    ((3, 258, 5, 5), 6), ((2, 1024, 2, 2), 16), ((1, 4160, 4, 4), 32), ((2, 512, 40, 40), 32), ((9, 3, 8, 8), 1),
]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,groups", NORM_SHAPES)
def test_group_norm_shapes(shape, groups, dtype):
    act = [None, "relu", "silu", "gelu"][(shape[0] + shape[1] + groups) % 4]
    c = shape[1]
    x = channels_last(shape, 1, dtype, 1.5, 0.5)
    res = channels_last(shape, 2, dtype) if (shape[-1] + groups) % 2 else None
    dy = channels_last(shape, 3, dtype)
    check_norm(x, groups, rand(c, 4, shift=1.0, scale=0.3), rand(c, 5), 1e-5, act, res, dy)


@gpu
@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("weight_dtype", [None, F32, BF16, F16])
def test_group_norm_forms(act, residual, weight_dtype):
    shape, dtype = (3, 48, 19, 6), BF16 if weight_dtype != F16 else F16
    x, dy = channels_last(shape, 1, dtype), channels_last(shape, 2, dtype)
    w, b = (None, None) if weight_dtype is None else (rand(48, 3, weight_dtype), rand(48, 4, weight_dtype))
    res = channels_last(shape, 5, dtype) if residual else None
    check_norm(x, 12, w, b, 1e-5, act, res, dy)
    if w is not None:
        check_norm(x, 12, w, None, 1e-3, act, res, dy)
        check_norm(x, 12, None, b, 0.1, act, res, dy)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_group_norm_layouts(dtype):
    shape, w, b = (3, 24, 10, 7), rand(24, 4), rand(24, 5)
    dense = rand(shape, 1, dtype)                                       # channels first: copied
    wide = channels_last((3, 72, 10, 7), 2, dtype)[:, 24:48]            # rows further apart
    odd = channels_last((3, 73, 10, 7), 2, dtype)[:, 1:25]              # and at odd addresses
    inner = channels_last((3, 24, 12, 9), 3, dtype)[:, :, 1:11, 1:8]    # rows of two strides: copied
    skip = channels_last((6, 24, 10, 7), 6, dtype)[::2]                 # every other image
    turned = rand((3, 24, 70), 7, dtype).view(shape).transpose(2, 3).contiguous().transpose(2, 3)
    grads = [rand(shape, 8, dtype), channels_last((3, 25, 10, 7), 9, dtype)[:, 1:],
             torch.ones((), dtype=dtype, device=cuda).expand(shape)]
    for i, x in enumerate((dense, wide, odd, inner, skip, turned)):
        res = (wide, dense, None)[i % 3]
        check_norm(x, 6, w, b, 1e-5, (None, "silu", "relu")[i % 3], res, grads[i % 3])


@gpu
@pytest.mark.parametrize("shape", [(3, 24, 10, 7), (1, 8, 201, 307)])  # clusters; two launches
def test_group_norm_gradients_that_nobody_wants(shape):
    x, res, dy = (channels_last(shape, s, BF16) for s in (1, 2, 3))
    args = [x, res, rand(shape[1], 4), rand(shape[1], 5)]

    def call(*a):
        return ops.group_norm(a[0], 4, a[2], a[3], activation="silu", residual=a[1])

    leaves = [t.clone().requires_grad_() for t in args]
    full = torch.autograd.grad(call(*leaves), leaves, dy)
    for i in range(4):
        some = [t.clone().requires_grad_(j == i) for j, t in enumerate(args)]
        g, = torch.autograd.grad(call(*some), some[i], dy)
        assert torch.equal(g, full[i])
    with torch.no_grad():
        assert torch.equal(call(*leaves), call(*args))


@gpu
@pytest.mark.parametrize("channels,groups", [(5000, 1), (1600, 1600), (8192, 2)])
def test_group_norm_wide_and_narrow_groups(channels, groups):
    shape = (2, channels, 3, 5)
    x, dy = channels_last(shape, 1, F32), channels_last(shape, 2, F32)
    check_norm(x, groups, rand(channels, 3), rand(channels, 4), 1e-2, "silu", None, dy)


@gpu
def test_group_norm_refuses_the_widest_groups():
    with pytest.raises(ValueError, match="8192 channels"):
        ops.group_norm(torch.zeros(1, 8200, 2, 2, device=cuda), 1)


@gpu
@pytest.mark.parametrize("shape", [(0, 8, 3, 3), (2, 8, 0, 3), (0, 8)])
def test_group_norm_of_nothing(shape):
    x = torch.empty(shape, device=cuda, requires_grad=True)
    w, b = (torch.ones(8, device=cuda, requires_grad=True) for _ in range(2))
    y = ops.group_norm(x, 2, w, b, activation="silu")
    assert y.shape == x.shape
    dx, dw, db = torch.autograd.grad(y.sum(), (x, w, b))
    assert dx.shape == x.shape and not dw.any() and not db.any()


@gpu
def test_group_norm_far_from_zero_and_constant():
    # a group of one value everywhere: no deviation, the bias is what is left
    x = torch.full((2, 8, 5, 5), 3.0, device=cuda, dtype=BF16)
    b = rand(8, 1)
    y = ops.group_norm(x, 2, rand(8, 2), b)
    assert torch.equal(y, b.to(BF16).view(1, 8, 1, 1).expand_as(y))
    # values 1000 times as far from zero as from each other
    x, dy = channels_last((2, 64, 21, 21), 3, F32, 1.0, 1000.0), channels_last((2, 64, 21, 21), 4, F32)
    check_norm(x, 8, rand(64, 5), rand(64, 6), 1e-5, "gelu", None, dy)


@gpu
def test_group_norm_infinities_stay_in_their_group():
    x = channels_last((2, 16, 6, 6), 1, BF16)
    y0 = ops.group_norm(x, 4)
    x[1, 5, 2, 3] = math.inf
    y = ops.group_norm(x, 4)
    assert y[1, 4:8].isnan().any()
    y[1, 4:8] = y0[1, 4:8]
    assert torch.equal(y, y0)


# ------------------------------------------------------------------------- distillation loss
def plain_distill(z, top, index, labels, t, alpha, ignore):
    """Loss of each row, its weight (1 or 0) and the gradient of each row's loss, in 64 bits, with the
    size of the terms that were summed."""
    z = z.double()
    rows, classes = z.shape
    there = (index >= 0) & (index < classes)
    at = index.long().clamp(0, classes - 1)
    v = torch.where(there, top.double() / t, -math.inf)
    some = (v != -math.inf).any(1) if v.shape[1] else torch.zeros(rows, dtype=torch.bool, device=z.device)
    logp = torch.where(some[:, None], v - torch.logsumexp(torch.where(some[:, None], v, 0.0), 1, keepdim=True), -math.inf)
    p = logp.exp()
    q = torch.log_softmax(z / t, 1)
    term = torch.where(p > 0, p * (logp - q.gather(1, at)), 0.0)
    size = torch.where(p > 0, p * (logp.abs() + (z / t).gather(1, at).abs() + torch.logsumexp(z / t, 1, keepdim=True).abs()), 0.0)
    a, b = (alpha, 1 - alpha) if labels is not None else (0.0, 1.0)
    loss, size = b * t * t * term.sum(1), b * t * t * size.sum(1)
    pt = torch.zeros_like(z).scatter_add_(1, at, p)
    grad = b * t * (q.exp() * some[:, None] - pt)
    gsize = b * t * (q.exp() + pt)
    counts = some
    if labels is not None:
        counts = (labels >= 0) & (labels < classes) & (labels != ignore)
        y = labels.long().clamp(0, classes - 1)[:, None]
        lp = torch.log_softmax(z, 1)
        loss = loss - a * lp.gather(1, y)[:, 0]
        size = size + a * (z.gather(1, y)[:, 0].abs() + torch.logsumexp(z, 1).abs())
        one = torch.zeros_like(z).scatter_(1, y, 1.0)
        grad = grad + a * (lp.exp() - one)
        gsize = gsize + a * (lp.exp() + one)
    c = counts.double()
    return (torch.where(counts, loss, 0.0), c, torch.where(counts[:, None], grad, 0.0),
            torch.where(counts, size, 0.0), torch.where(counts[:, None], gsize, 0.0))


def check_distill(z, top, index, labels=None, t=1.0, alpha=0.5, ignore=-100):
    classes, k = z.shape[-1], top.shape[-1]
    rows = z.numel() // classes
    flat = (z.reshape(rows, classes), top.reshape(rows, k), index.reshape(rows, k),
            None if labels is None else labels.reshape(rows))
    loss, c, grad, size, gsize = plain_distill(*flat, t, alpha, ignore)
    # sums of the exponentials: a thread adds at most classes / 128 of them, then a tree; an
    # exponential is off by two steps and what its argument is: z / t and the logarithm
    reach = float((flat[0].double()[flat[0].double().abs() < 1e30].abs().max() / min(t, 1.0)).cpu()) if z.numel() else 0.0
    e = (classes / 128 + 64 + 8 * reach) * U
    weight = (1 - alpha + alpha if labels is not None else 1.0) * (t * t if labels is None else max(1.0, t * t))
    for reduction in ("none", "sum", "mean"):
        x = z.detach().requires_grad_()
        got = ops.distill_loss(x, top, index, labels, temperature=t, alpha=alpha, ignore_index=ignore, reduction=reduction)
        assert got.dtype == F32
        row_tol = 8 * U * size + e * weight * c
        if reduction == "none":
            up = rand(z.shape[:-1], 77)
            within(got.reshape(rows), loss, row_tol)
            each = up.reshape(rows).double()
        else:
            many = max(1.0, float(c.sum())) if reduction == "mean" else 1.0
            within(got, loss.sum() / many, (row_tol.sum() + 4 * U * loss.abs().sum()) / many)
            up = torch.tensor(0.75, device=cuda)
            each = up.double().expand(len(c)) / many
        dz, = torch.autograd.grad(got, x, up)
        assert dz.dtype == z.dtype and dz.shape == z.shape
        # (16-bit gradients of 32-bit products may be rounded twice)
        want = grad * each[:, None]
        within(dz.reshape(rows, classes), want, gsize * each.abs()[:, None] * (e + 16 * U) + half(dz.dtype) * want.abs() * (dz.dtype == BF16))


def teacher(z, k, seed, dtype):
    top = torch.topk(z.float() + rand(z.shape, seed), k, dim=-1)
    return top.values.to(dtype), top.indices


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,classes,k", [
    (1, 1, 1), (3, 7, 7), (1, 50257, 20), (5, 1000, 5), (33, 513, 1), (2, 30522, 64), (300, 129, 12), (1, 200003, 128),
    (4, 65536, 3), (150, 4099, 0),
])
def test_distill_loss_sizes(rows, classes, k, dtype):
    z = rand((rows, classes), rows + classes, dtype, 2.0)
    top, index = teacher(z, k, 3, dtype)
    check_distill(z, top, index)
    labels = torch.randint(0, classes, (rows,), device=cuda, generator=torch.Generator(device=cuda).manual_seed(4))
    check_distill(z, top, index.int(), labels, t=2.0, alpha=0.3)


@gpu
@pytest.mark.parametrize("t,alpha", [(0.5, 0.0), (1.0, 1.0), (4.0, 0.9), (20.0, 0.5)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_distill_loss_weights(t, alpha, dtype):
    z = rand((6, 777), 1, dtype, 3.0)
    top, index = teacher(z, 9, 2, F32)
    labels = torch.tensor([0, 776, -100, 5, 700, 3], device=cuda, dtype=torch.int32)
    check_distill(z, top, index, labels, t, alpha)
    check_distill(z, top, index, None, t, alpha)
    check_distill(z, top, index, labels, t, alpha, ignore=5)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_distill_loss_rows_without_entries(dtype):
    z = rand((7, 40), 1, dtype)
    top, index = teacher(z, 4, 2, dtype)
    index[0] = -1                  # none
    index[1, 2:] = -1              # two
    index[2, 0] = 40               # one past the end
    index[3, 1] = index[3, 0]      # the same class twice
    top[4] = -math.inf             # none with any weight
    top[5, 1] = -math.inf          # one without
    index[6] = torch.tensor([1 << 40, -(1 << 40), 0, 39], device=cuda)
    check_distill(z, top, index)
    check_distill(z, top, index, torch.tensor([3, -100, 0, 39, 7, -1, 40], device=cuda), 2.0, 0.4)
    nothing = torch.full((7,), -100, device=cuda)
    check_distill(z, top, index, nothing)
    check_distill(z, top, torch.full_like(index, -1))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_distill_loss_masked_classes(dtype):
    z = rand((4, 300), 1, dtype)
    top, index = teacher(z, 6, 2, dtype)
    labels = index[:, 0].clone()
    masked = torch.ones(300, dtype=torch.bool, device=cuda)
    masked[index.flatten()] = False
    z[0, masked] = -math.inf
    z[1, masked] = torch.finfo(dtype).min
    z[2, masked & (torch.arange(300, device=cuda) < 290)] = -math.inf
    check_distill(z, top, index, labels, 2.0, 0.5)
    check_distill(z, top, index, None, 1.0)
    # a class that the teacher wants and the mask forbids costs infinitely much
    z[3, index[3, 1]] = -math.inf
    got = ops.distill_loss(z, top, index, reduction="none")
    assert got[3] == math.inf and got[:3].isfinite().all()
    # NaN stays in its row
    z[0, 0] = math.nan
    x = z.detach().requires_grad_()
    got = ops.distill_loss(x, top, index, reduction="none")
    dz, = torch.autograd.grad(got, x, torch.ones_like(got))
    assert got[0].isnan() and got[1:3].isfinite().all() and dz[1:3].isfinite().all()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_distill_loss_layouts(dtype):
    wide = rand((2, 9, 210), 1, dtype)
    top, index = teacher(wide[..., :201], 8, 2, dtype)
    labels = torch.randint(0, 201, (2, 9), device=cuda)
    check_distill(wide[..., :201], top, index, labels)                                # rows further apart
    check_distill(wide[..., 1:202], top[..., ::2], index[..., ::2], labels)           # at odd addresses
    check_distill(rand((9, 2, 201), 3, dtype).transpose(0, 1), top, index, labels)    # rows in another order
    check_distill(rand((2, 201, 9), 4, dtype).transpose(1, 2), top, index, labels)    # classes apart: copied
    check_distill(wide[0, 0, :201], top[0, 0], index[0, 0], labels[0, 0])             # one row, no leading dimension
    check_distill(wide[:, :1, :201].expand(2, 9, 201), top, index, labels)            # one row many times


@gpu
def test_distill_loss_of_nothing():
    z = torch.zeros(0, 11, device=cuda, requires_grad=True)
    top, index = torch.zeros(0, 3, device=cuda), torch.zeros(0, 3, dtype=torch.long, device=cuda)
    for reduction in ("mean", "sum", "none"):
        loss = ops.distill_loss(z, top, index, reduction=reduction)
        assert loss.shape == (torch.Size([0]) if reduction == "none" else torch.Size([])) and not loss.any()
        g, = torch.autograd.grad(loss.sum(), z)
        assert g.shape == z.shape


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_distill_loss_gradient_of_a_graph_used_twice(dtype):
    z = rand((17, 3001), 1, dtype).requires_grad_()
    top, index = teacher(z.detach(), 10, 2, dtype)
    loss = ops.distill_loss(z, top, index, torch.arange(17, device=cuda))
    g1, = torch.autograd.grad(loss, z, torch.tensor(1.0, device=cuda), retain_graph=True)
    kept = g1.clone()
    g3, = torch.autograd.grad(loss, z, torch.tensor(4.0, device=cuda), retain_graph=True)
    assert torch.equal(g1, kept) and torch.equal(g3, 4 * g1)
    g1.fill_(7)
    again, = torch.autograd.grad(loss, z)
    assert torch.equal(again, kept)


@gpu
def test_distill_loss_small_f16_gradients_survive_a_loss_scale():
    # 1 / (rows * classes) is below the smallest 16-bit number; times the scale it is not
    z = torch.zeros(500, 2000, device=cuda, dtype=F16, requires_grad=True)
    top, index = torch.zeros(500, 1, device=cuda), torch.zeros(500, 1, dtype=torch.long, device=cuda)
    loss = ops.distill_loss(z, top, index)
    g, = torch.autograd.grad(loss * 65536.0, z)
    want = torch.full((500, 1999), 65536.0 / 500 / 2000, device=cuda, dtype=torch.float64)
    within(g[:, 1:], want, 256 * U * want)


# ------------------------------------------------------------------------- gated projection
def check_gated(x, wg, wu, bg, bu, act, dh, call=ops.gated_linear):
    dt = x.dtype
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, wg, wu, bg, bu)]
    h = call(*leaves, activation=act)
    given = [t for t in leaves if t is not None]
    grads = torch.autograd.grad(h, given, dh)

    X, G, W = x.double().reshape(-1, x.shape[-1]), wg.double(), wu.double()
    BG, BU = (torch.zeros(len(wg), device=cuda).double() if b is None else b.double() for b in (bg, bu))
    D = dh.double().reshape(len(X), len(wg))
    g = (X @ G.t() + BG).requires_grad_()
    u = X @ W.t() + BU
    a = ACTS[act](g)
    da, = torch.autograd.grad(a.sum(), g)
    g, a = g.detach(), a.detach()
    # a product of K terms summed in 32 bits, each addition off by at most a whole step
    step, k = 2 * U, X.shape[1]
    eg = (k + 16) * step * (X.abs() @ G.abs().t() + BG.abs())
    eu = (k + 16) * step * (X.abs() @ W.abs().t() + BU.abs())
    ea = 1.13 * eg + 16 * U * (g.abs() + a.abs())
    eda = 1.2 * eg + 32 * U * (1 + g.abs())
    assert h.dtype == dt and h.shape == (*x.shape[:-1], len(wg))
    within(h.reshape(g.shape), a * u, ea * (u.abs() + eu) + a.abs() * eu + 4 * U * (a * u).abs())
    # dg and du are rounded to the type that the matrix instructions take, the saved g and u to 24 bits
    dg, du = D * u * da, D * a
    sg, su = 2.0 ** -16 * (g.abs() + eg), 2.0 ** -16 * (u.abs() + eu)
    if dt == F32:
        sg, su = 0 * sg, 0 * su
    r = half(dt) + 8 * U
    edg = D.abs() * ((u.abs() + eu + su) * (eda + 1.2 * sg) + (eu + su) * da.abs())
    edu = D.abs() * (ea + 1.13 * sg)
    edg, edu = edg + r * (dg.abs() + edg) + least(dt), edu + r * (du.abs() + edu) + least(dt)
    f, m = g.shape[1], g.shape[0]
    dx = dg @ G + du @ W
    sx = (dg.abs() + edg) @ G.abs() + (du.abs() + edu) @ W.abs()
    want = [(dx, edg @ G.abs() + edu @ W.abs() + (2 * f + 16) * step * sx)]
    for d, e in ((dg, edg), (du, edu)):
        want.append((d.t() @ X, e.t() @ X.abs() + (m + 16) * step * ((d.abs() + e).t() @ X.abs())))
    if bg is not None:
        for d, e in ((dg, edg), (du, edu)):
            want.append((d.sum(0), e.sum(0) + (m + 16) * U * (d.abs() + e).sum(0)))
    for got, (exact, tol) in zip(grads, want):
        within(got.reshape(exact.shape), exact, tol)
        if exact.norm() > 0:
            # errors of a sum's terms are of either sign: together they grow with its root.  Two roundings of
            # the terms and one of the result in 16 bits; in 32, sqrt(terms) of the steps
            rel = float((got.double().reshape(exact.shape) - exact).norm() / exact.norm())
            size = float(sx.norm() / dx.norm()) if exact is dx else 1.0
            terms = max(2 * f, m, k)
            if dt == F32 and exact.numel() > 100:
                assert rel < 16 * U * math.sqrt(terms) * max(1.0, size), rel


def gated_inputs(tokens, hidden, ffn, dtype, bias, seed=1):
    x, dh = rand((tokens, hidden), seed, dtype), rand((tokens, ffn), seed + 1, dtype)
    wg, wu = (rand((ffn, hidden), seed + 2 + i, dtype, hidden ** -0.5) for i in range(2))
    bg, bu = (rand((ffn,), seed + 4 + i, dtype, 0.3) if bias else None for i in range(2))
    return x, wg, wu, bg, bu, dh


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,hidden,ffn", [
    (1, 1, 1), (1, 768, 2048), (2, 64, 64), (3, 100, 7), (7, 257, 130), (8, 128, 384), (9, 72, 200), (16, 40, 513),
    (17, 1000, 96), (63, 33, 65), (64, 64, 128), (65, 136, 127), (128, 256, 256), (129, 72, 300), (300, 520, 264),
    (517, 200, 1111), (1024, 384, 512), (2, 4096, 33), (257, 8, 8),
])
def test_gated_linear_sizes(tokens, hidden, ffn, dtype):
    act = ["gelu", "gelu_tanh", "silu"][(tokens + ffn) % 3]
    *ins, dh = gated_inputs(tokens, hidden, ffn, dtype, bias=hidden % 3 != 1)
    check_gated(*ins, act, dh)


@gpu
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("tokens", [1, 5, 77])
def test_gated_linear_activations_over_their_range(act, tokens):
    x = torch.linspace(-30, 30, tokens * 16, device=cuda).view(tokens, 16)
    eye = torch.eye(16, device=cuda)
    for dtype in TYPES:
        dh = rand((tokens, 16), 3, dtype)
        check_gated(x.to(dtype), eye.to(dtype), 2 * eye.to(dtype), None, None, act, dh)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [2, 6, 150])
def test_gated_linear_layouts(dtype, tokens):
    x, wg, wu, bg, bu, dh = gated_inputs(2 * tokens, 88, 56, dtype, True)
    fused = torch.cat([wg, wu])
    check_gated(x, fused[:56], fused[56:], bg, bu, "silu", dh)                          # halves of one weight
    check_gated(x.view(2, tokens, 88), wg, wu, bg, bu, "gelu", dh.view(2, tokens, 56))   # leading dimensions
    wide, tall = rand((2 * tokens, 200), 7, dtype), rand((56, 300), 8, dtype, 0.1)
    check_gated(wide[:, 8:96], tall[:, 16:104], wu, bg, bu, "silu", dh)                 # rows further apart
    check_gated(wide[:, 3:91], tall[:, 1:89], tall[:, 5:93], None, None, "silu", dh)    # at odd addresses
    check_gated(wide.t().contiguous().t()[:, :88], wg.t().contiguous().t(), wu, bg, bu, "gelu", dh)
    check_gated(x, wg, wu, bg, bu, "gelu", torch.ones((), dtype=dtype, device=cuda).expand(dh.shape))
    check_gated(x, wg, wu, bg, bu, "gelu", rand((2 * tokens, 61), 9, dtype)[:, 2:58])
    check_gated(x, wg, wg, bg, bg, "gelu", dh)                                          # one weight twice
    check_gated(x[:1].expand(4, 88), wg, wu, bg, bu, "gelu", dh[:4])                    # one token four times


@gpu
def test_gated_linear_of_nothing():
    x = torch.empty(2, 0, 24, device=cuda, dtype=BF16, requires_grad=True)
    wg, wu = (torch.ones(40, 24, device=cuda, dtype=BF16, requires_grad=True) for _ in range(2))
    h = ops.gated_linear(x, wg, wu)
    assert h.shape == (2, 0, 40)
    dx, dwg, dwu = torch.autograd.grad(h.sum(), (x, wg, wu))
    assert dx.shape == x.shape and not dwg.any() and not dwu.any()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [4, 200])
def test_gated_linear_gradients_that_nobody_wants(dtype, tokens):
    x, wg, wu, bg, bu, dh = gated_inputs(tokens, 64, 72, dtype, True)
    all_of = [t.clone().requires_grad_() for t in (x, wg, wu, bg, bu)]
    full = torch.autograd.grad(ops.gated_linear(*all_of), all_of, dh)
    for i in range(5):
        some = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, wg, wu, bg, bu))]
        g, = torch.autograd.grad(ops.gated_linear(*some), some[i], dh)
        assert torch.equal(g, full[i])
    with torch.no_grad():
        assert torch.equal(ops.gated_linear(*all_of), ops.gated_linear(x, wg, wu, bg, bu))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [3, 140])
def test_gated_linear_infinities_stay_in_their_rows(dtype, tokens):
    x, wg, wu, bg, bu, _ = gated_inputs(tokens, 96, 80, dtype, True)
    h0 = ops.gated_linear(x, wg, wu, bg, bu)
    x[1, 7], x[2, 5] = math.inf, math.nan
    h = ops.gated_linear(x, wg, wu, bg, bu)
    assert not h[1].isfinite().all() and h[2].isnan().all()
    h[1:3] = h0[1:3]
    assert torch.equal(h, h0)


@gpu
def test_gated_linear_large_and_small_f32():
    # 24 bits of operands of any size count
    x, wg, wu, bg, bu, dh = gated_inputs(20, 64, 48, F32, True)
    check_gated(x * 2.0 ** 60, wg * 2.0 ** -60, wu * 2.0 ** -70, bg, bu, "silu", dh)
    check_gated(x * 2.0 ** -60, wg * 2.0 ** 61, wu * 2.0 ** 58, bg, bu, "silu", dh)


# ------------------------------------------------------------------------- differences
@gpu
def test_gradients_against_differences():
    """Central differences of the f32 operators themselves, along random directions: h = 2^-8, so the
    formula is off by h^2 / 6 of third derivatives (below 2 in size here) and by what 32 bits lose over 2h."""
    def slope(f, leaves, seed):
        out = f(*leaves)
        up = rand(out.shape, seed)
        grads = torch.autograd.grad(out, leaves, up)
        for i, t in enumerate(leaves):
            d = rand(t.shape, seed + 1 + i)
            d = d / d.norm()
            with torch.no_grad():
                moved = [f(*[v + s * d if j == i else v for j, v in enumerate(leaves)]) for s in (2.0 ** -8, -(2.0 ** -8))]
            diff = float(((moved[0].double() - moved[1].double()) * up.double()).sum() / 2 ** -7)
            want = float((grads[i].double() * d.double()).sum())
            size = float(out.double().norm() * up.double().norm())
            assert abs(diff - want) <= 4 * 2.0 ** -16 * size + 64 * U * size / 2 ** -7, (i, diff, want)

    w, b = rand(12, 1, shift=1.0).requires_grad_(), rand(12, 2).requires_grad_()
    x, r = (channels_last((2, 12, 5, 4), s, F32).requires_grad_() for s in (3, 4))
    for act in (None, "silu", "gelu"):
        slope(lambda x, r, w, b: ops.group_norm(x, 3, w, b, activation=act, residual=r), [x, r, w, b], 5)
    ins = [t.requires_grad_() for t in gated_inputs(11, 24, 18, F32, True)[:5]]
    for act in ("gelu", "gelu_tanh", "silu"):
        slope(lambda *a: ops.gated_linear(*a, activation=act), ins, 9)
    z = rand((4, 50), 6).requires_grad_()
    top, index = teacher(z.detach(), 5, 7, F32)
    slope(lambda z: ops.distill_loss(z, top, index, torch.arange(4, device=cuda), 2.0, 0.4, reduction="none"), [z], 11)


# ------------------------------------------------------------------------- streams, graphs, together
def a_step(seed, dtype=BF16):
    """The three in a row, as a small student has them; (function of the leaves, leaves)."""
    n, c, hw, ffn, classes = 6, 32, 9, 88, 151
    x = channels_last((n, c, hw, hw), seed, dtype).requires_grad_()
    w, b = rand(c, seed + 1, shift=1.0).requires_grad_(), rand(c, seed + 2).requires_grad_()
    wg, wu = (rand((ffn, c), seed + 3 + i, dtype, c ** -0.5).requires_grad_() for i in range(2))
    out = rand((classes, ffn), seed + 5, dtype, ffn ** -0.5).requires_grad_()
    top, index = torch.topk(rand((n * hw * hw, classes), seed + 6), 7)
    labels = torch.arange(n * hw * hw, device=cuda) % classes
    labels[::5] = -100

    def step(x, w, b, wg, wu, out):
        y = ops.group_norm(x, 8, w, b, activation="silu", residual=x)
        h = ops.gated_linear(y.permute(0, 2, 3, 1).reshape(-1, c), wg, wu)
        return ops.distill_loss(h @ out.t(), top, index, labels, 2.0, 0.5)
    return step, [x, w, b, wg, wu, out]


def run_step(step, leaves):
    loss = step(*leaves)
    return [loss.detach(), *torch.autograd.grad(loss, leaves)]


@gpu
def test_same_bits_again_and_on_another_stream():
    step, leaves = a_step(1)
    want = run_step(step, leaves)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    other, theirs = a_step(50)
    for _ in range(4):
        with torch.cuda.stream(side):  # two calls at once
            on_side = run_step(other, theirs)
        got = run_step(step, leaves)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        with torch.cuda.stream(side):
            got = run_step(step, leaves)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    here = run_step(other, theirs)
    assert all(torch.equal(a, b) for a, b in zip(on_side, here))


@gpu
def test_captured_and_replayed_with_new_inputs():
    step, leaves = a_step(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager_loss = step(*leaves)  # an eager graph of the same leaves that lives on
        run_step(step, leaves)
        graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
        outs = []
        for g in graphs:
            with torch.cuda.graph(g, stream=side):
                outs.append(run_step(step, leaves))
    torch.cuda.current_stream().wait_stream(side)
    for seed in (1, 20, 30):
        _, fresh = a_step(seed)
        with torch.no_grad():
            for t, f in zip(leaves, fresh):
                t.copy_(f)
        want = run_step(step, leaves)
        for g, out in zip(graphs, outs):
            g.replay()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    del eager_loss


@gpu
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_on_another_gpu_than_the_current_one():
    step, leaves = a_step(1)
    want = run_step(step, leaves)
    there = [t.detach().to("cuda:1").requires_grad_() for t in leaves[:3]]
    torch.cuda.set_device(0)
    y = ops.group_norm(*there[:1], 8, *there[1:], activation="silu", residual=there[0])
    assert y.device.index == 1 and torch.cuda.current_device() == 0
    assert torch.equal(y.to(cuda), ops.group_norm(leaves[0], 8, *leaves[1:3], activation="silu", residual=leaves[0]))
    assert len(want) == 7


@gpu
def test_calls_from_several_threads():
    """Each on a stream of its own, with sizes of its own."""
    import threading
    jobs = [a_step(10 * i, dtype) for i, dtype in enumerate((BF16, F32, F16, BF16))]
    want = [run_step(*job) for job in jobs]
    torch.cuda.synchronize()
    got, errors = [None] * len(jobs), []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got[i] = run_step(*jobs[i])
                    ops.group_norm(torch.randn(1, 64 * (i + 1), 9, 9, device=cuda), 2 ** i)
            torch.cuda.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))


@gpu
def test_second_derivatives_are_refused():
    step, leaves = a_step(1)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(step(*leaves), leaves, create_graph=True)
    x, w = leaves[0], leaves[1]
    for out in (ops.group_norm(x, 8, w), ops.gated_linear(x.movedim(1, -1), *leaves[3:5])):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(out.sum(), x, create_graph=True)
