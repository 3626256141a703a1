"""The operators of ops.train at inputs, sizes and uses where they can go wrong that test_train_ops.py does not reach: values far
from the others, long sums, derivatives that they do not have, hooks, captures, waits that run out.  Bounds as there."""
import ctypes

import pytest
import torch
from test_train_ops import (ACTS, BF16, F16, F32, U, channels_last, check_distill, check_gated, check_norm, cuda, gated_inputs, gpu,
                            plain_distill, rand, within)

from stdml_collective_experimental_b200 import ops


# ------------------------------------------------------------------------- group norm: statistics
@gpu
@pytest.mark.parametrize("mean,spread", [(100.0, 1.0), (1000.3, 0.1), (1000.7, 0.0), (-3.0, 1.0)])
@pytest.mark.parametrize("shape,groups", [((2, 8, 112, 112), 4), ((1, 32, 90, 77), 8), ((3, 512, 20, 20), 32), ((16, 8, 512, 512), 4)])
@pytest.mark.parametrize("place", ["corner", "border", "scattered"])
def test_group_norm_with_values_far_from_the_others(place, shape, groups, mean, spread):
    """A masked or padded position, in the first place of an image or of a slice above all, takes no bits from the rest."""
    x = channels_last(shape, 1, F32, spread, mean)
    if place == "corner":
        x[:, :, 0, 0] = 0
    elif place == "border":
        x[:, :, :, 0] = 0
    else:
        x.movedim(1, -1).view(shape[0], -1, shape[1])[:, ::257] = 0
    check_norm(x, groups, rand(shape[1], 2, shift=1.0, scale=0.3), rand(shape[1], 3), 1e-5, "silu", None, channels_last(shape, 4, F32))


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_group_norm_sums_over_many_positions(dtype):
    """Of one and the same value, whose roundings would all point the same way: 1024 positions to a thread."""
    shape = (10, 4, 1024, 1024)
    x = channels_last(shape, 1, dtype)
    dy = torch.full((shape[0], *shape[2:], shape[1]), 0.7, device=cuda, dtype=dtype).movedim(-1, 1)
    check_norm(x, 2, rand(4, 2, shift=1.0), rand(4, 3), 1e-5, None, None, dy)


# ------------------------------------------------------------------------- derivatives that they do not have
def calls():
    """Of each operator: (what it takes, the call), on whatever device the tensors get."""
    return [
        ([torch.ones(2, 4, 3), torch.ones(4), torch.ones(4), torch.ones(2, 4, 3)],
         lambda x, w, b, r: ops.group_norm(x, 2, w, b, residual=r)),
        ([torch.ones(3, 8), torch.ones(5, 8), torch.ones(5, 8), torch.ones(5), torch.ones(5)], ops.gated_linear),
        ([torch.ones(3, 8), torch.ones(3, 2)], lambda z, top: ops.distill_loss(z, top, torch.zeros(3, 2, dtype=torch.long, device=z.device))),
    ]


@pytest.mark.parametrize("which", range(3))
def test_tangents_are_refused(native_lib, which):
    from torch.autograd import forward_ad
    args, call = calls()[which]
    for i in range(len(args)):
        with forward_ad.dual_level(), torch.no_grad():
            dual = [forward_ad.make_dual(t, t) if j == i else t for j, t in enumerate(args)]
            with pytest.raises(ValueError, match="forward-mode"):
                call(*dual)
    with pytest.raises(ValueError, match="CUDA tensor expected"):
        call(*args)


# ------------------------------------------------------------------------- hooks on saved tensors
def on_gpu(which, dtype=F32):
    """The same calls on a GPU: (leaves, the call)."""
    if which == 0:
        return ([channels_last((2, 8, 5, 5), 1, dtype), rand(8, 2), rand(8, 3), channels_last((2, 8, 5, 5), 4, dtype)],
                lambda x, w, b, r: ops.group_norm(x, 2, w, b, activation="silu", residual=r))
    if which == 1:
        return [rand((9, 24), 1, dtype), rand((16, 24), 2, dtype), rand((16, 24), 3, dtype), rand(16, 4, dtype), rand(16, 5, dtype)], ops.gated_linear
    top, index = torch.topk(rand((9, 40), 2), 5)
    return [rand((9, 40), 1, dtype)], lambda z: ops.distill_loss(z, top, index, torch.arange(9, device=cuda), 2.0)


@gpu
@pytest.mark.parametrize("which", range(3))
def test_an_exception_of_a_hook_is_the_callers(which):
    class Mine(Exception):
        pass

    def pack(_):
        raise Mine("packed")

    args, call = on_gpu(which)
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t), pytest.raises(Mine, match="packed"):
        call(*[t.requires_grad_() for t in args])
    with torch.no_grad():
        call(*args)


@gpu
@pytest.mark.parametrize("which", range(3))
def test_checkpointed(which):
    """The second pass of a checkpoint stops with an exception out of the last operator that saves anything."""
    from torch.utils.checkpoint import checkpoint
    args, call = on_gpu(which)
    leaves = [t.requires_grad_() for t in args]
    want = torch.autograd.grad(call(*leaves).square().sum(), leaves)
    got = torch.autograd.grad(checkpoint(call, *leaves, use_reentrant=False).square().sum(), leaves)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------------- distillation: the gradient of the forward pass
@gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_distill_loss_backward_captured_apart_and_replayed_again(dtype):
    z = rand((17, 3001), 1, dtype).requires_grad_()
    top, index = torch.topk(z.detach().float(), 10)
    labels, up = torch.arange(17, device=cuda), torch.tensor(4.0, device=cuda)

    def loss_of():
        return ops.distill_loss(z, top, index, labels, 2.0)

    first, = torch.autograd.grad(loss_of(), z, up)
    forward, backward = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(forward):
        loss = loss_of()
    with torch.cuda.graph(backward, pool=forward.pool()):
        dz, = torch.autograd.grad(loss, z, up)
    for seed in (1, 5):
        with torch.no_grad():
            z.copy_(rand((17, 3001), seed, dtype))
        want, = torch.autograd.grad(loss_of(), z, up)
        forward.replay()
        for _ in range(3):  # (an accumulation step that asks again)
            backward.replay()
            assert torch.equal(dz, want)
    del first


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("up", [0.75, 1 / 3, 24.0, 1.0, -1.0, 0.0])
@pytest.mark.parametrize("rows,classes", [(17, 3001), (1500, 700), (3, 40000)])
def test_distill_loss_gradient_is_rounded_once(rows, classes, up, dtype):
    """Whatever the loss's own gradient is, the first backward pass over a graph gives the bits of the second, and those of the
    definition but for what 32 bits lose and half a step of the logits' type."""
    z = rand((rows, classes), 1, dtype, 2.0).requires_grad_()
    top, index = torch.topk(z.detach().float() + rand((rows, classes), 2), 9)
    labels = torch.arange(rows, device=cuda) % classes
    labels[::5] = -100
    loss = ops.distill_loss(z, top, index, labels, temperature=2.0, alpha=0.3)
    first, = torch.autograd.grad(loss, z, torch.tensor(up, device=cuda), retain_graph=True)
    second, = torch.autograd.grad(loss, z, torch.tensor(up, device=cuda))
    assert torch.equal(first, second)
    _, counts, grad, _, gsize = plain_distill(z.detach(), top, index, labels, 2.0, 0.3, -100)
    each = abs(float(torch.tensor(up))) / float(counts.sum())
    e = (classes / 128 + 64 + 8 * float(z.detach().abs().max())) * U  # (as check_distill)
    within(first, grad * (each if up >= 0 else -each), gsize * each * (e + 16 * U))


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("t", [1.0, 0.5])
@pytest.mark.parametrize("low", [-300.0, -60000.0])
def test_distill_loss_of_an_entry_without_weight_that_the_student_masks(low, t, dtype):
    """A teacher's entry far below its first weighs exp(-300) or less: nothing, and a student that forbids the class is not
    wrong."""
    z, top, index = rand((4, 200), 1, dtype), rand((4, 3), 2, dtype), torch.tensor([[5, 9, 30]], device=cuda).repeat(4, 1)
    top[1:, 1] = low
    z[1, 9] = -torch.inf
    z[2, 9] = torch.finfo(dtype).min
    check_distill(z, top, index, None, t)
    check_distill(z, top, index, torch.tensor([5, 30, 0, 199], device=cuda), t, 0.4)


@gpu
@pytest.mark.parametrize("t", [0.7, 1.0, 2.0, 3.0, 4.0])
@pytest.mark.parametrize("rows,classes", [(256, 1000), (300, 30522), (2, 50001)])
def test_distill_loss_in_f32_is_as_near_as_elementary_operations(rows, classes, t):
    """Neither takes more than a subtraction, a quotient, an exponential, a sum and a product of 32 bits, so that neither is further
    from 64 bits than the other but for chance, which over thousands of values is small."""
    z = rand((rows, classes), 1, F32, 2.0).requires_grad_()
    top, index = torch.topk(z.detach() + rand((rows, classes), 2), 5)
    labels = torch.arange(rows, device=cuda)
    dz, = torch.autograd.grad(ops.distill_loss(z, top, index, labels, t, 0.5, reduction="sum"), z)
    exact = plain_distill(z.detach(), top, index, labels, t, 0.5, -100)[2]
    with torch.no_grad():
        p = torch.exp(top / t - (top / t).amax(1, keepdim=True))
        plain = 0
        for scale, at, off, weight in ((1.0, labels[:, None], 1.0, 0.5), (t, index, p / p.sum(1, keepdim=True), 0.5 * t)):
            e = torch.exp(z / scale - (z / scale).amax(1, keepdim=True))
            plain = plain + weight * (e / e.sum(1, keepdim=True)).scatter_add_(1, at, torch.zeros_like(at, dtype=F32) - off)
    mine, theirs = (float((g.double() - exact).norm() / exact.norm()) for g in (dz, plain))
    assert mine <= 1.5 * theirs, (mine, theirs)


# ------------------------------------------------------------------------- the report of waits that ran out
@gpu
def test_check_waits_for_every_stream():
    args, call = on_gpu(1)
    with torch.no_grad():
        call(*args)  # (a kernel's first launch may wait by itself)
    ops.check()
    side, done = torch.cuda.Stream(), torch.cuda.Event()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        torch.cuda._sleep(1 << 30)  # (half a second of a kernel that waits for nobody)
        call(*args)
        done.record()
    ops.check()
    assert done.query()


def test_check_asks_the_gpu_that_is_meant(monkeypatch):
    from stdml_collective_experimental_b200.ops import train
    asked = []

    class Lib:
        @staticmethod
        def stdmlc_train_status(index, _):
            asked.append(index)
            return 0

    monkeypatch.setattr(train._native, "lib", lambda: Lib)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    for device in (None, "cuda", torch.device("cuda"), "cuda:0", torch.device("cuda", 1), 2):
        ops.check(device)
    assert asked == [3, 3, 3, 0, 1, 2]
    with pytest.raises(ValueError, match="CUDA device"):
        ops.check("cpu")


@gpu
@pytest.mark.parametrize("model", ["resnet50", "bert-base"])
def test_the_benchmark_asks_after_its_steps(monkeypatch, model):
    import argparse

    from stdml_collective_experimental_b200.benchmarks import resnet50_dp
    asked = []
    monkeypatch.setattr(resnet50_dp, "check", asked.append, raising=False)
    args = argparse.Namespace(model=model, batch=2, seq=8, steps=1, warmup=1, buckets=2, norm="group", ffn="gated", teacher=4)
    out = resnet50_dp.run_mode("local", args, None, 0, 1, cuda)
    assert asked == [cuda] and out["loss"] == out["loss"]


class GatedCall(ctypes.Structure):
    """stdmlc_gated of capi_train.h."""
    _fields_ = [("x", ctypes.c_void_p), ("x_row", ctypes.c_longlong), ("w_gate", ctypes.c_void_p), ("w_up", ctypes.c_void_p),
                ("w_gate_row", ctypes.c_longlong), ("w_up_row", ctypes.c_longlong), ("b_gate", ctypes.c_void_p),
                ("b_up", ctypes.c_void_p), ("h", ctypes.c_void_p), ("tokens", ctypes.c_longlong), ("hidden", ctypes.c_longlong),
                ("ffn", ctypes.c_longlong), ("dt", ctypes.c_int), ("act", ctypes.c_int), ("saved", ctypes.c_void_p),
                ("workspace", ctypes.c_void_p), ("dh", ctypes.c_void_p), ("dh_row", ctypes.c_longlong), ("dx", ctypes.c_void_p),
                ("dw_gate", ctypes.c_void_p), ("dw_up", ctypes.c_void_p), ("db_gate", ctypes.c_void_p), ("db_up", ctypes.c_void_p),
                ("wait_limit_ns", ctypes.c_longlong)]


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tokens,hidden,ffn", [(77, 64, 96), (300, 520, 264), (1024, 384, 512), (2100, 768, 2048)])
def test_gated_linear_reports_a_wait_that_may_not_last(native_lib, tokens, hidden, ffn, dtype):
    """Through the C ABI, whose callers may limit the waits: the kernel gives up with its first loads under way, says so, and the
    next call is whole."""
    from stdml_collective_experimental_b200 import _native
    lib = _native.lib()
    lib.stdmlc_gated_saved.restype = lib.stdmlc_gated_workspace.restype = ctypes.c_longlong
    x, wg, wu, _, _, dh = gated_inputs(tokens, hidden, ffn, dtype, False)
    leaves = [t.requires_grad_() for t in (x, wg, wu)]
    h = ops.gated_linear(*leaves)
    want = [h, *torch.autograd.grad(h, leaves, dh)]
    outs = [torch.zeros_like(t) for t in want]
    a = GatedCall(x=x.data_ptr(), x_row=hidden, w_gate=wg.data_ptr(), w_up=wu.data_ptr(), w_gate_row=hidden, w_up_row=hidden,
                  h=outs[0].data_ptr(), tokens=tokens, hidden=hidden, ffn=ffn, dt=8 if dtype == BF16 else 10, act=3, dh=dh.data_ptr(),
                  dh_row=ffn, dx=outs[1].data_ptr(), dw_gate=outs[2].data_ptr(), dw_up=outs[3].data_ptr())
    saved = torch.empty(lib.stdmlc_gated_saved(ctypes.byref(a)), dtype=torch.uint8, device=cuda)
    a.saved = saved.data_ptr()

    def run(backward, limit):
        work = torch.empty(lib.stdmlc_gated_workspace(ctypes.byref(a), backward), dtype=torch.uint8, device=cuda)
        a.workspace, a.wait_limit_ns = work.data_ptr(), limit
        f = lib.stdmlc_gated_backward if backward else lib.stdmlc_gated_forward
        _native.check(f(ctypes.byref(a), 0, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
        torch.cuda.synchronize()

    ops.check()
    for backward in (0, 1):
        run(backward, -1)
        assert not any(o.any() for o in (outs[1:] if backward else outs))
        with pytest.raises(_native.DeviceTimeoutError, match="ran out"):
            ops.check()
        ops.check()  # (once)
        run(backward, 1_000_000_000)
        run(backward, 0)
        ops.check()
        assert all(torch.equal(o, w) for o, w in zip(outs, want[:4 if backward else 1]))


# ------------------------------------------------------------------------- gelu left of zero
@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tokens", [4, 257])
def test_gelu_of_16_bits_is_near_where_it_is_small(tokens, dtype):
    """Relative to its own size, which vanishes like exp(-z^2 / 2): 2^-14 of it and half a step.  (5.2e-6 of the fit, three roundings
    of z^2 / 2 in an exponent of up to 104 powers of two, two quotients: 1.9e-5.)"""
    z = -torch.linspace(0, 12, 16 * tokens, device=cuda).to(dtype).view(tokens, 16)
    one, nothing = torch.ones(16, device=cuda, dtype=dtype), torch.zeros(16, 16, device=cuda, dtype=dtype)
    x = z.clone().requires_grad_()
    h = ops.gated_linear(x, torch.eye(16, device=cuda, dtype=dtype), nothing, 0 * one, one, activation="gelu")  # gelu(z) * 1
    z = z.double()
    phi, cdf = torch.exp(-0.5 * z * z) / (2 * torch.pi) ** 0.5, 0.5 * torch.special.erfc(-z / 2 ** 0.5)
    within(h, z * cdf, 2.0 ** -14 * (z * cdf).abs())
    dz, = torch.autograd.grad(h, x, torch.ones_like(h))
    within(dz, cdf + z * phi, 2.0 ** -14 * (cdf + z.abs() * phi))


# ------------------------------------------------------------------------- group norm: gradients that nobody wants
@gpu
def test_group_norm_walks_once_for_parameters_alone():
    """One large image is worked on in two launches, of which the second writes dx: for weight and bias the first is all."""
    from torch.profiler import ProfilerActivity, profile
    x, dy = (channels_last((1, 8, 201, 307), s, F32) for s in (1, 2))
    w, b = rand(8, 3, shift=1.0).requires_grad_(), rand(8, 4).requires_grad_()

    def launches(leaves):
        y = ops.group_norm(x, 4, w, b, activation="silu", residual=dy)
        torch.cuda.synchronize()
        with profile(activities=[ProfilerActivity.CUDA]) as p:
            torch.autograd.grad(y, leaves, dy)
            torch.cuda.synchronize()
        return sum("backward_kernel" in e.name for e in p.events())

    launches([w, b])
    assert launches([w, b]) == 1 and launches([w]) == 1
    x.requires_grad_()
    assert launches([x, w, b]) == 2


# ------------------------------------------------------------------------- views of negatives
@gpu
@pytest.mark.parametrize("which", range(3))
def test_memory_that_holds_negatives(which):
    """Imaginary parts of conjugates are views with a sign of their own, as operands and as gradients."""
    args, call = on_gpu(which)
    leaves = [t.requires_grad_() for t in args]
    y = call(*leaves)
    dy = torch.randn_like(y)
    want = [y, *torch.autograd.grad(y, leaves, dy)]
    theirs = [torch._neg_view(-t.detach()) for t in args]
    assert all(t.is_neg() for t in theirs)
    with torch.no_grad():
        assert torch.equal(call(*theirs), y)
    for t in theirs:
        t.requires_grad_()
    y = call(*theirs)
    got = [y, *torch.autograd.grad(y, theirs, torch._neg_view(-dy))]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------------- gated projection: the wide tiles
@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tokens,hidden,ffn", [(4096, 768, 2048), (2100, 768, 2048), (1037, 1000, 2730), (2561, 520, 1300), (700, 2048, 5000)])
def test_gated_linear_in_wide_tiles(tokens, hidden, ffn, dtype):
    """Sizes of use: tiles 256 wide, more of them than there are pairs of SMs (tensor memory is taken in turns), more than eight
    tile rows (bands), parts of long reductions."""
    from torch.profiler import ProfilerActivity, profile
    *ins, dh = gated_inputs(tokens, hidden, ffn, dtype, bias=tokens % 2 == 0)
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        check_gated(*ins, ["gelu", "silu", "gelu_tanh"][tokens % 3], dh)
        torch.cuda.synchronize()
    names = [e.name for e in p.events() if "product_kernel" in e.name]
    assert len(names) == 2 and any("<false, 256," in n for n in names), names


# ------------------------------------------------------------------------- gated projection: the range of f16
@gpu
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("tokens,hidden,ffn", [(3, 64, 72), (20, 64, 64), (600, 72, 264)])
@pytest.mark.parametrize("x_size,w_size,up_size,dh_size", [
    (1e-3, 1e-3, 30.0, 2e4),          # dh u is beyond 65504, its products with w and x are not
    (100.0, 1e-3, 2.0 ** -9, 2.0 ** -16),  # dh u is below 2^-24, its sums with x over the tokens are not
    (1.0, 0.1, 1.0, 1.0),
])
def test_gated_linear_in_f16_beyond_the_range_of_what_it_multiplies(x_size, w_size, up_size, dh_size, tokens, hidden, ffn, act):
    x, wg, wu, bg, bu, dh = gated_inputs(tokens, hidden, ffn, F32, True)
    x, dh = (x * x_size).to(F16), (dh.clamp(-3, 3) * dh_size).to(F16)
    wg, wu = ((w.sign() * w_size * (0.5 + 0.1 * w.abs())).to(F16) for w in (wg, wu))
    bg, bu = bg.to(F16), (up_size * (1 + 0.1 * bu)).to(F16)
    dh[1] = 0  # (and a row of nothing)
    leaves = [t.requires_grad_() for t in (x, wg, wu)]
    grads = torch.autograd.grad(ops.gated_linear(*leaves, bg, bu, activation=act), leaves, dh)
    X, G, W, D = (t.detach().double() for t in (x, wg, wu, dh))
    g, u = (X @ G.t() + bg.double()).requires_grad_(), X @ W.t() + bu.double()
    a = ACTS[act](g)
    da, = torch.autograd.grad(a.sum(), g)
    dg, du = D * u * da, D * a.detach()
    # half a step of f16 for dg and du, 2^-15 for each of g and u as they are kept (the derivatives follow by 1.2 at most), some 2^-20 for
    # sums of few hundred terms in 32 bits: below 2^-11 (1 + 1/4) of the terms' sizes
    rel = 1.25 * 2.0 ** -11
    eg = D.abs() * (u.abs() * (da.abs() + 2.0 ** -4) + 2.0 ** -4)  # (2^-15 of g and u, 2^-4 of the bound)
    eu = D.abs() * (a.detach().abs() + 2.0 ** -4 * g.detach().abs())
    within(grads[0], dg @ G + du @ W, rel * (eg @ G.abs() + eu @ W.abs()))
    within(grads[1], dg.t() @ X, rel * (eg.t() @ X.abs()))
    within(grads[2], du.t() @ X, rel * (eu.t() @ X.abs()))
    assert all(t.isfinite().all() for t in grads)


@gpu
def test_gated_linear_in_f16_infinite_gradients_stay_in_their_rows():
    x, wg, wu, bg, bu, dh = gated_inputs(140, 96, 80, F16, True)
    x = x.requires_grad_()
    want, = torch.autograd.grad(ops.gated_linear(x, wg, wu, bg, bu), x, dh)
    dh[3, 7], dh[9, 1] = torch.inf, torch.nan
    got, = torch.autograd.grad(ops.gated_linear(x, wg, wu, bg, bu), x, dh)
    rest = torch.ones(140, dtype=torch.bool, device=cuda)
    rest[[3, 9]] = False
    assert torch.equal(got[rest], want[rest]) and not got[3].isfinite().any() and got[9].isnan().all()


@gpu
def test_gelu_of_every_f16_number():
    """4 U |z| of the formula in 32 bits, an exponential and a quotient of the hardware (4 U each of a value that is below |z| / 2); left of
    zero in relation to the value: 1.5e-6, and z^2 / 2 times 1.5 roundings of the exponent."""
    z = torch.arange(0x4800 + 1, dtype=torch.int16, device=cuda).view(F16)  # 0 .. 8
    z = torch.cat([z, -z])
    z = z[:z.numel() // 16 * 16].view(-1, 16)
    one, nothing = torch.ones(16, device=cuda, dtype=F16), torch.zeros(16, 16, device=cuda, dtype=F16)
    with torch.no_grad():
        h = ops.gated_linear(z, torch.eye(16, device=cuda, dtype=F16), nothing, 0 * one, one, activation="gelu")
    z = z.double()
    cdf = 0.5 * torch.special.erfc(-z / 2 ** 0.5)
    within(h, z * cdf, torch.where(z > 0, 8 * U * z, (1.5e-6 + 1.5 * U * z * z) * (z * cdf).abs()))


# ------------------------------------------------------------------------- tensors that are not plain
class Wrapped(torch.Tensor):
    """A subclass around another tensor, without memory of its own."""

    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device, strides=inner.stride())

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise AssertionError(f"{func} was asked of a wrapper")


@pytest.mark.parametrize("which", range(3))
def test_tensors_without_memory_are_refused(native_lib, which):
    args, call = calls()[which]
    with torch.no_grad():
        for i in range(len(args)):
            with pytest.raises(TypeError, match="without memory"):
                call(*[Wrapped(t) if j == i else t for j, t in enumerate(args)])


@gpu
@pytest.mark.parametrize("which", range(3))
def test_tensors_without_memory_are_refused_on_a_gpu(which):
    args, call = on_gpu(which)
    for i in range(len(args)):
        with torch.no_grad(), pytest.raises(TypeError, match="without memory"):
            call(*[Wrapped(t) if j == i else t for j, t in enumerate(args)])
