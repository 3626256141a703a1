// The way from an operator on tensors (ops/train.py) to the C ABI: checks of the
// arguments, layouts that the kernels take, results and workspaces from PyTorch's
// allocator, the current stream of the tensors' GPU, and the gradients.  All of it native, the backward pass too,
// which autograd calls from threads of its own: through Python's Function a training step of small
// tensors took 85 us, five times what the GPU works.  What is wrong with the arguments raises
// ValueError / TypeError, before anything is launched; sizes and types are
// looked at before the place of the data, so that they are refused on any machine.
#include "train.hpp"

#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/DeviceGuardImplInterface.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>
#include <string>
#include <utility>
#include <vector>

#include "capi_cuda.h"
#include "capi_train.h"

namespace
{
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;

[[noreturn]] void refuse(const char *call, const std::string &what) { TORCH_CHECK_VALUE(false, call, ": ", what); }
[[noreturn]] void refuse_type(const char *call, const std::string &what) { TORCH_CHECK_TYPE(false, call, ": ", what); }

// Second derivatives would silently lack what goes through the operator.
void first_order(const char *call)
{
    TORCH_CHECK(!at::GradMode::is_enabled(), call, " is differentiable once: backward with create_graph=True is refused");
}

int float_code(const Tensor &t, const char *call)
{
    switch (t.scalar_type()) {
    case c10::ScalarType::BFloat16:
        return 8;
    case c10::ScalarType::Half:
        return 9;
    case c10::ScalarType::Float:
        return 10;
    default:
        refuse_type(call, std::string("bfloat16, float16 or float32 expected, got ") + c10::toString(t.scalar_type()));
    }
}

std::string shape_of(const Tensor &t)
{
    std::string s = "(";
    for (int64_t v : t.sizes()) { s += (s.size() > 1 ? ", " : "") + std::to_string(v); }
    return s + ")";
}

// The GPU that all tensors of a call lie on is current, its stream the one to enqueue on.
class OnDevice
{
  public:
    OnDevice(const char *call, const Tensor &first, std::initializer_list<const Tensor *> others)
        : device_(checked(call, first, others)), guard_(device_),
          stream_(c10::impl::getDeviceGuardImpl(c10::DeviceType::CUDA)->getStream(device_).native_handle())
    {
    }
    int index() const { return device_.index(); }
    void *stream() const { return stream_; }

  private:
    static c10::Device checked(const char *call, const Tensor &first, std::initializer_list<const Tensor *> others)
    {
        if (!first.is_cuda()) { refuse(call, "CUDA tensor expected"); }
        for (const Tensor *t : others) {
            if (t->defined() && t->device() != first.device()) { refuse(call, "all tensors must lie on one GPU"); }
        }
        return first.device();
    }
    c10::Device device_;
    c10::DeviceGuard guard_;
    void *stream_;
};

// The C ABI's refusals and errors as exceptions.
void done(int rc)
{
    if (rc == STDMLC_OK) { return; }
    if (rc == STDMLC_ERR_ARGS) { TORCH_CHECK_VALUE(false, stdmlc_last_error()); }
    TORCH_CHECK(false, stdmlc_last_error());
}

Tensor bytes_like(const Tensor &t, long long n)
{
    TORCH_CHECK(n >= 0, stdmlc_last_error());
    return at::empty({n}, t.options().dtype(at::kByte).requires_grad(false).memory_format(std::nullopt));
}

// Memory that holds the values' negatives (a view of a conjugate's imaginary part) is not read as it lies.
Tensor plain(const Tensor &t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }

void *ptr_of(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

// A tensor without memory of its own (a subclass that wraps others, a fake one) would pass for an operand that is not there.
void has_memory(const char *call, std::initializer_list<const Tensor *> all)
{
    for (const Tensor *t : all) {
        if (t->defined() && t->numel() > 0 && (!t->has_storage() || t->storage().data() == nullptr)) {
            refuse_type(call, "a plain tensor expected, got one without memory of its own");
        }
    }
}

// Operands that a call may lack: autograd's Function knows them as empty optionals, the code here as undefined tensors.
using Maybe = std::optional<Tensor>;
Maybe maybe(const Tensor &t) { return t.defined() ? Maybe(t) : Maybe(); }
Tensor given(const Maybe &t) { return t ? *t : Tensor(); }

bool wanted(std::initializer_list<const Tensor *> all)
{
    if (!at::GradMode::is_enabled()) { return false; }
    for (const Tensor *t : all) {
        if (t->defined() && t->requires_grad()) { return true; }
    }
    return false;
}

// A tangent would be dropped without a word where no gradient is wanted, and in the constants always.
void no_tangent(const char *call, std::initializer_list<const Tensor *> all)
{
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) { return; }
    for (const Tensor *t : all) {
        if (t->defined() && t->_fw_grad(0).defined()) { refuse(call, "has no forward-mode derivative: a tensor without a tangent expected"); }
    }
}

// ------------------------------------------------------------ group normalisation
// (N, C, spatial...) as rows of channels: the channels side by side, all positions of an image
// one stride apart.  False: in another layout.
bool rows_of(const Tensor &t, stdmlc_rows *r)
{
    const int64_t c = t.size(1);
    if (c > 1 && t.stride(1) != 1) { return false; }
    int64_t row = 0, extent = 0;  // stride of a position, and of all those inside the next dimension
    for (int64_t d = t.dim() - 1; d >= 2; --d) {
        if (t.size(d) == 1) { continue; }
        if (row == 0) {
            row = t.stride(d);
        } else if (t.stride(d) != extent) {
            return false;
        }
        extent = t.stride(d) * t.size(d);
        if (row == 0) { return false; }  // expanded
    }
    *r = {t.data_ptr(), t.size(0) > 1 ? t.stride(0) : 0, row};
    return true;
}

Tensor empty_rows(const Tensor &like)
{
    std::vector<int64_t> strides(like.dim());
    int64_t step = like.size(1);
    strides[1] = 1;
    for (int64_t d = like.dim() - 1; d >= 2; --d) {
        strides[d] = step;
        step *= like.size(d);
    }
    strides[0] = step;
    return at::empty_strided(like.sizes(), strides, like.options().requires_grad(false));
}

Tensor in_rows(const Tensor &t, stdmlc_rows *r)
{
    if (rows_of(t, r)) { return t; }
    Tensor copy = empty_rows(t);
    copy.copy_(t);
    rows_of(copy, r);
    return copy;
}

// What both directions of a call have in common.
struct Norm {
    static constexpr const char *kCall = "group_norm";
    stdmlc_norm a{};
    Tensor x, residual, weight, bias;

    void take(const Tensor &x_, const Tensor &residual_, const Tensor &weight_, const Tensor &bias_, long long groups,
              double eps, int act)
    {
        x = x_;
        if (x.dim() < 2) { refuse(kCall, "(N, C, ...) expected, got " + shape_of(x)); }
        const int64_t c = x.size(1);
        if (groups < 1 || c < 1 || c % groups != 0) {
            refuse(kCall, std::to_string(groups) + " groups do not divide " + std::to_string(c) + " channels");
        }
        if (!(eps >= 0)) { refuse(kCall, "eps must not be negative"); }
        a.dt = float_code(x, kCall);
        a.weight_dt = 10;
        for (const Tensor *p : {&weight_, &bias_}) {
            if (!p->defined()) { continue; }
            if (p->dim() != 1 || p->size(0) != c) {
                refuse(kCall, "weight and bias of " + std::to_string(c) + " channels expected, got " + shape_of(*p));
            }
            a.weight_dt = float_code(*p, kCall);
        }
        if (weight_.defined() && bias_.defined() && weight_.scalar_type() != bias_.scalar_type()) {
            refuse_type(kCall, "weight and bias must have one dtype");
        }
        if (residual_.defined()) {
            if (residual_.sizes() != x.sizes()) {
                refuse(kCall, "residual of " + shape_of(x) + " expected, got " + shape_of(residual_));
            }
            if (residual_.scalar_type() != x.scalar_type()) { refuse_type(kCall, "residual must have the input's dtype"); }
        }
        residual = residual_;
        weight = weight_;
        bias = bias_;
        a.images = x.size(0);
        a.positions = c * a.images > 0 ? x.numel() / (c * a.images) : 0;
        a.channels = static_cast<int>(c);
        a.groups = static_cast<int>(groups);
        a.eps = eps;
        a.act = act;
    }
    // (on the GPU: may copy)
    void lay_out()
    {
        x = in_rows(x, &a.x);
        if (residual.defined()) { residual = in_rows(residual, &a.residual); }
        for (Tensor *p : {&weight, &bias}) {
            if (p->defined()) { *p = p->contiguous(); }
        }
        a.weight = ptr_of(weight);
        a.bias = ptr_of(bias);
    }
    // y and the statistics
    std::pair<Tensor, Tensor> forward()
    {
        const OnDevice on(kCall, x, {&residual, &weight, &bias});
        lay_out();
        Tensor y = empty_rows(x);
        Tensor stats = at::empty({a.images, a.groups, 2}, x.options().dtype(at::kDouble).requires_grad(false));
        rows_of(y, &a.y);
        a.stats = stats.data_ptr<double>();
        const Tensor work = bytes_like(x, stdmlc_norm_workspace(&a, 0));
        a.workspace = work.data_ptr();
        done(stdmlc_norm_forward(&a, on.index(), on.stream()));
        return {y, stats};
    }
};

struct NormFunction : torch::autograd::Function<NormFunction> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Maybe &residual_, const Maybe &weight_, const Maybe &bias_,
                          int64_t groups, double eps, int64_t act)
    {
        const Tensor residual = given(residual_), weight = given(weight_), bias = given(bias_);
        Norm op;
        op.take(x, residual, weight, bias, groups, eps, static_cast<int>(act));
        const auto [y, stats] = op.forward();
        // (x and the residual as the kernels read them; without an activation the residual does not matter)
        ctx->save_for_backward({op.x, act != STDMLC_ACT_NONE ? op.residual : Tensor(), weight, bias, stats});
        ctx->saved_data["residual"] = residual.defined();
        ctx->saved_data["groups"] = groups;
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["act"] = act;
        return y;
    }
    static tensor_list backward(AutogradContext *ctx, tensor_list grads)
    {
        first_order(Norm::kCall);
        const auto saved = ctx->get_saved_variables();
        Norm op;
        const Tensor &weight = saved[2], &bias = saved[3], &stats = saved[4];
        op.take(saved[0], saved[1], weight, bias, ctx->saved_data["groups"].toInt(), ctx->saved_data["eps"].toDouble(),
                static_cast<int>(ctx->saved_data["act"].toInt()));
        const OnDevice on(Norm::kCall, op.x, {&grads[0]});
        op.lay_out();
        const Tensor dy = in_rows(plain(grads[0]), &op.a.dy);
        op.a.stats = stats.data_ptr<double>();
        Tensor dx, dres, dw, db;
        size_t edge = 0;  // (autograd counts the operands that there are)
        if (ctx->needs_input_grad(edge++)) {
            dx = empty_rows(op.x);
            rows_of(dx, &op.a.dx);
        }
        if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(edge++)) {
            dres = empty_rows(op.x);
            rows_of(dres, &op.a.dresidual);
        }
        if (weight.defined() && ctx->needs_input_grad(edge++)) { dw = at::empty_like(op.weight); }
        if (bias.defined() && ctx->needs_input_grad(edge++)) { db = at::empty_like(op.bias); }
        op.a.dweight = ptr_of(dw);
        op.a.dbias = ptr_of(db);
        const Tensor work = bytes_like(op.x, stdmlc_norm_workspace(&op.a, 1));
        op.a.workspace = work.data_ptr();
        done(stdmlc_norm_backward(&op.a, on.index(), on.stream()));
        return {dx, dres, dw, db, {}, {}, {}};
    }
};

// ------------------------------------------------------------ rows of a matrix
// (..., n) as rows with a stride, copied where it does not lie like that.
Tensor matrix_of(const Tensor &t, const void **ptr, long long *row)
{
    const Tensor &d = t;
    const int64_t n = d.size(-1);
    int64_t step = 0, extent = 0;
    bool fits = n <= 1 || d.stride(-1) == 1;
    for (int64_t i = d.dim() - 2; fits && i >= 0; --i) {
        if (d.size(i) == 1) { continue; }
        if (step == 0) {
            step = d.stride(i);
            fits = step != 0;
        } else {
            fits = d.stride(i) == extent;
        }
        extent = d.stride(i) * d.size(i);
    }
    if (!fits) {
        const Tensor copy = d.contiguous();
        *ptr = copy.data_ptr();
        *row = n;
        return copy;
    }
    *ptr = d.data_ptr();
    *row = step;
    return d;
}

bool same_rows(const Tensor &a, const Tensor &b)
{
    return a.dim() == b.dim() && a.sizes().slice(0, a.dim() - 1) == b.sizes().slice(0, b.dim() - 1);
}

// ------------------------------------------------------------ distillation loss
struct Distill {
    static constexpr const char *kCall = "distill_loss";
    stdmlc_distill d{};
    Tensor logits, top, index, labels;

    void take(const Tensor &logits_, const Tensor &top_, const Tensor &index_, const Tensor &labels_, double temperature,
              double alpha, long long ignore, int reduction)
    {
        logits = logits_;
        top = top_;
        index = index_;
        labels = labels_;
        if (logits.dim() < 1 || logits.size(-1) < 1) {
            refuse(kCall, "logits of (..., classes) expected, got " + shape_of(logits));
        }
        d.dt = float_code(logits, kCall);
        d.top_dt = float_code(top, kCall);
        if (top.dim() < 1 || !same_rows(top, logits)) {
            refuse(kCall, "teacher_logits of the logits' rows expected, got " + shape_of(top) + " for " + shape_of(logits));
        }
        if (index.sizes() != top.sizes()) {
            refuse(kCall, "teacher_index of " + shape_of(top) + " expected, got " + shape_of(index));
        }
        if (index.scalar_type() != at::kLong && index.scalar_type() != at::kInt) {
            refuse_type(kCall, "teacher_index must be int32 or int64");
        }
        if (labels.defined()) {
            if (labels.sizes() != logits.sizes().slice(0, logits.dim() - 1)) {
                refuse(kCall, "one label for each row expected, got " + shape_of(labels) + " for " + shape_of(logits));
            }
            if (labels.scalar_type() != at::kLong && labels.scalar_type() != at::kInt) {
                refuse_type(kCall, "labels must be int32 or int64");
            }
        }
        if (!(temperature > 0) || !(temperature < 1e30)) { refuse(kCall, "temperature must be positive"); }
        if (!(alpha >= 0 && alpha <= 1)) { refuse(kCall, "alpha must lie between 0 and 1"); }
        d.classes = logits.size(-1);
        d.rows = logits.numel() / d.classes;
        if (d.rows >= (1ll << 31) || d.classes >= (1ll << 31)) { refuse(kCall, "too many rows or classes"); }
        if (top.size(-1) > 4096) { refuse(kCall, "at most 4096 teacher entries in a row"); }
        d.top_count = static_cast<int>(top.size(-1));
        d.temperature = static_cast<float>(temperature);
        d.alpha = static_cast<float>(alpha);
        d.ignore = ignore;
        d.reduction = reduction;
    }
    void lay_out()
    {
        logits = matrix_of(logits, &d.logits, &d.logits_row);
        top = matrix_of(top, &d.top, &d.top_row);
        index = matrix_of(index, &d.index, &d.index_row);
        d.index_bytes = index.scalar_type() == at::kLong ? 8 : 4;
        if (labels.defined()) {
            labels = labels.to(at::kLong).contiguous();
            d.labels = labels.data_ptr();
        }
    }
    Tensor empty_grad() const
    {
        return at::empty(logits.sizes(), logits.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous));
    }
    // The loss and the rows' statistics; `grad`: where the gradient goes that the forward pass writes.
    std::pair<Tensor, Tensor> forward(bool with_grad, Tensor &grad)
    {
        const OnDevice on(kCall, logits, {&top, &index, &labels});
        const auto rows = logits.sizes().slice(0, logits.dim() - 1);
        lay_out();
        const auto f32 = logits.options().dtype(at::kFloat).requires_grad(false).memory_format(std::nullopt);
        Tensor stats = at::empty({d.rows, 5}, f32);
        Tensor loss = d.reduction == 0 ? at::empty(rows, f32) : at::empty({}, f32);
        d.row_stats = stats.data_ptr<float>();
        d.loss = loss.data_ptr<float>();
        // (f16 logits come with a loss scale, whose gradient is not one: theirs waits for the backward pass)
        if (with_grad && d.reduction != 0 && d.dt != 9) {
            grad = empty_grad();
            d.dlogits = grad.data_ptr();
        }
        const Tensor work = bytes_like(logits, stdmlc_distill_workspace(&d));
        d.workspace = work.data_ptr();
        done(stdmlc_distill_forward(&d, on.index(), on.stream()));
        capture = stdmlc_stream_capturing(on.stream());
        return {loss, stats};
    }
    int64_t capture = 0;  // that the call is part of
};

struct DistillFunction : torch::autograd::Function<DistillFunction> {
    static Tensor forward(AutogradContext *ctx, const Tensor &logits, const Tensor &top, const Tensor &index, const Maybe &labels_,
                          double temperature, double alpha, int64_t ignore, int64_t reduction)
    {
        const Tensor labels = given(labels_);
        Distill op;
        op.take(logits, top, index, labels, temperature, alpha, ignore, static_cast<int>(reduction));
        Tensor grad;
        const auto [loss, stats] = op.forward(true, grad);
        ctx->save_for_backward({logits, top, index, labels, stats});
        ctx->saved_data["temperature"] = temperature;
        ctx->saved_data["alpha"] = alpha;
        ctx->saved_data["ignore"] = ignore;
        ctx->saved_data["reduction"] = reduction;
        if (grad.defined()) {
            ctx->saved_data["grad"] = grad;
            ctx->saved_data["capture"] = op.capture;
        }
        return loss;
    }
    static tensor_list backward(AutogradContext *ctx, tensor_list grads)
    {
        first_order(Distill::kCall);
        const auto saved = ctx->get_saved_variables();
        Distill op;
        op.take(saved[0], saved[1], saved[2], saved[3], ctx->saved_data["temperature"].toDouble(),
                ctx->saved_data["alpha"].toDouble(), ctx->saved_data["ignore"].toInt(),
                static_cast<int>(ctx->saved_data["reduction"].toInt()));
        const OnDevice on(Distill::kCall, op.logits, {&grads[0]});
        const Tensor dloss = plain(grads[0]).to(at::kFloat).contiguous();
        Tensor dlogits;
        const auto held = ctx->saved_data.find("grad");
        // The forward pass's gradient, for the first who asks: as it is for a loss of gradient one, which the kernel looks at.  For
        // another it is written over, so a graph that is captured takes only one that its own replays write anew: of the same capture.
        if (held != ctx->saved_data.end() && stdmlc_stream_capturing(on.stream()) == ctx->saved_data["capture"].toInt()) {
            dlogits = held->second.toTensor();
            ctx->saved_data.erase("grad");
            op.d.written = 1;
        } else {
            dlogits = op.empty_grad();
        }
        op.lay_out();
        op.d.dloss = dloss.data_ptr<float>();
        op.d.dloss_row = op.d.reduction == 0 ? 1 : 0;
        op.d.row_stats = saved[4].data_ptr<float>();
        op.d.dlogits = dlogits.data_ptr();
        done(stdmlc_distill_backward(&op.d, on.index(), on.stream()));
        return {dlogits, {}, {}, {}, {}, {}, {}, {}};
    }
};

// ------------------------------------------------------------ gated projection
struct Gated {
    static constexpr const char *kCall = "gated_linear";
    stdmlc_gated a{};
    Tensor x, w_gate, w_up, b_gate, b_up;

    void take(const Tensor &x_, const Tensor &w_gate_, const Tensor &w_up_, const Tensor &b_gate_, const Tensor &b_up_,
              int act)
    {
        x = x_;
        w_gate = w_gate_;
        w_up = w_up_;
        b_gate = b_gate_;
        b_up = b_up_;
        a.dt = float_code(x, kCall);
        if (x.dim() < 1) { refuse(kCall, "(..., hidden) expected, got " + shape_of(x)); }
        if (w_gate.dim() != 2 || w_up.sizes() != w_gate.sizes()) {
            refuse(kCall, "two weights of (ffn, hidden) expected, got " + shape_of(w_gate) + " and " + shape_of(w_up));
        }
        a.hidden = x.size(-1);
        a.ffn = w_gate.size(0);
        if (w_gate.size(1) != a.hidden) {
            refuse(kCall, "weights of (ffn, " + std::to_string(a.hidden) + ") expected, got " + shape_of(w_gate));
        }
        if (a.hidden < 1 || a.ffn < 1) { refuse(kCall, "hidden and ffn must not be empty"); }
        a.tokens = x.numel() / a.hidden;
        if (a.hidden > (1ll << 20) || a.ffn > (1ll << 20) || a.tokens > (1ll << 22)) {
            refuse(kCall, "at most 2^22 tokens, 2^20 hidden and 2^20 ffn");
        }
        if (b_gate.defined() != b_up.defined()) { refuse(kCall, "both biases or none"); }
        for (const Tensor *b : {&b_gate, &b_up}) {
            if (b->defined() && (b->dim() != 1 || b->size(0) != a.ffn)) {
                refuse(kCall, "biases of (" + std::to_string(a.ffn) + ",) expected, got " + shape_of(*b));
            }
        }
        for (const Tensor *t : {&w_gate, &w_up, &b_gate, &b_up}) {
            if (t->defined() && t->scalar_type() != x.scalar_type()) {
                refuse_type(kCall, "weights and biases must have the input's dtype");
            }
        }
        a.act = act;
    }
    void lay_out()
    {
        x = matrix_of(x, &a.x, &a.x_row);
        w_gate = matrix_of(w_gate, &a.w_gate, &a.w_gate_row);
        w_up = matrix_of(w_up, &a.w_up, &a.w_up_row);
        for (Tensor *b : {&b_gate, &b_up}) {
            if (b->defined()) { *b = b->contiguous(); }
        }
        a.b_gate = ptr_of(b_gate);
        a.b_up = ptr_of(b_up);
    }
    // h, and what a backward pass needs, if one follows
    std::pair<Tensor, Tensor> forward(bool follows)
    {
        const OnDevice on(kCall, x, {&w_gate, &w_up, &b_gate, &b_up});
        std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
        shape.back() = a.ffn;
        const Tensor like = x;
        lay_out();
        Tensor h = at::empty(shape, like.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous)), saved;
        a.h = h.data_ptr();
        if (follows) {
            saved = bytes_like(like, stdmlc_gated_saved(&a));
            a.saved = saved.data_ptr();
        }
        const Tensor work = bytes_like(like, stdmlc_gated_workspace(&a, 0));
        a.workspace = work.data_ptr();
        done(stdmlc_gated_forward(&a, on.index(), on.stream()));
        return {h, saved};
    }
};

struct GatedFunction : torch::autograd::Function<GatedFunction> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w_gate, const Tensor &w_up, const Maybe &b_gate_,
                          const Maybe &b_up_, int64_t act)
    {
        const Tensor b_gate = given(b_gate_), b_up = given(b_up_);
        Gated op;
        op.take(x, w_gate, w_up, b_gate, b_up, static_cast<int>(act));
        const auto [h, saved] = op.forward(true);
        ctx->save_for_backward({x, w_gate, w_up, b_gate, b_up, saved});
        ctx->saved_data["act"] = act;
        return h;
    }
    static tensor_list backward(AutogradContext *ctx, tensor_list grads)
    {
        first_order(Gated::kCall);
        const auto saved = ctx->get_saved_variables();
        Gated op;
        op.take(saved[0], saved[1], saved[2], saved[3], saved[4], static_cast<int>(ctx->saved_data["act"].toInt()));
        const OnDevice on(Gated::kCall, op.x, {&grads[0]});
        op.lay_out();
        const Tensor dh = matrix_of(plain(grads[0]), &op.a.dh, &op.a.dh_row);
        op.a.saved = saved[5].data_ptr();
        const auto packed = saved[0].options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous);
        tensor_list out(6);
        for (size_t i = 0; i < 5; ++i) {
            if (saved[i].defined() && ctx->needs_input_grad(i)) { out[i] = at::empty(saved[i].sizes(), packed); }
        }
        op.a.dx = ptr_of(out[0]);
        op.a.dw_gate = ptr_of(out[1]);
        op.a.dw_up = ptr_of(out[2]);
        op.a.db_gate = ptr_of(out[3]);
        op.a.db_up = ptr_of(out[4]);
        const Tensor work = bytes_like(saved[0], stdmlc_gated_workspace(&op.a, 1));
        op.a.workspace = work.data_ptr();
        done(stdmlc_gated_backward(&op.a, on.index(), on.stream()));
        return out;
    }
};

// ------------------------------------------------------------ from Python
struct Raised {
};  // a Python exception is set

struct Args {
    const char *call;
    PyObject *const *a;
    Py_ssize_t n;
    int i = 0;

    void expect(Py_ssize_t want) const
    {
        if (n != want) { refuse_type(call, std::to_string(want) + " arguments expected"); }
    }
    Tensor optional()  // undefined for None
    {
        PyObject *o = a[i++];
        if (o == Py_None) { return {}; }
        if (!THPVariable_Check(o)) { refuse_type(call, std::string("tensor expected, got ") + Py_TYPE(o)->tp_name); }
        return plain(THPVariable_Unpack(o));
    }
    Tensor tensor()
    {
        const Tensor t = optional();
        if (!t.defined()) { refuse_type(call, "tensor expected, got None"); }
        return t;
    }
    long long integer()
    {
        const long long v = PyLong_AsLongLong(a[i++]);
        if (v == -1 && PyErr_Occurred()) { throw Raised{}; }
        return v;
    }
    double real()
    {
        const double v = PyFloat_AsDouble(a[i++]);
        if (v == -1.0 && PyErr_Occurred()) { throw Raised{}; }
        return v;
    }
};

struct WithoutGil {
    PyThreadState *state = PyEval_SaveThread();
    ~WithoutGil() { PyEval_RestoreThread(state); }
};

template <typename F>
PyObject *guarded(F f)
{
    try {
        return THPVariable_Wrap(f());
    } catch (const Raised &) {
    } catch (python_error &e) {  // of a hook on saved tensors: a checkpoint ends its second pass like that
        e.restore();
    } catch (const c10::ValueError &e) {
        PyErr_SetString(PyExc_ValueError, e.what_without_backtrace());
    } catch (const c10::TypeError &e) {
        PyErr_SetString(PyExc_TypeError, e.what_without_backtrace());
    } catch (const c10::OutOfMemoryError &e) {
        PyObject *torch = PyImport_ImportModule("torch"), *kind = nullptr;
        if (torch != nullptr) { kind = PyObject_GetAttrString(torch, "OutOfMemoryError"); }
        if (kind != nullptr) { PyErr_SetString(kind, e.what_without_backtrace()); }
        Py_XDECREF(kind);
        Py_XDECREF(torch);
    } catch (const c10::Error &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
    }
    return nullptr;
}

// (x, residual | None, weight | None, bias | None, groups, eps, activation) -> y
PyObject *group_norm(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return guarded([&] {
        Args g{Norm::kCall, args, n};
        g.expect(7);
        const Tensor x = g.tensor(), residual = g.optional(), weight = g.optional(), bias = g.optional();
        const long long groups = g.integer();
        const double eps = g.real();
        const long long act = g.integer();
        const WithoutGil free;
        has_memory(Norm::kCall, {&x, &residual, &weight, &bias});
        no_tangent(Norm::kCall, {&x, &residual, &weight, &bias});
        if (wanted({&x, &residual, &weight, &bias})) { return NormFunction::apply(x, maybe(residual), maybe(weight), maybe(bias), groups, eps, act); }
        Norm op;
        op.take(x, residual, weight, bias, groups, eps, static_cast<int>(act));
        return op.forward().first;
    });
}

// (logits, teacher_logits, teacher_index, labels | None, temperature, alpha, ignore_index, reduction) -> loss
PyObject *distill_loss(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return guarded([&] {
        Args g{Distill::kCall, args, n};
        g.expect(8);
        const Tensor logits = g.tensor(), top = g.tensor(), index = g.tensor(), labels = g.optional();
        const double temperature = g.real(), alpha = g.real();
        const long long ignore = g.integer(), reduction = g.integer();
        const WithoutGil free;
        has_memory(Distill::kCall, {&logits, &top, &index, &labels});
        no_tangent(Distill::kCall, {&logits, &top});
        if (top.requires_grad()) { refuse(Distill::kCall, "teacher_logits are constants: a tensor without gradient expected"); }
        if (wanted({&logits})) {
            return DistillFunction::apply(logits, top, index, maybe(labels), temperature, alpha, ignore, reduction);
        }
        Distill op;
        op.take(logits, top, index, labels, temperature, alpha, ignore, static_cast<int>(reduction));
        Tensor none;
        return op.forward(false, none).first;
    });
}

// (x, w_gate, w_up, b_gate | None, b_up | None, activation) -> h
PyObject *gated_linear(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return guarded([&] {
        Args g{Gated::kCall, args, n};
        g.expect(6);
        const Tensor x = g.tensor(), wg = g.tensor(), wu = g.tensor(), bg = g.optional(), bu = g.optional();
        const long long act = g.integer();
        const WithoutGil free;
        has_memory(Gated::kCall, {&x, &wg, &wu, &bg, &bu});
        no_tangent(Gated::kCall, {&x, &wg, &wu, &bg, &bu});
        if (wanted({&x, &wg, &wu, &bg, &bu})) { return GatedFunction::apply(x, wg, wu, maybe(bg), maybe(bu), act); }
        Gated op;
        op.take(x, wg, wu, bg, bu, static_cast<int>(act));
        return op.forward(false).first;
    });
}

PyMethodDef kMethods[] = {
    {"group_norm", reinterpret_cast<PyCFunction>(group_norm), METH_FASTCALL, nullptr},
    {"distill_loss", reinterpret_cast<PyCFunction>(distill_loss), METH_FASTCALL, nullptr},
    {"gated_linear", reinterpret_cast<PyCFunction>(gated_linear), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
}  // namespace

PyMethodDef *train_methods() { return kMethods; }
