// The way from an operator on tensors (ops/train.py) to the C ABI: checks of the
// arguments, layouts that the kernels take, results and workspaces from PyTorch's
// allocator, the current stream of the tensors' GPU.  What is wrong with the arguments raises
// ValueError / TypeError, before anything is launched; sizes and types are
// looked at before the place of the data, so that they are refused on any machine.
#include "train.hpp"

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/DeviceGuardImplInterface.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>
#include <string>
#include <vector>

#include "capi_cuda.h"
#include "capi_train.h"

namespace
{
using at::Tensor;
using Maybe = std::optional<Tensor>;

struct Raised {
};  // a Python exception is set

[[noreturn]] void refuse(const char *call, const std::string &what, PyObject *kind = PyExc_ValueError)
{
    PyErr_SetString(kind, (std::string(call) + ": " + what).c_str());
    throw Raised{};
}

struct Args {
    const char *call;
    PyObject *const *a;
    Py_ssize_t n;
    int i = 0;

    void expect(Py_ssize_t want) const
    {
        if (n != want) { refuse(call, std::to_string(want) + " arguments expected", PyExc_TypeError); }
    }
    Maybe maybe()
    {
        PyObject *o = a[i++];
        if (o == Py_None) { return {}; }
        if (!THPVariable_Check(o)) {
            refuse(call, std::string("tensor expected, got ") + Py_TYPE(o)->tp_name, PyExc_TypeError);
        }
        return THPVariable_Unpack(o);
    }
    Tensor tensor()
    {
        Maybe t = maybe();
        if (!t) { refuse(call, "tensor expected, got None", PyExc_TypeError); }
        return *t;
    }
    long long integer()
    {
        const long long v = PyLong_AsLongLong(a[i++]);
        if (v == -1 && PyErr_Occurred()) { throw Raised{}; }
        return v;
    }
    bool truth() { return PyObject_IsTrue(a[i++]) == 1; }
    double real()
    {
        const double v = PyFloat_AsDouble(a[i++]);
        if (v == -1.0 && PyErr_Occurred()) { throw Raised{}; }
        return v;
    }
};

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
        refuse(call, std::string("bfloat16, float16 or float32 expected, got ") + c10::toString(t.scalar_type()),
               PyExc_TypeError);
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
    OnDevice(const char *call, const Tensor &first, std::initializer_list<const Maybe *> others)
        : device_(checked(call, first, others)), guard_(device_),
          stream_(c10::impl::getDeviceGuardImpl(c10::DeviceType::CUDA)->getStream(device_).native_handle())
    {
    }
    int index() const { return device_.index(); }
    void *stream() const { return stream_; }

  private:
    static c10::Device checked(const char *call, const Tensor &first, std::initializer_list<const Maybe *> others)
    {
        if (!first.is_cuda()) { refuse(call, "CUDA tensor expected"); }
        for (const Maybe *t : others) {
            if (*t && (*t)->device() != first.device()) { refuse(call, "all tensors must lie on one GPU"); }
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
    PyErr_SetString(rc == STDMLC_ERR_ARGS ? PyExc_ValueError : PyExc_RuntimeError, stdmlc_last_error());
    throw Raised{};
}

#define WITHOUT_GIL(rc, call)                                                  \
    do {                                                                       \
        Py_BEGIN_ALLOW_THREADS rc = (call);                                    \
        Py_END_ALLOW_THREADS                                                   \
    } while (0)

template <typename F>
PyObject *guarded(F f)
{
    try {
        return f();
    } catch (const Raised &) {
        return nullptr;
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

PyObject *tuple_of(std::initializer_list<Maybe> all)
{
    PyObject *t = PyTuple_New(static_cast<Py_ssize_t>(all.size()));
    if (t == nullptr) { throw Raised{}; }
    Py_ssize_t i = 0;
    for (const Maybe &m : all) {
        PyObject *o = Py_None;
        if (m) {
            o = THPVariable_Wrap(*m);
        } else {
            Py_INCREF(o);
        }
        PyTuple_SET_ITEM(t, i++, o);
    }
    return t;
}

Tensor bytes_like(const Tensor &t, long long n)
{
    return at::empty({n}, t.options().dtype(at::kByte).requires_grad(false).memory_format(std::nullopt));
}

void *ptr_of(const Maybe &t) { return t ? t->data_ptr() : nullptr; }

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
    Tensor x;
    Maybe residual, weight, bias;

    void take(const Tensor &x_, const Maybe &residual_, const Maybe &weight_, const Maybe &bias_, long long groups,
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
        for (const Maybe *p : {&weight_, &bias_}) {
            if (!*p) { continue; }
            if ((*p)->dim() != 1 || (*p)->size(0) != c) {
                refuse(kCall, "weight and bias of " + std::to_string(c) + " channels expected, got " + shape_of(**p));
            }
            a.weight_dt = float_code(**p, kCall);
        }
        if (weight_ && bias_ && weight_->scalar_type() != bias_->scalar_type()) {
            refuse(kCall, "weight and bias must have one dtype", PyExc_TypeError);
        }
        if (residual_) {
            if (residual_->sizes() != x.sizes()) {
                refuse(kCall, "residual of " + shape_of(x) + " expected, got " + shape_of(*residual_));
            }
            if (residual_->scalar_type() != x.scalar_type()) {
                refuse(kCall, "residual must have the input's dtype", PyExc_TypeError);
            }
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
        if (residual) { residual = in_rows(*residual, &a.residual); }
        for (Maybe *p : {&weight, &bias}) {
            if (*p) { *p = (*p)->contiguous(); }
        }
        a.weight = ptr_of(weight);
        a.bias = ptr_of(bias);
    }
};

// (x, residual | None, weight | None, bias | None, groups, eps, activation) ->
// (y, statistics, x and residual as the kernels read them)
PyObject *norm_forward(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return guarded([&] {
        Args g{Norm::kCall, args, n};
        g.expect(7);
        Norm op;
        const Tensor x = g.tensor();
        const Maybe residual = g.maybe(), weight = g.maybe(), bias = g.maybe();
        const long long groups = g.integer();
        const double eps = g.real();
        op.take(x, residual, weight, bias, groups, eps, static_cast<int>(g.integer()));
        const OnDevice on(Norm::kCall, x, {&residual, &weight, &bias});
        op.lay_out();
        Tensor y = empty_rows(x);
        Tensor stats = at::empty({op.a.images, groups, 2}, x.options().dtype(at::kDouble).requires_grad(false));
        rows_of(y, &op.a.y);
        op.a.stats = stats.data_ptr<double>();
        Tensor work = bytes_like(x, stdmlc_norm_workspace(&op.a, 0));
        op.a.workspace = work.data_ptr();
        int rc;
        WITHOUT_GIL(rc, stdmlc_norm_forward(&op.a, on.index(), on.stream()));
        done(rc);
        return tuple_of({y, stats, op.x, op.residual});
    });
}

// (dy, x, residual | None, weight | None, bias | None, statistics, groups, eps, activation,
// want dx, want dresidual, want dweight, want dbias) -> (dx, dresidual, dweight, dbias), None where not wanted
PyObject *norm_backward(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return guarded([&] {
        Args g{Norm::kCall, args, n};
        g.expect(13);
        Norm op;
        Tensor dy = g.tensor();
        const Tensor x = g.tensor();
        const Maybe residual = g.maybe(), weight = g.maybe(), bias = g.maybe();
        Tensor stats = g.tensor();
        const long long groups = g.integer();
        const double eps = g.real();
        op.take(x, residual, weight, bias, groups, eps, static_cast<int>(g.integer()));
        const Maybe dy_ = dy, stats_ = stats;
        const OnDevice on(Norm::kCall, x, {&residual, &weight, &bias, &dy_, &stats_});
        op.lay_out();
        dy = in_rows(dy, &op.a.dy);
        op.a.stats = stats.data_ptr<double>();
        Maybe dx, dres, dw, db;
        if (g.truth()) {
            dx = empty_rows(x);
            rows_of(*dx, &op.a.dx);
        }
        if (g.truth()) {
            dres = empty_rows(x);
            rows_of(*dres, &op.a.dresidual);
        }
        if (g.truth()) { dw = at::empty_like(*op.weight); }
        if (g.truth()) { db = at::empty_like(*op.bias); }
        op.a.dweight = ptr_of(dw);
        op.a.dbias = ptr_of(db);
        Tensor work = bytes_like(x, stdmlc_norm_workspace(&op.a, 1));
        op.a.workspace = work.data_ptr();
        int rc;
        WITHOUT_GIL(rc, stdmlc_norm_backward(&op.a, on.index(), on.stream()));
        done(rc);
        return tuple_of({dx, dres, dw, db});
    });
}

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
    Tensor logits, top, index;
    Maybe labels;

    void take(const Tensor &logits_, const Tensor &top_, const Tensor &index_, const Maybe &labels_, double temperature,
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
            refuse(kCall, "teacher_index must be int32 or int64", PyExc_TypeError);
        }
        if (labels) {
            if (labels->sizes() != logits.sizes().slice(0, logits.dim() - 1)) {
                refuse(kCall, "one label for each row expected, got " + shape_of(*labels) + " for " + shape_of(logits));
            }
            if (labels->scalar_type() != at::kLong && labels->scalar_type() != at::kInt) {
                refuse(kCall, "labels must be int32 or int64", PyExc_TypeError);
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
        if (labels) {
            labels = labels->to(at::kLong).contiguous();
            d.labels = labels->data_ptr();
        }
    }
};

// (logits, teacher_logits, teacher_index, labels | None, temperature, alpha, ignore_index, reduction) ->
// (loss, row statistics)
PyObject *distill_forward(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return guarded([&] {
        Args g{Distill::kCall, args, n};
        g.expect(8);
        Distill op;
        const Tensor logits = g.tensor(), top = g.tensor(), index = g.tensor();
        const Maybe labels = g.maybe(), top_ = top, index_ = index;
        const double temperature = g.real(), alpha = g.real();
        const long long ignore = g.integer();
        op.take(logits, top, index, labels, temperature, alpha, ignore, static_cast<int>(g.integer()));
        const OnDevice on(Distill::kCall, logits, {&top_, &index_, &labels});
        op.lay_out();
        const auto f32 = logits.options().dtype(at::kFloat).requires_grad(false);
        Tensor stats = at::empty({op.d.rows, 4}, f32);
        Tensor loss = op.d.reduction == 0 ? at::empty(logits.sizes().slice(0, logits.dim() - 1), f32) : at::empty({}, f32);
        op.d.row_stats = stats.data_ptr<float>();
        op.d.loss = loss.data_ptr<float>();
        Tensor work = bytes_like(logits, stdmlc_distill_workspace(&op.d));
        op.d.workspace = work.data_ptr();
        int rc;
        WITHOUT_GIL(rc, stdmlc_distill_forward(&op.d, on.index(), on.stream()));
        done(rc);
        return tuple_of({loss, stats});
    });
}

// (dloss, logits, teacher_logits, teacher_index, labels | None, row statistics, temperature, alpha, ignore_index,
// reduction) -> dlogits
PyObject *distill_backward(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return guarded([&] {
        Args g{Distill::kCall, args, n};
        g.expect(10);
        Distill op;
        Tensor dloss = g.tensor();
        const Tensor logits = g.tensor(), top = g.tensor(), index = g.tensor();
        const Maybe labels = g.maybe();
        Tensor stats = g.tensor();
        const Maybe dloss_ = dloss, top_ = top, index_ = index, stats_ = stats;
        const double temperature = g.real(), alpha = g.real();
        const long long ignore = g.integer();
        op.take(logits, top, index, labels, temperature, alpha, ignore, static_cast<int>(g.integer()));
        const OnDevice on(Distill::kCall, logits, {&dloss_, &top_, &index_, &labels, &stats_});
        op.lay_out();
        dloss = dloss.to(at::kFloat).contiguous();
        Tensor dlogits = at::empty(logits.sizes(), logits.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous));
        op.d.dloss = dloss.data_ptr<float>();
        op.d.dloss_row = op.d.reduction == 0 ? 1 : 0;
        op.d.row_stats = stats.data_ptr<float>();
        op.d.dlogits = dlogits.data_ptr();
        int rc;
        WITHOUT_GIL(rc, stdmlc_distill_backward(&op.d, on.index(), on.stream()));
        done(rc);
        return THPVariable_Wrap(dlogits);
    });
}

// ------------------------------------------------------------ gated projection
struct Gated {
    static constexpr const char *kCall = "gated_linear";
    stdmlc_gated a{};
    Tensor x, w_gate, w_up;
    Maybe b_gate, b_up;

    void take(const Tensor &x_, const Tensor &w_gate_, const Tensor &w_up_, const Maybe &b_gate_, const Maybe &b_up_,
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
        if (b_gate.has_value() != b_up.has_value()) { refuse(kCall, "both biases or none"); }
        for (const Maybe *b : {&b_gate, &b_up}) {
            if (*b && ((*b)->dim() != 1 || (*b)->size(0) != a.ffn)) {
                refuse(kCall, "biases of (" + std::to_string(a.ffn) + ",) expected, got " + shape_of(**b));
            }
        }
        const Maybe wg = w_gate, wu = w_up;
        for (const Maybe *t : std::initializer_list<const Maybe *>{&wg, &wu, &b_gate, &b_up}) {
            if (*t && (*t)->scalar_type() != x.scalar_type()) {
                refuse(kCall, "weights and biases must have the input's dtype", PyExc_TypeError);
            }
        }
        a.act = act;
    }
    void lay_out()
    {
        const void *p;
        x = matrix_of(x, &p, &a.x_row);
        a.x = p;
        w_gate = matrix_of(w_gate, &p, &a.w_gate_row);
        a.w_gate = p;
        w_up = matrix_of(w_up, &p, &a.w_up_row);
        a.w_up = p;
        for (Maybe *b : {&b_gate, &b_up}) {
            if (*b) { *b = (*b)->contiguous(); }
        }
        a.b_gate = ptr_of(b_gate);
        a.b_up = ptr_of(b_up);
    }
};

// (x, w_gate, w_up, b_gate | None, b_up | None, activation, whether a backward pass follows) -> (h, saved | None)
PyObject *gated_forward(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return guarded([&] {
        Args g{Gated::kCall, args, n};
        g.expect(7);
        Gated op;
        const Tensor x = g.tensor(), wg = g.tensor(), wu = g.tensor();
        const Maybe bg = g.maybe(), bu = g.maybe(), wg_ = wg, wu_ = wu;
        op.take(x, wg, wu, bg, bu, static_cast<int>(g.integer()));
        const OnDevice on(Gated::kCall, x, {&wg_, &wu_, &bg, &bu});
        op.lay_out();
        std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
        shape.back() = op.a.ffn;
        Tensor h = at::empty(shape, x.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous));
        op.a.h = h.data_ptr();
        Maybe saved;
        if (g.truth()) {
            saved = bytes_like(x, stdmlc_gated_saved(&op.a));
            op.a.saved = saved->data_ptr();
        }
        Tensor work = bytes_like(x, stdmlc_gated_workspace(&op.a, 0));
        op.a.workspace = work.data_ptr();
        int rc;
        WITHOUT_GIL(rc, stdmlc_gated_forward(&op.a, on.index(), on.stream()));
        done(rc);
        return tuple_of({h, saved});
    });
}

// (dh, x, w_gate, w_up, b_gate | None, b_up | None, saved, activation, want dx, want dw_gate, want dw_up, want
// db_gate, want db_up) -> those
PyObject *gated_backward(PyObject *, PyObject *const *args, Py_ssize_t n)
{
    return guarded([&] {
        Args g{Gated::kCall, args, n};
        g.expect(13);
        Gated op;
        Tensor dh = g.tensor();
        const Tensor x = g.tensor(), wg = g.tensor(), wu = g.tensor();
        const Maybe bg = g.maybe(), bu = g.maybe();
        Tensor saved = g.tensor();
        const Maybe dh_ = dh, wg_ = wg, wu_ = wu, saved_ = saved;
        op.take(x, wg, wu, bg, bu, static_cast<int>(g.integer()));
        const OnDevice on(Gated::kCall, x, {&dh_, &wg_, &wu_, &bg, &bu, &saved_});
        op.lay_out();
        dh = matrix_of(dh, &op.a.dh, &op.a.dh_row);
        op.a.saved = saved.data_ptr();
        const auto packed = x.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous);
        Maybe dx, dwg, dwu, dbg, dbu;
        if (g.truth()) { dx = at::empty(x.sizes(), packed); }
        if (g.truth()) { dwg = at::empty(wg.sizes(), packed); }
        if (g.truth()) { dwu = at::empty(wg.sizes(), packed); }
        if (g.truth()) { dbg = at::empty({op.a.ffn}, packed); }
        if (g.truth()) { dbu = at::empty({op.a.ffn}, packed); }
        op.a.dx = ptr_of(dx);
        op.a.dw_gate = ptr_of(dwg);
        op.a.dw_up = ptr_of(dwu);
        op.a.db_gate = ptr_of(dbg);
        op.a.db_up = ptr_of(dbu);
        Tensor work = bytes_like(x, stdmlc_gated_workspace(&op.a, 1));
        op.a.workspace = work.data_ptr();
        int rc;
        WITHOUT_GIL(rc, stdmlc_gated_backward(&op.a, on.index(), on.stream()));
        done(rc);
        return tuple_of({dx, dwg, dwu, dbg, dbu});
    });
}

PyMethodDef kMethods[] = {
    {"norm_forward", reinterpret_cast<PyCFunction>(norm_forward), METH_FASTCALL, nullptr},
    {"norm_backward", reinterpret_cast<PyCFunction>(norm_backward), METH_FASTCALL, nullptr},
    {"distill_forward", reinterpret_cast<PyCFunction>(distill_forward), METH_FASTCALL, nullptr},
    {"distill_backward", reinterpret_cast<PyCFunction>(distill_backward), METH_FASTCALL, nullptr},
    {"gated_forward", reinterpret_cast<PyCFunction>(gated_forward), METH_FASTCALL, nullptr},
    {"gated_backward", reinterpret_cast<PyCFunction>(gated_backward), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
}  // namespace

PyMethodDef *train_methods() { return kMethods; }
