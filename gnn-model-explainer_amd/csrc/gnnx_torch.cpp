// gnnx_torch.cpp — the encoder-layer operators (include/gnnx.h, csrc/gnnx_ops.hip) as functions of torch tensors and nodes of its autograd graph: checks of
// arguments, outputs and scratch from torch's allocator, the current stream of the tensor's device.  The smallest calls take microseconds on the GPU; the same in
// Python (checks, ctypes, autograd.Function) took 12 to 15 us a call and 150 us a training step on the host, this takes a third.  ops.py is the public face.
#include <torch/extension.h>

#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <dlfcn.h>

#include <cstdint>
#include <mutex>
#include <optional>
#include <sstream>
#include <string>
#include <tuple>

#include "../../include/gnnx.h"

namespace {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

// ---- the library behind the calls ----
struct Library {
    decltype(&gnnx_layer_norm_forward) norm_forward = nullptr;
    decltype(&gnnx_layer_norm_backward) norm_backward = nullptr;
    decltype(&gnnx_layer_norm_workspace_bytes) workspace_bytes = nullptr;
    decltype(&gnnx_dropout) dropout = nullptr;
    decltype(&gnnx_last_error) last_error = nullptr;
    bool host = false;      // the emulator build: host tensors
} g_lib;
PyObject* g_error_class = nullptr;      // engine.GnnxError

template <class F>
void symbol(void* handle, const char* name, F* out) {
    *out = reinterpret_cast<F>(dlsym(handle, name));
    if (!*out) throw py::value_error(std::string(name) + " is not in the library");
}
void use_library(const std::string& path, bool host, py::object error_class) {
    void* h = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
    if (!h) throw std::runtime_error(dlerror());
    Library l;
    symbol(h, "gnnx_layer_norm_forward", &l.norm_forward);
    symbol(h, "gnnx_layer_norm_backward", &l.norm_backward);
    symbol(h, "gnnx_layer_norm_workspace_bytes", &l.workspace_bytes);
    symbol(h, "gnnx_dropout", &l.dropout);
    symbol(h, "gnnx_last_error", &l.last_error);
    l.host = host;
    g_lib = l;
    g_error_class = error_class.release().ptr();
}

// one call into the library with x's device current, on its current stream
template <class F>
void call(const Tensor& x, F&& f) {
    int rc;
    if (x.is_cuda()) {
        const c10::DeviceGuard guard(x.device());
        rc = f(static_cast<void*>(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(x.device().index()).stream()));
    } else {
        rc = f(nullptr);
    }
    if (rc == 0) return;
    if (PyGILState_Check()) {
        PyErr_SetString(g_error_class, g_lib.last_error());
        throw py::error_already_set();
    }
    TORCH_CHECK(false, g_lib.last_error());      // (a thread of the autograd engine)
}

// ---- arguments ----
template <class... A>
std::string text(const A&... a) {
    std::ostringstream s;
    (s << ... << a);
    return s.str();
}

int type_of(const Tensor& x) {
    switch (x.scalar_type()) {
        case at::kFloat: return GNNX_F32;
        case at::kBFloat16: return GNNX_BF16;
        case at::kHalf: return GNNX_F16;
        default: return -1;
    }
}

[[noreturn]] void not_implemented(const std::string& what) {
    if (PyGILState_Check()) {
        PyErr_SetString(PyExc_NotImplementedError, what.c_str());
        throw py::error_already_set();
    }
    C10_THROW_ERROR(NotImplementedError, what);      // (a thread of the autograd engine)
}

// forward-mode derivatives would be lost without a word
void no_tangent(const char* name, const Tensor& t) {
    if (t._fw_grad(/*level=*/0).defined()) not_implemented(text(name, " carries a forward-mode derivative, which the operators do not propagate"));
}

// A tensor that stands for others or for a computation (torch.func's batched and differentiated tensors, fake and functional ones, wrapper subclasses), or a sparse one,
// has no memory of its own on its device; its null pointer would be read as an argument that is not there.
bool has_memory(const Tensor& t) {
    const c10::TensorImpl* impl = t.unsafeGetTensorImpl();
    return !impl->key_set().has(c10::DispatchKey::Functionalize) && impl->has_storage() && impl->storage().device() == t.device();
}
void needs_memory(const char* name, const Tensor& t) {
    if (!has_memory(t)) not_implemented(text(name, " is a tensor without memory of its own (sparse, batched, fake, functional or wrapped), which the operators cannot read"));
}
// ... nor has torch's zero tensor, whose elements are known without it; and a view like the imaginary part of a conjugate has its elements' signs elsewhere.
Tensor materialized(const Tensor& t) { return !t.defined() ? t : t._is_zerotensor() ? at::zeros(t.sizes(), t.options()) : t.resolve_neg(); }

Tensor input(const char* name, const py::object& o) {
    if (!THPVariable_Check(o.ptr()) || type_of(THPVariable_Unpack(o.ptr())) < 0)
        throw py::type_error(text(name, " must be a float32, bfloat16 or float16 tensor, got ",
                                  THPVariable_Check(o.ptr()) ? std::string(c10::toString(THPVariable_Unpack(o.ptr()).scalar_type())) : std::string(Py_TYPE(o.ptr())->tp_name)));
    const Tensor& x = THPVariable_Unpack(o.ptr());
    if (x.dim() < 1) throw py::value_error(text(name, " needs at least one dimension"));
    if (g_lib.host ? !x.is_cpu() : !x.is_cuda()) throw std::runtime_error(text("the operators run on MI355X only (no CPU fallback): got a tensor on ", x.device()));
    if (x.layout() != at::kStrided || x.is_nested()) throw py::type_error(text(name, " must be a dense tensor"));
    needs_memory(name, x);
    no_tangent(name, x);
    return x;
}

Tensor parameter(const char* name, const py::object& o, const Tensor& x) {
    if (o.is_none()) return Tensor();
    if (!THPVariable_Check(o.ptr())) throw py::type_error(text(name, " must be float32 or of x's type, got ", Py_TYPE(o.ptr())->tp_name));
    const Tensor& p = THPVariable_Unpack(o.ptr());
    if (p.scalar_type() != at::kFloat && p.scalar_type() != x.scalar_type())
        throw py::type_error(text(name, " must be float32 or of x's type ", x.scalar_type(), ", got ", p.scalar_type()));
    if (p.dim() != 1 || p.size(0) != x.size(-1)) throw py::value_error(text(name, " must have shape (", x.size(-1), ",), got ", p.sizes()));
    if (p.device() != x.device()) throw py::value_error(text(name, " is on ", p.device(), ", x on ", x.device()));
    needs_memory(name, p);
    no_tangent(name, p);
    return p;
}

Tensor like(const char* name, const py::object& o, const Tensor& x, at::IntArrayRef shape, at::ScalarType type) {
    if (o.is_none()) return Tensor();
    if (!THPVariable_Check(o.ptr())) throw py::type_error(text(name, " must be a tensor, got ", Py_TYPE(o.ptr())->tp_name));
    const Tensor& t = THPVariable_Unpack(o.ptr());
    if (t.sizes() != shape || t.scalar_type() != type || t.device() != x.device())
        throw py::value_error(text(name, " must be ", shape, " ", type, " on ", x.device(), ", got ", t.sizes(), " ", t.scalar_type(), " on ", t.device()));
    needs_memory(name, t);
    no_tangent(name, t);
    return t;
}

int64_t integer(const char* name, const py::object& o, int64_t most) {
    const py::object n = py::reinterpret_steal<py::object>(PyNumber_Index(o.ptr()));
    if (!n) throw py::error_already_set();
    int over = 0;
    const long long v = PyLong_AsLongLongAndOverflow(n.ptr(), &over);
    if (over || v < 0 || v > most) throw py::value_error(text(name, " must be in [0, ", most, "], got ", std::string(py::str(n))));
    return v;
}

struct Drop {
    gnnx_drop c{};
    Tensor state;      // (seed, step) on the device, or undefined
    const gnnx_drop* get() {
        c.state = state.defined() ? state.const_data_ptr<int64_t>() : nullptr;
        return &c;
    }
};
Drop drop_of(const Tensor& x, double p, const py::object& seed, const py::object& step, const py::object& row_offset) {
    Drop d;
    if (!(p >= 0.0 && p <= 1.0)) throw py::value_error(text("p must be in [0, 1], got ", p));
    d.c.p = p;
    d.c.step = (uint32_t)integer("step", step, UINT32_MAX);
    d.c.row_offset = integer("row_offset", row_offset, (int64_t(1) << 62) - 1);
    if (THPVariable_Check(seed.ptr())) {
        d.state = THPVariable_Unpack(seed.ptr());
        if (d.state.scalar_type() != at::kLong || d.state.dim() != 1 || d.state.size(0) != 2 || !d.state.is_contiguous() || d.state.device() != x.device())
            throw py::value_error(text("a seed tensor must be two contiguous int64 (seed, step) on x's device ", x.device(), ", got ", d.state.sizes(), " ",
                                       d.state.scalar_type(), " on ", d.state.device()));
        needs_memory("a seed tensor", d.state);
        d.state = materialized(d.state);
    } else {
        d.c.seed = (uint64_t)integer("seed", seed, INT64_MAX);
    }
    return d;
}

// x as a matrix over its last dimension; a copy where its rows are not evenly spaced
struct Rows {
    Tensor t;
    int64_t rows = 0, cols = 0, stride = 0;
    const void* data() const { return t.defined() ? t.const_data_ptr() : nullptr; }
};
Rows rows_of(const Tensor& given) {
    Rows m;
    if (!given.defined()) return m;
    const Tensor x = materialized(given);
    m.cols = x.size(-1);
    m.rows = m.cols ? x.numel() / m.cols : 0;
    m.stride = m.cols;
    m.t = x;
    if (x.is_contiguous()) return m;
    if (m.cols == 1 || x.stride(-1) == 1) {
        int64_t size = 1, step = 0;      // rows so far, from the innermost leading dimension outwards, and their spacing
        bool even = true;
        for (int64_t i = x.dim() - 2; i >= 0 && even; --i) {
            if (x.size(i) == 1) continue;
            if (size == 1) step = x.stride(i);
            else if (x.stride(i) != step * size) even = false;
            size *= x.size(i);
        }
        if (even) {
            if (size > 1) m.stride = step;
            return m;
        }
    }
    m.t = x.contiguous();
    return m;
}

Tensor empty_as(const Tensor& x) { return at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous)); }
Tensor workspace(const Tensor& x, size_t bytes) { return bytes ? at::empty({(int64_t)bytes}, x.options().dtype(at::kByte)) : Tensor(); }

// ---- layer norm (drop: with the dropped output) ----
struct NormCall {
    gnnx_norm n{};
    Rows x;
    Tensor w, b;
    NormCall(const Tensor& xt, const Tensor& weight, const Tensor& bias, at::ScalarType param_type, bool relu) : x(rows_of(xt)) {
        n.type = type_of(xt);
        n.w_is_f32 = param_type == at::kFloat;
        n.rows = x.rows;
        n.cols = x.cols;
        n.x_stride = x.stride;
        n.x = x.data();
        if (weight.defined()) {
            w = materialized(weight).contiguous();
            n.w = w.const_data_ptr();
        }
        if (bias.defined()) {
            b = materialized(bias).contiguous();
            n.b = b.const_data_ptr();
        }
        n.relu = relu;
    }
};

struct NormOut { Tensor y, d; };
NormOut norm_forward(const Tensor& x, const Tensor& w, const Tensor& b, double eps, bool relu, Drop* drop, float* mean, float* rstd) {
    NormCall c(x, w, b, (w.defined() ? w : b.defined() ? b : x).scalar_type(), relu);
    NormOut out{empty_as(x), drop ? empty_as(x) : Tensor()};
    c.n.y = out.y.data_ptr();
    c.n.d = drop ? out.d.data_ptr() : nullptr;
    c.n.mean = mean;
    c.n.rstd = rstd;
    c.n.eps = (float)eps;
    const size_t bytes = g_lib.workspace_bytes(c.n.type, c.n.rows, c.n.cols, 0);
    const Tensor ws = workspace(x, bytes);
    call(x, [&](void* s) { return g_lib.norm_forward(&c.n, drop ? drop->get() : nullptr, bytes ? ws.data_ptr() : nullptr, bytes, s); });
    return out;
}

struct NormGrads { Tensor dx, dw, db; };
NormGrads norm_backward(const Tensor& dy, const Tensor& dd, const Tensor& x, const float* mean, const float* rstd, const Tensor& w, bool relu, Drop* drop, bool need_dw,
                        bool need_db, at::ScalarType param_type) {
    NormCall c(x, w, Tensor(), param_type, relu);
    const Rows g = rows_of(dy), e = rows_of(dd);
    c.n.dy = g.data();
    c.n.dy_stride = g.stride;
    c.n.dd = e.data();
    c.n.dd_stride = e.stride;
    c.n.mean = const_cast<float*>(mean);
    c.n.rstd = const_cast<float*>(rstd);
    NormGrads out;
    out.dx = empty_as(x);
    c.n.dx = out.dx.data_ptr();
    const auto params = x.options().dtype(param_type);
    if (need_dw) c.n.dw = (out.dw = at::empty({c.n.cols}, params)).data_ptr();
    if (need_db) c.n.db = (out.db = at::empty({c.n.cols}, params)).data_ptr();
    const size_t bytes = g_lib.workspace_bytes(c.n.type, c.n.rows, c.n.cols, 1);
    const Tensor ws = workspace(x, bytes);
    const gnnx_drop* d = e.t.defined() ? drop->get() : nullptr;
    call(x, [&](void* s) { return g_lib.norm_backward(&c.n, d, bytes ? ws.data_ptr() : nullptr, bytes, s); });
    return out;
}

Tensor dropout_of(const Tensor& x, Drop& d) {
    const Rows m = rows_of(x);
    const Tensor y = empty_as(x);
    call(x, [&](void* s) { return g_lib.dropout(type_of(x), m.rows, m.cols, m.data(), m.stride, y.data_ptr(), d.get(), s); });
    return y;
}

// ---- autograd ----
// Gradients that were asked for with create_graph: right as they are, an error where they would be differentiated.
variable_list once_differentiable(variable_list&& grads, const char* name) {
    if (!at::GradMode::is_enabled()) return std::move(grads);
    for (auto& g : grads)
        if (g.defined()) g = g.detach().requires_grad_();
    auto error = std::make_shared<torch::autograd::DelayedError>(text("trying to differentiate twice a function that was marked with once_differentiable: ", name),
                                                                 (int64_t)grads.size());
    return (*error)(std::move(grads));
}

struct NormNode : torch::autograd::Node {
    SavedVariable x, w, seed;
    Tensor stats;      // [2, rows]: the node's own
    gnnx_drop drop{};
    bool relu = false, dropped = false;
    at::ScalarType param_type = at::kFloat;
    std::string name() const override { return dropped ? "GnnxLayerNormDropoutBackward" : "GnnxLayerNormBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        x.reset_data();
        w.reset_data();
        seed.reset_data();
        stats.reset();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        const Tensor dy = grads[0], dd = dropped ? grads[1] : Tensor();
        if (!dy.defined() && !dd.defined()) return variable_list(3);
        for (const Tensor& g : {dy, dd})
            if (g.defined()) {
                needs_memory("a gradient", g);
                no_tangent("a gradient", g);
            }
        const Tensor xs = x.unpack(), ws = w.unpack();
        Drop d;
        d.c = drop;
        if (dropped) d.state = seed.unpack();
        const float* st = stats.const_data_ptr<float>();
        NormGrads g = norm_backward(dy, dd, xs, st, st + stats.size(1), ws, relu, &d, task_should_compute_output(1), task_should_compute_output(2), param_type);
        if (!task_should_compute_output(0)) g.dx.reset();
        return once_differentiable({g.dx, g.dw, g.db}, "layer_norm");
    }
};

struct DropoutNode : torch::autograd::Node {
    SavedVariable seed;
    gnnx_drop drop{};
    std::string name() const override { return "GnnxDropoutBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        seed.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        if (!grads[0].defined()) return variable_list(1);
        needs_memory("a gradient", grads[0]);
        no_tangent("a gradient", grads[0]);
        Drop d;
        d.c = drop;
        d.state = seed.unpack();
        return once_differentiable({dropout_of(grads[0], d)}, "dropout");
    }
};

NormOut norm_differentiable(const Tensor& x, const Tensor& w, const Tensor& b, double eps, bool relu, Drop* drop) {
    if (!torch::autograd::compute_requires_grad(x, w, b)) return norm_forward(x, w, b, eps, relu, drop, nullptr, nullptr);
    const int64_t rows = x.numel() / x.size(-1);
    std::shared_ptr<NormNode> node(new NormNode(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, w, b));
    node->stats = at::empty({2, rows}, x.options().dtype(at::kFloat));
    float* st = node->stats.data_ptr<float>();
    NormOut out;
    {
        const at::AutoDispatchBelowADInplaceOrView below;
        out = norm_forward(x, w, b, eps, relu, drop, st, st + rows);
    }
    node->x = SavedVariable(x, false);
    node->w = SavedVariable(w, false);
    if (drop) {
        node->dropped = true;
        node->drop = drop->c;
        node->seed = SavedVariable(drop->state, false);      // a seed tensor that was advanced before the backward pass is an error, like any saved tensor
    }
    node->relu = relu;
    node->param_type = (w.defined() ? w : b.defined() ? b : x).scalar_type();
    torch::autograd::set_history(out.y, node);
    if (drop) torch::autograd::set_history(out.d, node);
    return out;
}

// ---- the functions of ops.py ----
struct NormInputs { Tensor x, w, b; };
NormInputs norm_inputs(const py::object& x, const py::object& weight, const py::object& bias, double eps) {
    NormInputs i{input("x", x)};
    if (i.x.size(-1) < 1) throw py::value_error("layer norm over rows of no elements");
    i.w = parameter("weight", weight, i.x);
    i.b = parameter("bias", bias, i.x);
    if (i.w.defined() && i.b.defined() && i.w.scalar_type() != i.b.scalar_type())
        throw py::type_error(text("weight and bias must have one type, got ", i.w.scalar_type(), " and ", i.b.scalar_type()));
    if (!(eps >= 0.0)) throw py::value_error(text("eps must not be negative, got ", eps));
    return i;
}

Tensor layer_norm(const py::object& x, const py::object& weight, const py::object& bias, double eps, bool relu) {
    const NormInputs i = norm_inputs(x, weight, bias, eps);
    return norm_differentiable(i.x, i.w, i.b, eps, relu, nullptr).y;
}

std::tuple<Tensor, Tensor> layer_norm_dropout(const py::object& x, const py::object& weight, const py::object& bias, double p, const py::object& seed,
                                              const py::object& step, double eps, bool relu, const py::object& row_offset) {
    const NormInputs i = norm_inputs(x, weight, bias, eps);
    Drop d = drop_of(i.x, p, seed, step, row_offset);
    NormOut out = norm_differentiable(i.x, i.w, i.b, eps, relu, &d);
    return {out.y, out.d};
}

Tensor dropout(const py::object& x, double p, const py::object& seed, const py::object& step, const py::object& row_offset) {
    const Tensor t = input("x", x);
    Drop d = drop_of(t, p, seed, step, row_offset);
    if (!torch::autograd::compute_requires_grad(t)) return dropout_of(t, d);
    std::shared_ptr<DropoutNode> node(new DropoutNode(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(t));
    Tensor y;
    {
        const at::AutoDispatchBelowADInplaceOrView below;
        y = dropout_of(t, d);
    }
    node->drop = d.c;
    node->seed = SavedVariable(d.state, false);
    torch::autograd::set_history(y, node);
    return y;
}

struct Stats {
    Tensor mean, rstd;
    explicit Stats(const Tensor& x)
        : mean(at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat))), rstd(at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat))) {}
};

std::tuple<Tensor, Tensor, Tensor> layer_norm_forward(const py::object& x, const py::object& weight, const py::object& bias, double eps, bool relu) {
    const at::NoGradGuard guard;
    const NormInputs i = norm_inputs(x, weight, bias, eps);
    Stats s(i.x);
    NormOut out = norm_forward(i.x, i.w, i.b, eps, relu, nullptr, s.mean.data_ptr<float>(), s.rstd.data_ptr<float>());
    return {out.y, s.mean, s.rstd};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> layer_norm_dropout_forward(const py::object& x, const py::object& weight, const py::object& bias, double p, const py::object& seed,
                                                                      const py::object& step, double eps, bool relu, const py::object& row_offset) {
    const at::NoGradGuard guard;
    const NormInputs i = norm_inputs(x, weight, bias, eps);
    Drop d = drop_of(i.x, p, seed, step, row_offset);
    Stats s(i.x);
    NormOut out = norm_forward(i.x, i.w, i.b, eps, relu, &d, s.mean.data_ptr<float>(), s.rstd.data_ptr<float>());
    return {out.y, out.d, s.mean, s.rstd};
}

using MaybeTensor = std::optional<Tensor>;
MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : std::nullopt; }

std::tuple<MaybeTensor, MaybeTensor, MaybeTensor> backward_of(const py::object& dy, const py::object& dd, const py::object& x, const py::object& mean, const py::object& rstd,
                                                              const py::object& weight, bool relu, Drop* d, const NormInputs& i) {
    const Tensor g = like(d ? "dh" : "dy", dy, i.x, i.x.sizes(), i.x.scalar_type()), e = like("dd", dd, i.x, i.x.sizes(), i.x.scalar_type());
    if (!g.defined() && !e.defined()) throw py::value_error(d ? "dh and dd are both None" : "dy is None");
    if (mean.is_none() || rstd.is_none()) throw py::value_error("mean and rstd must be given");
    const auto lead = i.x.sizes().slice(0, i.x.dim() - 1);
    const Tensor m = materialized(like("mean", mean, i.x, lead, at::kFloat)).contiguous(), r = materialized(like("rstd", rstd, i.x, lead, at::kFloat)).contiguous();
    const bool params = i.w.defined();
    NormGrads out = norm_backward(g, e, i.x, m.const_data_ptr<float>(), r.const_data_ptr<float>(), i.w, relu, d, params, params, params ? i.w.scalar_type() : at::kFloat);
    return {maybe(out.dx), maybe(out.dw), maybe(out.db)};
}

std::tuple<MaybeTensor, MaybeTensor, MaybeTensor> layer_norm_backward(const py::object& dy, const py::object& x, const py::object& mean, const py::object& rstd,
                                                                      const py::object& weight, bool relu) {
    const at::NoGradGuard guard;
    return backward_of(dy, py::none(), x, mean, rstd, weight, relu, nullptr, norm_inputs(x, weight, py::none(), 0.0));
}

std::tuple<MaybeTensor, MaybeTensor, MaybeTensor> layer_norm_dropout_backward(const py::object& dh, const py::object& dd, const py::object& x, const py::object& mean,
                                                                              const py::object& rstd, const py::object& weight, double p, const py::object& seed,
                                                                              const py::object& step, bool relu, const py::object& row_offset) {
    const at::NoGradGuard guard;
    const NormInputs i = norm_inputs(x, weight, py::none(), 0.0);
    Drop d = drop_of(i.x, p, seed, step, row_offset);
    return backward_of(dh, dd, x, mean, rstd, weight, relu, &d, i);
}

}  // namespace

PYBIND11_MODULE(gnnx_torch, m) {
    m.def("use_library", &use_library);
    m.def("layer_norm", &layer_norm);
    m.def("layer_norm_forward", &layer_norm_forward);
    m.def("layer_norm_backward", &layer_norm_backward);
    m.def("dropout", &dropout);
    m.def("layer_norm_dropout", &layer_norm_dropout);
    m.def("layer_norm_dropout_forward", &layer_norm_dropout_forward);
    m.def("layer_norm_dropout_backward", &layer_norm_dropout_backward);
}
