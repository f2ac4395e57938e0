// The common call of each layer (fuselse_amd/layers.py) without the Python between
// it and the C ABI: contiguous tensors on the current device, of types that need no
// conversion.  Every function returns None for any other call, which the Python
// layer then takes (checks it, converts or refuses); results are the same, since
// both end in the same entry points.  A backward is a node of its own that runs
// without the interpreter, whose lock and cold code are most of a small one's time:
// layer norm of (129, 200) in fp32, both directions, 104 us in Python and 64 here, of
// which 50 are autograd's own; its forward alone 9.8 and 4.4.
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include "../../../include/fuselse_amd.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int code_of(at::ScalarType t) {
    switch (t) {
    case at::kFloat: return 0;
    case at::kHalf: return 1;
    case at::kBFloat16: return 2;
    default: return -1;
    }
}
int code_of(const Tensor& t) { return code_of(t.scalar_type()); }

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void check(int rc) { TORCH_CHECK(rc == 0, fl_last_error()); }

Tensor make(const Tensor& like, at::IntArrayRef sizes) { return at::empty(sizes, like.options()); }
Tensor make(const Tensor& like, at::IntArrayRef sizes, at::ScalarType type) {
    return at::empty(sizes, like.options().dtype(type));
}
Tensor workspace(const Tensor& like, size_t bytes) { return make(like, {(int64_t)bytes}, at::kByte); }
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* mut(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

// A plain tensor or parameter, not empty, contiguous, on the current device, without a
// forward-mode derivative.
bool plain(PyObject* o, Tensor& t) {
    if (!THPVariable_CheckExact(o)) return false;
    t = THPVariable_Unpack(o);
    return t.is_cuda() && t.layout() == at::kStrided && !t.is_neg() && t.is_contiguous() && t.numel() > 0 &&
           t.device().index() == c10::hip::current_device() && !t._fw_grad(0).defined();
}
bool floating(PyObject* o, Tensor& t) { return plain(o, t) && t.dim() >= 1 && code_of(t) >= 0; }
// Whether torch may follow calls by more than autograd's nodes.
bool followed() { return c10::impl::TorchDispatchModeTLS::any_modes_set() || torch::jit::tracer::isTracing(); }
bool absent(PyObject* o) { return o == Py_None; }

// A gradient as the kernels read it.
Tensor in_memory(const Tensor& g) { return g.resolve_neg().contiguous(); }

// Size of t's leading dimensions, its last, and whether both have these leading ones.
int64_t last(const Tensor& t) { return t.size(-1); }
int64_t lead(const Tensor& t) { return t.numel() / t.size(-1); }
bool same_lead(const Tensor& a, const Tensor& b) {
    return a.dim() == b.dim() && a.sizes().slice(0, a.dim() - 1) == b.sizes().slice(0, b.dim() - 1);
}
std::vector<int64_t> with_last(const Tensor& t, int64_t n) {
    std::vector<int64_t> s(t.sizes().begin(), t.sizes().end());
    s.back() = n;
    return s;
}

// Results of a backward are constants: with create_graph, those that depend on what
// requires a gradient (the upstream one, or, where `saved` says so, saved tensors) are an
// error where they are differentiated again.
variable_list once(variable_list&& out, const variable_list& grads, std::initializer_list<bool> saved = {}) {
    if (!at::GradMode::is_enabled()) return std::move(out);
    bool all = false;
    for (const Tensor& g : grads) all = all || (g.defined() && g.requires_grad());
    for (size_t i = 0; i < out.size(); ++i) {
        if (!out[i].defined() || !(all || (i < saved.size() && saved.begin()[i]))) continue;
        const auto error = std::make_shared<torch::autograd::DelayedError>(
            "trying to differentiate twice a function that is differentiable once", 1);
        out[i] = error->apply({out[i].detach().set_requires_grad(true)})[0];
    }
    return std::move(out);
}

// ---------------------------------------------------------------------------
Tensor embedding_fwd(const Tensor& weight, const Tensor& index, double scale) {
    const int64_t D = weight.size(1);
    std::vector<int64_t> sizes(index.sizes().begin(), index.sizes().end());
    sizes.push_back(D);
    Tensor out = make(weight, sizes);
    check(fl_embedding_fwd(ptr(weight), D, weight.size(0), D, code_of(weight), index.const_data_ptr<int64_t>(),
                           index.numel(), (float)scale, mut(out), stream_of(weight)));
    return out;
}

struct Embedding : torch::autograd::Function<Embedding> {
    static Tensor forward(AutogradContext* ctx, const Tensor& weight, const Tensor& index, double scale,
                          int64_t padding) {
        ctx->save_for_backward({index});
        ctx->saved_data["rows"] = weight.size(0);
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["padding"] = padding;
        return embedding_fwd(weight, index, scale);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Tensor index = ctx->get_saved_variables()[0].contiguous(), g = in_memory(grads[0]);
        const c10::DeviceGuard guard(g.device());
        const int64_t V = ctx->saved_data["rows"].toInt(), D = last(g), N = index.numel();
        Tensor dw = make(g, {V, D});
        const Tensor ws = workspace(g, fl_embedding_bwd_workspace_bytes(N, V, D));
        check(fl_embedding_bwd(ptr(g), D, index.const_data_ptr<int64_t>(), N, V, D, code_of(g),
                               (float)ctx->saved_data["scale"].toDouble(), ctx->saved_data["padding"].toInt(), mut(dw),
                               mut(ws), (size_t)ws.numel(), stream_of(g)));
        return once({dw, Tensor(), Tensor(), Tensor()}, grads);
    }
};

// embedding(index, weight, scale, padding): padding within the rows or -1
PyObject* embedding(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Tensor index, weight;
    if (n != 4 || followed() || !plain(a[0], index) || index.scalar_type() != at::kLong || !floating(a[1], weight) ||
        weight.dim() != 2)
        Py_RETURN_NONE;
    const double scale = PyFloat_AsDouble(a[2]);
    const int64_t padding = PyLong_AsLongLong(a[3]);
    if (PyErr_Occurred()) return nullptr;
    if (weight.requires_grad() && at::GradMode::is_enabled())
        return THPVariable_Wrap(Embedding::apply(weight, index, scale, padding));
    return THPVariable_Wrap(embedding_fwd(weight, index, scale));
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------
Tensor norm_fwd(const Tensor& x, const Tensor& w, const Tensor& b, double eps, Tensor* stats) {
    const int64_t N = lead(x), D = last(x);
    Tensor y = at::empty_like(x);
    if (stats) *stats = make(x, {N, 4}, at::kFloat);
    const int params = w.defined() ? code_of(w) : b.defined() ? code_of(b) : 0;
    check(fl_layer_norm_fwd(ptr(x), D, N, D, code_of(x), ptr(w), ptr(b), params, (float)eps, mut(y),
                            stats ? stats->mutable_data_ptr<float>() : nullptr, stream_of(x)));
    return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b,
                          double eps) {
        Tensor stats;
        const Tensor weight = w.value_or(Tensor()), bias = b.value_or(Tensor());
        Tensor y = norm_fwd(x, weight, bias, eps, &stats);
        ctx->save_for_backward({x, weight, stats});
        ctx->saved_data["x_grad"] = x.requires_grad();
        ctx->saved_data["w_grad"] = weight.defined() && weight.requires_grad();
        ctx->saved_data["weight"] = w.has_value();
        ctx->saved_data["bias"] = b.has_value();
        ctx->saved_data["type"] =
            (int64_t)(w ? weight.scalar_type() : b ? bias.scalar_type() : at::kFloat);
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor g = in_memory(grads[0]), x = saved[0].contiguous(), st = saved[2].contiguous();
        const Tensor w = saved[1].defined() ? saved[1].contiguous() : saved[1];
        const c10::DeviceGuard guard(g.device());
        const int64_t N = lead(x), D = last(x);
        const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
        const bool has_w = ctx->saved_data["weight"].toBool(), has_b = ctx->saved_data["bias"].toBool();
        Tensor dx, dw, db, ws;
        if (ctx->needs_input_grad(0)) dx = at::empty_like(x);
        if (has_w && ctx->needs_input_grad(1)) dw = make(x, {D}, type);
        if (has_b && ctx->needs_input_grad(has_w ? 2 : 1)) db = make(x, {D}, type);
        if (dw.defined() || db.defined()) ws = workspace(x, fl_layer_norm_bwd_workspace_bytes(N, D, code_of(x)));
        check(fl_layer_norm_bwd(ptr(g), D, ptr(x), D, N, D, code_of(x), ptr(w), code_of(type),
                                st.const_data_ptr<float>(), mut(dx), mut(dw), mut(db), mut(ws),
                                ws.defined() ? (size_t)ws.numel() : 0, stream_of(x)));
        const bool of_x = ctx->saved_data["x_grad"].toBool(), of_w = ctx->saved_data["w_grad"].toBool();
        return once({dx, dw, db, Tensor()}, grads, {of_x || of_w, of_x});
    }
};

// layer_norm(input, weight or None, bias or None, eps)
PyObject* layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Tensor x, w, b;
    if (n != 4 || followed() || !floating(a[0], x)) Py_RETURN_NONE;
    for (int i = 1; i < 3; ++i) {
        Tensor& t = i == 1 ? w : b;
        if (absent(a[i])) continue;
        if (!floating(a[i], t) || t.dim() != 1 || t.size(0) != last(x) ||
            (t.scalar_type() != x.scalar_type() && t.scalar_type() != at::kFloat))
            Py_RETURN_NONE;
    }
    if (w.defined() && b.defined() && w.scalar_type() != b.scalar_type()) Py_RETURN_NONE;
    const double eps = PyFloat_AsDouble(a[3]);
    if (PyErr_Occurred()) return nullptr;
    if (!(eps >= 0)) Py_RETURN_NONE;
    const bool needs = x.requires_grad() || (w.defined() && w.requires_grad()) || (b.defined() && b.requires_grad());
    if (needs && at::GradMode::is_enabled())
        return THPVariable_Wrap(LayerNorm::apply(x, w.defined() ? optional<Tensor>(w) : std::nullopt,
                                                 b.defined() ? optional<Tensor>(b) : std::nullopt, eps));
    return THPVariable_Wrap(norm_fwd(x, w, b, eps, nullptr));
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------
// expert_order(index, num_experts, mask or None): (position, counts, offsets)
PyObject* expert_order(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Tensor index, mask;
    if (n != 3 || followed() || !plain(a[0], index) || index.scalar_type() != at::kLong || index.dim() < 1)
        Py_RETURN_NONE;
    if (!absent(a[2]) && (!plain(a[2], mask) || mask.scalar_type() != at::kBool ||
                          mask.sizes() != index.sizes().slice(0, index.dim() - 1)))
        Py_RETURN_NONE;
    int overflow = 0;
    const int64_t experts = PyLong_AsLongLongAndOverflow(a[1], &overflow);
    if (PyErr_Occurred()) return nullptr;
    if (overflow || experts < 1 || experts > 1024) Py_RETURN_NONE;  // before results of that size are made
    const int64_t T = lead(index), K = last(index);
    Tensor position = make(index, index.sizes(), at::kInt), counts = make(index, {experts});
    Tensor offsets = make(index, {experts + 1}, at::kInt), ws;
    const size_t bytes = fl_expert_order_workspace_bytes(T, K, experts);
    if (bytes) ws = workspace(index, bytes);
    check(fl_expert_order(index.const_data_ptr<int64_t>(), T, K, experts, static_cast<const uint8_t*>(ptr(mask)),
                          position.mutable_data_ptr<int32_t>(), counts.mutable_data_ptr<int64_t>(),
                          offsets.mutable_data_ptr<int32_t>(), mut(ws), bytes, stream_of(index)));
    PyObject* out = PyTuple_New(3);
    if (!out) return nullptr;
    PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(position));
    PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(counts));
    PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(offsets));
    return out;
    END_HANDLE_TH_ERRORS
}

bool places(PyObject* o, Tensor& position) {
    return plain(o, position) && position.scalar_type() == at::kInt && position.dim() >= 1;
}

Tensor dispatch(const Tensor& x, const Tensor& position) {
    const int64_t T = lead(position), K = last(position), D = last(x);
    Tensor rows = make(x, {T * K, D});
    check(fl_expert_dispatch(ptr(x), D, T, D, code_of(x), position.const_data_ptr<int32_t>(), K, mut(rows),
                             stream_of(x)));
    return rows;
}

Tensor combine(const Tensor& rows, const Tensor& weights, const Tensor& position) {
    const int64_t T = lead(position), K = last(position), D = rows.size(1);
    Tensor out = make(rows, with_last(position, D));
    check(fl_expert_combine(ptr(rows), D, T, D, code_of(rows), position.const_data_ptr<int32_t>(), K, ptr(weights),
                            weights.defined() ? code_of(weights) : 0, mut(out), stream_of(rows)));
    return out;
}

struct Dispatch : torch::autograd::Function<Dispatch> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& position) {
        ctx->save_for_backward({position});
        return dispatch(x, position);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Tensor position = ctx->get_saved_variables()[0].contiguous(), g = in_memory(grads[0]);
        const c10::DeviceGuard guard(g.device());
        return once({combine(g, Tensor(), position), Tensor()}, grads);
    }
};

struct Combine : torch::autograd::Function<Combine> {
    static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Tensor& weights, const Tensor& position) {
        ctx->save_for_backward({rows, weights, position});
        ctx->saved_data["rows_grad"] = rows.requires_grad();
        ctx->saved_data["weights_grad"] = weights.requires_grad();
        return combine(rows, weights, position);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor g = in_memory(grads[0]), rows = saved[0].contiguous(), weights = saved[1].contiguous();
        const Tensor position = saved[2].contiguous();
        const c10::DeviceGuard guard(g.device());
        const int64_t T = lead(position), K = last(position), D = rows.size(1);
        Tensor d_rows, d_weights;
        if (ctx->needs_input_grad(0)) d_rows = at::empty_like(rows);
        if (ctx->needs_input_grad(1)) d_weights = at::empty_like(weights);
        check(fl_expert_combine_bwd(ptr(g), D, ptr(rows), D, T, D, code_of(rows), position.const_data_ptr<int32_t>(),
                                    K, ptr(weights), code_of(weights), mut(d_rows), mut(d_weights), stream_of(rows)));
        return once({d_rows, d_weights, Tensor()}, grads,
                    {ctx->saved_data["weights_grad"].toBool(), ctx->saved_data["rows_grad"].toBool()});
    }
};

// expert_dispatch(input, position)
PyObject* expert_dispatch(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Tensor x, position;
    if (n != 2 || followed() || !floating(a[0], x) || !places(a[1], position) || !same_lead(x, position))
        Py_RETURN_NONE;
    if (x.requires_grad() && at::GradMode::is_enabled()) return THPVariable_Wrap(Dispatch::apply(x, position));
    return THPVariable_Wrap(dispatch(x, position));
    END_HANDLE_TH_ERRORS
}

// expert_combine(rows, weights, position)
PyObject* expert_combine(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Tensor rows, weights, position;
    if (n != 3 || followed() || !floating(a[0], rows) || rows.dim() != 2 || !floating(a[1], weights) ||
        !places(a[2], position) || weights.sizes() != position.sizes() ||
        rows.size(0) != position.numel() ||
        (weights.scalar_type() != rows.scalar_type() && weights.scalar_type() != at::kFloat))
        Py_RETURN_NONE;
    if ((rows.requires_grad() || weights.requires_grad()) && at::GradMode::is_enabled())
        return THPVariable_Wrap(Combine::apply(rows, weights, position));
    return THPVariable_Wrap(combine(rows, weights, position));
    END_HANDLE_TH_ERRORS
}

#define FL_METHOD(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FL_METHOD(embedding),       FL_METHOD(layer_norm),     FL_METHOD(expert_order),
                         FL_METHOD(expert_dispatch), FL_METHOD(expert_combine), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_layers", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__layers(void) { return PyModule_Create(&module); }
