// Python module _train: the training-side operators (norm.hip, linear.hip) as
// torch functions with their gradients.  The C ABI does the work; this is the
// argument checks, the allocations and the autograd nodes around it, which in
// Python cost 112 us for a small layer norm with its gradients and 10 for one
// without; here 32 or 55 to 67, by process, most of it torch's engine and its
// threads, and 5.
//
// The reference forms these operators from MLX operations under valueAndGrad
// (RWKVBlock.swift:163-307).

#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/Exceptions.h>
#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>

#include <algorithm>
#include <cstring>
#include <string>

#include "../../include/rwkv_hip.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using Guard = c10::hip::OptionalHIPGuardMasqueradingAsCUDA;

PyObject* hip_error = nullptr;   // _lib.RwkvHipError
constexpr int MAX_D = 65536;

// ───────────────────────────── checks ─────────────────────────────

[[noreturn]] void raise(PyObject* type, const std::string& msg) {
    PyErr_SetString(type, msg.c_str());
    throw python_error();
}

// A refused or failed C call, as _lib.check raises it; the backward pass runs
// without the interpreter's lock on a thread of the engine.
void check(rwkv_status st) {
    if (st == RWKV_OK) return;
    const std::string msg = rwkv_last_error();
    pybind11::gil_scoped_acquire gil;
    if (PyObject* e = PyObject_CallFunction(hip_error, "is", (int)st, msg.c_str())) {
        PyErr_SetObject(hip_error, e);
        Py_DECREF(e);
    }
    python_error err;
    err.persist();
    throw err;
}

std::string shape_of(at::IntArrayRef s) {
    std::string r = "(";
    for (size_t i = 0; i < s.size(); ++i) r += std::to_string(s[i]) + (s.size() == 1 ? "," : i + 1 < s.size() ? ", " : "");
    return r + ")";
}
std::string shape_of(const Tensor& t) { return shape_of(t.sizes()); }

const char* type_of(at::ScalarType t) {
    return t == at::kFloat ? "float32" : t == at::kBFloat16 ? "bfloat16" : t == at::kHalf ? "float16" : at::toString(t);
}

bool float_ok(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf; }

rwkv_dtype dt_of(at::ScalarType t) { return t == at::kFloat ? RWKV_F32 : t == at::kBFloat16 ? RWKV_BF16 : RWKV_F16; }

bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw python_error();   // an array of several, say
    return v == 1;
}

// The tensor behind an argument; undefined for None where that is allowed.
Tensor tensor_arg(PyObject* o, const char* what, bool optional = false) {
    if (optional && o == Py_None) return {};
    if (!THPVariable_Check(o)) raise(PyExc_TypeError, std::string(what) + " must be a tensor, got " + Py_TYPE(o)->tp_name);
    Tensor t = THPVariable_Unpack(o);
    if (!float_ok(t.scalar_type()))
        raise(PyExc_TypeError, std::string(what) + " must be float32, bfloat16 or float16, got " + type_of(t.scalar_type()));
    return t;
}

// A result without a tangent would read as a derivative of zero; for a
// gradient's input as for the call's.
void no_tangent(const char* what, std::initializer_list<const Tensor*> inputs) {
    for (const Tensor* t : inputs)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), what,
                                    ": forward-mode derivatives are not available");
}

// Calls here go past torch's dispatcher: a traced one would be a constant, and
// a tensor of a transform or of a class with a dispatch of its own is not the
// memory that it stands for.
void plain_call(const char* what, std::initializer_list<const Tensor*> inputs) {
    using c10::DispatchKey;
    using c10::impl::TorchDispatchModeKey;
    constexpr c10::DispatchKeySet wrapped({DispatchKey::Python, DispatchKey::Functionalize, DispatchKey::FuncTorchBatched,
                                           DispatchKey::FuncTorchGradWrapper});
    bool ok = !c10::impl::tls_is_dispatch_key_included(DispatchKey::Tracer);
    for (const TorchDispatchModeKey k : {TorchDispatchModeKey::FAKE, TorchDispatchModeKey::PROXY, TorchDispatchModeKey::FUNCTIONAL})
        ok = ok && !c10::impl::TorchDispatchModeTLS::get_mode(k).has_value();
    for (const Tensor* t : inputs) ok = ok && (!t->defined() || !t->key_set().has_any(wrapped));
    TORCH_CHECK_NOT_IMPLEMENTED(ok, what, ": not available under tracing or function transforms");
}

void need_device(const Tensor& x, const char* what) {
    if (!x.is_cuda())
        raise(PyExc_ValueError, std::string(what) + " must live on a ROCm device, got " + x.device().str());
}

void same_device(const Tensor& x, const Tensor& t, const char* what) {
    if (t.device() != x.device())
        raise(PyExc_ValueError, std::string(what) + " is on " + t.device().str() + ", the input on " + x.device().str());
}

// ───────────────────────────── memory ─────────────────────────────

void* stream_of(const Tensor& t) {
    return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

Tensor empty(at::IntArrayRef size, at::ScalarType dt, c10::Device dev) {
    return Tensor(at::detail::empty_cuda(size, dt, dev, std::nullopt));
}

// A tensor as rows [N, D] of a pitch: where it lies if the last axis is
// contiguous and the rows evenly apart, else a copy.
struct Rows {
    Tensor t;   // holds the memory
    int64_t N, D, ld;
    const void* p() const { return t.const_data_ptr(); }
};

Rows rows_of(const Tensor& x, bool dense = false) {
    const at::IntArrayRef size = x.sizes(), stride = x.strides();
    const int64_t k = x.dim(), D = size[k - 1];
    int64_t N = 1;
    for (int64_t i = 0; i + 1 < k; ++i) N *= size[i];
    bool ok = D == 1 || stride[k - 1] == 1;
    int64_t ld = D, span = 0;   // span: where the axis above has to step
    for (int64_t i = k - 2; i >= 0 && N > 1; --i) {
        if (size[i] == 1) continue;
        if (span == 0) ld = stride[i];
        else ok = ok && stride[i] == span;
        span = stride[i] * size[i];
        if (span == 0) ok = false;
    }
    if (ok && ld >= D && !(dense && ld != D)) return {x, N, D, ld};
    return {x.detach().contiguous(), N, D, D};
}

// Operands of the products, which take rows up to a pitch; others are copied.
Rows product_rows(const Tensor& x) {
    Rows r = rows_of(x);
    if (r.ld > RWKV_LINEAR_MAX_PITCH) r = {r.t.detach().contiguous(), r.N, r.D, r.D};
    return r;
}

// Rows for the products: 16-byte aligned ones as they lie, others as a copy
// whose width is rounded up to 8, with zeros behind.
Rows aligned_rows(Rows r) {
    if (r.D % 8 == 0 && r.ld % 8 == 0 && (uintptr_t)r.p() % 16 == 0) return r;
    const int64_t W = (r.D + 7) / 8 * 8;
    Tensor t = empty({r.N, W}, r.t.scalar_type(), r.t.device());
    check(rwkv_linear_pad(r.p(), r.ld, t.data_ptr(), r.N, r.D, stream_of(r.t)));
    return {std::move(t), r.N, W, W};
}

struct Ws {
    Tensor t;
    int64_t bytes;
    Ws(int64_t n, c10::Device dev) : bytes(n) {
        if (n) t = empty({n}, at::kByte, dev);
    }
    void* p() const { return bytes ? t.data_ptr() : nullptr; }
};

template <typename T = void>
T* ptr(const Tensor& t) {
    return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}

const void* cptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }

struct Codes {
    Tensor codes, scales;
};

Codes codes_for(int64_t N, int64_t D, c10::Device dev) {
    const int64_t W = rwkv_act8_width(D);
    return {empty({N, W}, at::kChar, dev), empty({N, W / 32}, at::kByte, dev)};
}

Codes pack(const Rows& x) {
    Codes c = codes_for(x.N, x.D, x.t.device());
    check(rwkv_act8_pack(x.p(), dt_of(x.t.scalar_type()), x.ld, ptr<int8_t>(c.codes), ptr<uint8_t>(c.scales), x.N, x.D,
                         stream_of(x.t)));
    return c;
}

Tensor unpack(const Tensor& codes, const Tensor& scales, at::IntArrayRef shape, at::ScalarType dt) {
    Tensor y = empty(shape, dt, codes.device());
    check(rwkv_act8_unpack(ptr<int8_t>(codes), ptr<uint8_t>(scales), ptr(y), dt_of(dt), codes.size(0), shape.back(),
                           stream_of(codes)));
    return y;
}

bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }

// Gradients of gradients: the kernels leave no graph, so a graph through
// their results raises instead of missing a term, on the way to every input
// and to what dy was made of.
variable_list once(variable_list&& g, const Tensor& dy, const Node& node, const char* what) {
    if (!at::GradMode::is_enabled()) return std::move(g);
    torch::autograd::edge_list edges(node.next_edges());
    if (wants(dy)) edges.push_back(torch::autograd::impl::gradient_edge(dy));
    const std::shared_ptr<Node> err(
        new torch::autograd::Error(std::string(what) + ": gradients of its gradients are not available", std::move(edges)),
        torch::autograd::deleteNode);
    for (Tensor& t : g)
        if (t.defined()) {
            t = t.detach();
            torch::autograd::set_history(t, err);
        }
    return std::move(g);
}

// ───────────────────────────── layer norm ─────────────────────────────

struct NormNode : Node {
    SavedVariable x, codes, scales, stats, w;
    std::vector<int64_t> shape;
    at::ScalarType x_dt, y_dt;
    int64_t N, D;
    bool keep8;

    std::string name() const override { return "LayerNormBackward"; }

    void release_variables() override {
        for (SavedVariable* v : {&x, &codes, &scales, &stats, &w}) v->reset_data();
    }

    variable_list apply(variable_list&& grads) override {
        const bool need_x = task_should_compute_output(0), need_w = task_should_compute_output(1),
                   need_b = num_outputs() > 2 && task_should_compute_output(2);
        no_tangent("layer_norm", {&grads[0]});
        const auto self = shared_from_this();
        const Tensor st = stats.unpack(self), wt = w.unpack(self), xt = x.unpack(self), ct = codes.unpack(self),
                     sc = scales.unpack(self);
        const Guard guard(st.device());
        const auto dev = st.device();
        Tensor dyt = grads[0].defined() ? grads[0] : at::zeros(shape, st.options().dtype(y_dt));
        const Rows dy = rows_of(dyt, true);
        int64_t ld = D;
        Rows xr;
        if (!keep8) {
            xr = rows_of(xt);
            ld = xr.ld;
        }
        variable_list out(num_outputs());
        Tensor dw;
        if (need_x) out[0] = empty(shape, x_dt, dev);
        if (need_w || need_b) dw = empty({D}, wt.scalar_type(), dev);
        if (need_w) out[1] = dw;
        if (need_b) out[2] = empty({D}, wt.scalar_type(), dev);
        const Ws ws(dw.defined() ? rwkv_norm_bwd_workspace(N, D) : 0, dev);
        check(rwkv_norm_bwd(dy.p(), dt_of(y_dt), keep8 ? nullptr : xr.p(), dt_of(x_dt), ld, ptr<int8_t>(ct),
                            ptr<uint8_t>(sc), ptr<float>(st), ptr(wt), dt_of(wt.scalar_type()), ptr(out[0]), ptr(dw),
                            need_b ? ptr(out[2]) : nullptr, N, D, ws.p(), ws.bytes, stream_of(st)));
        return once(std::move(out), grads[0], *this, "layer_norm");
    }
};

// layer_norm(x, weight, bias, eps, out_dtype, keep8)
PyObject* py_layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6) raise(PyExc_TypeError, "layer_norm: six arguments");
    const Tensor x = tensor_arg(a[0], "layer_norm: x");
    Tensor w = tensor_arg(a[1], "layer_norm: weight"), b = tensor_arg(a[2], "layer_norm: bias", true);
    plain_call("layer_norm", {&x, &w, &b});
    no_tangent("layer_norm", {&x, &w, &b});
    const double eps = PyFloat_AsDouble(a[3]);
    if (PyErr_Occurred()) throw python_error();
    const auto xt = x.scalar_type();
    auto yt = xt;
    if (a[4] != Py_None) {
        if (!THPDtype_Check(a[4])) raise(PyExc_TypeError, "layer_norm: out_dtype must be a torch.dtype");
        yt = reinterpret_cast<THPDtype*>(a[4])->scalar_type;
    }
    const bool keep8 = truth(a[5]);
    if (x.dim() < 1 || x.size(-1) < 1 || x.size(-1) > MAX_D)
        raise(PyExc_ValueError, "layer_norm: the last axis must hold 1 to 65536 values, got " + shape_of(x));
    const int64_t D = x.size(-1);
    if (!float_ok(yt) || (yt != xt && xt != at::kFloat))
        raise(PyExc_TypeError, std::string("layer_norm: ") + type_of(xt) + " rows give " + type_of(xt) + ", not " + type_of(yt));
    for (const Tensor* t : {&w, &b}) {
        if (!t->defined()) continue;
        const char* name = t == &w ? "weight" : "bias";
        if (t->dim() != 1 || t->size(0) != D)
            raise(PyExc_ValueError, std::string("layer_norm: ") + name + " must be [" + std::to_string(D) + "], got " + shape_of(*t));
        if ((t->scalar_type() != at::kFloat && t->scalar_type() != xt) || t->scalar_type() != w.scalar_type())
            raise(PyExc_TypeError, std::string("layer_norm: weight and bias must share float32 or ") + type_of(xt) + ", got " +
                                       type_of(t->scalar_type()));
    }
    need_device(x, "layer_norm: x");
    same_device(x, w, "layer_norm: weight");
    if (b.defined()) same_device(x, b, "layer_norm: bias");

    const bool train = at::GradMode::is_enabled() && (wants(x) || wants(w) || wants(b));
    std::shared_ptr<NormNode> node;
    if (train) {
        node = std::shared_ptr<NormNode>(new NormNode(), torch::autograd::deleteNode);
        node->set_next_edges(b.defined() ? torch::autograd::collect_next_edges(x, w, b)
                                         : torch::autograd::collect_next_edges(x, w));
    }
    const Guard guard(x.device());
    const auto dev = x.device();
    const Rows xr = rows_of(x);
    const Tensor wc = w.is_contiguous() ? w : w.detach().contiguous();
    const Tensor bc = !b.defined() || b.is_contiguous() ? b : b.detach().contiguous();
    Tensor y = empty(x.sizes(), yt, dev), st;
    Codes c;
    if (train) {
        st = empty({xr.N, 2}, at::kFloat, dev);
        if (keep8) c = codes_for(xr.N, D, dev);
    }
    check(rwkv_norm_fwd(xr.p(), dt_of(xt), xr.ld, cptr(wc), cptr(bc), dt_of(w.scalar_type()), ptr(y), dt_of(yt),
                        ptr<float>(st), ptr<int8_t>(c.codes), ptr<uint8_t>(c.scales), xr.N, D, (float)eps, stream_of(x)));
    if (train) {
        node->shape = x.sizes().vec();
        node->x_dt = xt;
        node->y_dt = yt;
        node->N = xr.N;
        node->D = D;
        node->keep8 = keep8;
        if (!keep8) node->x = SavedVariable(xr.t, false);
        if (keep8) {
            node->codes = SavedVariable(c.codes, false);
            node->scales = SavedVariable(c.scales, false);
        }
        node->stats = SavedVariable(st, false);
        node->w = SavedVariable(wc, false);
        torch::autograd::set_history(y, node);
    }
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// ───────────────────────────── dense products ─────────────────────────────

constexpr int RELU2 = RWKV_ACT_RELU2;

// Keeps x (or its checkpoint), W, and for the activation's slope, with 8 bits
// more than the type's 16: nothing for "none"; y for bfloat16 relu² without a
// residual (relu(z) = √y); else an extra buffer of relu(z) (float16 relu² too:
// its squares underflow early) or, for tanh and sigmoid, of z; or with keep8
// the 8-bit checkpoint of z.  A result of tanh and sigmoid without a residual
// that was changed in place is refused, as torch does for its own, though only
// the count of its changes is kept.
struct LinearNode : Node {
    SavedVariable x, xc, xs, w, kept, rem, zc, zs;
    c10::VariableVersion y_version;
    int64_t y_was = -1;   // its value after the forward pass, if it is looked at
    std::vector<int64_t> x_shape, y_shape, res_shape;
    at::ScalarType dt, y_dt;
    int64_t M, N, K;
    int act, bias_at, res_at;   // outputs of the bias' and the residual's gradient, or -1
    bool from_y, x8;

    std::string name() const override { return "LinearBackward"; }

    void release_variables() override {
        for (SavedVariable* v : {&x, &xc, &xs, &w, &kept, &rem, &zc, &zs}) v->reset_data();
    }

    variable_list apply(variable_list&& grads) override {
        const bool need_x = task_should_compute_output(0), need_w = task_should_compute_output(1),
                   need_b = bias_at >= 0 && task_should_compute_output(bias_at),
                   need_r = res_at >= 0 && task_should_compute_output(res_at);
        no_tangent("linear", {&grads[0]});
        const auto self = shared_from_this();
        const Tensor wt = w.unpack(self);
        TORCH_CHECK(y_was < 0 || (int64_t)y_version.current_version() == y_was,
                    "linear: its result has been modified by an inplace operation before the backward pass");
        const auto dev = wt.device();
        const Guard guard(dev);
        const Tensor dyt = grads[0].defined() ? grads[0] : at::zeros(y_shape, wt.options().dtype(y_dt));
        variable_list out(num_outputs());
        if (need_r) out[res_at] = dyt;
        if (!need_x && !need_w && !need_b) return once(std::move(out), grads[0], *this, "linear");
        const Rows dy = rows_of(dyt);
        const Rows wr = product_rows(wt);
        const bool need_z = need_x || need_w;
        Tensor dzt = dy.t;
        int64_t ldz = dy.ld;
        // dy itself serves as dz unless it has to be multiplied, narrowed,
        // brought closer together, or laid out in whole 16-byte chunks (with
        // zeros behind an odd N)
        const bool own_z = need_z && (act != 0 || y_dt != dt || N % 8 || dy.ld % 8 || (uintptr_t)dy.p() % 16 ||
                                      dy.ld > RWKV_LINEAR_MAX_PITCH);
        if (own_z) {
            ldz = (N + 7) / 8 * 8;
            dzt = empty({M, ldz}, dt, dev);
        }
        // one workspace for the launches, which run one after another
        const Ws ws(std::max({need_b ? rwkv_linear_dact_workspace(M, N) : 0,
                              need_x ? rwkv_linear_dgrad_workspace(M, N, K) : 0,
                              need_w && M > 0 ? rwkv_linear_wgrad_workspace(M, N, K) : 0}), dev);
        void* const s = stream_of(wt);
        if (need_b) out[bias_at] = empty({N}, dt, dev);
        if (own_z || need_b) {
            const Tensor k = kept.unpack(self), r = rem.unpack(self), c = zc.unpack(self), sc = zs.unpack(self);
            check(rwkv_linear_dact(dy.p(), dy.ld, dt_of(y_dt), cptr(k), ptr<uint8_t>(r), from_y,
                                   ptr<int8_t>(c), ptr<uint8_t>(sc), (rwkv_activation)act, own_z ? ptr(dzt) : nullptr,
                                   ldz, need_b ? ptr(out[bias_at]) : nullptr, dt_of(dt), M, N, ws.p(), ws.bytes, s));
        }
        if (need_x) {
            out[0] = empty(x_shape, dt, dev);
            check(rwkv_linear_dgrad(cptr(dzt), ldz, wr.p(), wr.ld, ptr(out[0]), dt_of(dt), M, N, K, ws.p(), ws.bytes, s));
        }
        if (need_w && M == 0) {
            out[1] = at::zeros({N, K}, wt.options());
        } else if (need_w) {
            // codes hold zeros up to a multiple of 32
            const Tensor xt = x8 ? unpack(xc.unpack(self), xs.unpack(self), {M, (K + 7) / 8 * 8}, dt) : x.unpack(self);
            const Rows xr = product_rows(xt);   // (columns from K on, of a padded x, are not asked for)
            out[1] = empty({N, K}, dt, dev);
            check(rwkv_linear_wgrad(cptr(dzt), ldz, xr.p(), xr.ld, ptr(out[1]), dt_of(dt), M, N, K, ws.p(), ws.bytes, s));
        }
        return once(std::move(out), grads[0], *this, "linear");
    }
};

const char* const ACTIVATIONS[] = {"none", "relu2", "tanh", "sigmoid"};

// linear(x, weight, bias, activation, residual, keep8)
PyObject* py_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6) raise(PyExc_TypeError, "linear: six arguments");
    const Tensor x = tensor_arg(a[0], "linear: x"), w = tensor_arg(a[1], "linear: weight"),
                 b = tensor_arg(a[2], "linear: bias", true), res = tensor_arg(a[4], "linear: residual", true);
    plain_call("linear", {&x, &w, &b, &res});
    no_tangent("linear", {&x, &w, &b, &res});
    const auto dt = x.scalar_type();
    if (dt == at::kFloat) raise(PyExc_TypeError, "linear: x must be bfloat16 or float16, got float32");
    const char* name = PyUnicode_Check(a[3]) ? PyUnicode_AsUTF8(a[3]) : nullptr;
    int act = -1;
    for (int i = 0; name && i < 4; ++i)
        if (std::strcmp(name, ACTIVATIONS[i]) == 0) act = i;
    if (act < 0) raise(PyExc_ValueError, std::string("linear: activation '") + (name ? name : "?") + "' is none of none, relu2, tanh, sigmoid");
    const bool keep8 = truth(a[5]);
    if (x.dim() < 1 || w.dim() != 2 || w.size(1) != x.size(-1) || w.numel() == 0)
        raise(PyExc_ValueError, "linear: x " + shape_of(x) + " and weight " + shape_of(w) + " must be [..., K] and [N, K]");
    const int64_t N = w.size(0), K = w.size(1);
    for (const Tensor* t : {&w, &b})
        if (t->defined() && t->scalar_type() != dt)
            raise(PyExc_TypeError, std::string("linear: ") + (t == &w ? "weight" : "bias") + " is " + type_of(t->scalar_type()) +
                                       ", x " + type_of(dt));
    if (b.defined() && (b.dim() != 1 || b.size(0) != N))
        raise(PyExc_ValueError, "linear: bias must be [" + std::to_string(N) + "], got " + shape_of(b));
    c10::SmallVector<int64_t, 6> ysize(x.sizes().begin(), x.sizes().end());
    ysize.back() = N;
    auto yt = dt;
    if (res.defined()) {
        yt = res.scalar_type();
        if (yt != dt && yt != at::kFloat)
            raise(PyExc_TypeError, std::string("linear: residual must be ") + type_of(dt) + " or float32, got " + type_of(yt));
        if (res.sizes() != at::IntArrayRef(ysize))
            raise(PyExc_ValueError, "linear: residual must be " + shape_of(ysize) + ", got " + shape_of(res));
    }
    need_device(x, "linear: x");
    same_device(x, w, "linear: weight");
    if (b.defined()) same_device(x, b, "linear: bias");
    if (res.defined()) same_device(x, res, "linear: residual");

    const bool train = at::GradMode::is_enabled() && (wants(x) || wants(w) || wants(b) || wants(res));
    std::shared_ptr<LinearNode> node;
    if (train) {
        node = std::shared_ptr<LinearNode>(new LinearNode(), torch::autograd::deleteNode);
        torch::autograd::edge_list edges = torch::autograd::collect_next_edges(x, w);
        node->bias_at = node->res_at = -1;
        if (b.defined()) {
            node->bias_at = (int)edges.size();
            edges.push_back(torch::autograd::impl::gradient_edge(b));
        }
        if (res.defined()) {
            node->res_at = (int)edges.size();
            edges.push_back(torch::autograd::impl::gradient_edge(res));
        }
        node->set_next_edges(std::move(edges));
    }
    const auto dev = x.device();
    const Guard guard(dev);
    const Rows x0 = product_rows(x), w0 = product_rows(w);
    // Aligned copies, for all three products.  Not for small ones: two more
    // launches and buffers take the host 10 us, about what the pass loses on the
    // GPU at 2^30 products.  Nor for few rows, where W's copy costs more than
    // the product: 64 rows through 14000 x 4099 bf16 as they lie 51 us forward,
    // 112 backward; copied 69 (39 of them the copies) and 80; 128 rows 50 and
    // 132, 74 and 101; 512 rows 117 and 251, 104 and 176.
    const bool pad = x0.N > 128 && (double)x0.N * N * K >= 1073741824.0;
    const Rows xr = pad ? aligned_rows(x0) : x0, wr = pad ? aligned_rows(w0) : w0;
    const Tensor bc = !b.defined() || b.is_contiguous() ? b : b.detach().contiguous();
    Rows rr{};
    if (res.defined()) rr = rows_of(res);
    const int64_t M = xr.N;
    const bool z8 = train && keep8 && act != 0;
    const bool from_y = train && !z8 && act == RELU2 && !res.defined() && dt == at::kBFloat16;
    Tensor y = empty(ysize, yt, dev), aux, rem;
    Codes z;
    if (train && act != 0 && !z8) {
        rem = empty({M, N}, at::kByte, dev);
        if (!from_y) aux = empty({M, N}, dt, dev);
    }
    if (z8) z = codes_for(M, N, dev);
    const int64_t KK = xr.D;   // K, or K rounded up to 8 in both
    const Ws ws(rwkv_linear_fwd_workspace(M, N, KK), dev);
    check(rwkv_linear_fwd(xr.p(), xr.ld, wr.p(), wr.ld, cptr(bc), rr.t.defined() ? rr.p() : nullptr, rr.ld, ptr(y),
                          dt_of(yt), ptr(aux), ptr<uint8_t>(rem), ptr<int8_t>(z.codes), ptr<uint8_t>(z.scales),
                          (rwkv_activation)act, dt_of(dt), M, N, KK, ws.p(), ws.bytes, stream_of(x)));
    if (train) {
        node->x_shape = x.sizes().vec();
        node->y_shape.assign(ysize.begin(), ysize.end());
        node->dt = dt;
        node->y_dt = yt;
        node->M = M;
        node->N = N;
        node->K = K;
        node->act = act;
        node->from_y = from_y;
        node->x8 = keep8;
        node->w = SavedVariable(wr.t, false);
        if (wants(w)) {
            if (keep8) {
                const Codes c = pack(x0);
                node->xc = SavedVariable(c.codes, false);
                node->xs = SavedVariable(c.scales, false);
            } else {
                node->x = SavedVariable(xr.t, false);
            }
        }
        if (z8) {
            node->zc = SavedVariable(z.codes, false);
            node->zs = SavedVariable(z.scales, false);
        }
        if (rem.defined()) node->rem = SavedVariable(rem, false);
        if (aux.defined()) node->kept = SavedVariable(aux, false);
        torch::autograd::set_history(y, node);
        if (from_y) node->kept = SavedVariable(y, true);
        if (aux.defined() && act != RELU2 && !res.defined()) {
            node->y_version = y.unsafeGetTensorImpl()->version_counter();
            node->y_was = node->y_version.current_version();
        }
    }
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// ───────────────────────────── checkpoints ─────────────────────────────

// checkpoint8(x): (codes, scales)
PyObject* py_checkpoint8(PyObject*, PyObject* o) {
    HANDLE_TH_ERRORS
    const Tensor x = tensor_arg(o, "checkpoint8: x");
    plain_call("checkpoint8", {&x});
    if (x.dim() < 1 || x.size(-1) < 1)
        raise(PyExc_ValueError, "checkpoint8: x must have a last axis of at least 1, got " + shape_of(x));
    need_device(x, "checkpoint8: x");
    const Guard guard(x.device());
    Codes c = pack(rows_of(x));
    PyObject* r = PyTuple_New(2);
    if (!r) throw python_error();
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(c.codes)));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(c.scales)));
    return r;
    END_HANDLE_TH_ERRORS
}

// restore8(codes, scales, shape, dtype)
PyObject* py_restore8(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 4 || !THPVariable_Check(a[0]) || !THPVariable_Check(a[1]) || !PyTuple_Check(a[2]))
        raise(PyExc_TypeError, "restore8: codes, scales, shape, dtype");
    const Tensor codes = THPVariable_Unpack(a[0]), scales = THPVariable_Unpack(a[1]);
    plain_call("restore8", {&codes, &scales});
    if (!THPDtype_Check(a[3]) || !float_ok(reinterpret_cast<THPDtype*>(a[3])->scalar_type))
        raise(PyExc_TypeError, "checkpoints restore to float32, bfloat16 or float16");
    c10::SmallVector<int64_t, 6> shape;
    int64_t rows = 1;
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(a[2]); ++i) {
        shape.push_back(PyLong_AsLongLong(PyTuple_GET_ITEM(a[2], i)));
        if (PyErr_Occurred()) throw python_error();
        if (i + 1 < PyTuple_GET_SIZE(a[2])) rows *= shape.back();
    }
    if (shape.empty() || codes.dim() != 2 || scales.dim() != 2 || codes.scalar_type() != at::kChar ||
        scales.scalar_type() != at::kByte || codes.size(0) != rows || scales.size(0) != rows ||
        codes.size(1) != rwkv_act8_width(shape.back()) || scales.size(1) * 32 != codes.size(1) ||
        !codes.is_contiguous() || !scales.is_contiguous())
        raise(PyExc_ValueError, "checkpoint of " + shape_of(codes) + " codes and " + shape_of(scales) +
                                    " scales does not hold " + shape_of(shape));
    need_device(codes, "checkpoint codes");
    same_device(codes, scales, "checkpoint scales");
    const Guard guard(codes.device());
    return THPVariable_Wrap(unpack(codes, scales, shape, reinterpret_cast<THPDtype*>(a[3])->scalar_type));
    END_HANDLE_TH_ERRORS
}

// set_error(RwkvHipError)
PyObject* py_set_error(PyObject*, PyObject* type) {
    Py_INCREF(type);
    Py_XSETREF(hip_error, type);
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"layer_norm", (PyCFunction)(void (*)(void))py_layer_norm, METH_FASTCALL, nullptr},
    {"linear", (PyCFunction)(void (*)(void))py_linear, METH_FASTCALL, nullptr},
    {"checkpoint8", py_checkpoint8, METH_O, nullptr},
    {"restore8", (PyCFunction)(void (*)(void))py_restore8, METH_FASTCALL, nullptr},
    {"set_error", py_set_error, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_train", "Training-side operators with their gradients", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__train() { return PyModule_Create(&module); }
