// Python module _train: the training-side operators (norm.hip, linear.hip, block.hip) as
// torch functions with their gradients.  The C ABI does the work; this is the
// argument checks, the allocations and the autograd nodes around it, which in
// Python cost 112 us for a small layer norm with its gradients and 10 for one
// without; here 32 or 55 to 67, by process, most of it torch's engine and its
// threads, and 5.
//
// Of these operators the reference forms the norms, the dense products, the
// residual sums and the recurrence's tail from MLX operations under valueAndGrad
// (RWKVBlock.swift:163-307).

#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
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
#include <cmath>
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
    return t.is_neg() ? t.resolve_neg() : t;   // (a view whose memory holds its negative)
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
    if (x.is_neg()) return rows_of(x.detach().resolve_neg(), dense);   // (a gradient; arguments are none)
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

// Operands of dropout, likewise.
Rows dropout_rows(const Tensor& x) {
    Rows r = rows_of(x);
    if (r.ld > RWKV_DROPOUT_MAX_PITCH) r = {r.t.detach().contiguous(), r.N, r.D, r.D};
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

// What a node keeps of a call.  A hook on saved tensors may give it back laid out
// otherwise; of another type, shape or device it is refused, before a kernel reads
// past it.
struct Saved {
    Saved() = default;
    explicit Saved(const Tensor& t, bool output = false) : v(t, output), size(t.sizes()), dt(t.scalar_type()), dev(t.device()) {}
    void reset_data() { v.reset_data(); }
    Tensor unpack(const std::shared_ptr<Node>& node) const {
        Tensor t = v.unpack(node);
        TORCH_CHECK(!t.defined() || (t.sizes() == at::IntArrayRef(size) && t.scalar_type() == dt && t.device() == dev), node->name(),
                    ": a saved tensor came back as ", type_of(t.scalar_type()), " ", shape_of(t), " on ", t.device().str(), ", not ", type_of(dt), " ",
                    shape_of(size), " on ", dev.str());
        return t;
    }
    // for what the kernels take as it lies (rows_of sees to the rest)
    Tensor dense(const std::shared_ptr<Node>& node) const {
        const Tensor t = unpack(node);
        return t.defined() && (!t.is_contiguous() || t.is_neg()) ? t.detach().resolve_neg().contiguous() : t;
    }

private:
    SavedVariable v;
    c10::SmallVector<int64_t, 4> size;
    at::ScalarType dt{};
    c10::Device dev{at::kCPU};
};

bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }

// A leaf's gradient belongs to the stream under which its node came to be.  If
// an eager graph still holds that node, a captured backward pass on another
// stream would have the engine make the one wait for the other, which the
// capture does not survive, nor the process.  Every node here looks at the leaves
// next to it, those alone that the pass goes to.
void capture_ok(const char* what, const Node& node, c10::Device dev) {
    using Stream = c10::hip::HIPStreamMasqueradingAsCUDA;
    const auto captured = [](const Stream& s) {
        if (!s.stream()) return false;   // (the default stream never is; to ask it while another is captured is an error)
        hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
        return hipStreamIsCapturing(s.stream(), &status) == hipSuccess && status != hipStreamCaptureStatusNone;
    };
    const Stream stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index());
    if (!captured(stream)) return;
    const torch::autograd::edge_list& edges = node.next_edges();
    for (size_t i = 0; i < edges.size(); ++i) {
        const torch::autograd::Edge& e = edges[i];
        if (!e.function || !node.task_should_compute_output(i)) continue;
        if (!dynamic_cast<torch::autograd::AccumulateGrad*>(e.function.get())) continue;
        const std::optional<c10::Stream> leaf = e.function->stream();
        if (!leaf || *leaf == stream.unwrap()) continue;
        TORCH_CHECK(captured(Stream(*leaf)), what,
                    ": its captured backward pass reaches a leaf that an eager graph on another stream still holds; "
                    "free that graph, or capture with leaves of their own");
    }
}

// Gradients of gradients: the kernels leave no graph, so a graph through
// their results raises instead of missing a term, on the way to every input
// and to what dy was made of.
variable_list once(variable_list&& g, std::initializer_list<const Tensor*> dys, const Node& node, const char* what) {
    if (!at::GradMode::is_enabled()) return std::move(g);
    torch::autograd::edge_list edges(node.next_edges());
    for (const Tensor* dy : dys)
        if (wants(*dy)) edges.push_back(torch::autograd::impl::gradient_edge(*dy));
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
variable_list once(variable_list&& g, const Tensor& dy, const Node& node, const char* what) {
    return once(std::move(g), {&dy}, node, what);
}

// ───────────────────────────── layer norm ─────────────────────────────

struct NormNode : Node {
    Saved x, codes, scales, stats, w;
    std::vector<int64_t> shape;
    at::ScalarType x_dt, y_dt;
    int64_t N, D;
    bool keep8;

    std::string name() const override { return "LayerNormBackward"; }

    void release_variables() override {
        for (Saved* v : {&x, &codes, &scales, &stats, &w}) v->reset_data();
    }

    variable_list apply(variable_list&& grads) override {
        const bool need_x = task_should_compute_output(0), need_w = task_should_compute_output(1),
                   need_b = num_outputs() > 2 && task_should_compute_output(2);
        no_tangent("layer_norm", {&grads[0]});
        const auto self = shared_from_this();
        const Tensor st = stats.dense(self), wt = w.dense(self), xt = x.unpack(self), ct = codes.dense(self),
                     sc = scales.dense(self);
        const auto dev = st.device();
        const Guard guard(dev);
        capture_ok("layer_norm", *this, dev);
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
        if (!keep8) node->x = Saved(xr.t);
        if (keep8) {
            node->codes = Saved(c.codes);
            node->scales = Saved(c.scales);
        }
        node->stats = Saved(st);
        node->w = Saved(wc);
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
    Saved x, xc, xs, w, kept, rem, zc, zs;
    c10::VariableVersion y_version;
    int64_t y_was = -1;   // its value after the forward pass, if it is looked at
    std::vector<int64_t> x_shape, y_shape, res_shape;
    at::ScalarType dt, y_dt;
    int64_t M, N, K;
    int act, bias_at, res_at;   // outputs of the bias' and the residual's gradient, or -1
    bool from_y, x8;

    std::string name() const override { return "LinearBackward"; }

    void release_variables() override {
        for (Saved* v : {&x, &xc, &xs, &w, &kept, &rem, &zc, &zs}) v->reset_data();
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
        capture_ok("linear", *this, dev);
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
            const Tensor k = kept.dense(self), r = rem.dense(self), c = zc.dense(self), sc = zs.dense(self);
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
            const Tensor xt = x8 ? unpack(xc.dense(self), xs.dense(self), {M, (K + 7) / 8 * 8}, dt) : x.unpack(self);
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
        node->w = Saved(wr.t);
        if (wants(w)) {
            if (keep8) {
                const Codes c = pack(x0);
                node->xc = Saved(c.codes);
                node->xs = Saved(c.scales);
            } else {
                node->x = Saved(xr.t);
            }
        }
        if (z8) {
            node->zc = Saved(z.codes);
            node->zs = Saved(z.scales);
        }
        if (rem.defined()) node->rem = Saved(rem);
        if (aux.defined()) node->kept = Saved(aux);
        torch::autograd::set_history(y, node);
        if (from_y) node->kept = Saved(y, true);
        if (aux.defined() && act != RELU2 && !res.defined()) {
            node->y_version = y.unsafeGetTensorImpl()->version_counter();
            node->y_was = node->y_version.current_version();
        }
    }
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// ───────────────────────────── gated products ─────────────────────────────

// Keeps x, W, and both pre-activations in 24 bits, as whole numbers: a hook that
// keeps floating point tensors in another type has no business with patterns.
struct GatedNode : Node {
    Saved x, w, kept, rem;
    std::vector<int64_t> x_shape, y_shape;
    at::ScalarType dt;
    int64_t M, F, K;
    rwkv_gate act;

    std::string name() const override { return "GatedLinearBackward"; }

    void release_variables() override {
        for (Saved* v : {&x, &w, &kept, &rem}) v->reset_data();
    }

    variable_list apply(variable_list&& grads) override {
        const bool need_x = task_should_compute_output(0), need_w = task_should_compute_output(1);
        no_tangent("gated_linear", {&grads[0]});
        const auto self = shared_from_this();
        const Tensor wt = w.unpack(self), k = kept.dense(self), r = rem.dense(self);
        const auto dev = wt.device();
        const Guard guard(dev);
        capture_ok("gated_linear", *this, dev);
        variable_list out(2);
        if (!need_x && !need_w) return once(std::move(out), grads[0], *this, "gated_linear");
        const Tensor dyt = grads[0].defined() ? grads[0] : at::zeros(y_shape, wt.options());
        const Rows dy = rows_of(dyt), wr = product_rows(wt);
        const int64_t N = 2 * F, ldz = (N + 7) / 8 * 8;
        const Tensor dz = empty({M, ldz}, dt, dev);
        const Ws ws(std::max(need_x ? rwkv_linear_dgrad_workspace(M, N, K) : 0,
                             need_w && M > 0 ? rwkv_linear_wgrad_workspace(M, N, K) : 0), dev);
        void* const s = stream_of(wt);
        check(rwkv_gated_dact(dy.p(), dy.ld, cptr(k), ptr<uint8_t>(r), act, ptr(dz), ldz, dt_of(dt), M, F, s));
        if (need_x) {
            out[0] = empty(x_shape, dt, dev);
            check(rwkv_linear_dgrad(cptr(dz), ldz, wr.p(), wr.ld, ptr(out[0]), dt_of(dt), M, N, K, ws.p(), ws.bytes, s));
        }
        if (need_w && M == 0) {
            out[1] = at::zeros({N, K}, wt.options());
        } else if (need_w) {
            const Rows xr = product_rows(x.unpack(self));   // (columns from K on, of a padded x, are not asked for)
            out[1] = empty({N, K}, dt, dev);
            check(rwkv_linear_wgrad(cptr(dz), ldz, xr.p(), xr.ld, ptr(out[1]), dt_of(dt), M, N, K, ws.p(), ws.bytes, s));
        }
        return once(std::move(out), grads[0], *this, "gated_linear");
    }
};

const char* const GATES[] = {"relu2", "sigmoid", "silu", "gelu_tanh"};

// gated_linear(x, weight, activation)
PyObject* py_gated_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 3) raise(PyExc_TypeError, "gated_linear: three arguments");
    const Tensor x = tensor_arg(a[0], "gated_linear: x"), w = tensor_arg(a[1], "gated_linear: weight");
    plain_call("gated_linear", {&x, &w});
    no_tangent("gated_linear", {&x, &w});
    const auto dt = x.scalar_type();
    if (dt == at::kFloat) raise(PyExc_TypeError, "gated_linear: x must be bfloat16 or float16, got float32");
    const char* name = PyUnicode_Check(a[2]) ? PyUnicode_AsUTF8(a[2]) : nullptr;
    int act = -1;
    for (int i = 0; name && i < 4; ++i)
        if (std::strcmp(name, GATES[i]) == 0) act = i;
    if (act < 0)
        raise(PyExc_ValueError, std::string("gated_linear: activation '") + (name ? name : "?") + "' is none of relu2, sigmoid, silu, gelu_tanh");
    if (x.dim() < 1 || w.dim() != 2 || w.size(1) != x.size(-1) || w.numel() == 0 || w.size(0) % 2)
        raise(PyExc_ValueError, "gated_linear: x " + shape_of(x) + " and weight " + shape_of(w) + " must be [..., K] and [2F, K]");
    const int64_t N = w.size(0), F = N / 2, K = w.size(1);
    if (w.scalar_type() != dt)
        raise(PyExc_TypeError, std::string("gated_linear: weight is ") + type_of(w.scalar_type()) + ", x " + type_of(dt));
    need_device(x, "gated_linear: x");
    same_device(x, w, "gated_linear: weight");

    const bool train = at::GradMode::is_enabled() && (wants(x) || wants(w));
    std::shared_ptr<GatedNode> node;
    if (train) {
        node = std::shared_ptr<GatedNode>(new GatedNode(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x, w));
    }
    const auto dev = x.device();
    const Guard guard(dev);
    const Rows x0 = product_rows(x), w0 = product_rows(w);
    const bool pad = x0.N > 128 && (double)x0.N * N * K >= 1073741824.0;   // as linear's
    const Rows xr = pad ? aligned_rows(x0) : x0, wr = pad ? aligned_rows(w0) : w0;
    const int64_t M = xr.N, KK = xr.D;
    c10::SmallVector<int64_t, 6> ysize(x.sizes().begin(), x.sizes().end());
    ysize.back() = F;
    Tensor y = empty(ysize, dt, dev), kept, rem;
    if (train) {
        kept = empty({M, N}, at::kShort, dev);
        rem = empty({M, N}, at::kByte, dev);
    }
    const Ws ws(rwkv_gated_fwd_workspace(M, F, KK), dev);
    check(rwkv_gated_fwd(xr.p(), xr.ld, wr.p(), wr.ld, ptr(y), ptr(kept), ptr<uint8_t>(rem), (rwkv_gate)act, dt_of(dt), M, F, KK,
                         ws.p(), ws.bytes, stream_of(x)));
    if (train) {
        node->x_shape = x.sizes().vec();
        node->y_shape.assign(ysize.begin(), ysize.end());
        node->dt = dt;
        node->M = M;
        node->F = F;
        node->K = K;
        node->act = (rwkv_gate)act;
        node->w = Saved(wr.t);
        if (wants(w)) node->x = Saved(xr.t);
        node->kept = Saved(kept);
        node->rem = Saved(rem);
        torch::autograd::set_history(y, node);
    }
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// ───────────────────────────── dropout ─────────────────────────────

// A probability and the two numbers that name its draw; the seed from a tensor
// is read by the kernels, so a captured call takes what it holds at the replay.
struct DropArgs {
    rwkv_drop d{};
    Tensor seed;
};

uint64_t count_arg(PyObject* o, const char* what) {
    // (numpy's integers too; not a tensor, whose value would have to be waited for)
    PyObject* n = THPVariable_Check(o) ? nullptr : PyNumber_Index(o);
    uint64_t v = 0;
    if (n) {
        v = PyLong_AsUnsignedLongLong(n);
        Py_DECREF(n);
    }
    if (n && !PyErr_Occurred()) return v;
    PyErr_Clear();
    raise(n ? PyExc_ValueError : PyExc_TypeError, std::string(what) + " must be an integer of 0 to 2^64 - 1");
}

// p, seed and offset, before anything is known of the device
DropArgs drop_args(PyObject* p, PyObject* seed, PyObject* offset, const std::string& what) {
    DropArgs r;
    const double v = PyFloat_AsDouble(p);
    if (PyErr_Occurred()) throw python_error();
    if (!(v >= 0.0 && v <= 1.0)) raise(PyExc_ValueError, what + ": p must be 0 to 1, got " + std::to_string(v));
    r.d.threshold = (int32_t)std::nearbyint(v * 65536.0);
    r.d.offset = count_arg(offset, (what + ": offset").c_str());
    if (THPVariable_Check(seed)) {
        r.seed = THPVariable_Unpack(seed);
        if (r.seed.scalar_type() != at::kLong || r.seed.numel() != 1)
            raise(PyExc_TypeError, what + ": a seed tensor holds one int64, got " + shape_of(r.seed) + " " + type_of(r.seed.scalar_type()));
    } else {
        r.d.seed = count_arg(seed, (what + ": seed").c_str());
    }
    return r;
}

// The call's argument; t, the seed's tensor, outlives it.
const rwkv_drop drop_of(const rwkv_drop& d, const Tensor& t) {
    rwkv_drop r = d;
    if (t.defined()) r.seed_dev = static_cast<const int64_t*>(t.const_data_ptr());
    return r;
}

// Keeps nothing but the numbers' names: the backward pass draws them again.
struct DropoutNode : Node {
    Saved seed;
    rwkv_drop drop;
    std::vector<int64_t> shape;
    at::ScalarType x_dt, y_dt;
    c10::Device dev{at::kCUDA};

    std::string name() const override { return "DropoutBackward"; }
    void release_variables() override { seed.reset_data(); }

    variable_list apply(variable_list&& grads) override {
        const bool need_x = task_should_compute_output(0), need_r = num_outputs() > 1 && task_should_compute_output(1);
        no_tangent("dropout", {&grads[0]});
        const Tensor st = seed.unpack(shared_from_this());
        const Guard guard(dev);
        capture_ok("dropout", *this, dev);
        const Tensor dyt = grads[0].defined() ? grads[0] : at::zeros(shape, at::TensorOptions().dtype(y_dt).device(dev));
        variable_list out(num_outputs());
        if (need_r) out[1] = dyt;
        if (need_x) {
            const Rows dy = dropout_rows(dyt);
            out[0] = empty(shape, x_dt, dev);
            const rwkv_drop d = drop_of(drop, st);
            check(rwkv_dropout(dy.p(), dt_of(y_dt), dy.ld, nullptr, 0, ptr(out[0]), dt_of(x_dt), &d, dy.N, dy.D, stream_of(dyt)));
        }
        return once(std::move(out), grads[0], *this, "dropout");
    }
};

// dropout(x, p, seed, offset, residual)
PyObject* py_dropout(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 5) raise(PyExc_TypeError, "dropout: five arguments");
    const Tensor x = tensor_arg(a[0], "dropout: x"), res = tensor_arg(a[4], "dropout: residual", true);
    const DropArgs drop = drop_args(a[1], a[2], a[3], "dropout");
    plain_call("dropout", {&x, &res, &drop.seed});
    no_tangent("dropout", {&x, &res});
    const auto xt = x.scalar_type(), yt = res.defined() ? res.scalar_type() : xt;
    if (x.dim() < 1 || x.size(-1) < 1 || x.size(-1) > (1 << 22))
        raise(PyExc_ValueError, "dropout: the last axis must hold 1 to 2^22 values, got " + shape_of(x));
    if (yt != xt && yt != at::kFloat)
        raise(PyExc_TypeError, std::string("dropout: residual must be ") + type_of(xt) + " or float32, got " + type_of(yt));
    if (res.defined() && res.sizes() != x.sizes())
        raise(PyExc_ValueError, "dropout: residual must be " + shape_of(x) + ", got " + shape_of(res));
    need_device(x, "dropout: x");
    if (res.defined()) same_device(x, res, "dropout: residual");
    if (drop.seed.defined()) same_device(x, drop.seed, "dropout: seed");

    std::shared_ptr<DropoutNode> node;
    if (at::GradMode::is_enabled() && (wants(x) || wants(res))) {
        node = std::shared_ptr<DropoutNode>(new DropoutNode(), torch::autograd::deleteNode);
        node->set_next_edges(res.defined() ? torch::autograd::collect_next_edges(x, res) : torch::autograd::collect_next_edges(x));
    }
    const Guard guard(x.device());
    const Rows xr = dropout_rows(x);
    Rows rr{};
    if (res.defined()) rr = dropout_rows(res);
    Tensor y = empty(x.sizes(), yt, x.device());
    const rwkv_drop d = drop_of(drop.d, drop.seed);
    check(rwkv_dropout(xr.p(), dt_of(xt), xr.ld, rr.t.defined() ? rr.p() : nullptr, rr.ld, ptr(y), dt_of(yt), &d, xr.N, xr.D,
                       stream_of(x)));
    if (node) {
        if (drop.seed.defined()) node->seed = Saved(drop.seed);
        node->drop = drop.d;
        node->shape = x.sizes().vec();
        node->x_dt = xt;
        node->y_dt = yt;
        node->dev = x.device();
        torch::autograd::set_history(y, node);
    }
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// ───────────────────────────── block join ─────────────────────────────

// The vectors of a call, [D] each (or `also`), of one type: float32 or `dt`.
struct Vector {
    const char* name;
    Tensor t;   // as given
    Tensor c;   // contiguous
};

at::ScalarType vectors_of(std::initializer_list<Vector*> all, const std::string& what, const Tensor& x, at::ScalarType dt,
                          int64_t D) {
    const auto wt = (*all.begin())->t.scalar_type();
    for (Vector* v : all) {
        if (!v->t.defined()) continue;
        if (v->t.dim() != 1 || v->t.size(0) != D)
            raise(PyExc_ValueError, what + ": " + v->name + " must be [" + std::to_string(D) + "], got " + shape_of(v->t));
        if (v->t.scalar_type() != wt || (wt != at::kFloat && wt != dt))
            raise(PyExc_TypeError, what + ": " + v->name + " is " + type_of(v->t.scalar_type()) + "; the vectors share float32 or " +
                                       type_of(dt));
    }
    need_device(x, (what + ": x").c_str());
    for (Vector* v : all)
        if (v->t.defined()) {
            same_device(x, v->t, (what + ": " + v->name).c_str());
            v->c = v->t.is_contiguous() ? v->t : v->t.detach().contiguous();
        }
    return wt;
}

// Keeps x' (its own result), the statistics, and o and gate where they reach a
// gradient; of a 16-bit stream x and o, from which x' is formed again.
struct JoinNode : Node {
    enum { X, O, GATE, W, B, PW, PB, SC, INPUTS };
    Saved xs, stats, seed, in[INPUTS];
    rwkv_drop drop;
    int at[INPUTS];                              // an input's gradient among the outputs, or -1
    std::vector<int64_t> shape;
    at::ScalarType x_dt, dt, w_dt;
    int64_t N, D;
    float post_eps, eps;

    std::string name() const override { return "BlockJoinBackward"; }

    void release_variables() override {
        for (Saved* v : {&xs, &stats, &seed}) v->reset_data();
        for (Saved& v : in) v.reset_data();
    }

    variable_list apply(variable_list&& grads) override {
        no_tangent("block_join", {&grads[0], &grads[1]});
        const auto self = shared_from_this();
        const Tensor x1 = xs.dense(self), st = stats.dense(self), sd = seed.unpack(self);
        Tensor t[INPUTS];
        for (int i = 0; i < INPUTS; ++i) t[i] = i < W ? in[i].unpack(self) : in[i].dense(self);
        const auto dev = st.device();
        const Guard guard(dev);
        capture_ok("block_join", *this, dev);
        Rows x{}, o{}, g{}, dx{}, dh{};
        if (t[X].defined()) x = rows_of(t[X]);
        if (t[O].defined()) o = rows_of(t[O]);
        if (t[GATE].defined()) g = rows_of(t[GATE]);
        if (grads[0].defined()) dx = rows_of(grads[0], true);
        if (grads[1].defined()) dh = rows_of(grads[1], true);
        const auto opt = [](const Rows& r) { return r.t.defined() ? r.p() : nullptr; };
        variable_list out(num_outputs());
        void* d[INPUTS] = {};
        bool sums = false;
        for (int i = 0; i < INPUTS; ++i) {
            if (at[i] < 0 || !task_should_compute_output(at[i])) continue;
            Tensor& r = out[at[i]];
            r = i < W ? empty(shape, i == X ? x_dt : dt, dev) : empty({D}, w_dt, dev);
            d[i] = ptr(r);
            sums = sums || i >= W;
        }
        const rwkv_join a{opt(x), opt(o), opt(g), x.ld, o.ld, g.ld, dt_of(x_dt), dt_of(dt), dt_of(w_dt), cptr(t[PW]), cptr(t[PB]),
                          cptr(t[SC]), cptr(t[W]), nullptr, post_eps, eps, drop_of(drop, sd), N, D};
        const Ws ws(sums ? rwkv_join_bwd_workspace(N, D) : 0, dev);
        check(rwkv_join_bwd(&a, cptr(x1), ptr<float>(st), opt(dx), opt(dh), d[X], d[O], d[GATE], d[W], d[B], d[PW], d[PB], d[SC],
                            ws.p(), ws.bytes, stream_of(st)));
        return once(std::move(out), {&grads[0], &grads[1]}, *this, "block_join");
    }
};

// block_join(x, o, weight, bias, post_weight, post_bias, gate, scale, p, seed, offset, eps, post_eps): (x', h)
PyObject* py_block_join(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 13) raise(PyExc_TypeError, "block_join: thirteen arguments");
    const Tensor x = tensor_arg(a[0], "block_join: x"), o = tensor_arg(a[1], "block_join: o"),
                 gate = tensor_arg(a[6], "block_join: gate", true);
    Vector w{"weight", tensor_arg(a[2], "block_join: weight"), {}}, b{"bias", tensor_arg(a[3], "block_join: bias", true), {}},
        pw{"post_weight", tensor_arg(a[4], "block_join: post_weight", true), {}},
        pb{"post_bias", tensor_arg(a[5], "block_join: post_bias", true), {}},
        sc{"scale", tensor_arg(a[7], "block_join: scale", true), {}};
    const DropArgs drop = drop_args(a[8], a[9], a[10], "block_join");
    const double eps = PyFloat_AsDouble(a[11]);
    if (PyErr_Occurred()) throw python_error();
    const double post_eps = PyFloat_AsDouble(a[12]);
    if (PyErr_Occurred()) throw python_error();
    plain_call("block_join", {&x, &o, &gate, &w.t, &b.t, &pw.t, &pb.t, &sc.t, &drop.seed});
    no_tangent("block_join", {&x, &o, &gate, &w.t, &b.t, &pw.t, &pb.t, &sc.t});
    if (x.dim() < 1 || x.size(-1) < 1 || x.size(-1) > 8192)
        raise(PyExc_ValueError, "block_join: the last axis must hold 1 to 8192 values, got " + shape_of(x));
    const int64_t D = x.size(-1);
    const auto xt = x.scalar_type(), dt = o.scalar_type();
    if (o.sizes() != x.sizes() || (gate.defined() && gate.sizes() != x.sizes()))
        raise(PyExc_ValueError, "block_join: o " + shape_of(o) + (gate.defined() ? " and gate " + shape_of(gate) : "") + " must be " + shape_of(x) + " as x");
    if (xt != dt && xt != at::kFloat)
        raise(PyExc_TypeError, std::string("block_join: x must be float32 or ") + type_of(dt) + " as o, got " + type_of(xt));
    if (gate.defined() && gate.scalar_type() != dt)
        raise(PyExc_TypeError, std::string("block_join: gate is ") + type_of(gate.scalar_type()) + ", o " + type_of(dt));
    if (pb.t.defined() && !pw.t.defined()) raise(PyExc_ValueError, "block_join: post_bias without post_weight");
    const auto wt = vectors_of({&w, &b, &pw, &pb, &sc}, "block_join", x, dt, D);
    same_device(x, o, "block_join: o");
    if (gate.defined()) same_device(x, gate, "block_join: gate");
    if (drop.seed.defined()) same_device(x, drop.seed, "block_join: seed");

    const Tensor* const inputs[JoinNode::INPUTS] = {&x, &o, &gate, &w.t, &b.t, &pw.t, &pb.t, &sc.t};
    bool train = false;
    for (const Tensor* t : inputs) train = train || wants(*t);
    train = train && at::GradMode::is_enabled();
    std::shared_ptr<JoinNode> node;
    if (train) {
        node = std::shared_ptr<JoinNode>(new JoinNode(), torch::autograd::deleteNode);
        torch::autograd::edge_list edges;
        for (int i = 0; i < JoinNode::INPUTS; ++i) {
            node->at[i] = inputs[i]->defined() ? (int)edges.size() : -1;
            if (inputs[i]->defined()) edges.push_back(wants(*inputs[i]) ? torch::autograd::impl::gradient_edge(*inputs[i]) : torch::autograd::Edge());
        }
        node->set_next_edges(std::move(edges));
    }
    const auto dev = x.device();
    const Guard guard(dev);
    const Rows xr = rows_of(x), orr = rows_of(o);
    Rows g{};
    if (gate.defined()) g = rows_of(gate);
    Tensor xs = empty(x.sizes(), xt, dev), h = empty(x.sizes(), dt, dev), st;
    if (train) st = empty({xr.N, 4}, at::kFloat, dev);
    const rwkv_join j{xr.p(), orr.p(), g.t.defined() ? g.p() : nullptr, xr.ld, orr.ld, g.ld, dt_of(xt), dt_of(dt), dt_of(wt),
                      cptr(pw.c), cptr(pb.c), cptr(sc.c), cptr(w.c), cptr(b.c), (float)post_eps, (float)eps,
                      drop_of(drop.d, drop.seed), xr.N, D};
    check(rwkv_join_fwd(&j, ptr(xs), ptr(h), ptr<float>(st), stream_of(x)));
    if (train) {
        node->drop = drop.d;
        node->shape = x.sizes().vec();
        node->x_dt = xt;
        node->dt = dt;
        node->w_dt = wt;
        node->N = xr.N;
        node->D = D;
        node->eps = (float)eps;
        node->post_eps = (float)post_eps;
        if (drop.seed.defined()) node->seed = Saved(drop.seed);
        node->stats = Saved(st);
        if (xt != at::kFloat || gate.defined() || pw.t.defined() || sc.t.defined()) node->in[JoinNode::O] = Saved(orr.t);
        if (xt != at::kFloat) node->in[JoinNode::X] = Saved(xr.t);
        if (gate.defined()) node->in[JoinNode::GATE] = Saved(g.t);
        node->in[JoinNode::W] = Saved(w.c);
        if (pw.c.defined()) node->in[JoinNode::PW] = Saved(pw.c);
        if (pb.c.defined()) node->in[JoinNode::PB] = Saved(pb.c);
        if (sc.c.defined()) node->in[JoinNode::SC] = Saved(sc.c);
        torch::autograd::set_history(std::vector<Tensor>{xs, h}, node);
        if (xt == at::kFloat) node->xs = Saved(xs, true);
    }
    PyObject* r = PyTuple_New(2);
    if (!r) throw python_error();
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(xs)));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(h)));
    return r;
    END_HANDLE_TH_ERRORS
}

// ───────────────────────────── the recurrence's tail ─────────────────────────────

struct TailNode : Node {
    enum { O, R, K, V, GATE, RK, W, B, INPUTS };
    Saved in[INPUTS];
    std::vector<int64_t> shape, rk_shape;
    at::ScalarType o_dt, dt, w_dt;
    int64_t N, H;
    float eps;

    std::string name() const override { return "WkvTailBackward"; }

    void release_variables() override {
        for (Saved& v : in) v.reset_data();
    }

    variable_list apply(variable_list&& grads) override {
        no_tangent("wkv_tail", {&grads[0]});
        const auto self = shared_from_this();
        Tensor t[INPUTS];
        Rows r[RK];
        for (int i = 0; i < INPUTS; ++i) t[i] = i < RK ? in[i].unpack(self) : in[i].dense(self);
        const auto dev = t[O].device();
        const Guard guard(dev);
        capture_ok("wkv_tail", *this, dev);
        for (int i = 0; i < RK; ++i) r[i] = rows_of(t[i]);
        const Tensor dyt = grads[0].defined() ? grads[0] : at::zeros(shape, t[R].options());
        const Rows dy = rows_of(dyt);
        variable_list out(INPUTS);
        void* d[INPUTS] = {};
        bool sums = false;
        for (int i = RK; i < INPUTS; ++i) sums = sums || task_should_compute_output(i);
        for (int i = 0; i < INPUTS; ++i) {
            if (i < RK ? !task_should_compute_output(i) : !sums) continue;   // the three sums go together
            out[i] = i < RK ? empty(shape, i == O ? o_dt : dt, dev) : empty(i == RK ? at::IntArrayRef(rk_shape) : at::IntArrayRef(shape.back()), w_dt, dev);
            d[i] = ptr(out[i]);
        }
        const rwkv_tail a{r[O].p(), r[R].p(), r[K].p(), r[V].p(), r[GATE].p(), r[O].ld, r[R].ld, r[K].ld, r[V].ld, r[GATE].ld,
                          dt_of(o_dt), dt_of(dt), dt_of(w_dt), cptr(t[RK]), cptr(t[W]), cptr(t[B]), eps, N, H};
        const Ws ws(sums ? rwkv_tail_bwd_workspace(N, H) : 0, dev);
        check(rwkv_tail_bwd(&a, dy.p(), dy.ld, d[O], d[R], d[K], d[V], d[GATE], d[RK], d[W], d[B], ws.p(), ws.bytes,
                            stream_of(dyt)));
        for (int i = RK; i < INPUTS; ++i)
            if (!task_should_compute_output(i)) out[i] = Tensor();
        return once(std::move(out), grads[0], *this, "wkv_tail");
    }
};

// wkv_tail(o, r, k, v, r_k, gate, weight, bias, eps)
PyObject* py_wkv_tail(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 9) raise(PyExc_TypeError, "wkv_tail: nine arguments");
    const Tensor in[5] = {tensor_arg(a[0], "wkv_tail: o"), tensor_arg(a[1], "wkv_tail: r"), tensor_arg(a[2], "wkv_tail: k"),
                          tensor_arg(a[3], "wkv_tail: v"), tensor_arg(a[5], "wkv_tail: gate")};
    const char* const names[5] = {"o", "r", "k", "v", "gate"};
    const Tensor &o = in[0], &r = in[1];
    const Tensor rk0 = tensor_arg(a[4], "wkv_tail: r_k");
    Vector w{"weight", tensor_arg(a[6], "wkv_tail: weight"), {}}, b{"bias", tensor_arg(a[7], "wkv_tail: bias"), {}}, rk{"r_k", rk0, {}};
    const double eps = PyFloat_AsDouble(a[8]);
    if (PyErr_Occurred()) throw python_error();
    plain_call("wkv_tail", {&in[0], &in[1], &in[2], &in[3], &in[4], &rk0, &w.t, &b.t});
    no_tangent("wkv_tail", {&in[0], &in[1], &in[2], &in[3], &in[4], &rk0, &w.t, &b.t});
    if (o.dim() < 1 || o.size(-1) < 64 || o.size(-1) % 64 || o.size(-1) > 65536)
        raise(PyExc_ValueError, "wkv_tail: the last axis must hold 1 to 1024 heads of 64, got " + shape_of(o));
    const int64_t C = o.size(-1);
    const auto ot = o.scalar_type(), dt = r.scalar_type();
    for (int i = 1; i < 5; ++i) {
        if (in[i].sizes() != o.sizes())
            raise(PyExc_ValueError, std::string("wkv_tail: ") + names[i] + " must be " + shape_of(o) + " as o, got " + shape_of(in[i]));
        if (in[i].scalar_type() != dt)
            raise(PyExc_TypeError, std::string("wkv_tail: ") + names[i] + " is " + type_of(in[i].scalar_type()) + ", r " + type_of(dt));
    }
    if (ot != dt && ot != at::kFloat)
        raise(PyExc_TypeError, std::string("wkv_tail: o must be float32 or ") + type_of(dt) + " as r, got " + type_of(ot));
    if (rk0.dim() == 2 && rk0.size(0) == C / 64 && rk0.size(1) == 64) rk.t = rk0.detach().reshape({C});
    const auto wt = vectors_of({&w, &b, &rk}, "wkv_tail", o, dt, C);
    for (int i = 1; i < 5; ++i) same_device(o, in[i], (std::string("wkv_tail: ") + names[i]).c_str());

    const Tensor* const inputs[TailNode::INPUTS] = {&in[0], &in[1], &in[2], &in[3], &in[4], &rk0, &w.t, &b.t};
    bool train = false;
    for (const Tensor* t : inputs) train = train || wants(*t);
    train = train && at::GradMode::is_enabled();
    std::shared_ptr<TailNode> node;
    if (train) {
        node = std::shared_ptr<TailNode>(new TailNode(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(in[0], in[1], in[2], in[3], in[4], rk0, w.t, b.t));
    }
    const auto dev = o.device();
    const Guard guard(dev);
    Rows rows[5];
    for (int i = 0; i < 5; ++i) rows[i] = rows_of(in[i]);
    Tensor y = empty(o.sizes(), dt, dev);
    const rwkv_tail j{rows[0].p(), rows[1].p(), rows[2].p(), rows[3].p(), rows[4].p(), rows[0].ld, rows[1].ld, rows[2].ld,
                      rows[3].ld, rows[4].ld, dt_of(ot), dt_of(dt), dt_of(wt), cptr(rk.c), cptr(w.c), cptr(b.c), (float)eps,
                      rows[0].N, C / 64};
    check(rwkv_tail_fwd(&j, ptr(y), stream_of(o)));
    if (train) {
        for (int i = 0; i < 5; ++i) node->in[i] = Saved(rows[i].t);
        node->in[TailNode::RK] = Saved(rk.c);
        node->in[TailNode::W] = Saved(w.c);
        node->in[TailNode::B] = Saved(b.c);
        node->shape = o.sizes().vec();
        node->rk_shape = rk0.sizes().vec();
        node->o_dt = ot;
        node->dt = dt;
        node->w_dt = wt;
        node->N = rows[0].N;
        node->H = C / 64;
        node->eps = (float)eps;
        torch::autograd::set_history(y, node);
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
    {"gated_linear", (PyCFunction)(void (*)(void))py_gated_linear, METH_FASTCALL, nullptr},
    {"dropout", (PyCFunction)(void (*)(void))py_dropout, METH_FASTCALL, nullptr},
    {"block_join", (PyCFunction)(void (*)(void))py_block_join, METH_FASTCALL, nullptr},
    {"wkv_tail", (PyCFunction)(void (*)(void))py_wkv_tail, METH_FASTCALL, nullptr},
    {"checkpoint8", py_checkpoint8, METH_O, nullptr},
    {"restore8", (PyCFunction)(void (*)(void))py_restore8, METH_FASTCALL, nullptr},
    {"set_error", py_set_error, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_train", "Training-side operators with their gradients", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__train() { return PyModule_Create(&module); }
