// decoder_shim.cpp -- the calls of svox_amd.decoder in native code: checks, outputs, workspaces, launches and their autograd nodes.
//
// A call on a few rows lasts as long as the host needs to make it, so the whole of it is here, the backward pass too.
#include <torch/extension.h>

#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <mutex>
#include <stdexcept>
#include <string>

#include "../../../include/svox_decoder.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

namespace {

#define SVOX_CALLS(X)                                                                                            \
    X(svox_decoder_last_error) X(svox_layer_norm) X(svox_layer_norm_backward) X(svox_layer_norm_workspace_bytes) \
    X(svox_gated_ffn) X(svox_gated_ffn_backward) X(svox_gated_ffn_workspace_bytes)
struct Library {
#define X(name) decltype(&::name) name = nullptr;
    SVOX_CALLS(X)
#undef X
} lib;

void init(const std::string& path) {
    void* const handle = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
    if (!handle) throw std::runtime_error(std::string("svox: ") + dlerror());
#define X(name)                                                                       \
    lib.name = reinterpret_cast<decltype(&::name)>(dlsym(handle, #name));             \
    if (!lib.name) throw std::runtime_error(path + " does not export " #name ": it was built from other sources, build it again");
    SVOX_CALLS(X)
#undef X
}

[[noreturn]] void fail(const std::string& what) { throw std::runtime_error(what); }
int64_t status(int64_t rc, const char* name) {
    if (rc < 0) fail(std::string("svox.") + name + ": " + lib.svox_decoder_last_error());
    return rc;
}
std::string dtype_text(at::ScalarType t) {
    if (t == at::kFloat) return "torch.float32";
    if (t == at::kDouble) return "torch.float64";
    if (t == at::kHalf) return "torch.float16";
    if (t == at::kBFloat16) return "torch.bfloat16";
    return std::string("torch.") + c10::toString(t);
}
int32_t dtype_code(const Tensor& x, const char* name) {
    switch (x.scalar_type()) {
        case at::kFloat: return SVOX_DECODER_F32;
        case at::kHalf: return SVOX_DECODER_F16;
        case at::kBFloat16: return SVOX_DECODER_BF16;
        default: fail(std::string(name) + " must be a float32, float16 or bfloat16 tensor, got " + dtype_text(x.scalar_type()));
    }
}
void check_like(const Tensor& x, const Tensor& with, const char* name) {
    if (!x.is_cuda()) fail(std::string(name) + " must be a CUDA tensor");
    if (x.layout() != at::kStrided) fail(std::string(name) + " must be a dense tensor");
    if (x.device() != with.device()) fail(std::string(name) + " must be on the device of x (" + with.device().str() + "), got " + x.device().str());
    if (x.scalar_type() != with.scalar_type())
        fail("expected scalar type " + dtype_text(with.scalar_type()) + " for " + name + " but found " + dtype_text(x.scalar_type()));
}
std::string shape_text(at::IntArrayRef s) {
    std::string t = "(";
    for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
    return t + (s.size() == 1 ? ",)" : ")");
}
void check_shape(const Tensor& x, at::IntArrayRef shape, const char* name) {
    if (x.sizes() != shape) fail(std::string(name) + " must have shape " + shape_text(shape) + ", got " + shape_text(x.sizes()));
}
int32_t size32(int64_t n, const char* name) {
    if (n < 1 || n > INT32_MAX) fail(std::string(name) + " must be between 1 and 2^31 - 1, got " + std::to_string(n));
    return (int32_t)n;
}

// x as rows of its last dimension: as it is where the rows lie one stride apart, else a copy
struct Rows {
    Tensor x;
    int64_t rows = 0, stride = 0;
};
Rows rows_of(const Tensor& x) {
    if (x.is_neg()) return rows_of(x.resolve_neg());   // (what memory holds is turned around)
    const int64_t d = x.size(-1), rows = d ? x.numel() / d : 0;
    if (x.is_contiguous()) return Rows{x, rows, d};
    if (rows > 0 && (x.stride(-1) == 1 || d == 1)) {
        int64_t stride = 0, reach = 0;   // of a row, and of what the dimensions seen so far cover
        bool seen = false, even = true;
        for (int64_t i = x.dim() - 2; i >= 0; --i) {
            if (x.size(i) == 1) continue;
            if (!seen) seen = true, stride = x.stride(i), reach = stride * x.size(i);
            else if (x.stride(i) == reach) reach *= x.size(i);
            else even = false;
        }
        if (!seen) stride = d;
        if (even && stride >= d) return Rows{x, rows, stride};
    }
    return Rows{x.contiguous(), rows, d};
}

// ---- what a call takes and makes
struct On {
    c10::DeviceGuard guard;
    void* stream;
    explicit On(const Tensor& x)
        : guard(x.device()), stream((void*)c10::hip::getCurrentHIPStream(x.device().index()).stream()) {}
};
Tensor make(at::IntArrayRef shape, at::ScalarType type, const Tensor& on) { return at::detail::empty_cuda(shape, type, on.device(), std::nullopt); }
Tensor make_like(const Tensor& x) { return make(x.sizes(), x.scalar_type(), x); }
Tensor bytes_on(const Tensor& x, int64_t bytes) { return bytes > 0 ? make({bytes}, at::kByte, x) : Tensor(); }
void* at_or_null(const Tensor& x) { return x.defined() ? x.data_ptr() : nullptr; }

// (A tracer does not see these calls: it would take their results for constants.)
void no_tracing(const char* name) {
    using namespace c10::impl;
    if (torch::jit::tracer::isTracing() || TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY)) fail(std::string("svox.") + name + " cannot be traced");
}
// Whether a call has to make an autograd node.  A tangent of forward mode has no node to go to.
template <size_t n>
bool wants_node(const Tensor* const (&inputs)[n], const char* name) {
    bool wants = false;
    for (const Tensor* x : inputs) {
        if (!x->defined()) continue;
        wants = wants || x->requires_grad();
        if (x->_fw_grad(0).defined()) fail(std::string("svox.") + name + " has no derivatives in forward mode");
    }
    return wants && at::GradMode::is_enabled();
}
void once(const char* name, const Tensor& grad_output) {
    if (at::GradMode::is_enabled()) fail(std::string("svox.") + name + ": its gradient cannot be differentiated again (create_graph)");
    if (grad_output._fw_grad(0).defined()) fail(std::string("svox.") + name + ": its gradient has no derivatives in forward mode");
}
// A node of the given inputs' graph, to which `y` is then tied.
template <class N, class... Inputs>
std::shared_ptr<N> node_of(const Inputs&... inputs) {
    std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(inputs...));
    return node;
}
void make_contiguous(Tensor& x) {
    if (!x.defined()) return;
    if (x.is_neg()) x = x.resolve_neg();
    if (!x.is_contiguous()) x = x.contiguous();
}

// ---- layer norm
SvoxLayerNorm norm_spec(const Rows& x, const Tensor& weight, const Tensor& bias, double eps) {
    SvoxLayerNorm s{};
    s.x = x.x.data_ptr();
    s.weight = at_or_null(weight);
    s.bias = at_or_null(bias);
    s.rows = x.rows;
    s.x_stride = x.stride;
    s.dim = (int32_t)x.x.size(-1);
    s.dtype = dtype_code(x.x, "x");
    s.eps = (float)eps;
    return s;
}
Tensor norm_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, Tensor* stats) {
    const On on(x);
    const Rows rows = rows_of(x);
    Tensor y = make_like(x);
    if (stats) *stats = make({rows.rows, 2}, at::kFloat, x);
    const SvoxLayerNorm s = norm_spec(rows, weight, bias, eps);
    status(lib.svox_layer_norm(&s, y.data_ptr(), stats ? (float*)stats->data_ptr() : nullptr, on.stream), "layer_norm");
    return y;
}

struct NormNode : torch::autograd::Node {
    SavedVariable x_, weight_, stats_;
    double eps = 0.0;

    std::string name() const override { return "SvoxLayerNormBackward"; }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        x_.reset_data();
        weight_.reset_data();
        stats_.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        const std::lock_guard<std::mutex> lock(mutex_);
        variable_list out(3);
        if (!grads[0].defined()) return out;
        once("layer_norm", grads[0]);
        const Tensor x = x_.unpack(), weight = weight_.unpack(), stats = stats_.unpack();
        const On on(x);
        check_like(grads[0], x, "grad_output");
        const Rows rows = rows_of(x), dy = rows_of(grads[0]);
        const SvoxLayerNorm s = norm_spec(rows, weight, Tensor(), eps);
        if (task_should_compute_output(0)) out[0] = make_like(x);
        if (task_should_compute_output(1)) out[1] = make({s.dim}, x.scalar_type(), x);
        if (task_should_compute_output(2)) out[2] = make({s.dim}, x.scalar_type(), x);
        const int64_t bytes = status(lib.svox_layer_norm_workspace_bytes(&s, out[1].defined() || out[2].defined()), "layer_norm");
        const Tensor space = bytes_on(x, bytes);
        status(lib.svox_layer_norm_backward(&s, (const float*)stats.data_ptr(), dy.x.data_ptr(), dy.stride, at_or_null(out[0]), at_or_null(out[1]),
                                            at_or_null(out[2]), at_or_null(space), bytes, on.stream),
               "layer_norm_backward");
        return out;
    }
};

Tensor layer_norm(const Tensor& x, Tensor weight, Tensor bias, double eps) {
    no_tracing("layer_norm");
    check_like(x, x, "x");
    dtype_code(x, "x");
    if (x.dim() < 1) fail("x must have at least one dimension");
    const int64_t d = size32(x.size(-1), "the size of x's rows");
    if (weight.defined()) check_like(weight, x, "weight"), check_shape(weight, {d}, "weight");
    if (bias.defined()) check_like(bias, x, "bias"), check_shape(bias, {d}, "bias");
    make_contiguous(weight);
    make_contiguous(bias);
    if (!wants_node({&x, &weight, &bias}, "layer_norm")) return norm_forward(x, weight, bias, eps, nullptr);
    const auto node = node_of<NormNode>(x, weight, bias);
    Tensor stats, y;
    {
        const at::AutoDispatchBelowADInplaceOrView guard;
        y = norm_forward(x, weight, bias, eps, &stats);
    }
    node->x_ = SavedVariable(x, false);
    node->weight_ = SavedVariable(weight, false);
    node->stats_ = SavedVariable(stats, false);
    node->eps = eps;
    torch::autograd::set_history(y, node);
    return y;
}

// ---- the gated feed-forward block
struct Ffn {
    Tensor x, w_gate, w_up, w_down, b_gate, b_up, b_down, residual;
};
SvoxGatedFfn ffn_spec(const Ffn& f, const Rows& x, int32_t activation) {
    SvoxGatedFfn s{};
    s.x = x.x.data_ptr();
    s.w_gate = f.w_gate.data_ptr();
    s.w_up = f.w_up.data_ptr();
    s.w_down = f.w_down.data_ptr();
    s.b_gate = at_or_null(f.b_gate);
    s.b_up = at_or_null(f.b_up);
    s.b_down = at_or_null(f.b_down);
    s.rows = x.rows;
    s.x_stride = x.stride;
    s.dim = (int32_t)f.w_gate.size(1);
    s.hidden = (int32_t)f.w_gate.size(0);
    s.out = (int32_t)f.w_down.size(0);
    s.dtype = dtype_code(f.x, "x");
    s.activation = activation;
    return s;
}
c10::SmallVector<int64_t, 6> out_shape(const Ffn& f) {
    c10::SmallVector<int64_t, 6> shape(f.x.sizes().begin(), f.x.sizes().end());
    shape.back() = f.w_down.size(0);
    return shape;
}
Tensor ffn_forward(const Ffn& f, int32_t activation) {
    const On on(f.x);
    const Rows x = rows_of(f.x);
    SvoxGatedFfn s = ffn_spec(f, x, activation);
    Rows residual;
    if (f.residual.defined()) {
        residual = rows_of(f.residual);
        s.residual = residual.x.data_ptr();
        s.residual_stride = residual.stride;
    }
    Tensor y = make(out_shape(f), f.x.scalar_type(), f.x);
    const int64_t bytes = status(lib.svox_gated_ffn_workspace_bytes(&s, 0), "gated_ffn");
    const Tensor space = bytes_on(f.x, bytes);
    status(lib.svox_gated_ffn(&s, y.data_ptr(), at_or_null(space), bytes, on.stream), "gated_ffn");
    return y;
}

struct FfnNode : torch::autograd::Node {
    SavedVariable saved_[6];   // x, w_gate, w_up, w_down, b_gate, b_up
    int32_t activation = 0;

    std::string name() const override { return "SvoxGatedFfnBackward"; }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        for (SavedVariable& v : saved_) v.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        const std::lock_guard<std::mutex> lock(mutex_);
        variable_list out(8);
        if (!grads[0].defined()) return out;
        once("gated_ffn", grads[0]);
        const Ffn f{saved_[0].unpack(), saved_[1].unpack(), saved_[2].unpack(), saved_[3].unpack(), saved_[4].unpack(), saved_[5].unpack(), Tensor(), Tensor()};
        const On on(f.x);
        check_like(grads[0], f.x, "grad_output");
        if (task_should_compute_output(7)) out[7] = grads[0];
        const Rows x = rows_of(f.x), dy = rows_of(grads[0]);
        const SvoxGatedFfn s = ffn_spec(f, x, activation);
        const Tensor* const shaped[6] = {&f.x, &f.w_gate, &f.w_up, &f.w_down, &f.b_gate, &f.b_up};
        bool any = false;
        for (int i = 0; i < 7; ++i)
            if (task_should_compute_output(i)) {
                out[i] = i == 6 ? make({s.out}, f.x.scalar_type(), f.x) : make_like(*shaped[i]);
                any = true;
            }
        if (!any) return out;
        const SvoxGatedFfnGrads g{at_or_null(out[0]), at_or_null(out[1]), at_or_null(out[2]), at_or_null(out[3]),
                                  at_or_null(out[4]), at_or_null(out[5]), at_or_null(out[6])};
        const int64_t bytes = status(lib.svox_gated_ffn_workspace_bytes(&s, 1), "gated_ffn");
        const Tensor space = bytes_on(f.x, bytes);
        status(lib.svox_gated_ffn_backward(&s, dy.x.data_ptr(), dy.stride, &g, at_or_null(space), bytes, on.stream), "gated_ffn_backward");
        return out;
    }
};

Tensor gated_ffn(Ffn& f, int64_t activation) {
    const Tensor& x = f.x;
    no_tracing("gated_ffn");
    check_like(x, x, "x");
    dtype_code(x, "x");
    if (x.dim() < 1) fail("x must have at least one dimension");
    check_like(f.w_gate, x, "w_gate");
    check_like(f.w_up, x, "w_up");
    check_like(f.w_down, x, "w_down");
    if (f.w_gate.dim() != 2 || f.w_down.dim() != 2) fail("w_gate, w_up and w_down must be 2-D");
    const int64_t d = size32(x.size(-1), "the size of x's rows"), h = size32(f.w_gate.size(0), "the number of hidden units"),
                  o = size32(f.w_down.size(0), "the size of the result's rows");
    check_shape(f.w_gate, {h, d}, "w_gate");
    check_shape(f.w_up, {h, d}, "w_up");
    check_shape(f.w_down, {o, h}, "w_down");
    if (f.b_gate.defined()) check_like(f.b_gate, x, "b_gate"), check_shape(f.b_gate, {h}, "b_gate");
    if (f.b_up.defined()) check_like(f.b_up, x, "b_up"), check_shape(f.b_up, {h}, "b_up");
    if (f.b_down.defined()) check_like(f.b_down, x, "b_down"), check_shape(f.b_down, {o}, "b_down");
    if (f.residual.defined()) check_like(f.residual, x, "residual"), check_shape(f.residual, out_shape(f), "residual");
    if (activation < SVOX_ACTIVATION_SILU || activation > SVOX_ACTIVATION_SIGMOID) fail("unknown activation " + std::to_string(activation));
    for (Tensor* t : {&f.w_gate, &f.w_up, &f.w_down, &f.b_gate, &f.b_up, &f.b_down}) make_contiguous(*t);
    if (!wants_node({&f.x, &f.w_gate, &f.w_up, &f.w_down, &f.b_gate, &f.b_up, &f.b_down, &f.residual}, "gated_ffn"))
        return ffn_forward(f, (int32_t)activation);
    const auto node = node_of<FfnNode>(f.x, f.w_gate, f.w_up, f.w_down, f.b_gate, f.b_up, f.b_down, f.residual);
    Tensor y;
    {
        const at::AutoDispatchBelowADInplaceOrView guard;
        y = ffn_forward(f, (int32_t)activation);
    }
    const Tensor* const saved[6] = {&f.x, &f.w_gate, &f.w_up, &f.w_down, &f.b_gate, &f.b_up};
    for (int i = 0; i < 6; ++i) node->saved_[i] = SavedVariable(*saved[i], false);
    node->activation = (int32_t)activation;
    torch::autograd::set_history(y, node);
    return y;
}

// ---- called from Python with positional arguments
struct WrongType {
    const char* name;
};
const Tensor& tensor(PyObject* x, const char* name) {
    if (!THPVariable_Check(x)) throw WrongType{name};
    return THPVariable_Unpack(x);
}
Tensor tensor_or_none(PyObject* x, const char* name) { return x == Py_None ? Tensor() : tensor(x, name); }

template <class F>
PyObject* call(Py_ssize_t given, Py_ssize_t wanted, F f) {
    if (given != wanted) {
        PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", wanted, given);
        return nullptr;
    }
    try {
        return THPVariable_Wrap(f());
    } catch (const WrongType& e) {
        PyErr_Format(PyExc_TypeError, "%s must be a tensor", e.name);
    } catch (py::error_already_set& e) {
        e.restore();
    } catch (...) {
        torch::translate_exception_to_python(std::current_exception());
    }
    return nullptr;
}
PyObject* layer_norm_py(PyObject*, PyObject* const* args, Py_ssize_t given) {
    return call(given, 4, [&] {
        const Tensor &x = tensor(args[0], "x"), weight = tensor_or_none(args[1], "weight"), bias = tensor_or_none(args[2], "bias");
        const double eps = PyFloat_AsDouble(args[3]);
        if (eps == -1.0 && PyErr_Occurred()) throw py::error_already_set();
        const py::gil_scoped_release unlocked;
        return layer_norm(x, weight, bias, eps);
    });
}
PyObject* gated_ffn_py(PyObject*, PyObject* const* args, Py_ssize_t given) {
    return call(given, 9, [&] {
        Ffn f{tensor(args[0], "x"), tensor(args[1], "w_gate"), tensor(args[2], "w_up"), tensor(args[3], "w_down"), tensor_or_none(args[4], "b_gate"),
              tensor_or_none(args[5], "b_up"), tensor_or_none(args[6], "b_down"), tensor_or_none(args[7], "residual")};
        const int64_t activation = PyLong_AsLongLong(args[8]);
        if (activation == -1 && PyErr_Occurred()) throw py::error_already_set();
        const py::gil_scoped_release unlocked;
        return gated_ffn(f, activation);
    });
}
PyMethodDef kCalls[] = {{"layer_norm", (PyCFunction)(void (*)())layer_norm_py, METH_FASTCALL, nullptr},
                        {"gated_ffn", (PyCFunction)(void (*)())gated_ffn_py, METH_FASTCALL, nullptr},
                        {nullptr, nullptr, 0, nullptr}};

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("init", &init);
    PyModule_AddFunctions(m.ptr(), kCalls);
}
