// operator_shim.h -- what the host extensions of the operators share: the checks of tensors, outputs and workspaces, what torch could get
// wrong silently, and calls from Python with positional arguments.
#pragma once
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

#include "../../include/svox_decoder.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

namespace {

// The calls of a C ABI, `SVOX_CALLS(X)`, as pointers, looked up in the library by their names.
#define SVOX_LIBRARY                                                                                                                       \
    struct Library {                                                                                                                       \
        SVOX_CALLS(SVOX_POINTER)                                                                                                           \
    } lib;                                                                                                                                 \
    void init(const std::string& path) {                                                                                                   \
        void* const handle = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);                                                                  \
        if (!handle) throw std::runtime_error(std::string("svox: ") + dlerror());                                                          \
        SVOX_CALLS(SVOX_LOOK_UP)                                                                                                           \
    }
#define SVOX_POINTER(name) decltype(&::name) name = nullptr;
#define SVOX_LOOK_UP(name)                                                \
    lib.name = reinterpret_cast<decltype(&::name)>(dlsym(handle, #name)); \
    if (!lib.name) throw std::runtime_error(path + " does not export " #name ": it was built from other sources, build it again");

[[noreturn]] void fail(const std::string& what) { throw std::runtime_error(what); }
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
void check_like(const Tensor& x, const Tensor& with, const char* name, const char* of = "x") {
    if (!x.is_cuda()) fail(std::string(name) + " must be a CUDA tensor");
    if (x.layout() != at::kStrided) fail(std::string(name) + " must be a dense tensor");
    if (!x.has_storage()) fail(std::string(name) + " has no memory of its own: transforms of functions (vmap, torch.func) are not supported");
    if (x.device() != with.device()) fail(std::string(name) + " must be on the device of " + of + " (" + with.device().str() + "), got " + x.device().str());
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

// A tensor kept for the backward pass.  Hooks on saved tensors may give back another in its place: one of another device, type or shape is refused,
// any strides can be.
struct Kept {
    SavedVariable saved;
    at::DimVector shape;
    at::ScalarType type = at::kFloat;
    at::Device device = at::kCPU;
    bool defined = false;

    void keep(const Tensor& x, bool is_output = false) {
        saved = SavedVariable(x, is_output);
        defined = x.defined();
        if (!defined) return;
        shape.assign(x.sizes().begin(), x.sizes().end());
        type = x.scalar_type();
        device = x.device();
    }
    Tensor take(const char* name, std::shared_ptr<torch::autograd::Node> node = nullptr) const {
        const Tensor x = saved.unpack(std::move(node));
        if (!defined) return Tensor();
        if (!x.defined() || x.layout() != at::kStrided || x.device() != device || x.scalar_type() != type || x.sizes() != at::IntArrayRef(shape))
            fail(std::string("svox.") + name + ": a hook on saved tensors gave back another tensor than a " + dtype_text(type) + " one of shape " + shape_text(shape) + " on " +
                 device.str());
        return x;
    }
    Tensor take_contiguous(const char* name, std::shared_ptr<torch::autograd::Node> node = nullptr) const {
        Tensor x = take(name, std::move(node));
        make_contiguous(x);
        return x;
    }
    void reset() { saved.reset_data(); }
};

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
        if constexpr (std::is_same_v<decltype(f()), Tensor>) return THPVariable_Wrap(f());
        else return f();
    } catch (const WrongType& e) {
        PyErr_Format(PyExc_TypeError, "%s must be a tensor", e.name);
    } catch (py::error_already_set& e) {
        e.restore();
    } catch (...) {
        torch::translate_exception_to_python(std::current_exception());
    }
    return nullptr;
}

}  // namespace
