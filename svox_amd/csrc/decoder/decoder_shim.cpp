// decoder_shim.cpp -- the calls of svox_amd.decoder in native code: checks, outputs, workspaces, launches and their autograd nodes.
//
// A call on a few rows lasts as long as the host needs to make it, so the whole of it is here, the backward pass too.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>

#include <optional>
#include <stdexcept>
#include <string>

#include "../../../include/svox_decoder.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

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
    int64_t rows, stride;
};
Rows rows_of(const Tensor& x) {
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

struct On {
    c10::DeviceGuard guard;
    void* stream;
    explicit On(const Tensor& x)
        : guard(x.device()), stream((void*)c10::hip::getCurrentHIPStream(x.device().index()).stream()) {}
};
Tensor fresh_like(const Tensor& x) { return at::empty(x.sizes(), x.options().requires_grad(false)); }
Tensor bytes_on(const Tensor& x, int64_t bytes) {
    return bytes > 0 ? at::empty({bytes}, x.options().dtype(at::kByte).requires_grad(false)) : Tensor();
}
void* at_or_null(const Tensor& x) { return x.defined() ? x.data_ptr() : nullptr; }

// Whether a call has to make an autograd node.  (A tangent of forward mode does not show in requires_grad: the node refuses it, where
// the operator called by itself would drop it.)
bool wants_node(std::initializer_list<const Tensor*> inputs) {
    const bool grad = at::GradMode::is_enabled();
    for (const Tensor* x : inputs)
        if (x->defined() && ((grad && x->requires_grad()) || x->_fw_grad(0).defined())) return true;
    return false;
}
// A node has an edge for each tensor it was given: wanted(ctx, i) says whether the gradient of argument i is asked for.
void keep_edges(AutogradContext* ctx, std::initializer_list<const Tensor*> inputs) {
    int64_t given = 0, i = 0;
    for (const Tensor* x : inputs) given |= (int64_t)x->defined() << i++;
    ctx->saved_data["given"] = given;
}
bool wanted(AutogradContext* ctx, int argument) {
    const int64_t given = ctx->saved_data["given"].toInt();
    if (!(given >> argument & 1)) return false;
    return ctx->needs_input_grad((size_t)__builtin_popcountll(given & ((1ll << argument) - 1)));
}
Maybe given(const Tensor& x) { return x.defined() ? Maybe(x) : Maybe(); }
void once(const char* name) {
    if (at::GradMode::is_enabled()) fail(std::string("svox.") + name + ": its gradient cannot be differentiated again (create_graph)");
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
    Tensor y = fresh_like(x);
    if (stats) *stats = at::empty({rows.rows, 2}, x.options().dtype(at::kFloat).requires_grad(false));
    const SvoxLayerNorm s = norm_spec(rows, weight, bias, eps);
    status(lib.svox_layer_norm(&s, y.data_ptr(), stats ? (float*)stats->data_ptr() : nullptr, on.stream), "layer_norm");
    return y;
}

struct NormNode : torch::autograd::Function<NormNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& weight_, const Maybe& bias_, double eps) {
        const Tensor weight = weight_.value_or(Tensor()), bias = bias_.value_or(Tensor());
        Tensor stats;
        Tensor y = norm_forward(x, weight, bias, eps, &stats);
        ctx->save_for_backward({x, weight, stats});
        keep_edges(ctx, {&x, &weight, &bias});
        ctx->saved_data["eps"] = eps;
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list out(4);
        if (!grads[0].defined()) return out;
        once("layer_norm");
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1], &stats = saved[2];
        const On on(x);
        check_like(grads[0], x, "grad_output");
        const Rows rows = rows_of(x), dy = rows_of(grads[0]);
        const SvoxLayerNorm s = norm_spec(rows, weight, Tensor(), ctx->saved_data["eps"].toDouble());
        Tensor dw, db;
        if (wanted(ctx, 0)) out[0] = fresh_like(x);
        if (wanted(ctx, 1)) out[1] = dw = at::empty({s.dim}, x.options().requires_grad(false));
        if (wanted(ctx, 2)) out[2] = db = at::empty({s.dim}, x.options().requires_grad(false));
        const int64_t bytes = status(lib.svox_layer_norm_workspace_bytes(&s, dw.defined() || db.defined()), "layer_norm");
        const Tensor space = bytes_on(x, bytes);
        status(lib.svox_layer_norm_backward(&s, (const float*)stats.data_ptr(), dy.x.data_ptr(), dy.stride, at_or_null(out[0]), at_or_null(dw),
                                            at_or_null(db), at_or_null(space), bytes, on.stream),
               "layer_norm_backward");
        return out;
    }
};

Tensor layer_norm(const Tensor& x, const Maybe& weight_, const Maybe& bias_, double eps) {
    const Tensor weight = weight_.value_or(Tensor()), bias = bias_.value_or(Tensor());
    check_like(x, x, "x");
    dtype_code(x, "x");
    if (x.dim() < 1) fail("x must have at least one dimension");
    const int64_t d = size32(x.size(-1), "the size of x's rows");
    if (weight.defined()) check_like(weight, x, "weight"), check_shape(weight, {d}, "weight");
    if (bias.defined()) check_like(bias, x, "bias"), check_shape(bias, {d}, "bias");
    const py::gil_scoped_release unlocked;
    const Tensor w = weight.defined() ? weight.contiguous() : weight, b = bias.defined() ? bias.contiguous() : bias;
    if (wants_node({&x, &w, &b})) return NormNode::apply(x, given(w), given(b), eps);
    return norm_forward(x, w, b, eps, nullptr);
}

// ---- the gated feed-forward block
struct Ffn {
    Tensor x, w_gate, w_up, w_down, b_gate, b_up, b_down, residual;
};
SvoxGatedFfn ffn_spec(const Ffn& f, const Rows& x, int64_t activation) {
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
    s.activation = (int32_t)activation;
    return s;
}
std::vector<int64_t> out_shape(const Ffn& f) {
    std::vector<int64_t> shape = f.x.sizes().vec();
    shape.back() = f.w_down.size(0);
    return shape;
}
Tensor ffn_forward(const Ffn& f, int64_t activation) {
    const On on(f.x);
    const Rows x = rows_of(f.x);
    SvoxGatedFfn s = ffn_spec(f, x, activation);
    Rows residual;
    if (f.residual.defined()) {
        residual = rows_of(f.residual);
        s.residual = residual.x.data_ptr();
        s.residual_stride = residual.stride;
    }
    Tensor y = at::empty(out_shape(f), f.x.options().requires_grad(false));
    const int64_t bytes = status(lib.svox_gated_ffn_workspace_bytes(&s, 0), "gated_ffn");
    const Tensor space = bytes_on(f.x, bytes);
    status(lib.svox_gated_ffn(&s, y.data_ptr(), at_or_null(space), bytes, on.stream), "gated_ffn");
    return y;
}

struct FfnNode : torch::autograd::Function<FfnNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const Tensor& w_down, const Maybe& b_gate,
                          const Maybe& b_up, const Maybe& b_down, const Maybe& residual, int64_t activation) {
        const Tensor none;
        const Ffn f{x, w_gate, w_up, w_down, b_gate.value_or(none), b_up.value_or(none), b_down.value_or(none), residual.value_or(none)};
        Tensor y = ffn_forward(f, activation);
        ctx->save_for_backward({x, w_gate, w_up, w_down, f.b_gate, f.b_up});
        keep_edges(ctx, {&f.x, &f.w_gate, &f.w_up, &f.w_down, &f.b_gate, &f.b_up, &f.b_down, &f.residual});
        ctx->saved_data["activation"] = activation;
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list out(9);
        if (!grads[0].defined()) return out;
        once("gated_ffn");
        const variable_list saved = ctx->get_saved_variables();
        const Ffn f{saved[0], saved[1], saved[2], saved[3], saved[4], saved[5], Tensor(), Tensor()};
        const On on(f.x);
        check_like(grads[0], f.x, "grad_output");
        if (wanted(ctx, 7)) out[7] = grads[0];
        const Rows x = rows_of(f.x), dy = rows_of(grads[0]);
        const SvoxGatedFfn s = ffn_spec(f, x, ctx->saved_data["activation"].toInt());
        const Tensor shaped[7] = {f.x, f.w_gate, f.w_up, f.w_down, f.b_gate, f.b_up, Tensor()};
        bool any = false;
        for (int i = 0; i < 7; ++i)
            if (wanted(ctx, i)) {
                out[i] = i == 6 ? at::empty({s.out}, f.x.options().requires_grad(false)) : fresh_like(shaped[i]);
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

Tensor gated_ffn(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const Tensor& w_down, const Maybe& b_gate, const Maybe& b_up,
                 const Maybe& b_down, const Maybe& residual, int64_t activation) {
    Ffn f{x, w_gate, w_up, w_down, b_gate.value_or(Tensor()), b_up.value_or(Tensor()), b_down.value_or(Tensor()), residual.value_or(Tensor())};
    check_like(x, x, "x");
    dtype_code(x, "x");
    if (x.dim() < 1) fail("x must have at least one dimension");
    check_like(w_gate, x, "w_gate");
    check_like(w_up, x, "w_up");
    check_like(w_down, x, "w_down");
    if (w_gate.dim() != 2 || w_down.dim() != 2) fail("w_gate, w_up and w_down must be 2-D");
    const int64_t d = size32(x.size(-1), "the size of x's rows"), h = size32(w_gate.size(0), "the number of hidden units"),
                  o = size32(w_down.size(0), "the size of the result's rows");
    check_shape(w_gate, {h, d}, "w_gate");
    check_shape(w_up, {h, d}, "w_up");
    check_shape(w_down, {o, h}, "w_down");
    if (f.b_gate.defined()) check_like(f.b_gate, x, "b_gate"), check_shape(f.b_gate, {h}, "b_gate");
    if (f.b_up.defined()) check_like(f.b_up, x, "b_up"), check_shape(f.b_up, {h}, "b_up");
    if (f.b_down.defined()) check_like(f.b_down, x, "b_down"), check_shape(f.b_down, {o}, "b_down");
    if (f.residual.defined()) check_like(f.residual, x, "residual"), check_shape(f.residual, out_shape(f), "residual");
    if (activation < SVOX_ACTIVATION_SILU || activation > SVOX_ACTIVATION_SIGMOID) fail("unknown activation " + std::to_string(activation));
    const py::gil_scoped_release unlocked;
    for (Tensor* t : {&f.w_gate, &f.w_up, &f.w_down, &f.b_gate, &f.b_up, &f.b_down})
        if (t->defined()) *t = t->contiguous();
    if (wants_node({&f.x, &f.w_gate, &f.w_up, &f.w_down, &f.b_gate, &f.b_up, &f.b_down, &f.residual}))
        return FfnNode::apply(f.x, f.w_gate, f.w_up, f.w_down, given(f.b_gate), given(f.b_up), given(f.b_down), given(f.residual), activation);
    return ffn_forward(f, activation);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("init", &init);
    m.def("layer_norm", &layer_norm);
    m.def("gated_ffn", &gated_ffn);
}
