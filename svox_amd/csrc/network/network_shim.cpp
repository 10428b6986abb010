// network_shim.cpp -- the calls of svox_amd.network in native code: checks, outputs, workspaces, launches and their autograd nodes.
#include "../operator_shim.h"

#include <algorithm>
#include <cmath>
#include <vector>

#include "../../../include/svox_network.h"

namespace {

#define SVOX_CALLS(X)                                                                           \
    X(svox_network_last_error) X(svox_clip_norm) X(svox_clip_norm_workspace_bytes)              \
    X(svox_rotate_heads) X(svox_rotate_heads_backward) X(svox_rotate_heads_workspace_bytes)     \
    X(svox_attention) X(svox_attention_backward) X(svox_attention_workspace_bytes)
SVOX_LIBRARY

int64_t status(int64_t rc, const char* name) {
    if (rc < 0) fail(std::string("svox.") + name + ": " + lib.svox_network_last_error());
    return rc;
}

// x (rows, heads, dim) as it is where a head's numbers lie side by side and rows and heads forward, else a copy
Tensor heads_of(const Tensor& x) {
    if (x.is_neg()) return heads_of(x.resolve_neg());   // (what memory holds is turned around)
    if ((x.stride(2) == 1 || x.size(2) == 1) && x.stride(0) >= 0 && x.stride(1) >= 0) return x;
    return x.contiguous();
}
void check_3d(const Tensor& x, const char* name) {
    if (x.dim() != 3) fail(std::string(name) + " must be 3-D (rows, heads, numbers of a head), got " + shape_text(x.sizes()));
}

// ---- the norm of many tensors, and clipping
std::vector<Tensor> tensors_of(PyObject* list, const char* name) {
    PyObject* const fast = PySequence_Fast(list, "expected a sequence of tensors");
    if (!fast) throw py::error_already_set();
    const py::object hold = py::reinterpret_steal<py::object>(fast);
    std::vector<Tensor> all;
    for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(fast); ++i) all.push_back(tensor(PySequence_Fast_GET_ITEM(fast, i), name));
    return all;
}
void check_clipped(const std::vector<Tensor>& all, const char* name, double max_norm) {
    no_tracing(name);
    if (all.empty()) fail(std::string("svox.") + name + ": no tensors");
    if (!(max_norm >= 0.0)) fail("max_norm must be >= 0, got " + std::to_string(max_norm));
    for (const Tensor& x : all) {
        if (!x.is_cuda()) fail("every tensor must be a CUDA tensor");
        if (x.layout() != at::kStrided) fail("every tensor must be a dense tensor");
        if (!x.has_storage()) fail("every tensor must have memory of its own: transforms of functions (vmap, torch.func) are not supported");
        if (x.device() != all[0].device()) fail("every tensor must be on the same device, got " + all[0].device().str() + " and " + x.device().str());
        dtype_code(x, "every tensor");
        if (x._fw_grad(0).defined()) fail(std::string("svox.") + name + " has no derivatives in forward mode");
    }
}
Tensor clip(const std::vector<SvoxClipTensor>& table, const Tensor& on_device, double max_norm, const char* name) {
    const On on(on_device);
    Tensor norm = make({}, at::kFloat, on_device);
    const int64_t bytes = status(lib.svox_clip_norm_workspace_bytes(table.data(), (int64_t)table.size()), name);
    const Tensor space = bytes_on(on_device, bytes);
    status(lib.svox_clip_norm(table.data(), (int64_t)table.size(), max_norm, (float*)norm.data_ptr(), at_or_null(space), bytes, on.stream), name);
    return norm;
}
SvoxClipTensor clip_entry(const Tensor& from, const Tensor& to) {
    SvoxClipTensor e{};
    e.from = from.data_ptr();
    e.to = to.data_ptr();
    e.count = from.numel();
    e.dtype = dtype_code(from, "every tensor");
    return e;
}
// As it lies in memory, in whatever order, if every number lies there once and none lies between.
Tensor dense(const Tensor& x) {
    if (x.is_neg()) return dense(x.resolve_neg());
    return x.is_non_overlapping_and_dense() ? x : x.contiguous();
}

Tensor clip_norm(const std::vector<Tensor>& all, double max_norm, std::vector<Tensor>& out) {
    check_clipped(all, "clip_norm", max_norm);
    if (at::GradMode::is_enabled())
        for (const Tensor& x : all)
            if (x.requires_grad()) fail("svox.clip_norm has no gradient: give it tensors that need none (x.detach())");
    std::vector<SvoxClipTensor> table;
    std::vector<Tensor> hold;
    const c10::DeviceGuard guard(all[0].device());
    for (const Tensor& x : all) {
        hold.push_back(dense(x));
        const Tensor& from = hold.back();
        const bool plain = from.is_contiguous();
        out.push_back(plain ? make_like(from) : at::empty_strided(from.sizes(), from.strides(), from.options()));
        table.push_back(clip_entry(from, out.back()));
    }
    return clip(table, all[0], max_norm, "clip_norm");
}

// Gradients where they lie.  What two of them share, whole, is one gradient; those that reach into one another otherwise are refused.
Tensor clip_in_place(const std::vector<Tensor>& all, double max_norm) {
    const char* const name = "clip_grad_norm";
    check_clipped(all, name, max_norm);
    const at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard guard(all[0].device());
    struct Part {
        const Tensor* x;
        Tensor copy;   // where the gradient's numbers do not lie side by side: of them
        const char *from, *to;
    };
    std::vector<Part> parts;
    for (const Tensor& x : all) {
        if (x.numel() == 0) continue;
        if (x.is_neg()) fail("svox.clip_grad_norm: a gradient is a view of the negatives of its memory");
        int64_t reach = 1;
        for (int64_t i = 0; i < x.dim(); ++i) {
            if (x.size(i) > 1 && x.stride(i) == 0) fail("svox.clip_grad_norm: a gradient has several numbers in one place (expand)");
            reach += (x.size(i) - 1) * x.stride(i);
        }
        const char* const from = (const char*)x.data_ptr();
        parts.push_back(Part{&x, Tensor(), from, from + reach * x.element_size()});
    }
    std::stable_sort(parts.begin(), parts.end(), [](const Part& a, const Part& b) { return a.from < b.from; });
    std::vector<Part> once;
    for (Part& p : parts) {
        if (!once.empty() && p.from < once.back().to) {
            const Tensor &a = *once.back().x, &b = *p.x;
            if (p.from == once.back().from && a.sizes() == b.sizes() && a.strides() == b.strides() && a.scalar_type() == b.scalar_type()) continue;
            fail("svox.clip_grad_norm: two gradients share memory, or one lies between the numbers of another");
        }
        once.push_back(p);
    }
    std::vector<SvoxClipTensor> table;
    for (Part& p : once) {
        if (!p.x->is_non_overlapping_and_dense()) p.copy = p.x->contiguous();
        const Tensor& x = p.copy.defined() ? p.copy : *p.x;
        table.push_back(clip_entry(x, x));
    }
    const Tensor norm = clip(table, all[0], max_norm, name);
    for (Part& p : once) {
        if (p.copy.defined()) p.x->copy_(p.copy);
        if (!p.x->is_inference()) p.x->unsafeGetTensorImpl()->bump_version();   // (nothing below this call does)
    }
    return norm;
}

// ---- heads, their norms and rotation
struct Heads {
    Tensor q, k, positions, frequencies, q_weight, k_weight;
    bool interleaved = false;
    double eps = 0.0;
};
SvoxRotateHeads rotate_spec(const Heads& h) {
    SvoxRotateHeads s{};
    s.q = h.q.data_ptr();
    s.k = h.k.data_ptr();
    s.q_weight = at_or_null(h.q_weight);
    s.k_weight = at_or_null(h.k_weight);
    s.positions = h.positions.data_ptr();
    s.frequencies = (const float*)h.frequencies.data_ptr();
    s.rows = h.q.size(0);
    s.q_stride = h.q.stride(0), s.q_head = h.q.stride(1);
    s.k_stride = h.k.stride(0), s.k_head = h.k.stride(1);
    s.heads = (int32_t)h.q.size(1);
    s.kv_heads = (int32_t)h.k.size(1);
    s.dim = (int32_t)h.q.size(2);
    s.rotated = 2 * (int32_t)h.frequencies.size(1);
    s.axes = (int32_t)h.positions.size(1);
    s.interleaved = h.interleaved;
    s.dtype = dtype_code(h.q, "q");
    s.position_type = h.positions.scalar_type() == at::kFloat    ? SVOX_POSITIONS_F32
                      : h.positions.scalar_type() == at::kDouble ? SVOX_POSITIONS_F64
                      : h.positions.scalar_type() == at::kInt    ? SVOX_POSITIONS_I32
                                                                 : SVOX_POSITIONS_I64;
    s.eps = (float)h.eps;
    return s;
}
std::pair<Tensor, Tensor> rotate_forward(const Heads& h) {
    const On on(h.q);
    Tensor y_q = make_like(h.q), y_k = make_like(h.k);
    const SvoxRotateHeads s = rotate_spec(h);
    status(lib.svox_rotate_heads(&s, y_q.data_ptr(), y_k.data_ptr(), on.stream), "rotate_heads");
    return {y_q, y_k};
}

struct RotateNode : torch::autograd::Node {
    Kept saved_[6];   // q, k, positions, frequencies and the weights
    bool interleaved = false;
    double eps = 0.0;

    std::string name() const override { return "SvoxRotateHeadsBackward"; }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        for (Kept& v : saved_) v.reset();
    }
    variable_list apply(variable_list&& grads) override {
        const std::lock_guard<std::mutex> lock(mutex_);
        variable_list out(4);
        if (!grads[0].defined() && !grads[1].defined()) return out;
        const auto kept = [&](int i) { return saved_[i].take_contiguous("rotate_heads"); };
        Heads h{saved_[0].take("rotate_heads"), saved_[1].take("rotate_heads"), kept(2), kept(3), kept(4), kept(5), interleaved, eps};
        const On on(h.q);
        h.q = heads_of(h.q), h.k = heads_of(h.k);
        for (int i = 0; i < 2; ++i) {
            if (!grads[i].defined()) {
                grads[i] = at::zeros((i ? h.k : h.q).sizes(), h.q.options());
                continue;
            }
            once("rotate_heads", grads[i]);
            check_like(grads[i], h.q, "grad_output", "q");
            grads[i] = heads_of(grads[i]);
        }
        const SvoxRotateHeads s = rotate_spec(h);
        if (task_should_compute_output(0)) out[0] = make_like(h.q);
        if (task_should_compute_output(1)) out[1] = make_like(h.k);
        if (task_should_compute_output(2)) out[2] = make({s.dim}, h.q.scalar_type(), h.q);
        if (task_should_compute_output(3)) out[3] = make({s.dim}, h.q.scalar_type(), h.q);
        const int64_t strides[4] = {grads[0].stride(0), grads[0].stride(1), grads[1].stride(0), grads[1].stride(1)};
        const int64_t bytes = status(lib.svox_rotate_heads_workspace_bytes(&s, out[2].defined() || out[3].defined()), "rotate_heads");
        const Tensor space = bytes_on(h.q, bytes);
        status(lib.svox_rotate_heads_backward(&s, grads[0].data_ptr(), grads[1].data_ptr(), strides, at_or_null(out[0]), at_or_null(out[1]),
                                              at_or_null(out[2]), at_or_null(out[3]), at_or_null(space), bytes, on.stream),
               "rotate_heads_backward");
        return out;
    }
};

std::pair<Tensor, Tensor> rotate_heads(Heads h) {
    no_tracing("rotate_heads");
    const Tensor q = h.q, k = h.k;
    check_like(q, q, "q", "q");
    dtype_code(q, "q");
    check_like(k, q, "k", "q");
    check_3d(q, "q");
    check_3d(k, "k");
    if (k.size(0) != q.size(0) || k.size(2) != q.size(2))
        fail("q and k must have the same rows and numbers of a head, got " + shape_text(q.sizes()) + " and " + shape_text(k.sizes()));
    const int64_t d = size32(q.size(2), "the numbers of a head");
    size32(q.size(1), "the number of heads");
    size32(k.size(1), "the number of k's heads");
    const Tensor &p = h.positions, &f = h.frequencies;
    if (!p.is_cuda() || p.device() != q.device() || p.layout() != at::kStrided) fail("positions must be a dense tensor on the device of q (" + q.device().str() + ")");
    if (p.scalar_type() != at::kFloat && p.scalar_type() != at::kDouble && p.scalar_type() != at::kInt && p.scalar_type() != at::kLong)
        fail("positions must be a float32, float64, int32 or int64 tensor, got " + dtype_text(p.scalar_type()));
    if (p.dim() < 1 || p.dim() > 2 || p.size(0) != q.size(0)) fail("positions must have shape (rows of q,) or (rows of q, axes), got " + shape_text(p.sizes()));
    if (!f.is_cuda() || f.device() != q.device() || f.layout() != at::kStrided) fail("frequencies must be a dense tensor on the device of q (" + q.device().str() + ")");
    if (f.scalar_type() != at::kFloat) fail("expected scalar type torch.float32 for frequencies but found " + dtype_text(f.scalar_type()));
    const int64_t axes = p.dim() == 2 ? p.size(1) : 1;
    if (f.dim() < 1 || f.dim() > 2 || f.dim() != p.dim() || (f.dim() == 2 && f.size(0) != axes))
        fail("frequencies must have shape (axes, pairs), or (pairs,) for positions of one axis, got " + shape_text(f.sizes()) + " for positions " + shape_text(p.sizes()));
    if (2 * f.size(-1) > d) fail("frequencies are of " + std::to_string(f.size(-1)) + " pairs, more than a head of " + std::to_string(d) + " numbers has");
    if (at::GradMode::is_enabled() && (p.requires_grad() || f.requires_grad())) fail("svox.rotate_heads has no gradient of positions or frequencies");
    if (p._fw_grad(0).defined() || f._fw_grad(0).defined()) fail("svox.rotate_heads has no derivatives in forward mode");
    if (h.q_weight.defined()) check_like(h.q_weight, q, "q_weight", "q"), check_shape(h.q_weight, {d}, "q_weight");
    if (h.k_weight.defined()) check_like(h.k_weight, q, "k_weight", "q"), check_shape(h.k_weight, {d}, "k_weight");
    if (p.dim() == 1) h.positions = p.unsqueeze(1);
    if (f.dim() == 1) h.frequencies = f.unsqueeze(0);
    for (Tensor* t : {&h.positions, &h.frequencies, &h.q_weight, &h.k_weight}) make_contiguous(*t);
    const bool wants = wants_node({&q, &k, &h.q_weight, &h.k_weight}, "rotate_heads");
    std::shared_ptr<RotateNode> node;
    if (wants) node = node_of<RotateNode>(q, k, h.q_weight, h.k_weight);
    std::pair<Tensor, Tensor> y;
    {
        const at::AutoDispatchBelowADInplaceOrView guard;
        Heads dense = h;
        dense.q = heads_of(q), dense.k = heads_of(k);
        y = rotate_forward(dense);
    }
    if (!wants) return y;
    const Tensor* const saved[6] = {&q, &k, &h.positions, &h.frequencies, &h.q_weight, &h.k_weight};
    for (int i = 0; i < 6; ++i) node->saved_[i].keep(*saved[i]);
    node->interleaved = h.interleaved;
    node->eps = h.eps;
    torch::autograd::set_history(std::vector<Tensor>{y.first, y.second}, node);
    return y;
}

// ---- attention
constexpr double kDefaultScale = -HUGE_VAL;   // 1 / sqrt(numbers of a head)
struct Attend {
    Tensor q, k, v, offsets, key_offsets;
    bool causal = false;
    double scale = 0.0;
};
SvoxAttention attention_spec(const Attend& a) {
    SvoxAttention s{};
    s.q = a.q.data_ptr(), s.k = a.k.data_ptr(), s.v = a.v.data_ptr();
    s.offsets = at_or_null(a.offsets);
    s.key_offsets = at_or_null(a.key_offsets);
    s.queries = a.q.size(0);
    s.keys = a.k.size(0);
    s.sequences = a.offsets.defined() ? a.offsets.numel() - 1 : 1;
    s.q_stride = a.q.stride(0), s.q_head = a.q.stride(1);
    s.k_stride = a.k.stride(0), s.k_head = a.k.stride(1);
    s.v_stride = a.v.stride(0), s.v_head = a.v.stride(1);
    s.heads = (int32_t)a.q.size(1);
    s.kv_heads = (int32_t)a.k.size(1);
    s.dim = (int32_t)a.q.size(2);
    s.dtype = dtype_code(a.q, "q");
    s.wide_offsets = a.offsets.defined() && a.offsets.scalar_type() == at::kLong;
    s.causal = a.causal;
    s.scale = (float)a.scale;
    return s;
}
Attend dense_heads(Attend a) {
    a.q = heads_of(a.q), a.k = heads_of(a.k), a.v = heads_of(a.v);
    return a;
}
// `lse` and `rest`: what a backward pass needs; rest only of 16-bit types
Tensor attention_forward(const Attend& a, Tensor* lse, Tensor* rest) {
    const On on(a.q);
    Tensor y = make_like(a.q);
    if (lse) *lse = make({a.q.size(0) * a.q.size(1)}, at::kFloat, a.q);
    if (rest && a.q.scalar_type() != at::kFloat) *rest = make_like(a.q);
    const SvoxAttention s = attention_spec(a);
    const int64_t bytes = status(lib.svox_attention_workspace_bytes(&s, 0), "attention");
    const Tensor space = bytes_on(a.q, bytes);
    status(lib.svox_attention(&s, y.data_ptr(), lse ? (float*)lse->data_ptr() : nullptr, rest ? at_or_null(*rest) : nullptr, at_or_null(space), bytes, on.stream), "attention");
    return y;
}

struct AttendNode : torch::autograd::Node {
    Kept saved_[5], out_, lse_, rest_;   // q, k, v and the offsets
    bool causal = false;
    double scale = 0.0;

    std::string name() const override { return "SvoxAttentionBackward"; }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        for (Kept& v : saved_) v.reset();
        out_.reset();
        lse_.reset();
        rest_.reset();
    }
    variable_list apply(variable_list&& grads) override {
        const std::lock_guard<std::mutex> lock(mutex_);
        variable_list out(3);
        if (!grads[0].defined()) return out;
        once("attention", grads[0]);
        const auto kept = [&](int i) { return saved_[i].take("attention"); };
        Attend a{kept(0), kept(1), kept(2), saved_[3].take_contiguous("attention"), saved_[4].take_contiguous("attention"), causal, scale};
        const Tensor y = out_.take_contiguous("attention", shared_from_this()), lse = lse_.take_contiguous("attention"), rest = rest_.take_contiguous("attention");
        const On on(a.q);
        check_like(grads[0], a.q, "grad_output", "q");
        a = dense_heads(a);
        const Tensor dy = heads_of(grads[0]);
        const SvoxAttention s = attention_spec(a);
        const Tensor* const like[3] = {&a.q, &a.k, &a.v};
        for (int i = 0; i < 3; ++i)
            if (task_should_compute_output(i)) out[i] = make_like(*like[i]);
        SvoxAttentionGrads g{};
        g.out = y.data_ptr();
        g.lse = (const float*)lse.data_ptr();
        g.rest = at_or_null(rest);
        g.grad = dy.data_ptr();
        g.grad_stride = dy.stride(0), g.grad_head = dy.stride(1);
        g.q = at_or_null(out[0]), g.k = at_or_null(out[1]), g.v = at_or_null(out[2]);
        const int64_t bytes = status(lib.svox_attention_workspace_bytes(&s, 1), "attention");
        const Tensor space = bytes_on(a.q, bytes);
        status(lib.svox_attention_backward(&s, &g, at_or_null(space), bytes, on.stream), "attention_backward");
        return out;
    }
};

void check_offsets(const Tensor& x, const Tensor& q, const char* name) {
    if (!x.is_cuda() || x.device() != q.device() || x.layout() != at::kStrided) fail(std::string(name) + " must be a dense tensor on the device of q (" + q.device().str() + ")");
    if (x.scalar_type() != at::kInt && x.scalar_type() != at::kLong) fail(std::string(name) + " must be an int32 or int64 tensor, got " + dtype_text(x.scalar_type()));
    if (x.dim() != 1 || x.numel() < 2) fail(std::string(name) + " must have shape (sequences + 1,), got " + shape_text(x.sizes()));
}

Tensor attention(Attend a) {
    no_tracing("attention");
    const Tensor &q = a.q, &k = a.k, &v = a.v;
    check_like(q, q, "q", "q");
    dtype_code(q, "q");
    check_like(k, q, "k", "q");
    check_like(v, q, "v", "q");
    check_3d(q, "q");
    check_3d(k, "k");
    check_shape(v, k.sizes(), "v");
    if (k.size(2) != q.size(2)) fail("q and k must have the same numbers of a head, got " + shape_text(q.sizes()) + " and " + shape_text(k.sizes()));
    const int64_t h = size32(q.size(1), "the number of heads"), g = size32(k.size(1), "the number of k's heads");
    size32(q.size(2), "the numbers of a head");
    if (h % g) fail("the number of heads must be a multiple of that of k's, got " + std::to_string(h) + " and " + std::to_string(g));
    if (a.offsets.defined()) check_offsets(a.offsets, q, "offsets");
    if (a.key_offsets.defined()) {
        if (!a.offsets.defined()) fail("key_offsets need offsets");
        check_offsets(a.key_offsets, q, "key_offsets");
        if (a.key_offsets.numel() != a.offsets.numel() || a.key_offsets.scalar_type() != a.offsets.scalar_type())
            fail("offsets and key_offsets must have the same shape and type, got " + shape_text(a.offsets.sizes()) + " " + dtype_text(a.offsets.scalar_type()) + " and " +
                 shape_text(a.key_offsets.sizes()) + " " + dtype_text(a.key_offsets.scalar_type()));
    } else if (a.offsets.defined() && q.size(0) != k.size(0)) {
        fail("without key_offsets there must be as many keys as queries, got " + std::to_string(k.size(0)) + " and " + std::to_string(q.size(0)));
    }
    if (a.scale == kDefaultScale) a.scale = 1.0 / std::sqrt((double)q.size(2));
    if (!(a.scale > 0.0) || std::isinf(a.scale)) fail("scale must be > 0 and finite, got " + std::to_string(a.scale));
    make_contiguous(a.offsets);
    make_contiguous(a.key_offsets);
    if (!wants_node({&q, &k, &v}, "attention")) return attention_forward(dense_heads(a), nullptr, nullptr);
    const auto node = node_of<AttendNode>(q, k, v);
    Tensor lse, rest, y;
    {
        const at::AutoDispatchBelowADInplaceOrView guard;
        y = attention_forward(dense_heads(a), &lse, &rest);
    }
    const Tensor* const saved[5] = {&q, &k, &v, &a.offsets, &a.key_offsets};
    for (int i = 0; i < 5; ++i) node->saved_[i].keep(*saved[i]);
    node->lse_.keep(lse);
    node->rest_.keep(rest);
    node->causal = a.causal;
    node->scale = a.scale;
    torch::autograd::set_history(y, node);
    node->out_.keep(y, true);
    return y;
}

// ---- called from Python with positional arguments
double number(PyObject* x) {
    const double v = PyFloat_AsDouble(x);
    if (v == -1.0 && PyErr_Occurred()) throw py::error_already_set();
    return v;
}
double scale_of(PyObject* x) {
    const double v = number(x);
    return v == kDefaultScale ? HUGE_VAL : v;   // (refused alike)
}
bool truth(PyObject* x) {
    const int v = PyObject_IsTrue(x);
    if (v < 0) throw py::error_already_set();
    return v != 0;
}
PyObject* pair_of(PyObject* a, PyObject* b) {
    if (!a || !b) {
        Py_XDECREF(a);
        Py_XDECREF(b);
        return nullptr;
    }
    PyObject* const both = PyTuple_Pack(2, a, b);
    Py_DECREF(a);
    Py_DECREF(b);
    return both;
}
PyObject* clip_norm_py(PyObject*, PyObject* const* args, Py_ssize_t given) {
    return call(given, 2, [&]() -> PyObject* {
        const std::vector<Tensor> all = tensors_of(args[0], "every one of tensors");
        const double most = number(args[1]);
        std::vector<Tensor> out;
        Tensor norm;
        {
            const py::gil_scoped_release unlocked;
            norm = clip_norm(all, most, out);
        }
        PyObject* const list = PyList_New((Py_ssize_t)out.size());
        if (!list) return nullptr;
        for (size_t i = 0; i < out.size(); ++i) PyList_SET_ITEM(list, (Py_ssize_t)i, THPVariable_Wrap(out[i]));
        return pair_of(THPVariable_Wrap(norm), list);
    });
}
PyObject* clip_in_place_py(PyObject*, PyObject* const* args, Py_ssize_t given) {
    return call(given, 2, [&]() -> PyObject* {
        const std::vector<Tensor> all = tensors_of(args[0], "every gradient");
        const double most = number(args[1]);
        Tensor norm;
        {
            const py::gil_scoped_release unlocked;
            norm = clip_in_place(all, most);
        }
        return THPVariable_Wrap(norm);
    });
}
PyObject* rotate_heads_py(PyObject*, PyObject* const* args, Py_ssize_t given) {
    return call(given, 8, [&]() -> PyObject* {
        const Heads h{tensor(args[0], "q"), tensor(args[1], "k"), tensor(args[2], "positions"), tensor(args[3], "frequencies"),
                      tensor_or_none(args[4], "q_weight"), tensor_or_none(args[5], "k_weight"), truth(args[6]), number(args[7])};
        std::pair<Tensor, Tensor> y;
        {
            const py::gil_scoped_release unlocked;
            y = rotate_heads(h);
        }
        return pair_of(THPVariable_Wrap(y.first), THPVariable_Wrap(y.second));
    });
}
PyObject* attention_py(PyObject*, PyObject* const* args, Py_ssize_t given) {
    return call(given, 7, [&] {
        const Attend a{tensor(args[0], "q"), tensor(args[1], "k"), tensor(args[2], "v"), tensor_or_none(args[3], "offsets"), tensor_or_none(args[4], "key_offsets"),
                       truth(args[5]), args[6] == Py_None ? kDefaultScale : scale_of(args[6])};
        const py::gil_scoped_release unlocked;
        return attention(a);
    });
}
PyMethodDef kCalls[] = {{"attention", (PyCFunction)(void (*)())attention_py, METH_FASTCALL, nullptr},
                        {"clip_norm", (PyCFunction)(void (*)())clip_norm_py, METH_FASTCALL, nullptr},
                        {"clip_in_place", (PyCFunction)(void (*)())clip_in_place_py, METH_FASTCALL, nullptr},
                        {"rotate_heads", (PyCFunction)(void (*)())rotate_heads_py, METH_FASTCALL, nullptr},
                        {nullptr, nullptr, 0, nullptr}};

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("init", &init);
    PyModule_AddFunctions(m.ptr(), kCalls);
}
