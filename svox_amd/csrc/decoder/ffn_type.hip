// ffn_type.hip -- the kernels of the gated feed-forward block of one type (SVOX_DECODER_TYPE) and their launches.
#include "ffn_plan.h"

namespace svox_decoder {

using T = SVOX_DECODER_TYPE;

namespace {

constexpr int kPlanes = Form<T>::planes;
constexpr int64_t kMostLd = TileOf<true, 64, 64, 256>::most_ld;
using R = Rules<kPlanes>;
using Small = R::Small;
using Deep = R::Deep;
using Medium = R::Medium;
using Large = R::Large;
template <class F>
void by_size(Size size, F f) {
    if (size == kSmall) f(Small());
    else if (size == kDeep) f(Deep());
    else if (size == kMedium) f(Medium());
    else f(Large());
}

// ---- operands: where they are if the tiles can be read from there, else laid out in the workspace
bool tiles_read(const void* at, int64_t ld, int64_t cols) {
    return kPlanes == 1 && (uintptr_t)at % 16 == 0 && ld % 8 == 0 && cols % 8 == 0 && ld <= kMostLd;
}
struct Lays {
    LayArgs<T> args{};
    int count = 0;
    int64_t blocks = 0;
    Planes operand(Room& room, const void* at, int64_t ld, int64_t rows, int64_t cols) {
        if (tiles_read(at, ld, cols)) return Planes{(const u16*)at, ld, 0, rows, cols};
        const int64_t wide = up_to(cols, 8);
        Planes to{nullptr, wide, rows * wide, rows, wide};
        to.at = room.take<u16>(kPlanes * rows * wide);
        LayJob<T>& job = args.job[count++];
        const int lanes = wide >= 1024 ? 256 : wide >= 256 ? 64 : 16;
        // (some 4096 numbers to a block, and all of its lanes' rows at least)
        const int64_t each = up_to(pieces(4096, wide), kLayThreads / lanes);
        job = LayJob<T>{(const T*)at, ld, to, cols, pieces(rows, each), each, lanes};
        blocks += job.blocks;
        return to;
    }
    void launch(hipStream_t stream) const {
        if (blocks > 0) hipLaunchKernelGGL((lay_kernel<T>), grid_of(blocks, kLayThreads), dim3(kLayThreads), 0, stream, args);
    }
};
Planes hidden_numbers(Room& room, const SvoxGatedFfn& s) {
    const int64_t wide = up_to(s.hidden, 8);
    Planes h{nullptr, wide, s.rows * wide, s.rows, wide};
    h.at = room.take<u16>(kPlanes * s.rows * wide);
    return h;
}

// ---- few rows
template <bool backward>
void launch_few(const FewArgs<T>& p, bool result, hipStream_t stream) {
    const auto launch = [&](auto tiles) {
        constexpr int MT = decltype(tiles)::value;
        const unsigned down = (unsigned)pieces(p.rows, 16 * MT);
        hipLaunchKernelGGL((few_hidden_kernel<T, MT, backward>), dim3((unsigned)pieces(p.ldh, 16), down), dim3(kFewHiddenWaves * kWave), 0, stream, p);
        if (result)
            hipLaunchKernelGGL((few_output_kernel<T, MT, backward>), dim3((unsigned)pieces(backward ? p.dim : p.out, 16), down),
                               dim3(kFewOutputWaves * kWave), 0, stream, p);
    };
    if (p.rows <= 16) launch(std::integral_constant<int, 1>());
    else if (p.rows <= 32) launch(std::integral_constant<int, 2>());
    else launch(std::integral_constant<int, 4>());
}
FewArgs<T> few_args(const SvoxGatedFfn& s, const Planes& h) {
    FewArgs<T> p{};
    p.x = (const T*)s.x;
    p.w_gate = (const T*)s.w_gate;
    p.w_up = (const T*)s.w_up;
    p.w_down = (const T*)s.w_down;
    p.b_gate = (const T*)s.b_gate;
    p.b_up = (const T*)s.b_up;
    p.x_ld = s.x_stride;
    p.h = const_cast<u16*>(h.at);
    p.ldh = h.ld;
    p.plane = h.plane;
    p.rows = s.rows;
    p.dim = s.dim;
    p.hidden = s.hidden;
    p.out = s.out;
    p.activation = s.activation;
    return p;
}
int launch_few_forward(const SvoxGatedFfn& s, void* y, void* workspace, hipStream_t stream) {
    Room room(workspace);
    FewArgs<T> p = few_args(s, hidden_numbers(room, s));
    p.b_down = (const T*)s.b_down;
    p.residual = (const T*)s.residual;
    p.residual_ld = s.residual_stride;
    p.y = (T*)y;
    launch_few<false>(p, true, stream);
    return check_launch("gated_ffn");
}

// ---- narrow layers
template <class F>
int by_activation(int activation, F f) {
    switch (activation) {
        case kSilu: return f(std::integral_constant<int, kSilu>());
        case kGelu: return f(std::integral_constant<int, kGelu>());
        case kRelu: return f(std::integral_constant<int, kRelu>());
        default: return f(std::integral_constant<int, kSigmoid>());
    }
}

// ---- what a call keeps in its workspace
struct Forward {
    Lays lays;
    Planes x, w_gate, w_up, w_down, h;
    int64_t bytes;
    Forward(const SvoxGatedFfn& s, void* workspace) {
        Room room(workspace);
        x = lays.operand(room, s.x, s.x_stride, s.rows, s.dim);
        w_gate = lays.operand(room, s.w_gate, s.dim, s.hidden, s.dim);
        w_up = lays.operand(room, s.w_up, s.dim, s.hidden, s.dim);
        w_down = lays.operand(room, s.w_down, s.hidden, s.out, s.hidden);
        h = hidden_numbers(room, s);
        bytes = room.used;
    }
};

// The rows of the biases' sums of hidden_kernel.
int64_t hidden_parts(const SvoxGatedFfn& s) {
    int64_t parts = 0;
    by_size(R::hidden_size(s.rows, up_to(s.hidden, 8)), [&](auto shapes) {
        using S = typename decltype(shapes)::Hidden;
        parts = pieces(s.rows, S::BM) * S::WM;
    });
    return parts;
}
struct Backward {
    Lays lays;
    Planes x, w_gate, w_up, w_down, dy, h, dgate, dup;
    R::Split split;
    float* part;
    int64_t bytes, bias_parts;
    bool few;
    Backward(const SvoxGatedFfn& s, const void* grad_output, int64_t grad_stride, void* workspace, bool any_grad) {
        Room room(workspace);
        // (grad_output's address is not known when its workspace is asked for: there is room to lay it out)
        x = lays.operand(room, s.x, s.x_stride, s.rows, s.dim);
        few = R::few_rows(s, true);
        if (!few) {
            w_gate = lays.operand(room, s.w_gate, s.dim, s.hidden, s.dim);
            w_up = lays.operand(room, s.w_up, s.dim, s.hidden, s.dim);
            w_down = lays.operand(room, s.w_down, s.hidden, s.out, s.hidden);
        }
        h = hidden_numbers(room, s);
        dgate = hidden_numbers(room, s);
        dup = hidden_numbers(room, s);
        split = R::weight_split(s);
        bias_parts = few ? pieces(s.rows, 16) : hidden_parts(s);
        part = room.take<float>((split.splits > 1 ? split.splits * (2 * (int64_t)s.hidden * s.dim + (int64_t)s.hidden * s.out + s.out) : 0) +
                                bias_parts * 2 * s.hidden);
        if (any_grad)
            room.take<u16>(kPlanes * s.rows * up_to(s.out, 8));
        else
            dy = lays.operand(room, grad_output, grad_stride, s.rows, s.out);
        bytes = room.used;
    }
};

HiddenArgs<T> hidden_args(const SvoxGatedFfn& s, const Planes& x, const Planes& w_gate, const Planes& w_up, const Planes& h) {
    HiddenArgs<T> p{};
    p.x = x;
    p.w_gate = w_gate;
    p.w_up = w_up;
    p.b_gate = (const T*)s.b_gate;
    p.b_up = (const T*)s.b_up;
    p.h = const_cast<u16*>(h.at);
    p.ldh = h.ld;
    p.plane = h.plane;
    p.rows = s.rows;
    p.dim = s.dim;
    p.hidden = s.hidden;
    p.out = s.out;
    p.activation = s.activation;
    return p;
}

template <class S, bool backward>
void launch_hidden_as(HiddenArgs<T> p, hipStream_t stream) {
    p.tiles_m = pieces(p.rows, S::BM);
    p.tiles_n = pieces(p.ldh, S::BN);
    hipLaunchKernelGGL((hidden_kernel<T, S, backward>), grid_of(p.tiles_m * p.tiles_n, S::threads), dim3(S::threads), 0, stream, p);
}
template <bool backward>
void launch_hidden(const HiddenArgs<T>& p, hipStream_t stream) {
    by_size(R::hidden_size(p.rows, p.ldh), [&](auto shapes) { launch_hidden_as<typename decltype(shapes)::Hidden, backward>(p, stream); });
}
template <class S, bool along_b>
void launch_output_as(OutputArgs<T> p, hipStream_t stream) {
    p.tiles_m = pieces(p.rows, S::BM);
    p.tiles_n = pieces(p.cols, S::BN);
    hipLaunchKernelGGL((output_kernel<T, S, along_b>), grid_of(p.tiles_m * p.tiles_n, S::threads), dim3(S::threads), 0, stream, p);
}
template <bool along_b>
void launch_output(const OutputArgs<T>& p, hipStream_t stream) {
    by_size(R::output_size(p.rows, p.cols),
            [&](auto shapes) { launch_output_as<typename decltype(shapes)::Output, along_b>(p, stream); });
}

template <class S>
void launch_weight_as(WeightArgs<T> w, hipStream_t stream) {
    int64_t blocks = 0;
    for (WeightJob<T>& job : w.job) {   // (one that is not there has no columns)
        job.tiles_m = pieces(job.m, S::BM);
        job.tiles_n = pieces(job.n, S::BN);
        blocks += job.tiles_m * job.tiles_n;
    }
    hipLaunchKernelGGL((weight_kernel<T, S>), grid_of(blocks * w.splits, S::threads), dim3(S::threads), 0, stream, w);
}

}  // namespace

template <>
int64_t ffn_workspace<T>(const SvoxGatedFfn& s, bool backward) {
    if (backward && !R::few_rows(s, true) && R::narrow(s, true)) return NarrowBackward<T>(s, nullptr).bytes;
    if (backward) return Backward(s, nullptr, 0, nullptr, true).bytes;
    if (R::few_rows(s, false)) {
        Room room(nullptr);
        hidden_numbers(room, s);
        return room.used;
    }
    if (R::narrow(s, false)) {
        Room room(nullptr);
        room.take<u16>(narrow_numbers<T>(s, false));
        return room.used;
    }
    return Forward(s, nullptr).bytes;
}

template <>
int launch_ffn<T>(const SvoxGatedFfn& s, void* y, void* workspace, hipStream_t stream) {
    if (R::few_rows(s, false)) return launch_few_forward(s, y, workspace, stream);
    if (R::narrow(s, false)) return by_activation(s.activation, [&](auto a) { return Narrow<T, decltype(a)::value>::forward(s, y, workspace, stream); });
    const Forward f(s, workspace);
    f.lays.launch(stream);
    const HiddenArgs<T> p = hidden_args(s, f.x, f.w_gate, f.w_up, f.h);
    launch_hidden<false>(p, stream);
    OutputArgs<T> o{};
    o.a[0] = f.h;
    o.b[0] = f.w_down;
    o.bias = (const T*)s.b_down;
    o.residual = (const T*)s.residual;
    o.residual_ld = s.residual_stride;
    o.y = (T*)y;
    o.rows = s.rows;
    o.cols = s.out;
    launch_output<true>(o, stream);
    return check_launch("gated_ffn");
}

template <>
int launch_ffn_backward<T>(const SvoxGatedFfn& s, const void* grad_output, int64_t grad_stride, const SvoxGatedFfnGrads& grads, void* workspace,
                           hipStream_t stream) {
    if (!R::few_rows(s, true) && R::narrow(s, true))
        return by_activation(s.activation, [&](auto a) {
            return Narrow<T, decltype(a)::value>::backward(s, grad_output, grad_stride, grads, workspace, stream);
        });
    Backward b(s, grad_output, grad_stride, workspace, false);
    b.lays.launch(stream);
    Parts<T> parts(b.part);
    float* const b_gate_part = grads.b_gate ? parts.take(s.hidden, b.bias_parts, grads.b_gate) : nullptr;
    float* const b_up_part = grads.b_up ? parts.take(s.hidden, b.bias_parts, grads.b_up) : nullptr;
    if (b.few) {
        FewArgs<T> p = few_args(s, b.h);
        p.dy = (const T*)grad_output;
        p.dy_ld = grad_stride;
        p.dgate = const_cast<u16*>(b.dgate.at);
        p.dup = const_cast<u16*>(b.dup.at);
        p.b_gate_part = b_gate_part;
        p.b_up_part = b_up_part;
        p.y = (T*)grads.x;
        launch_few<true>(p, grads.x != nullptr, stream);
    } else {
        HiddenArgs<T> p = hidden_args(s, b.x, b.w_gate, b.w_up, b.h);
        p.dy = b.dy;
        p.w_down = b.w_down;
        p.dgate = const_cast<u16*>(b.dgate.at);
        p.dup = const_cast<u16*>(b.dup.at);
        p.b_gate_part = b_gate_part;
        p.b_up_part = b_up_part;
        launch_hidden<true>(p, stream);
        if (grads.x) {
            OutputArgs<T> o{};
            o.a[0] = b.dgate;
            o.a[1] = b.dup;
            o.b[0] = b.w_gate;
            o.b[1] = b.w_up;
            o.y = (T*)grads.x;
            o.rows = s.rows;
            o.cols = s.dim;
            launch_output<false>(o, stream);
        }
    }
    WeightArgs<T> w{};
    const int64_t H = s.hidden, D = s.dim, O = s.out;
    void* const outs[3] = {grads.w_gate, grads.w_up, grads.w_down};
    void* const sums[3] = {nullptr, nullptr, grads.b_down};
    const Planes left[3] = {b.dgate, b.dup, b.dy}, right[3] = {b.x, b.x, b.h};
    int jobs = 0;
    for (int j = 0; j < 3; ++j) {
        if (!outs[j] && !sums[j]) continue;
        WeightJob<T>& job = w.job[jobs++];
        job.a = left[j];
        job.b = right[j];
        job.m = j < 2 ? H : O;
        job.n = j < 2 ? D : H;
        job.out = (T*)outs[j];
        job.sums_out = (T*)sums[j];
        if (b.split.splits > 1) {
            if (outs[j]) job.part = parts.take(job.m * job.n, b.split.splits, outs[j]);
            if (sums[j]) job.sums_part = parts.take(job.m, b.split.splits, sums[j]);
        }
    }
    if (jobs) {
        w.rows = s.rows;
        w.each = b.split.each;
        w.splits = b.split.splits;
        by_size(b.split.size, [&](auto shapes) { launch_weight_as<typename decltype(shapes)::Weight>(w, stream); });
    }
    parts.launch(stream);
    return check_launch("gated_ffn_backward");
}

}  // namespace svox_decoder
