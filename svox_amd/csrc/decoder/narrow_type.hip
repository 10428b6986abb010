// narrow_type.hip -- the kernels of narrow layers of one type (SVOX_DECODER_TYPE) with one activation (SVOX_DECODER_ACTIVATION), and
// their launches.
#include "ffn_plan.h"

namespace svox_decoder {

using T = SVOX_DECODER_TYPE;
constexpr int kActivation = SVOX_DECODER_ACTIVATION;

namespace {

NarrowArgs<T> narrow_args(const SvoxGatedFfn& s, const u16* chunks) {
    NarrowArgs<T> p{};
    p.x = (const T*)s.x;
    p.x_ld = s.x_stride;
    p.chunks = chunks;
    p.rows = s.rows;
    p.dim = s.dim;
    p.hidden = s.hidden;
    p.out = s.out;
    return p;
}
template <class F>
void by_rows(int64_t rows, F launch) {
    if constexpr (Form<T>::planes == 1) {
        if (Rules<1>::narrow_tiles(rows) == 2) return launch(std::integral_constant<int, 2>());
    }
    launch(std::integral_constant<int, 1>());
}

// `launch` for all rows, 2^28 of them at a time: four lanes to a row or two, and a launch has less than 2^32.  cols: numbers of a row of y
template <class F>
void in_launches(NarrowArgs<T> p, int64_t cols, F launch) {
    constexpr int64_t most = (int64_t)1 << 28;
    for (int64_t left = p.rows; left > 0; left -= most) {
        p.rows = least(left, most);
        launch(p);
        p.x += p.rows * p.x_ld;
        p.y += p.rows * cols;
        if (p.dy) p.dy += p.rows * p.dy_ld;
        if (p.residual) p.residual += p.rows * p.residual_ld;
    }
}

template <int KD, int KO, bool backward>
void launch_narrow_lay(const SvoxGatedFfn& s, u16* to, hipStream_t stream) {
    using C = Chunk<KD, KO, backward>;
    NarrowLayArgs<T> p{(const T*)s.w_gate, (const T*)s.w_up, (const T*)s.w_down, (const T*)s.b_gate, (const T*)s.b_up, s.dim, s.hidden, s.out, to};
    hipLaunchKernelGGL((narrow_lay_kernel<T, KD, KO, backward>), grid_of(pieces(pieces(s.hidden, 32) * (C::fragments + 1), 4), 256), dim3(256), 0, stream,
                       p);
}
int narrow_forward(const SvoxGatedFfn& s, void* y, void* workspace, hipStream_t stream) {
    Room room(workspace);
    u16* const chunks = room.take<u16>(narrow_numbers<T>(s, false));
    NarrowArgs<T> p = narrow_args(s, chunks);
    p.b_down = (const T*)s.b_down;
    p.residual = (const T*)s.residual;
    p.residual_ld = s.residual_stride;
    p.y = (T*)y;
    SVOX_NARROW_STEPS(s.dim, KD, SVOX_NARROW_STEPS(s.out, KO, {
        launch_narrow_lay<KD, KO, false>(s, chunks, stream);
        const auto launch = [&](auto rows) {
            constexpr int QT = decltype(rows)::value;
            in_launches(p, s.out, [&](const NarrowArgs<T>& some) {
                hipLaunchKernelGGL((narrow_kernel<T, KD, KO, QT, kActivation>), grid_of(pieces(some.rows, 16 * QT * kNarrowWaves), kNarrowWaves * kWave),
                                   dim3(kNarrowWaves * kWave), 0, stream, some);
            });
        };
        by_rows(s.rows, launch);
    }));
    return check_launch("gated_ffn");
}

int narrow_backward(const SvoxGatedFfn& s, const void* grad_output, int64_t grad_stride, const SvoxGatedFfnGrads& grads, void* workspace,
                           hipStream_t stream) {
    const NarrowBackward<T> b(s, workspace);
    NarrowArgs<T> p = narrow_args(s, b.chunks);
    p.dy = (const T*)grad_output;
    p.dy_ld = grad_stride;
    p.y = (T*)grads.x;
    Parts<T> parts(b.part);
    NarrowWeightArgs<T> w{};
    w.x = p.x;
    w.x_ld = p.x_ld;
    w.dy = p.dy;
    w.dy_ld = p.dy_ld;
    w.chunks = b.chunks;
    w.gate = parts.take((int64_t)s.hidden * s.dim, b.split.splits, grads.w_gate);
    w.up = parts.take((int64_t)s.hidden * s.dim, b.split.splits, grads.w_up);
    w.down = parts.take((int64_t)s.hidden * s.out, b.split.splits, grads.w_down);
    w.b_gate = parts.take(s.hidden, b.split.splits, grads.b_gate);
    w.b_up = parts.take(s.hidden, b.split.splits, grads.b_up);
    w.b_down = parts.take(s.out, b.split.splits, grads.b_down);
    w.rows = s.rows;
    w.each = b.split.each;
    w.dim = s.dim;
    w.hidden = s.hidden;
    w.out = s.out;
    SVOX_NARROW_STEPS(s.dim, KD, SVOX_NARROW_STEPS(s.out, KO, {
        launch_narrow_lay<KD, KO, true>(s, b.chunks, stream);
        const auto launch = [&](auto rows) {
            constexpr int QT = decltype(rows)::value;
            in_launches(p, s.dim, [&](const NarrowArgs<T>& some) {
                hipLaunchKernelGGL((narrow_backward_kernel<T, KD, KO, QT, kActivation>),
                                   grid_of(pieces(some.rows, 16 * QT * kNarrowWaves), kNarrowWaves * kWave), dim3(kNarrowWaves * kWave), 0, stream, some);
            });
        };
        if (grads.x) by_rows(s.rows, launch);
        if (parts.jobs)
            hipLaunchKernelGGL((narrow_weight_kernel<T, KD, KO, kActivation>), dim3((unsigned)b.split.splits, (unsigned)b.split.down),
                               dim3((kNarrowWeightWaves<T, KD, KO>) * kWave), 0, stream, w);
    }));
    parts.launch(stream);
    return check_launch("gated_ffn_backward");
}

}  // namespace

template <>
int Narrow<T, kActivation>::forward(const SvoxGatedFfn& s, void* y, void* workspace, hipStream_t stream) {
    return narrow_forward(s, y, workspace, stream);
}
template <>
int Narrow<T, kActivation>::backward(const SvoxGatedFfn& s, const void* grad_output, int64_t grad_stride, const SvoxGatedFfnGrads& grads,
                                     void* workspace, hipStream_t stream) {
    return narrow_backward(s, grad_output, grad_stride, grads, workspace, stream);
}

}  // namespace svox_decoder
