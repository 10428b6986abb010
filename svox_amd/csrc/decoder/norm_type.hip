// norm_type.hip -- the layer norm kernels of one type (SVOX_DECODER_TYPE) and their launches.
#include "entry.h"
#include "norm_kernels.h"

namespace svox_decoder {

using T = SVOX_DECODER_TYPE;

namespace {

// The lanes that hold a row: as few as do it with one or two pieces each, up to a wavefront; then more pieces, then a block.
#define SVOX_NORM_SHAPE(pieces, ...)                                                          \
    if ((pieces) <= 4) { constexpr int kLanes = 4, kPieces = 1; __VA_ARGS__; }                \
    else if ((pieces) <= 8) { constexpr int kLanes = 8, kPieces = 1; __VA_ARGS__; }           \
    else if ((pieces) <= 16) { constexpr int kLanes = 16, kPieces = 1; __VA_ARGS__; }         \
    else if ((pieces) <= 32) { constexpr int kLanes = 32, kPieces = 1; __VA_ARGS__; }         \
    else if ((pieces) <= 64) { constexpr int kLanes = 64, kPieces = 1; __VA_ARGS__; }         \
    else if ((pieces) <= 128) { constexpr int kLanes = 64, kPieces = 2; __VA_ARGS__; }        \
    else if ((pieces) <= 256) { constexpr int kLanes = 64, kPieces = 4; __VA_ARGS__; }        \
    else if ((pieces) <= 512) { constexpr int kLanes = 256, kPieces = 2; __VA_ARGS__; }       \
    else if ((pieces) <= 1024) { constexpr int kLanes = 256, kPieces = 4; __VA_ARGS__; }      \
    else { constexpr int kLanes = 0, kPieces = 0; __VA_ARGS__; }

NormArgs<T> args(const SvoxLayerNorm& s) {
    NormArgs<T> p{};
    p.x = (const T*)s.x;
    p.weight = (const T*)s.weight;
    p.bias = (const T*)s.bias;
    p.x_ld = s.x_stride;
    p.rows = s.rows;
    p.dim = s.dim;
    p.eps = s.eps;
    return p;
}

}  // namespace

template <>
int launch_norm<T>(const SvoxLayerNorm& s, void* y, float* stats, hipStream_t stream) {
    NormArgs<T> p = args(s);
    p.y = (T*)y;
    p.stats = stats;
    const int64_t row_pieces = pieces(s.dim, kNormPiece<T>);
    SVOX_NORM_SHAPE(row_pieces, {
        if constexpr (kLanes > 0) {
            const int64_t blocks = least(pieces(s.rows, kNormThreads / kLanes), 2048);
            hipLaunchKernelGGL((norm_kernel<T, kLanes, kPieces>), dim3((unsigned)blocks), dim3(kNormThreads), 0, stream, p);
        } else {
            hipLaunchKernelGGL((norm_long_kernel<T, false>), dim3((unsigned)least(s.rows, 2048)), dim3(kNormThreads), 0, stream, p);
        }
    });
    return check_launch("layer_norm");
}

template <>
int launch_norm_backward<T>(const SvoxLayerNorm& s, const float* stats, const void* grad_output, int64_t grad_stride, void* grad_x,
                            void* grad_weight, void* grad_bias, float* part, hipStream_t stream) {
    NormArgs<T> p = args(s);
    p.dy = (const T*)grad_output;
    p.dy_ld = grad_stride;
    p.stats = const_cast<float*>(stats);
    p.y = (T*)grad_x;
    p.part = part;
    const int64_t row_pieces = pieces(s.dim, kNormPiece<T>);
    const int blocks = norm_backward_blocks(s.rows, s.dim, kNormPiece<T>);
    SVOX_NORM_SHAPE(row_pieces, {
        if constexpr (kLanes > 0)
            hipLaunchKernelGGL((norm_backward_kernel<T, kLanes, kPieces>), dim3(blocks), dim3(kNormThreads), 0, stream, p);
        else
            hipLaunchKernelGGL((norm_long_kernel<T, true>), dim3(blocks), dim3(kNormThreads), 0, stream, p);
    });
    if (part)
        hipLaunchKernelGGL((norm_join_kernel<T>), grid_of(least(pieces(2 * (int64_t)s.dim, kNormJoinColumns), 1 << 16), kNormJoinThreads),
                           dim3(kNormJoinThreads), 0, stream, part, blocks, s.dim, (T*)grad_weight, (T*)grad_bias);
    return check_launch("layer_norm_backward");
}

}  // namespace svox_decoder
