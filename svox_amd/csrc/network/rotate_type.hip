// rotate_type.hip -- the kernels of one type (SVOX_DECODER_TYPE) that rotate heads, and their launches.
#include "entry.h"
#include "rotate_kernels.h"

namespace svox_network {

using T = SVOX_DECODER_TYPE;

namespace {

int pieces_of(const SvoxRotateHeads& s) {
    const int pairs = s.rotated / 2, rest = (s.dim - s.rotated + 1) / 2;
    return (int)(pieces(pairs, kRotatePairs<T>) + pieces(rest, kRotatePairs<T>));
}
int lanes_of(const SvoxRotateHeads& s) {
    int lanes = 2;
    while (lanes < pieces_of(s)) lanes *= 2;
    return lanes;
}
// Rows of a block at a time: enough of them for two keys' heads of every lane group, as far as LDS holds their angles, and as long as there are
// rows for all blocks.  (262 144 rows of 8 + 2 heads of 32: 16 rows 105 us, 64 rows and more 98.)
int rows_at_once(const SvoxRotateHeads& s) {
    int64_t rows = pieces(2 * kRotateThreads / lanes_of(s), (int64_t)s.kv_heads);
    rows = least(least(rows, kRotateTurns / (s.rotated < 2 ? 1 : s.rotated / 2)), pieces(s.rows, 1024));
    return (int)(rows < 1 ? 1 : rows);
}
RotateArgs<T> args(const SvoxRotateHeads& s) {
    RotateArgs<T> p{};
    p.x[0] = (const T*)s.q, p.x[1] = (const T*)s.k;
    p.weight[0] = (const T*)s.q_weight, p.weight[1] = (const T*)s.k_weight;
    p.x_stride[0] = s.q_stride, p.x_stride[1] = s.k_stride;
    p.x_head[0] = s.q_head, p.x_head[1] = s.k_head;
    p.heads[0] = s.heads, p.heads[1] = s.kv_heads;
    p.positions = s.positions;
    p.frequencies = s.frequencies;
    p.rows = s.rows;
    p.dim = s.dim, p.rotated = s.rotated, p.axes = s.axes, p.position_type = s.position_type;
    p.rows_at_once = rows_at_once(s);
    p.eps = s.eps;
    return p;
}
template <bool interleaved, bool backward>
void launch(const RotateArgs<T>& p, int lanes, int blocks, hipStream_t stream) {
    const auto with = [&](auto n) {
        hipLaunchKernelGGL((rotate_kernel<T, decltype(n)::value, interleaved, backward>), dim3(blocks), dim3(kRotateThreads), 0, stream, p);
    };
    switch (lanes) {
        case 2: return with(std::integral_constant<int, 2>());
        case 4: return with(std::integral_constant<int, 4>());
        case 8: return with(std::integral_constant<int, 8>());
        case 16: return with(std::integral_constant<int, 16>());
        case 32: return with(std::integral_constant<int, 32>());
        default: return with(std::integral_constant<int, 64>());
    }
}

}  // namespace

template <>
int rotate_backward_blocks<T>(const SvoxRotateHeads& s) {
    return (int)least(pieces(s.rows, rows_at_once(s)), kRotateMostBlocks);
}

template <>
int launch_rotate<T>(const SvoxRotateHeads& s, void* y_q, void* y_k, hipStream_t stream) {
    RotateArgs<T> p = args(s);
    p.y[0] = (T*)y_q, p.y[1] = (T*)y_k;
    const int blocks = (int)least(pieces(s.rows, p.rows_at_once), 4096);
    if (s.interleaved) launch<true, false>(p, lanes_of(s), blocks, stream);
    else launch<false, false>(p, lanes_of(s), blocks, stream);
    return check_launch("rotate_heads");
}

template <>
int launch_rotate_backward<T>(const SvoxRotateHeads& s, const void* grad_q, const void* grad_k, const int64_t* grad, void* out_q, void* out_k,
                              void* out_q_weight, void* out_k_weight, float* part, hipStream_t stream) {
    RotateArgs<T> p = args(s);
    p.dy[0] = (const T*)grad_q, p.dy[1] = (const T*)grad_k;
    p.dy_stride[0] = grad[0], p.dy_head[0] = grad[1], p.dy_stride[1] = grad[2], p.dy_head[1] = grad[3];
    p.y[0] = (T*)out_q, p.y[1] = (T*)out_k;
    p.part = part;
    const int blocks = rotate_backward_blocks<T>(s);
    if (s.interleaved) launch<true, true>(p, lanes_of(s), blocks, stream);
    else launch<false, true>(p, lanes_of(s), blocks, stream);
    if (part)
        hipLaunchKernelGGL((rotate_join_kernel<T>), dim3((unsigned)pieces(2 * s.dim, 16)), dim3(1024), 0, stream, part, blocks, s.dim, (T*)out_q_weight,
                           (T*)out_k_weight);
    return check_launch("rotate_heads_backward");
}

}  // namespace svox_network
