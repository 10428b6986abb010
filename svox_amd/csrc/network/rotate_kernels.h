// rotate_kernels.h -- heads of queries and keys, divided by the root of the mean of their squares and rotated by their row's positions;
// and the gradients of that.
//
//   n = x r w,  r = 1 / sqrt(mean(x^2) + eps);   (y_a, y_b) = (n_a c - n_b s, n_b c + n_a s),  c, s = cos, sin of the row's angle of the pair
//   dn = dy rotated back,  dw = sum over rows and heads of dn x r,  g = dn w,  dx = r (g - x r mean(g x r))
//
// Every number is read once and written once, and some ten (backward: thirty) instructions lie between: bound by memory, if the angles
// are not computed too often.  They are the same for all heads of a row: a block takes a few rows, computes their sines and cosines into
// LDS and goes through the rows' heads with them.  A head lies in the registers of 1 to 64 lanes, each of which holds the two numbers of
// kRotatePairs pairs, 16 bytes of each side, so that the rotation is within a lane; what is not rotated is split into two sides
// the same way, with its last number alone where there is an odd one.
//
// Angles are multiplied out in 64 bits and brought within an eighth of a turn of a quarter before they become 32: a position of 2^20 loses as
// little as one of 1.  Sums are in 32 bits; weights' gradients are summed by lane over its rows and heads, over the block's lanes, and over
// the blocks by rotate_join_kernel, in an order of their own: the same call gives the same bits.
#pragma once
#include "../decoder/common.h"
#include "../../../include/svox_network.h"

namespace svox_network {

using namespace svox_decoder;

constexpr int kRotateThreads = 256, kRotateTurns = 2048, kRotateMostDim = 256, kRotateMostBlocks = 1024;

template <class T>
constexpr int kRotatePairs = 16 / (int)sizeof(T);

template <class T>
struct RotateArgs {
    const T* x[2];            // queries and keys
    const T* weight[2];
    const T* dy[2];
    T* y[2];                  // dense; backward: dx, or NULL
    int64_t x_stride[2], x_head[2], dy_stride[2], dy_head[2];
    int heads[2];
    const void* positions;
    const float* frequencies;
    float* part;              // backward: [blocks][2][dim], or NULL
    int64_t rows;
    int dim, rotated, axes, position_type, rows_at_once;
    float eps;
};

__device__ __forceinline__ double position(const void* at, int type, int64_t i) {
    switch (type) {
        case SVOX_POSITIONS_F32: return (double)((const float*)at)[i];
        case SVOX_POSITIONS_F64: return ((const double*)at)[i];
        case SVOX_POSITIONS_I32: return (double)((const int32_t*)at)[i];
        default: return (double)((const int64_t*)at)[i];
    }
}

// (cos, sin) of an angle.  For results of 16 bits by the hardware's functions of turns, good to 2^-20 or so; else float32's own.
template <bool accurate>
__device__ __forceinline__ float2 turn_of(double angle) {
    const double turns = angle * 0.15915494309189533577;
    const double quarters = rint(turns * 4.0);
    const float left = (float)__builtin_fma(quarters, -0.25, turns);   // within an eighth
    float c, s;
    if constexpr (accurate) {
        sincospif(2.0f * left, &s, &c);
    } else {
        s = __builtin_amdgcn_sinf(left);
        c = __builtin_amdgcn_cosf(left);
    }
    const int q = (int)(quarters - 4.0 * floor(quarters * 0.25));
    float2 v = q & 1 ? make_float2(-s, c) : make_float2(c, s);
    if (q & 2) v = make_float2(-v.x, -v.y);
    return v;
}

// Which numbers of a head a lane holds: `a` of one side from a_at on, `b` of the other from b_at on.
struct RotatePiece {
    int a_at, b_at, a, b, pair;   // pair: the first one's angle, or -1 where nothing is rotated
};
template <int W>
__device__ __forceinline__ RotatePiece piece_of(int piece, int dim, int rotated) {
    const int pairs = rotated / 2, turned = (pairs + W - 1) / W;
    if (piece < turned) {
        const int n = min(W, pairs - piece * W);
        return {piece * W, pairs + piece * W, n, n, piece * W};
    }
    const int i = (piece - turned) * W, first = (dim - rotated + 1) / 2;
    return {rotated + i, rotated + first + i, max(0, min(W, first - i)), max(0, min(W, dim - rotated - first - i)), -1};
}

// The two sides of a lane's pairs as they lie in memory, zeros beyond them, and as numbers.  (Interleaved pairs lie side by side.)
template <class T, int W>
struct RawPairs {
    typename Few<T, W>::vector first, second;
};
template <class T, bool interleaved, int W>
__device__ __forceinline__ RawPairs<T, W> load_pairs(const T* head, const RotatePiece& p) {
    if (interleaved && p.pair >= 0) return {load_some<T, W>(head + 2 * p.pair, 2 * p.a), load_some<T, W>(head + 2 * p.pair + W, 2 * p.a - W)};
    return {load_some<T, W>(head + p.a_at, p.a), load_some<T, W>(head + p.b_at, p.b)};
}
template <class T, bool interleaved, int W>
__device__ __forceinline__ void numbers_of(const RawPairs<T, W>& raw, const RotatePiece& p, float (&a)[W], float (&b)[W]) {
    const bool beside = interleaved && p.pair >= 0;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        const float x = (float)raw.first[i], y = (float)raw.second[i];
        if (!interleaved) {
            a[i] = x, b[i] = y;
        } else {
            const float even = 2 * i < W ? (float)raw.first[2 * i % W] : (float)raw.second[2 * i % W];
            const float odd = 2 * i + 1 < W ? (float)raw.first[(2 * i + 1) % W] : (float)raw.second[(2 * i + 1) % W];
            a[i] = beside ? even : x, b[i] = beside ? odd : y;
        }
    }
}
template <class T, int W>
__device__ __forceinline__ void store_some(T* at, int room, const float* v) {
    if (room >= W) {
        typename Few<T, W>::vector f;
#pragma unroll
        for (int i = 0; i < W; ++i) f[i] = (T)v[i];
        store_few<T, W>(at, f);
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i)
            if (i < room) at[i] = (T)v[i];
    }
}
template <class T, bool interleaved, int W>
__device__ __forceinline__ void write_pairs(T* head, const RotatePiece& p, const float (&a)[W], const float (&b)[W]) {
    if (interleaved && p.pair >= 0) {
        float v[2 * W];
#pragma unroll
        for (int i = 0; i < W; ++i) v[2 * i] = a[i], v[2 * i + 1] = b[i];
        store_some<T, W>(head + 2 * p.pair, 2 * p.a, v);
        store_some<T, W>(head + 2 * p.pair + W, 2 * p.a - W, v + W);
    } else {
        store_some<T, W>(head + p.a_at, p.a, a);
        store_some<T, W>(head + p.b_at, p.b, b);
    }
}

template <int lanes>
__device__ __forceinline__ float sum_over_lanes(float v) {
#pragma unroll
    for (int d = 1; d < lanes; d *= 2) v += __shfl_xor(v, d, kWave);
    return v;
}

// Measured under the profiler, bfloat16: 131 072 rows of 8 + 4 heads of 128 160 us (805 MB, 5.0 TB/s; a copy of 2 GiB 4.9), their gradients 288 us (1.2 GB,
// 4.2 TB/s); 262 144 rows of 8 + 2 heads of 32 91 us (339 MB, 3.7 TB/s: the angles of 16 pairs a row, three axes each, are a quarter of the instructions).
template <class T, int lanes, bool interleaved, bool backward>
__global__ __launch_bounds__(kRotateThreads) void rotate_kernel(RotateArgs<T> p) {
    constexpr int W = kRotatePairs<T>, groups = kRotateThreads / lanes;
    constexpr bool accurate = sizeof(T) == 4;
    __shared__ float2 turns[kRotateTurns];
    __shared__ float sums[backward ? kRotateThreads * 2 * W : 1];
    const int lane = threadIdx.x % lanes, group = threadIdx.x / lanes, pairs = p.rotated / 2;
    const RotatePiece piece = piece_of<W>(lane, p.dim, p.rotated);
    RawPairs<T, W> weight[2];
    float da[2][W], db[2][W];
#pragma unroll
    for (int o = 0; o < 2; ++o) {
#pragma unroll
        for (int i = 0; i < W; ++i) weight[o].first[i] = weight[o].second[i] = (T)1.0f, da[o][i] = db[o][i] = 0.0f;
        if (p.weight[o]) weight[o] = load_pairs<T, interleaved, W>(p.weight[o], piece);
    }
    const float dim = (float)p.dim;
    for (int64_t first = (int64_t)blockIdx.x * p.rows_at_once; first < p.rows; first += (int64_t)gridDim.x * p.rows_at_once) {
        const int rows = (int)least(p.rows_at_once, p.rows - first);
        __syncthreads();   // (the last rows' angles are read no more)
        for (int i = threadIdx.x; i < rows * pairs; i += kRotateThreads) {
            const int row = i / pairs, pair = i - row * pairs;
            double angle = 0.0;
            for (int x = 0; x < p.axes; ++x)
                angle = __builtin_fma(position(p.positions, p.position_type, (first + row) * p.axes + x), (double)p.frequencies[x * pairs + pair], angle);
            turns[i] = turn_of<accurate>(angle);
        }
        __syncthreads();
#pragma unroll
        for (int o = 0; o < 2; ++o) {
            const int heads = p.heads[o];
            const auto load = [&](int row, int head, RawPairs<T, W>& x, RawPairs<T, W>& g) {
                x = load_pairs<T, interleaved, W>(p.x[o] + (first + row) * p.x_stride[o] + head * p.x_head[o], piece);
                if constexpr (backward) g = load_pairs<T, interleaved, W>(p.dy[o] + (first + row) * p.dy_stride[o] + head * p.dy_head[o], piece);
            };
            RawPairs<T, W> x, g, next_x, next_g;     // (a head's numbers are on their way while the one before is computed)
            const int step_rows = groups / heads, step_heads = groups - step_rows * heads;
            int next_row = group / heads, next_head = group - next_row * heads;
            if (next_row < rows) load(next_row, next_head, next_x, next_g);
            while (next_row < rows) {
                const int row = next_row, head = next_head;
                x = next_x, g = next_g;
                next_row += step_rows, next_head += step_heads;
                if (next_head >= heads) ++next_row, next_head -= heads;
                if (next_row < rows) load(next_row, next_head, next_x, next_g);
                float a[W], b[W], ga[W], gb[W], wa[W], wb[W], c[W], s[W], squares = 0.0f;
                numbers_of<T, interleaved, W>(x, piece, a, b);
                if constexpr (backward) numbers_of<T, interleaved, W>(g, piece, ga, gb);
                numbers_of<T, interleaved, W>(weight[o], piece, wa, wb);
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    const bool turned = piece.pair >= 0 && i < piece.a;
                    const float2 t = turned ? turns[row * pairs + piece.pair + i] : make_float2(1.0f, 0.0f);
                    c[i] = t.x, s[i] = t.y;
                    squares = __builtin_fmaf(a[i], a[i], __builtin_fmaf(b[i], b[i], squares));
                }
                const float r = 1.0f / sqrtf(sum_over_lanes<lanes>(squares) / dim + p.eps);
                T* const to = p.y[o] ? p.y[o] + ((first + row) * heads + head) * p.dim : nullptr;
                if constexpr (!backward) {
#pragma unroll
                    for (int i = 0; i < W; ++i) {
                        const float na = a[i] * r * wa[i], nb = b[i] * r * wb[i];
                        a[i] = __builtin_fmaf(na, c[i], -(nb * s[i]));
                        b[i] = __builtin_fmaf(nb, c[i], na * s[i]);
                    }
                    write_pairs<T, interleaved, W>(to, piece, a, b);
                } else {
                    float dot = 0.0f;
#pragma unroll
                    for (int i = 0; i < W; ++i) {
                        const float na = __builtin_fmaf(ga[i], c[i], gb[i] * s[i]), nb = __builtin_fmaf(gb[i], c[i], -(ga[i] * s[i]));
                        a[i] *= r, b[i] *= r;
                        da[o][i] = __builtin_fmaf(na, a[i], da[o][i]), db[o][i] = __builtin_fmaf(nb, b[i], db[o][i]);
                        ga[i] = na * wa[i], gb[i] = nb * wb[i];
                        dot = __builtin_fmaf(ga[i], a[i], __builtin_fmaf(gb[i], b[i], dot));
                    }
                    dot = sum_over_lanes<lanes>(dot) / dim;
#pragma unroll
                    for (int i = 0; i < W; ++i) {
                        a[i] = r * __builtin_fmaf(-a[i], dot, ga[i]);
                        b[i] = r * __builtin_fmaf(-b[i], dot, gb[i]);
                    }
                    if (to) write_pairs<T, interleaved, W>(to, piece, a, b);
                }
            }
        }
    }
    if constexpr (backward) {
        if (!p.part) return;
#pragma unroll
        for (int o = 0; o < 2; ++o) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < W; ++i) {     // [number of a lane][thread]
                sums[i * kRotateThreads + threadIdx.x] = da[o][i];
                sums[(W + i) * kRotateThreads + threadIdx.x] = db[o][i];
            }
            __syncthreads();
            // thread (i, lane) of the first 2 W lanes adds up its number over the groups
            for (int j = threadIdx.x; j < 2 * W * lanes; j += kRotateThreads) {
                const int l = j % lanes, i = j / lanes, within = i % W;
                const RotatePiece q = piece_of<W>(l, p.dim, p.rotated);
                if (within >= (i < W ? q.a : q.b)) continue;
                float sum = 0.0f;
                for (int g = 0; g < groups; ++g) sum += sums[i * kRotateThreads + g * lanes + l];
                const int at = interleaved && q.pair >= 0 ? 2 * (q.pair + within) + (i < W ? 0 : 1) : (i < W ? q.a_at : q.b_at) + within;
                p.part[((int64_t)blockIdx.x * 2 + o) * p.dim + at] = sum;
            }
        }
    }
}

// The weights' gradients: columns of [blocks][2 dim], 16 to a block, by 64 threads each.  (1024 rows of 256: 29 us by 16 threads, 5 by 64.)
template <class T>
__global__ __launch_bounds__(1024) void rotate_join_kernel(const float* part, int blocks, int dim, T* q_weight, T* k_weight) {
    __shared__ float room[1024];
    const int column = blockIdx.x * 16 + threadIdx.x % 16, from = threadIdx.x / 16;
    float sum = 0.0f;
    if (column < 2 * dim)
#pragma unroll 8
        for (int b = from; b < blocks; b += 64) sum += part[(int64_t)b * 2 * dim + column];
    room[threadIdx.x] = sum;
    for (int n = 32; n > 0; n /= 2) {
        __syncthreads();
        if (from < n) room[threadIdx.x] = sum += room[threadIdx.x + n * 16];
    }
    if (from != 0 || column >= 2 * dim) return;
    T* const to = column < dim ? q_weight : k_weight;
    if (to) to[column < dim ? column : column - dim] = (T)sum;
}

}  // namespace svox_network
