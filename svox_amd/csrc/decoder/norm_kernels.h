// norm_kernels.h -- layer norm of the rows of a matrix and its gradients.
//
//   n = (x - mean) rstd, y = n w + b,   mean and variance over the row's D numbers, rstd = 1 / sqrt(variance + eps)
//   dn = dy w,  dx = rstd (dn - mean(dn) - n mean(dn n)),  dw = sum over rows of dy n,  db = sum over rows of dy
//
// A row is read once: `lanes` lanes hold it in registers, NV pieces of V numbers each (V numbers are 16 bytes), so that the
// variance is that of the differences from the mean and not of squares.  Every number is read once and written once, some ten
// flops in between: the kernels are bound by memory.  A group of lanes goes through rows with the weights in registers.
// Sums are held in 32 bits.  The gradients of w and b are summed by every group over its rows, by every block over its groups,
// and over the blocks by norm_join_kernel, in an order of their own: the same call gives the same bits.
#pragma once
#include "common.h"

namespace svox_decoder {

constexpr int kNormThreads = 256;

template <class T>
constexpr int kNormPiece = 16 / (int)sizeof(T);

// The sum over `lanes` neighbouring lanes, known to all of them.  Up to a wavefront by exchange; a whole block by LDS, where
// `slot` (of alternating calls) keeps one sum's numbers apart from the next one's.
template <int lanes>
__device__ __forceinline__ float sum_over(float v, float* room, int slot) {
#pragma unroll
    for (int d = 1; d < (lanes < kWave ? lanes : kWave); d *= 2) v += __shfl_xor(v, d, kWave);
    if constexpr (lanes > kWave) {
        constexpr int waves = lanes / kWave;
        room += slot * waves;
        if (threadIdx.x % kWave == 0) room[threadIdx.x / kWave] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < waves; ++w) v += room[w];
    }
    return v;
}

// One piece of a row: V numbers from column c on, zeros beyond the row.
template <class T, int V, class Column>
__device__ __forceinline__ void read_piece(const T* row, Column c, int dim, float* v) {
    const auto f = load_some<T, V>(row + c, dim - c);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (float)f[i];
}
template <class T, int V, class Column>
__device__ __forceinline__ void write_piece(T* row, Column c, int dim, const float* v) {
    if (c + V <= dim) {
        typename Few<T, V>::vector f;
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = (T)v[i];
        store_few<T, V>(row + c, f);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (c + i < dim) row[c + i] = (T)v[i];
    }
}

template <class T>
struct NormArgs {
    const T *x, *weight, *bias, *dy;
    int64_t x_ld, dy_ld, rows;
    int dim;
    float eps;
    T* y;              // dense; backward: dx
    float* stats;      // (rows, 2): mean and rstd; forward: may be NULL
    float* part;       // backward: [blocks][2][dim], NULL without weight and bias
};

// Measured, bfloat16: 262 144 rows of 128 25 us (134 MB, 5.3 TB/s), 65 536 rows of 1024 51 us (5.2 TB/s; a copy of 2 GiB 5.0 TB/s); one row of
// 256 in a queue of calls 4 us, the launch.  float32, 100 003 rows of 48 out of 49: 10 us (3.7 TB/s).
template <class T, int lanes, int NV>
__global__ __launch_bounds__(kNormThreads) void norm_kernel(NormArgs<T> p) {
    constexpr int V = kNormPiece<T>, groups = kNormThreads / lanes;
    __shared__ float room[2 * (kNormThreads / kWave)];
    const int lane = threadIdx.x % lanes, group = threadIdx.x / lanes;
    float w[NV][V], b[NV][V];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * lanes + lane) * V;
        for (int i = 0; i < V; ++i) w[j][i] = 1.0f, b[j][i] = 0.0f;
        if (p.weight) read_piece<T, V>(p.weight, c, p.dim, w[j]);
        if (p.bias) read_piece<T, V>(p.bias, c, p.dim, b[j]);
    }
    const float dim = (float)p.dim;   // (division: the mean of equal numbers is exactly theirs)
    for (int64_t first = (int64_t)blockIdx.x * groups; first < p.rows; first += (int64_t)gridDim.x * groups) {
        const int64_t row = first + group;
        const bool there = row < p.rows;    // (all lanes of a group alike; the last groups of a block go on for its barriers)
        const T* const x = p.x + (there ? row : first) * p.x_ld;
        float v[NV][V], sum = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            read_piece<T, V>(x, (j * lanes + lane) * V, p.dim, v[j]);
#pragma unroll
            for (int i = 0; i < V; ++i) sum += v[j][i];
        }
        const float mean = sum_over<lanes>(sum, room, 0) / dim;
        float squares = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[j][i] -= mean;
                if ((j * lanes + lane) * V + i < p.dim) squares += v[j][i] * v[j][i];
            }
        const float rstd = 1.0f / sqrtf(sum_over<lanes>(squares, room, 1) / dim + p.eps);
        if (!there) continue;
        T* const y = p.y + row * p.dim;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * lanes + lane) * V;
#pragma unroll
            for (int i = 0; i < V; ++i) v[j][i] = v[j][i] * rstd * w[j][i] + b[j][i];
            if (c < p.dim) write_piece<T, V>(y, c, p.dim, v[j]);
        }
        if (p.stats && lane == 0) {
            p.stats[row * 2] = mean;
            p.stats[row * 2 + 1] = rstd;
        }
    }
}

// Measured: 65 536 rows of 1024 in bfloat16 79 us (403 MB, 5.1 TB/s), 100 003 rows of 48 in float32 13 us (4.6 TB/s).
template <class T, int lanes, int NV>
__global__ __launch_bounds__(kNormThreads) void norm_backward_kernel(NormArgs<T> p) {
    constexpr int V = kNormPiece<T>, groups = kNormThreads / lanes;
    __shared__ float room[2 * (kNormThreads / kWave)];
    __shared__ float shared[groups > 1 ? kNormThreads * V : 1];
    const int lane = threadIdx.x % lanes, group = threadIdx.x / lanes;
    float w[NV][V], dw[NV][V], db[NV][V];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        for (int i = 0; i < V; ++i) w[j][i] = 1.0f, dw[j][i] = db[j][i] = 0.0f;
        if (p.weight) read_piece<T, V>(p.weight, (j * lanes + lane) * V, p.dim, w[j]);
    }
    const float dim = (float)p.dim;   // (division: the mean of equal numbers is exactly theirs)
    for (int64_t first = (int64_t)blockIdx.x * groups; first < p.rows; first += (int64_t)gridDim.x * groups) {
        const int64_t row = first + group;
        const bool there = row < p.rows;
        const int64_t from = there ? row : first;
        const float mean = p.stats[from * 2], rstd = p.stats[from * 2 + 1];
        float n[NV][V], dn[NV][V], sum = 0.0f, dot = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * lanes + lane) * V;
            read_piece<T, V>(p.x + from * p.x_ld, c, p.dim, n[j]);
            read_piece<T, V>(p.dy + from * p.dy_ld, c, p.dim, dn[j]);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                n[j][i] = (n[j][i] - mean) * rstd;
                if (there) {
                    dw[j][i] += dn[j][i] * n[j][i];
                    db[j][i] += dn[j][i];
                }
                dn[j][i] *= w[j][i];
                sum += dn[j][i];
                dot += dn[j][i] * n[j][i];
            }
        }
        sum = sum_over<lanes>(sum, room, 0) / dim;
        dot = sum_over<lanes>(dot, room, 1) / dim;
        if (!there || !p.y) continue;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * lanes + lane) * V;
#pragma unroll
            for (int i = 0; i < V; ++i) dn[j][i] = rstd * (dn[j][i] - sum - n[j][i] * dot);
            if (c < p.dim) write_piece<T, V>(p.y + row * p.dim, c, p.dim, dn[j]);
        }
    }
    if (!p.part) return;
    float* const part = p.part + (int64_t)blockIdx.x * 2 * p.dim;
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float* const mine = which ? db[j] : dw[j];
            const int c = (j * lanes + lane) * V;
            if constexpr (groups > 1) {
                __syncthreads();
#pragma unroll
                for (int i = 0; i < V; ++i) shared[threadIdx.x * V + i] = mine[i];
                __syncthreads();
                if (group == 0)
                    for (int g = 1; g < groups; ++g)
#pragma unroll
                        for (int i = 0; i < V; ++i) mine[i] += shared[(g * lanes + lane) * V + i];
            }
            if (group == 0 && c < p.dim) write_piece<float, V>(part + which * p.dim, c, p.dim, mine);
        }
}

// Rows longer than the registers of a block: a block to a row, which it reads again for every sum (from a cache).  Columns are counted in 64
// bits: the last step of a row of nearly 2^31 numbers goes beyond them.
template <class T, bool backward>
__global__ __launch_bounds__(kNormThreads) void norm_long_kernel(NormArgs<T> p) {
    constexpr int V = kNormPiece<T>, stride = kNormThreads * V;
    __shared__ float room[2 * (kNormThreads / kWave)];
    const float dim = (float)p.dim;   // (division: the mean of equal numbers is exactly theirs)
    float v[V], w[V], d[V];
    float* const part = backward && p.part ? p.part + (int64_t)blockIdx.x * 2 * p.dim : nullptr;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* const x = p.x + row * p.x_ld;
        T* const y = p.y + row * p.dim;
        if constexpr (!backward) {
            float sum = 0.0f, squares = 0.0f;
            for (int64_t c = threadIdx.x * V; c < p.dim; c += stride) {
                read_piece<T, V>(x, c, p.dim, v);
                for (int i = 0; i < V; ++i) sum += v[i];
            }
            const float mean = sum_over<kNormThreads>(sum, room, 0) / dim;
            for (int64_t c = threadIdx.x * V; c < p.dim; c += stride) {
                read_piece<T, V>(x, c, p.dim, v);
                for (int i = 0; i < V; ++i)
                    if (c + i < p.dim) squares += (v[i] - mean) * (v[i] - mean);
            }
            const float rstd = 1.0f / sqrtf(sum_over<kNormThreads>(squares, room, 1) / dim + p.eps);
            for (int64_t c = threadIdx.x * V; c < p.dim; c += stride) {
                read_piece<T, V>(x, c, p.dim, v);
                for (int i = 0; i < V; ++i) w[i] = 1.0f, d[i] = 0.0f;
                if (p.weight) read_piece<T, V>(p.weight, c, p.dim, w);
                if (p.bias) read_piece<T, V>(p.bias, c, p.dim, d);
                for (int i = 0; i < V; ++i) v[i] = (v[i] - mean) * rstd * w[i] + d[i];
                write_piece<T, V>(y, c, p.dim, v);
            }
            if (p.stats && threadIdx.x == 0) {
                p.stats[row * 2] = mean;
                p.stats[row * 2 + 1] = rstd;
            }
        } else {
            const T* const dy = p.dy + row * p.dy_ld;
            const float mean = p.stats[row * 2], rstd = p.stats[row * 2 + 1];
            float sum = 0.0f, dot = 0.0f;
            const bool first = row == blockIdx.x;
            for (int64_t c = threadIdx.x * V; c < p.dim; c += stride) {
                read_piece<T, V>(x, c, p.dim, v);
                read_piece<T, V>(dy, c, p.dim, d);
                for (int i = 0; i < V; ++i) w[i] = 1.0f;
                if (p.weight) read_piece<T, V>(p.weight, c, p.dim, w);
                float dw[V], db[V];
                for (int i = 0; i < V; ++i) dw[i] = db[i] = 0.0f;
                if (part && !first) {   // (a thread comes back to the same columns)
                    read_piece<float, V>(part, c, p.dim, dw);
                    read_piece<float, V>(part + p.dim, c, p.dim, db);
                }
                for (int i = 0; i < V; ++i) {
                    const float n = (v[i] - mean) * rstd;
                    dw[i] += d[i] * n;
                    db[i] += d[i];
                    sum += d[i] * w[i];
                    dot += d[i] * w[i] * n;
                }
                if (part) {
                    write_piece<float, V>(part, c, p.dim, dw);
                    write_piece<float, V>(part + p.dim, c, p.dim, db);
                }
            }
            sum = sum_over<kNormThreads>(sum, room, 0) / dim;
            dot = sum_over<kNormThreads>(dot, room, 1) / dim;
            if (!p.y) continue;
            for (int64_t c = threadIdx.x * V; c < p.dim; c += stride) {
                read_piece<T, V>(x, c, p.dim, v);
                read_piece<T, V>(dy, c, p.dim, d);
                for (int i = 0; i < V; ++i) w[i] = 1.0f;
                if (p.weight) read_piece<T, V>(p.weight, c, p.dim, w);
                for (int i = 0; i < V; ++i) v[i] = rstd * (d[i] * w[i] - sum - (v[i] - mean) * rstd * dot);
                write_piece<T, V>(y, c, p.dim, v);
            }
        }
    }
}

// The gradients of weight and bias from the blocks' sums: 16 columns a block at a time, the sums over its 64 groups of lanes.
// (1024 columns 5 us, 48 columns 4 us: a launch and its first loads.)
constexpr int kNormJoinThreads = 1024, kNormJoinColumns = 16;
template <class T>
__global__ __launch_bounds__(kNormJoinThreads) void norm_join_kernel(const float* part, int blocks, int dim, T* dweight, T* dbias) {
    constexpr int groups = kNormJoinThreads / kNormJoinColumns;
    __shared__ float shared[kNormJoinThreads];
    const int lane = threadIdx.x % kNormJoinColumns, group = threadIdx.x / kNormJoinColumns;
    const int64_t columns = 2 * (int64_t)dim;
    for (int64_t first = (int64_t)blockIdx.x * kNormJoinColumns; first < columns; first += (int64_t)gridDim.x * kNormJoinColumns) {
        const int64_t c = first + lane;
        float sum = 0.0f;
        if (c < columns)
#pragma unroll 4
            for (int b = group; b < blocks; b += groups) sum += part[b * columns + c];
        shared[threadIdx.x] = sum;
        __syncthreads();
        for (int half = groups / 2; half > 0; half /= 2) {
            if (group < half) shared[threadIdx.x] += shared[threadIdx.x + half * kNormJoinColumns];
            __syncthreads();
        }
        if (group == 0 && c < columns) {
            if (c < dim) {
                if (dweight) dweight[c] = (T)shared[lane];
            } else if (dbias) {
                dbias[c - dim] = (T)shared[lane];
            }
        }
        __syncthreads();
    }
}

}  // namespace svox_decoder
