// few_kernels.h -- the gated feed-forward block for few rows: points that are asked for one by one, small batches.
//
// With few rows the weights are the work: each is read once and used for some rows only, and what counts is that all of them are
// on their way at once.  A block takes 16 rows of a weight (16 hidden units, or 16 numbers of the result) and its wavefronts
// share the reduction, so that the weights come from memory straight into the matrix cores' registers, wherever they lie and
// however long their rows are, with no tile, no barrier and no load that waits for another.  Only the wavefronts' sums go
// through LDS.  (float32 is split into its planes in registers.)
#pragma once
#include "product_kernels.h"

namespace svox_decoder {

// 8 numbers of a row as the matrix cores take them
template <class T>
__device__ __forceinline__ void pieces_of(const T* from, u16x8* out) {
    if constexpr (Form<T>::planes == 1) {
        out[0] = load_few<u16, 8>(reinterpret_cast<const u16*>(from));
    } else {
        u16x4 half[2][3];
        Form<T>::split(load_few<float, 4>(from), half[0]);
        Form<T>::split(load_few<float, 4>(from + 4), half[1]);
#pragma unroll
        for (int p = 0; p < 3; ++p) out[p] = __builtin_shufflevector(half[0][p], half[1][p], 0, 1, 2, 3, 4, 5, 6, 7);
    }
}
// ... of which only the first `there` are in the row: zeros for the others
template <class T>
__device__ __forceinline__ void pieces_of(const T* from, int64_t there, u16x8* out) {
    if (there >= 8) return pieces_of(from, out);
    u16x4 half[2][Form<T>::planes];
    Form<T>::split(four_of(from, 0, there), half[0]);
    Form<T>::split(there > 4 ? four_of(from, 4, there - 4) : f32x4{0.0f, 0.0f, 0.0f, 0.0f}, half[1]);
#pragma unroll
    for (int p = 0; p < Form<T>::planes; ++p) out[p] = __builtin_shufflevector(half[0][p], half[1][p], 0, 1, 2, 3, 4, 5, 6, 7);
}

// Where a lane's 8 numbers of a reduction come from: along a row, down a column, or along a row that is laid out in planes.
// whole: all 8 are there, else as many as `count` goes.
template <class T>
struct AlongRow {
    const T* row;
    __device__ __forceinline__ void read(int64_t at, int64_t count, bool whole, u16x8 (&out)[Form<T>::planes]) const {
        if (whole) pieces_of(row + at, out);
        else pieces_of(row + at, count - at, out);
    }
};
template <class T>
struct DownColumn {
    const T* column;
    int64_t ld;
    __device__ __forceinline__ void read(int64_t at, int64_t count, bool whole, u16x8 (&out)[Form<T>::planes]) const {
        typename Few<T, 8>::vector v;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = whole || at + i < count ? column[(at + i) * ld] : (T)0.0f;
        planes_of<T>(v, out);
    }
};
template <class T>
struct LaidRow {
    const u16* row;
    int64_t plane;
    __device__ __forceinline__ void read(int64_t at, int64_t count, bool whole, u16x8 (&out)[Form<T>::planes]) const {
#pragma unroll
        for (int p = 0; p < Form<T>::planes; ++p)
            out[p] = whole || at < count ? *reinterpret_cast<const u16x8*>(row + p * plane + at) : u16x8{0, 0, 0, 0, 0, 0, 0, 0};
    }
};

// acc[i][m] += 16 of left[i] times 16 of right[m] over this wavefront's share of the reduction of `count` numbers: 32 at a time, one
// time in `waves`, the loads of several times together.
template <class T, int waves, int NB, int MT, class Left, class Right>
__device__ __forceinline__ void few_products(const Left (&left)[NB], const Right (&right)[MT], int64_t count, f32x4 (*acc)[MT]) {
    constexpr int planes = Form<T>::planes;
    constexpr int together = planes == 1 ? (MT == 4 ? 2 : 4) : (MT == 4 ? 1 : 2);   // as many as the registers hold
    const int wave = threadIdx.x / kWave, group = threadIdx.x % kWave / 16;
    auto some = [&](int64_t k, auto number, bool whole) {
        constexpr int n = decltype(number)::value;
        u16x8 a[n][NB][planes], b[n][MT][planes];
#pragma unroll
        for (int s = 0; s < n; ++s) {
            const int64_t at = k + s * 32 * waves;
#pragma unroll
            for (int i = 0; i < NB; ++i) left[i].read(at, count, whole, a[s][i]);
#pragma unroll
            for (int m = 0; m < MT; ++m) right[m].read(at, count, whole, b[s][m]);
        }
#pragma unroll
        for (int s = 0; s < n; ++s)
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int m = 0; m < MT; ++m) acc[i][m] = multiply<T>(a[s][i], b[s][m], acc[i][m]);
    };
    const int64_t steps = count / 32;
    int64_t s = wave;
    for (; s + (together - 1) * waves < steps; s += together * waves) some(s * 32 + group * 8, std::integral_constant<int, together>(), true);
    for (; s < steps; s += waves) some(s * 32 + group * 8, std::integral_constant<int, 1>(), true);
    if (count % 32 && wave == steps % waves) some(steps * 32 + group * 8, std::integral_constant<int, 1>(), false);
}

// The wavefronts' sums added up: afterwards wavefront m has those of tile m (m < MT <= waves).
template <int NB, int MT, int waves>
__device__ __forceinline__ void few_join(f32x4 (&acc)[NB][MT], f32x4 (&sum)[NB], f32x4* shared) {
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int m = 0; m < MT; ++m) shared[((wave * NB + i) * MT + m) * kWave + lane] = acc[i][m];
    __syncthreads();
    if (wave >= MT) return;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        sum[i] = shared[(i * MT + wave) * kWave + lane];
#pragma unroll
        for (int w = 1; w < waves; ++w) sum[i] += shared[((w * NB + i) * MT + wave) * kWave + lane];
    }
}

template <class T>
struct FewArgs {
    const T *x, *dy, *w_gate, *w_up, *w_down, *b_gate, *b_up, *b_down, *residual;
    int64_t x_ld, dy_ld, residual_ld;
    u16 *h, *dgate, *dup;   // planes of (rows, ldh)
    float *b_gate_part, *b_up_part;   // backward: sums over 16 rows each, or NULL
    int64_t ldh, plane;
    T* y;                   // backward: dx
    int64_t rows, dim, hidden, out;
    int activation;
};

constexpr int kFewHiddenWaves = 4, kFewOutputWaves = 8;

// Measured: one row of 512 -> 2048 -> 512 in bfloat16 8.1 us for this kernel and the next (6.3 MB, 0.8 TB/s), 37 rows of 256 -> 1024 -> 256
// in float16 10.2 us: two launches, one after the other's end, and two trips to memory each.
// Grid: 16 hidden units a block (the last ones to the end of h's rows), 16 MT rows.
template <class T, int MT, bool backward>
__global__ __launch_bounds__(kFewHiddenWaves* kWave, 2) void few_hidden_kernel(FewArgs<T> p) {
    constexpr int planes = Form<T>::planes, waves = kFewHiddenWaves, products = backward ? 3 : 2;
    __shared__ f32x4 shared[waves * products * MT * kWave];
    const int lane = threadIdx.x % kWave, l = lane & 15, wave = threadIdx.x / kWave;
    const int64_t h0 = (int64_t)blockIdx.x * 16, row0 = (int64_t)blockIdx.y * 16 * MT;
    // (a row beyond the last is the last one again: what comes of it is not stored)
    const int64_t unit = least(h0 + l, p.hidden - 1);
    f32x4 acc[products][MT], sum[products];
#pragma unroll
    for (int i = 0; i < products; ++i)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[i][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    {
        const AlongRow<T> w[2] = {{p.w_gate + unit * p.dim}, {p.w_up + unit * p.dim}};
        AlongRow<T> x[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) x[m].row = p.x + least(row0 + m * 16 + l, p.rows - 1) * p.x_ld;
        few_products<T, waves>(w, x, p.dim, acc);
    }
    if constexpr (backward) {
        const DownColumn<T> w[1] = {{p.w_down + unit, p.hidden}};
        AlongRow<T> dy[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) dy[m].row = p.dy + least(row0 + m * 16 + l, p.rows - 1) * p.dy_ld;
        few_products<T, waves>(w, dy, p.out, acc + 2);
    }
    few_join<products, MT, waves>(acc, sum, shared);
    const int64_t row = row0 + wave * 16 + l, col = h0 + lane / 16 * 4;
    if (wave >= MT || (backward ? row0 + wave * 16 : row) >= p.rows || col >= p.ldh) return;
    const f32x4 bg = four_of(p.b_gate, col, p.hidden - col), bu = four_of(p.b_up, col, p.hidden - col);
    f32x4 h, dg, du;
    with_activation(p.activation, [&](auto activation) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool there = col + i < p.hidden && row < p.rows;
            const float u = sum[1][i] + bu[i];
            float slope;
            const float a = activate<planes == 3, decltype(activation)::value>(sum[0][i] + bg[i], backward ? &slope : nullptr);
            h[i] = there ? a * u : 0.0f;
            if constexpr (backward) {
                dg[i] = there ? sum[2][i] * u * slope : 0.0f;
                du[i] = there ? sum[2][i] * a : 0.0f;
            }
        }
    });
    auto keep = [&](f32x4 v, u16* to) {
        u16x4 part[planes];
        Form<T>::split(v, part);
#pragma unroll
        for (int q = 0; q < planes; ++q) *reinterpret_cast<u16x4*>(to + q * p.plane + row * p.ldh + col) = part[q];
    };
    if (row < p.rows) keep(h, p.h);
    if constexpr (backward) {
        if (row < p.rows) {
            keep(dg, p.dgate);
            keep(du, p.dup);
        }
        if (p.b_gate_part || p.b_up_part) keep_bias_sums(dg, du, p.b_gate_part, p.b_up_part, row0 / 16 + wave, col, p.hidden);
    }
}

// Grid: 16 numbers of the result (backward: features) a block, 16 MT rows.
template <class T, int MT, bool backward>
__global__ __launch_bounds__(kFewOutputWaves* kWave, 2) void few_output_kernel(FewArgs<T> p) {
    constexpr int waves = kFewOutputWaves;
    __shared__ f32x4 shared[waves * MT * kWave];
    const int lane = threadIdx.x % kWave, l = lane & 15, wave = threadIdx.x / kWave;
    const int64_t o0 = (int64_t)blockIdx.x * 16, row0 = (int64_t)blockIdx.y * 16 * MT, cols = backward ? p.dim : p.out;
    const int64_t mine = least(o0 + l, cols - 1);
    f32x4 acc[1][MT], sum[1];
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[0][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    LaidRow<T> rows[MT];
    auto take = [&](const u16* laid) {
#pragma unroll
        for (int m = 0; m < MT; ++m) rows[m] = LaidRow<T>{laid + least(row0 + m * 16 + l, p.rows - 1) * p.ldh, p.plane};
    };
    if constexpr (backward) {
        const DownColumn<T> gate[1] = {{p.w_gate + mine, p.dim}}, up[1] = {{p.w_up + mine, p.dim}};
        take(p.dgate);
        few_products<T, waves>(gate, rows, p.hidden, acc);
        take(p.dup);
        few_products<T, waves>(up, rows, p.hidden, acc);
    } else {
        const AlongRow<T> w[1] = {{p.w_down + mine * p.hidden}};
        take(p.h);
        few_products<T, waves>(w, rows, p.hidden, acc);
    }
    few_join<1, MT, waves>(acc, sum, shared);
    const int64_t row = row0 + wave * 16 + l, col = o0 + lane / 16 * 4;
    if (wave >= MT || row >= p.rows || col >= cols) return;
    f32x4 v = sum[0];
    if constexpr (!backward) {
        v += four_of(p.b_down, col, p.out - col);
        if (p.residual) v += four_of(p.residual + row * p.residual_ld, col, p.out - col);
    }
    store_four(p.y + row * cols, v, col, cols);
}

}  // namespace svox_decoder
