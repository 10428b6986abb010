// few_kernels.h -- the forward pass of the gated feed-forward block for few rows: points that are asked for one by one.
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

// acc[i][m] += rows w[i] + (0..15) times rows x[m] + (0..15) over this wavefront's share of the reduction of `count` numbers: 32 at a
// time, one time in `waves`.  w[i], x[m]: the lane's row.  x is of type T, or laid out in planes (rows of whole 8).
template <class T, int NB, int MT, int waves, bool laid>
__device__ __forceinline__ void few_products(const T* const (&w)[NB], const T* const (&x)[MT], const u16* const (&h)[MT], int64_t plane, int64_t count,
                                             f32x4 (&acc)[NB][MT]) {
    constexpr int planes = Form<T>::planes;
    // steps whose loads go out together: as many as the registers hold
    constexpr int together = planes == 1 ? (MT == 4 ? 2 : 4) : (MT == 4 ? 1 : 2);
    const int wave = threadIdx.x / kWave, group = threadIdx.x % kWave / 16;
    auto some = [&](int64_t k, auto number, bool whole) {
        constexpr int n = decltype(number)::value;
        u16x8 a[n][NB][planes], b[n][MT][planes];
#pragma unroll
        for (int s = 0; s < n; ++s) {
            const int64_t at = k + s * 32 * waves;
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                if (whole) pieces_of(w[i] + at, a[s][i]);
                else pieces_of(w[i] + at, count - at, a[s][i]);
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                if constexpr (laid) {
#pragma unroll
                    for (int p = 0; p < planes; ++p)
                        b[s][m][p] = whole || at < count ? *reinterpret_cast<const u16x8*>(h[m] + p * plane + at) : u16x8{0, 0, 0, 0, 0, 0, 0, 0};
                } else {
                    if (whole) pieces_of(x[m] + at, b[s][m]);
                    else pieces_of(x[m] + at, count - at, b[s][m]);
                }
            }
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
    const T *x, *w_gate, *w_up, *w_down, *b_gate, *b_up, *b_down, *residual;
    int64_t x_ld, residual_ld;
    u16* h;              // planes of (rows, ldh)
    int64_t ldh, plane;
    T* y;
    int64_t rows, dim, hidden, out;
    int activation;
};

constexpr int kFewHiddenWaves = 4, kFewOutputWaves = 8;

// Grid: 16 hidden units a block (the last ones to the end of h's rows), 16 MT rows.
template <class T, int MT>
__global__ __launch_bounds__(kFewHiddenWaves* kWave, 2) void few_hidden_kernel(FewArgs<T> p) {
    constexpr int planes = Form<T>::planes, waves = kFewHiddenWaves;
    __shared__ f32x4 shared[waves * 2 * MT * kWave];
    const int lane = threadIdx.x % kWave, l = lane & 15, wave = threadIdx.x / kWave;
    const int64_t h0 = (int64_t)blockIdx.x * 16, row0 = (int64_t)blockIdx.y * 16 * MT;
    // (a row beyond the last is the last one again: what comes of it is not stored)
    const int64_t unit = least(h0 + l, p.hidden - 1);
    const T* const w[2] = {p.w_gate + unit * p.dim, p.w_up + unit * p.dim};
    const T* x[MT];
    const u16* none[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) x[m] = p.x + least(row0 + m * 16 + l, p.rows - 1) * p.x_ld, none[m] = nullptr;
    f32x4 acc[2][MT], sum[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[i][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    few_products<T, 2, MT, waves, false>(w, x, none, 0, p.dim, acc);
    few_join<2, MT, waves>(acc, sum, shared);
    const int64_t row = row0 + wave * 16 + l, col = h0 + lane / 16 * 4;
    if (wave >= MT || row >= p.rows || col >= p.ldh) return;
    const f32x4 bg = four_of(p.b_gate, col, p.hidden - col), bu = four_of(p.b_up, col, p.hidden - col);
    f32x4 v;
    with_activation(p.activation, [&](auto activation) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v[i] = col + i < p.hidden ? activate<planes == 3, decltype(activation)::value>(sum[0][i] + bg[i], nullptr) * (sum[1][i] + bu[i]) : 0.0f;
    });
    u16x4 part[planes];
    Form<T>::split(v, part);
#pragma unroll
    for (int q = 0; q < planes; ++q) *reinterpret_cast<u16x4*>(p.h + q * p.plane + row * p.ldh + col) = part[q];
}

// Grid: 16 numbers of the result a block, 16 MT rows.
template <class T, int MT>
__global__ __launch_bounds__(kFewOutputWaves* kWave, 2) void few_output_kernel(FewArgs<T> p) {
    constexpr int waves = kFewOutputWaves;
    __shared__ f32x4 shared[waves * MT * kWave];
    const int lane = threadIdx.x % kWave, l = lane & 15, wave = threadIdx.x / kWave;
    const int64_t o0 = (int64_t)blockIdx.x * 16, row0 = (int64_t)blockIdx.y * 16 * MT;
    const T* const w[1] = {p.w_down + least(o0 + l, p.out - 1) * p.hidden};
    const u16* h[MT];
    const T* none[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) h[m] = p.h + least(row0 + m * 16 + l, p.rows - 1) * p.ldh, none[m] = nullptr;
    f32x4 acc[1][MT], sum[1];
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[0][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    few_products<T, 1, MT, waves, true>(w, none, h, p.plane, p.hidden, acc);
    few_join<1, MT, waves>(acc, sum, shared);
    const int64_t row = row0 + wave * 16 + l, col = o0 + lane / 16 * 4;
    if (wave >= MT || row >= p.rows || col >= p.out) return;
    f32x4 v = sum[0] + four_of(p.b_down, col, p.out - col);
    if (p.residual) v += four_of(p.residual + row * p.residual_ld, col, p.out - col);
    store_four(p.y + row * p.out, v, col, p.out);
}

}  // namespace svox_decoder
