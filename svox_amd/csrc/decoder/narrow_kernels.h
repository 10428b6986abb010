// narrow_kernels.h -- the gated feed-forward block of narrow layers (up to 128 features in and out), where the hidden numbers of
// all rows would be most of what a call moves: they stay in registers.
//
// A wavefront keeps the features of some rows in registers and goes through the hidden units 32 at a time:
//
//   gate' = Wg x', up' = Wu x'      (hidden units down, rows across: a lane gets 4 neighbouring units of one row)
//   h'    = act(gate') up'          in place, rounded to the operands' type
//   y'   += Wd h'                   with h' as the matrix cores have just left it
//
// The last step needs 8 hidden numbers of a row in a lane, and a lane has 4 of each of two tiles: units 4 g..4 g + 3 of the first
// 16 and of the second.  Which 8 indices of a reduction a lane holds does not matter if both operands agree, so the weights
// are laid out for that order, and no number changes lanes between the two products.
//
// Weights come laid out in fragments: 64 lanes x 8 numbers, 1024 bytes, in the order in which a chunk of 32 hidden units uses them
// (narrow_lay_kernel).  A chunk goes to LDS in whole KiB while the one before it is used; reads from there are free of conflicts
// as they are.
#pragma once
#include "few_kernels.h"

namespace svox_decoder {

// What a fragment holds: rows of a weight and a part of the reduction, in the order above.
enum FragmentOf { kGate, kUp, kDown, kDownT, kGateT, kUpT };

// The fragments of a chunk of 32 hidden units, for KD * 32 features in and KO * 32 numbers out.
template <int KD, int KO, bool backward>
struct Chunk {
    // forward:  gate, up: [2 tiles of 16 units][KD], down: [2 KO tiles of 16 numbers]
    // backward: gate, up: the same, down turned: [2 tiles of units][KO], gate, up turned: [2 KD tiles of 16 features] each
    static constexpr int gate = 0, up = 2 * KD, down = 4 * KD, gate_t = down + 2 * KO, up_t = gate_t + 2 * KD;
    static constexpr int fragments = backward ? up_t + 2 * KD : down + 2 * KO;
    static constexpr int numbers(int planes) { return (fragments * planes + 1) * 512; }   // 16-bit; the last KiB: the biases, 2 x 32 floats
};

template <class T>
struct NarrowLayArgs {
    const T *w_gate, *w_up, *w_down, *b_gate, *b_up;
    int64_t dim, hidden, out;
    u16* to;
};
template <class T, int KD, int KO, bool backward>
__global__ __launch_bounds__(256) void narrow_lay_kernel(NarrowLayArgs<T> p) {
    using C = Chunk<KD, KO, backward>;
    constexpr int planes = Form<T>::planes;
    const int lane = threadIdx.x % kWave, l = lane & 15, g = lane >> 4;
    const int64_t piece = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave, chunk = piece / (C::fragments + 1);
    const int f = (int)(piece % (C::fragments + 1));
    const int64_t h0 = chunk * 32;
    if (h0 >= p.hidden) return;
    u16* const to = p.to + chunk * C::numbers(planes);
    if (f == C::fragments) {   // the biases
        float* const b = reinterpret_cast<float*>(to + C::fragments * planes * 512);
        const T* const from = lane < 32 ? p.b_gate : p.b_up;
        const int64_t h = h0 + lane % 32;
        b[lane] = from && h < p.hidden ? (float)from[h] : 0.0f;
        return;
    }
    f32x4 v[2];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int64_t turned = h0 + (j / 4) * 16 + 4 * g + j % 4;   // the hidden unit of a reduction over units
        float x = 0.0f;
        if (f < C::down) {
            const int of = f < C::up ? f : f - C::up;
            const int64_t h = h0 + of / KD * 16 + l, d = of % KD * 32 + 8 * g + j;
            if (h < p.hidden && d < p.dim) x = (float)(f < C::up ? p.w_gate : p.w_up)[h * p.dim + d];
        } else if (!backward) {
            const int64_t o = (f - C::down) * 16 + l;
            if (o < p.out && turned < p.hidden) x = (float)p.w_down[o * p.hidden + turned];
        } else if (f < C::gate_t) {
            const int of = f - C::down;
            const int64_t h = h0 + of / KO * 16 + l, o = of % KO * 32 + 8 * g + j;
            if (h < p.hidden && o < p.out) x = (float)p.w_down[o * p.hidden + h];
        } else {
            const int of = f < C::up_t ? f - C::gate_t : f - C::up_t;
            const int64_t d = of * 16 + l;
            if (d < p.dim && turned < p.hidden) x = (float)(f < C::up_t ? p.w_gate : p.w_up)[turned * p.dim + d];
        }
        v[j / 4][j % 4] = x;
    }
    u16x4 half[2][planes];
    Form<T>::split(v[0], half[0]);
    Form<T>::split(v[1], half[1]);
#pragma unroll
    for (int q = 0; q < planes; ++q)
        *reinterpret_cast<u16x8*>(to + ((int64_t)f * planes + q) * 512 + lane * 8) =
            __builtin_shufflevector(half[0][q], half[1][q], 0, 1, 2, 3, 4, 5, 6, 7);
}

// A chunk's KiB on their way to LDS, one of `waves` each.
template <int kib, int waves>
__device__ __forceinline__ void chunk_to_lds(const u16* from, u16* lds) {
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave), lane = threadIdx.x % kWave;
    const __amdgpu_buffer_rsrc_t buffer = __builtin_amdgcn_make_buffer_rsrc((void*)from, 0, kib * 1024, 0x00020000);
#pragma unroll
    for (int i = 0; i < (kib + waves - 1) / waves; ++i)
        if (i * waves + wave < kib)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer, (Lds*)(lds + (i * waves + wave) * 512), 16, lane * 16, (i * waves + wave) * 1024, 0, 0);
}

template <int planes>
__device__ __forceinline__ void fragment_of(const u16* lds, int f, u16x8 (&out)[planes]) {
#pragma unroll
    for (int q = 0; q < planes; ++q) out[q] = *reinterpret_cast<const u16x8*>(lds + (f * planes + q) * 512 + threadIdx.x % kWave * 8);
}

// Rows in fragments: K * 32 numbers of row `row` (as far as `count` goes; nothing of a row that is not there).
template <class T, int K>
__device__ __forceinline__ void row_fragments(const T* m, int64_t ld, int64_t row, int64_t rows, int64_t count, u16x8 (&out)[K][Form<T>::planes]) {
    const int g = threadIdx.x % kWave / 16;
    const T* const from = m + least(row, rows - 1) * ld;
#pragma unroll
    for (int s = 0; s < K; ++s) pieces_of(from + s * 32 + g * 8, row < rows ? count - (s * 32 + g * 8) : 0, out[s]);
}

template <class T>
struct NarrowArgs {
    const T *x, *dy;         // (rows, dim), (rows, out)
    int64_t x_ld, dy_ld;
    const u16* chunks;       // narrow_lay_kernel's
    const T *b_down, *residual;
    int64_t residual_ld;
    T* y;                    // (rows, out); backward: dx (rows, dim)
    int64_t rows, dim, hidden, out;
    int activation;
};

constexpr int kNarrowWaves = 4;

// the two tiles of 4 hidden numbers of a lane, as the 8 of a reduction over them
template <class T>
__device__ __forceinline__ void turn(const f32x4 (&v)[2], u16x8 (&out)[Form<T>::planes]) {
    u16x4 half[2][Form<T>::planes];
    Form<T>::split(v[0], half[0]);
    Form<T>::split(v[1], half[1]);
#pragma unroll
    for (int q = 0; q < Form<T>::planes; ++q) out[q] = __builtin_shufflevector(half[0][q], half[1][q], 0, 1, 2, 3, 4, 5, 6, 7);
}

// Rows go 16 QT to a wavefront.
template <class T, int KD, int KO, int QT>
__global__ __launch_bounds__(kNarrowWaves* kWave) void narrow_kernel(NarrowArgs<T> p) {
    using C = Chunk<KD, KO, false>;
    constexpr int planes = Form<T>::planes, kib = C::fragments * planes + 1, OT = 2 * KO;
    __shared__ __align__(16) u16 lds[2][kib * 512];
    const int lane = threadIdx.x % kWave, l = lane & 15, g = lane >> 4, wave = threadIdx.x / kWave;
    const int64_t row0 = ((int64_t)blockIdx.x * kNarrowWaves + wave) * 16 * QT;
    const int chunks = (int)((p.hidden + 31) / 32);
    chunk_to_lds<kib, kNarrowWaves>(p.chunks, lds[0]);
    u16x8 x[QT][KD][planes];
#pragma unroll
    for (int q = 0; q < QT; ++q) row_fragments<T, KD>(p.x, p.x_ld, row0 + q * 16 + l, p.rows, p.dim, x[q]);
    f32x4 y[QT][OT];
#pragma unroll
    for (int q = 0; q < QT; ++q)
#pragma unroll
        for (int o = 0; o < OT; ++o) y[q][o] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int c = 0; c < chunks; ++c) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (c + 1 < chunks) chunk_to_lds<kib, kNarrowWaves>(p.chunks + (int64_t)(c + 1) * kib * 512, lds[(c + 1) & 1]);
        const u16* const at = lds[c & 1];
        const float* const bias = reinterpret_cast<const float*>(at + C::fragments * planes * 512);
        f32x4 h[QT][2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const f32x4 bg = *reinterpret_cast<const f32x4*>(bias + t * 16 + g * 4), bu = *reinterpret_cast<const f32x4*>(bias + 32 + t * 16 + g * 4);
            f32x4 gate[QT], up[QT];
#pragma unroll
            for (int q = 0; q < QT; ++q) gate[q] = bg, up[q] = bu;
#pragma unroll
            for (int s = 0; s < KD; ++s) {
                u16x8 wg[planes], wu[planes];
                fragment_of<planes>(at, C::gate + t * KD + s, wg);
                fragment_of<planes>(at, C::up + t * KD + s, wu);
#pragma unroll
                for (int q = 0; q < QT; ++q) {
                    gate[q] = multiply<T>(wg, x[q][s], gate[q]);
                    up[q] = multiply<T>(wu, x[q][s], up[q]);
                }
            }
            with_activation(p.activation, [&](auto activation) {
#pragma unroll
                for (int q = 0; q < QT; ++q)
#pragma unroll
                    for (int i = 0; i < 4; ++i) h[q][t][i] = activate<planes == 3, decltype(activation)::value>(gate[q][i], nullptr) * up[q][i];
            });
        }
        u16x8 turned[QT][planes];
#pragma unroll
        for (int q = 0; q < QT; ++q) turn<T>(h[q], turned[q]);
#pragma unroll
        for (int o = 0; o < OT; ++o) {
            u16x8 wd[planes];
            fragment_of<planes>(at, C::down + o, wd);
#pragma unroll
            for (int q = 0; q < QT; ++q) y[q][o] = multiply<T>(wd, turned[q], y[q][o]);
        }
    }
#pragma unroll
    for (int o = 0; o < OT; ++o) {
        const int64_t col = o * 16 + g * 4;
        if (col >= p.out) continue;
        const f32x4 bias = four_of(p.b_down, col, p.out);
#pragma unroll
        for (int q = 0; q < QT; ++q) {
            const int64_t row = row0 + q * 16 + l;
            if (row >= p.rows) continue;
            f32x4 v = y[q][o] + bias;
            if (p.residual) v += four_of(p.residual + row * p.residual_ld, col, p.out);
            store_four(p.y + row * p.out, v, col, p.out);
        }
    }
}

}  // namespace svox_decoder
