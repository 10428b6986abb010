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
};

constexpr int kNarrowWaves = 4;

// the two tiles of 4 hidden numbers of a lane, as the 8 of a reduction over them
template <class T>
__device__ __forceinline__ void turn(const u16x4 (&half)[2][Form<T>::planes], u16x8 (&out)[Form<T>::planes]) {
#pragma unroll
    for (int q = 0; q < Form<T>::planes; ++q) out[q] = __builtin_shufflevector(half[0][q], half[1][q], 0, 1, 2, 3, 4, 5, 6, 7);
}
template <class T>
__device__ __forceinline__ void turn(const f32x4 (&v)[2], u16x8 (&out)[Form<T>::planes]) {
    u16x4 half[2][Form<T>::planes];
    Form<T>::split(v[0], half[0]);
    Form<T>::split(v[1], half[1]);
    turn<T>(half, out);
}

// The biases of a lane's 4 hidden units, as what their sums begin with: read for each tile anew, straight to where it adds up,
// since vector instructions are what these kernels run out of and reads of LDS are not.
__device__ __forceinline__ void biases(const float* bias, int unit, f32x4& gate, f32x4& up) {
    asm("" : "+v"(unit));   // (or one read would be copied to all tiles)
    gate = *reinterpret_cast<const f32x4*>(bias + unit);
    up = *reinterpret_cast<const f32x4*>(bias + 32 + unit);
}

// Rows go 16 QT to a wavefront.
template <class T, int KD, int KO, int QT, int activation>
__global__ __launch_bounds__(kNarrowWaves* kWave, 2) void narrow_kernel(NarrowArgs<T> p) {
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
            f32x4 gate[QT], up[QT];
#pragma unroll
            for (int q = 0; q < QT; ++q) biases(bias, t * 16 + g * 4, gate[q], up[q]);
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
#pragma unroll
            for (int q = 0; q < QT; ++q)
#pragma unroll
                for (int i = 0; i < 4; ++i) h[q][t][i] = activate<planes == 3, activation>(gate[q][i], nullptr) * up[q][i];
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

// dx: as narrow_kernel, with dh' = Wd' dy' and dx' = Wg' dgate' + Wu' dup' in place of y'.
template <class T, int KD, int KO, int QT, int activation>
__global__ __launch_bounds__(kNarrowWaves* kWave, 2) void narrow_backward_kernel(NarrowArgs<T> p) {
    using C = Chunk<KD, KO, true>;
    constexpr int planes = Form<T>::planes, kib = C::fragments * planes + 1, DT = 2 * KD;
    __shared__ __align__(16) u16 lds[2][kib * 512];
    const int lane = threadIdx.x % kWave, l = lane & 15, g = lane >> 4, wave = threadIdx.x / kWave;
    const int64_t row0 = ((int64_t)blockIdx.x * kNarrowWaves + wave) * 16 * QT;
    const int chunks = (int)((p.hidden + 31) / 32);
    chunk_to_lds<kib, kNarrowWaves>(p.chunks, lds[0]);
    u16x8 x[QT][KD][planes], dy[QT][KO][planes];
#pragma unroll
    for (int q = 0; q < QT; ++q) {
        row_fragments<T, KD>(p.x, p.x_ld, row0 + q * 16 + l, p.rows, p.dim, x[q]);
        row_fragments<T, KO>(p.dy, p.dy_ld, row0 + q * 16 + l, p.rows, p.out, dy[q]);
    }
    f32x4 dx[QT][DT];
#pragma unroll
    for (int q = 0; q < QT; ++q)
#pragma unroll
        for (int d = 0; d < DT; ++d) dx[q][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int c = 0; c < chunks; ++c) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (c + 1 < chunks) chunk_to_lds<kib, kNarrowWaves>(p.chunks + (int64_t)(c + 1) * kib * 512, lds[(c + 1) & 1]);
        const u16* const at = lds[c & 1];
        const float* const bias = reinterpret_cast<const float*>(at + C::fragments * planes * 512);
        f32x4 dg[QT][2], du[QT][2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            f32x4 gate[QT], up[QT], dh[QT];
#pragma unroll
            for (int q = 0; q < QT; ++q) biases(bias, t * 16 + g * 4, gate[q], up[q]), dh[q] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
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
#pragma unroll
            for (int s = 0; s < KO; ++s) {
                u16x8 wd[planes];
                fragment_of<planes>(at, C::down + t * KO + s, wd);
#pragma unroll
                for (int q = 0; q < QT; ++q) dh[q] = multiply<T>(wd, dy[q][s], dh[q]);
            }
#pragma unroll
            for (int q = 0; q < QT; ++q)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float slope;
                    const float a = activate<planes == 3, activation>(gate[q][i], &slope);
                    dg[q][t][i] = dh[q][i] * up[q][i] * slope;
                    du[q][t][i] = dh[q][i] * a;
                }
        }
        u16x8 turned_g[QT][planes], turned_u[QT][planes];
#pragma unroll
        for (int q = 0; q < QT; ++q) turn<T>(dg[q], turned_g[q]), turn<T>(du[q], turned_u[q]);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            u16x8 wg[planes], wu[planes];
            fragment_of<planes>(at, C::gate_t + d, wg);
            fragment_of<planes>(at, C::up_t + d, wu);
#pragma unroll
            for (int q = 0; q < QT; ++q) {
                dx[q][d] = multiply<T>(wg, turned_g[q], dx[q][d]);
                dx[q][d] = multiply<T>(wu, turned_u[q], dx[q][d]);
            }
        }
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) {
        const int64_t col = d * 16 + g * 4;
#pragma unroll
        for (int q = 0; q < QT; ++q) {
            const int64_t row = row0 + q * 16 + l;
            if (col < p.dim && row < p.rows) store_four(p.y + row * p.dim, dx[q][d], col, p.dim);
        }
    }
}

// 32 rows of K * 32 numbers in LDS, read along the rows and down the columns.  A row's pieces of 16 numbers lie at their index ^ a
// number of the row, so that neither the eight rows nor the four times 32 bytes that a clock serves meet on a bank.
template <int K, int planes>
struct RowTile {
    static constexpr int plane = 32 * K * 32, numbers = planes * plane, pieces = 32 * K * 4;   // (pieces: of 8 numbers)
    static __device__ __forceinline__ int turned(int row) { return K == 1 ? (row >> 2) & 1 : K == 2 ? (row >> 1) & 3 : row & 7; }
    static __device__ __forceinline__ u16* at(u16* lds, int row, int piece) {
        return lds + row * K * 32 + ((piece >> 1) ^ turned(row)) * 16 + (piece & 1) * 8;
    }
    // rows 16 tile..+15, numbers 32 step..+31, as the matrix cores take rows
    static __device__ __forceinline__ void along(u16* lds, int tile, int step, u16x8 (&out)[planes]) {
        const int lane = threadIdx.x % kWave;
#pragma unroll
        for (int q = 0; q < planes; ++q) out[q] = *reinterpret_cast<const u16x8*>(at(lds + q * plane, tile * 16 + (lane & 15), step * 4 + lane / 16));
    }
    // columns 16 tile..+15 over the 32 rows, in the order of `turn`
    static __device__ __forceinline__ void across(u16* lds, int tile, u16x8 (&out)[planes]) {
        const int lane = threadIdx.x % kWave, l = lane & 15;
#pragma unroll
        for (int q = 0; q < planes; ++q)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int row = half * 16 + lane / 16 * 4 + (l >> 2);
                const u16* const from = lds + q * plane + row * K * 32 + (tile ^ turned(row)) * 16 + (l & 3) * 4;
                const s16x4 four = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)from);
#pragma unroll
                for (int i = 0; i < 4; ++i) out[q][half * 4 + i] = (u16)four[i];
            }
    }
};

// 8 numbers of a row as they lie in memory, to be laid out when they have arrived
template <class T>
struct Raw {
    T v[8];
    __device__ __forceinline__ void read(const T* row, int64_t c, int64_t count, bool there) {
        if (there && c + 8 <= count) {
            const auto a = load_few<T, 8>(row + c);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = a[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = there && c + i < count ? row[c + i] : (T)0.0f;
        }
    }
    __device__ __forceinline__ void lay(u16x8 (&out)[Form<T>::planes]) const {
        f32x4 part[2];
#pragma unroll
        for (int i = 0; i < 8; ++i) part[i / 4][i % 4] = (float)v[i];
        turn<T>(part, out);
    }
};

template <class T>
struct NarrowWeightArgs {
    const T *x, *dy;
    int64_t x_ld, dy_ld;
    const u16* chunks;
    float *gate, *up, *down, *b_gate, *b_up, *b_down;   // [splits] of each gradient
    int64_t rows, each;                                 // rows of a split: a whole number of 32
    int64_t dim, hidden, out;
};

// The gradients of the weights over a share of the rows: a wavefront has 16 HT hidden units, their weights and their sums in
// registers, and a block's wavefronts go through the rows together, 32 at a time: gate, up and dh of those rows and units (rows down
// this time, a lane has 4 rows of a unit), and the products of what comes of them with the columns of x and dy.
constexpr int kNarrowWeightWaves = 8;
template <class T, int KD, int KO, int HT, int activation>
__global__ __launch_bounds__(kNarrowWeightWaves* kWave, 2) void narrow_weight_kernel(NarrowWeightArgs<T> p) {
    using C = Chunk<KD, KO, true>;
    constexpr int planes = Form<T>::planes, DT = 2 * KD, OT = 2 * KO, threads = kNarrowWeightWaves * kWave;
    using X = RowTile<KD, planes>;
    using Y = RowTile<KO, planes>;
    constexpr int nx = (X::pieces + threads - 1) / threads, ny = (Y::pieces + threads - 1) / threads;
    __shared__ __align__(16) u16 lds[2][X::numbers + Y::numbers];
    const int thread = threadIdx.x, lane = thread % kWave, l = lane & 15, g = lane >> 4, wave = thread / kWave;
    const int64_t tile0 = ((int64_t)blockIdx.y * kNarrowWeightWaves + wave) * HT, split = blockIdx.x;
    const int64_t first = split * p.each, end = least(first + p.each, p.rows);
    const bool works = tile0 * 16 < p.hidden;
    u16x8 wg[HT][KD][planes], wu[HT][KD][planes], wd[HT][KO][planes];
    float bg[HT], bu[HT];
    if (works) {
#pragma unroll
        for (int t = 0; t < HT; ++t) {
            // (HT 2: the last chunk has both of its tiles, zeros beyond the hidden units)
            const int64_t tile = tile0 + t;
            const int half = (int)(tile % 2);
            const u16* const at = p.chunks + tile / 2 * C::numbers(planes);
#pragma unroll
            for (int s = 0; s < KD; ++s) fragment_of<planes>(at, C::gate + half * KD + s, wg[t][s]), fragment_of<planes>(at, C::up + half * KD + s, wu[t][s]);
#pragma unroll
            for (int s = 0; s < KO; ++s) fragment_of<planes>(at, C::down + half * KO + s, wd[t][s]);
            const float* const bias = reinterpret_cast<const float*>(at + C::fragments * planes * 512);
            bg[t] = bias[half * 16 + l];
            bu[t] = bias[32 + half * 16 + l];
        }
    }
    f32x4 gate_sum[HT][DT], up_sum[HT][DT], down_sum[HT][OT];
    float bg_sum[HT], bu_sum[HT], bd_sum[ny][8];
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int t = 0; t < HT; ++t) {
        bg_sum[t] = bu_sum[t] = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; ++d) gate_sum[t][d] = up_sum[t][d] = zero;
#pragma unroll
        for (int o = 0; o < OT; ++o) down_sum[t][o] = zero;
    }
#pragma unroll
    for (int i = 0; i < ny; ++i)
        for (int j = 0; j < 8; ++j) bd_sum[i][j] = 0.0f;
    Raw<T> rx[nx], ry[ny];
    auto read = [&](int64_t row0) {
#pragma unroll
        for (int i = 0; i < nx; ++i) {
            const int piece = i * threads + thread, row = piece / (KD * 4);
            if (X::pieces % threads == 0 || piece < X::pieces) rx[i].read(p.x + (row0 + row) * p.x_ld, piece % (KD * 4) * 8, p.dim, row0 + row < end);
        }
#pragma unroll
        for (int i = 0; i < ny; ++i) {
            const int piece = i * threads + thread, row = piece / (KO * 4);
            if (Y::pieces % threads == 0 || piece < Y::pieces) ry[i].read(p.dy + (row0 + row) * p.dy_ld, piece % (KO * 4) * 8, p.out, row0 + row < end);
        }
    };
    read(first);
    int which = 0;
    for (int64_t row0 = first; row0 < end; row0 += 32, which ^= 1) {
        u16 *const x = lds[which], *const dy = lds[which] + X::numbers;
#pragma unroll
        for (int i = 0; i < nx; ++i) {
            const int piece = i * threads + thread;
            if (X::pieces % threads != 0 && piece >= X::pieces) continue;
            u16x8 laid[planes];
            rx[i].lay(laid);
            for (int q = 0; q < planes; ++q) *reinterpret_cast<u16x8*>(X::at(x + q * X::plane, piece / (KD * 4), piece % (KD * 4))) = laid[q];
        }
#pragma unroll
        for (int i = 0; i < ny; ++i) {
            const int piece = i * threads + thread;
            if (Y::pieces % threads != 0 && piece >= Y::pieces) continue;
            u16x8 laid[planes];
            ry[i].lay(laid);
            for (int q = 0; q < planes; ++q) *reinterpret_cast<u16x8*>(Y::at(dy + q * Y::plane, piece / (KO * 4), piece % (KO * 4))) = laid[q];
            for (int j = 0; j < 8; ++j) bd_sum[i][j] += (float)ry[i].v[j];
        }
        __syncthreads();
        if (row0 + 32 < end) read(row0 + 32);
        if (!works) continue;
        u16x4 h[HT][2][planes], dg[HT][2][planes], du[HT][2][planes];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            f32x4 gate[HT], up[HT], dh[HT];
#pragma unroll
            for (int t = 0; t < HT; ++t) gate[t] = zero + bg[t], up[t] = zero + bu[t], dh[t] = zero;
#pragma unroll
            for (int s = 0; s < KD; ++s) {
                u16x8 a[planes];
                X::along(x, q, s, a);
#pragma unroll
                for (int t = 0; t < HT; ++t) gate[t] = multiply<T>(a, wg[t][s], gate[t]), up[t] = multiply<T>(a, wu[t][s], up[t]);
            }
#pragma unroll
            for (int s = 0; s < KO; ++s) {
                u16x8 a[planes];
                Y::along(dy, q, s, a);
#pragma unroll
                for (int t = 0; t < HT; ++t) dh[t] = multiply<T>(a, wd[t][s], dh[t]);
            }
#pragma unroll
            for (int t = 0; t < HT; ++t) {
                f32x4 vh, vg, vu;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float slope;
                    const float a = activate<planes == 3, activation>(gate[t][i], &slope);
                    vh[i] = a * up[t][i];
                    vg[i] = dh[t][i] * up[t][i] * slope;
                    vu[i] = dh[t][i] * a;
                    bg_sum[t] += vg[i];
                    bu_sum[t] += vu[i];
                }
                Form<T>::split(vh, h[t][q]);
                Form<T>::split(vg, dg[t][q]);
                Form<T>::split(vu, du[t][q]);
            }
        }
        u16x8 th[HT][planes], tg[HT][planes], tu[HT][planes];
#pragma unroll
        for (int t = 0; t < HT; ++t) turn<T>(h[t], th[t]), turn<T>(dg[t], tg[t]), turn<T>(du[t], tu[t]);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            u16x8 a[planes];
            X::across(x, d, a);
#pragma unroll
            for (int t = 0; t < HT; ++t) gate_sum[t][d] = multiply<T>(a, tg[t], gate_sum[t][d]), up_sum[t][d] = multiply<T>(a, tu[t], up_sum[t][d]);
        }
#pragma unroll
        for (int o = 0; o < OT; ++o) {
            u16x8 a[planes];
            Y::across(dy, o, a);
#pragma unroll
            for (int t = 0; t < HT; ++t) down_sum[t][o] = multiply<T>(th[t], a, down_sum[t][o]);
        }
    }
    if (works) {
#pragma unroll
        for (int t = 0; t < HT; ++t) {
            const int64_t h = (tile0 + t) * 16 + l, h4 = (tile0 + t) * 16 + g * 4;
            if (h < p.hidden) {   // (a lane has 4 features of a unit)
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const int64_t col = d * 16 + g * 4;
                    if (col >= p.dim) continue;
                    store_four(p.gate + (split * p.hidden + h) * p.dim, gate_sum[t][d], col, p.dim);
                    store_four(p.up + (split * p.hidden + h) * p.dim, up_sum[t][d], col, p.dim);
                }
            }
#pragma unroll
            for (int o = 0; o < OT; ++o)   // (4 units of a number of the result)
                if (o * 16 + l < p.out && h4 < p.hidden) store_four(p.down + (split * p.out + o * 16 + l) * p.hidden, down_sum[t][o], h4, p.hidden);
            float sg = bg_sum[t], su = bu_sum[t];
            sg += __shfl_xor(sg, 16, kWave), su += __shfl_xor(su, 16, kWave);
            sg += __shfl_xor(sg, 32, kWave), su += __shfl_xor(su, 32, kWave);
            if (g == 0 && h < p.hidden) p.b_gate[split * p.hidden + h] = sg, p.b_up[split * p.hidden + h] = su;
        }
    }
    if (blockIdx.y != 0) return;
    // the sums of dy: a thread has 8 columns of a row in 32, its piece's
    float* const sums = reinterpret_cast<float*>(lds);
    static_assert(sizeof(lds) >= KO * 32 * sizeof(float), "room");
    __syncthreads();
    for (int c = thread; c < KO * 32; c += threads) sums[c] = 0.0f;
    __syncthreads();
    for (int turn_of = 0; turn_of < 32; ++turn_of) {   // (row by row, in one order)
#pragma unroll
        for (int i = 0; i < ny; ++i) {
            const int piece = i * threads + thread;
            if ((Y::pieces % threads == 0 || piece < Y::pieces) && piece / (KO * 4) == turn_of)
                for (int j = 0; j < 8; ++j) sums[piece % (KO * 4) * 8 + j] += bd_sum[i][j];
        }
        __syncthreads();
    }
    for (int c = thread; c < p.out; c += threads) p.b_down[split * p.out + c] = sums[c];
}

}  // namespace svox_decoder
