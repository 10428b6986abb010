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

// 8 numbers of a row as they lie in memory, to be laid out when they have arrived.  `there` of them are the row's (all that is read
// beyond is taken for zeros), `room` can be read.
template <class T>
struct Raw {
    typename Few<T, 8>::vector v;
    __device__ __forceinline__ void read(const T* at, int64_t there, int64_t room) {
        if (there > 0)
            v = load_some<T, 8>(at, room);
        else
            v = 0.0f;
    }
    // as the matrix cores take them; ragged: rows are not of whole 8 numbers
    __device__ __forceinline__ void lay(u16x8 (&out)[Form<T>::planes], int64_t there, bool ragged) {
        if (ragged) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = i < there ? v[i] : (T)0.0f;
        }
        planes_of<T>(v, out);
    }
};

// A matrix of rows `ld` apart, and 8 numbers of it from column c of row r on.
template <class T>
struct Matrix {
    const T* at;
    int64_t ld, rows, cols;
    __device__ __forceinline__ void read(Raw<T>& raw, int64_t r, int64_t c) const {
        raw.read(at + r * ld + c, r < rows ? cols - c : 0, (rows - 1 - r) * ld + cols - c);
    }
    __device__ __forceinline__ bool ragged() const { return cols % 8 != 0; }
};

// K * 32 numbers of 16 QT rows on their way; a lane has 8 of each 32 of its rows.
template <class T, int K, int QT>
struct RowsRaw {
    Raw<T> v[QT][K];
    __device__ __forceinline__ void read(const Matrix<T>& m, int64_t row0) {
        const int lane = threadIdx.x % kWave;
#pragma unroll
        for (int q = 0; q < QT; ++q)
#pragma unroll
            for (int s = 0; s < K; ++s) m.read(v[q][s], row0 + q * 16 + (lane & 15), s * 32 + (lane >> 4) * 8);
    }
    __device__ __forceinline__ void lay(const Matrix<T>& m, u16x8 (&out)[QT][K][Form<T>::planes]) {
#pragma unroll
        for (int q = 0; q < QT; ++q)
#pragma unroll
            for (int s = 0; s < K; ++s) v[q][s].lay(out[q][s], m.cols - (s * 32 + threadIdx.x % kWave / 16 * 8), m.ragged());
    }
};

// The rows' results: a lane has 4 numbers of each 16 of its rows.
template <class T, int QT, int tiles>
__device__ __forceinline__ void store_rows(const f32x4 (&v)[QT][tiles], T* to, int64_t cols, const T* bias, const T* residual, int64_t residual_ld,
                                           int64_t row0, int64_t rows) {
    const int lane = threadIdx.x % kWave;
    // (all that is read, before any of it is used)
    typename Few<T, 4>::vector r[QT][tiles];
    if (residual) {
#pragma unroll
        for (int q = 0; q < QT; ++q)
#pragma unroll
            for (int o = 0; o < tiles; ++o) {
                const int64_t row = row0 + q * 16 + (lane & 15), col = o * 16 + lane / 16 * 4;
                if (col < cols && row < rows) r[q][o] = load_some<T, 4>(residual + row * residual_ld + col, (rows - 1 - row) * residual_ld + cols - col);
            }
    }
#pragma unroll
    for (int o = 0; o < tiles; ++o) {
        const int64_t col = o * 16 + lane / 16 * 4;
        if (col >= cols) continue;
        const f32x4 b = four_of(bias, col, cols - col);
#pragma unroll
        for (int q = 0; q < QT; ++q) {
            const int64_t row = row0 + q * 16 + (lane & 15);
            if (row >= rows) continue;
            f32x4 sum = v[q][o] + b;
            if (residual)
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] += (float)r[q][o][i];
            store_four(to + row * cols, sum, col, cols);
        }
    }
}
template <int QT, int tiles>
__device__ __forceinline__ void clear_rows(f32x4 (&v)[QT][tiles]) {
#pragma unroll
    for (int q = 0; q < QT; ++q)
#pragma unroll
        for (int i = 0; i < tiles; ++i) v[q][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
}

// The biases of a lane's 4 hidden units, as what their sums begin with: read for each tile anew, straight to where it adds up,
// since vector instructions are what these kernels run out of and reads of LDS are not.
__device__ __forceinline__ void biases(const float* bias, int unit, f32x4& gate, f32x4& up) {
    asm("" : "+v"(unit));   // (or one read would be copied to all tiles)
    gate = *reinterpret_cast<const f32x4*>(bias + unit);
    up = *reinterpret_cast<const f32x4*>(bias + 32 + unit);
}

// Zeros for the hidden units from `left` on that pad the last chunk (a row of infinities has made NaN of them).
template <int QT>
__device__ __forceinline__ void clear_padding(f32x4 (&v)[QT][2], int64_t left) {
    const int unit = threadIdx.x % kWave / 16 * 4;
#pragma unroll
    for (int q = 0; q < QT; ++q)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[q][t][i] = t * 16 + unit + i < left ? v[q][t][i] : 0.0f;
}

// Bound by vector instructions: a hidden number costs an exponential and a reciprocal, 16 cycles of a SIMD each for 64 lanes, and some
// ten others of 4.  Measured, bfloat16, silu: 262 144 rows of 64 -> 256 -> 49 in 39.6 us, 67 million hidden numbers, 600 TFLOP/s of
// products (59 MB, for which a copy takes 12 us); 65 537 rows of 32 -> 128 -> 28 in float32 21 us.
// Rows go 16 QT to a wavefront.
template <class T, int KD, int KO, int QT, int activation>
__global__ __launch_bounds__(kNarrowWaves* kWave, 2) void narrow_kernel(NarrowArgs<T> p) {
    using C = Chunk<KD, KO, false>;
    constexpr int planes = Form<T>::planes, kib = C::fragments * planes + 1, OT = 2 * KO;
    __shared__ __align__(16) u16 lds[2][kib * 512];
    const int g = threadIdx.x % kWave / 16, wave = threadIdx.x / kWave;
    const int64_t row0 = ((int64_t)blockIdx.x * kNarrowWaves + wave) * 16 * QT;
    const int chunks = (int)((p.hidden + 31) / 32);
    chunk_to_lds<kib, kNarrowWaves>(p.chunks, lds[0]);
    u16x8 x[QT][KD][planes];
    {
        const Matrix<T> m{p.x, p.x_ld, p.rows, p.dim};
        RowsRaw<T, KD, QT> raw;
        raw.read(m, row0);
        raw.lay(m, x);
    }
    f32x4 y[QT][OT];
    clear_rows(y);
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
        if (p.hidden - c * 32 < 32) clear_padding(h, p.hidden - c * 32);
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
    store_rows<T>(y, p.y, p.out, p.b_down, p.residual, p.residual_ld, row0, p.rows);
}

// dx: as narrow_kernel, with dh' = Wd' dy' and dx' = Wg' dgate' + Wu' dup' in place of y'.
// Bound as that is.  131 072 rows of 64 -> 256 -> 64 in bfloat16 35 us, 614 TFLOP/s of products.
template <class T, int KD, int KO, int QT, int activation>
__global__ __launch_bounds__(kNarrowWaves* kWave, 2) void narrow_backward_kernel(NarrowArgs<T> p) {
    using C = Chunk<KD, KO, true>;
    constexpr int planes = Form<T>::planes, kib = C::fragments * planes + 1, DT = 2 * KD;
    __shared__ __align__(16) u16 lds[2][kib * 512];
    const int g = threadIdx.x % kWave / 16, wave = threadIdx.x / kWave;
    const int64_t row0 = ((int64_t)blockIdx.x * kNarrowWaves + wave) * 16 * QT;
    const int chunks = (int)((p.hidden + 31) / 32);
    chunk_to_lds<kib, kNarrowWaves>(p.chunks, lds[0]);
    u16x8 x[QT][KD][planes], dy[QT][KO][planes];
    {
        const Matrix<T> mx{p.x, p.x_ld, p.rows, p.dim}, my{p.dy, p.dy_ld, p.rows, p.out};
        RowsRaw<T, KD, QT> raw_x;
        RowsRaw<T, KO, QT> raw_y;
        raw_x.read(mx, row0);
        raw_y.read(my, row0);
        raw_x.lay(mx, x);
        raw_y.lay(my, dy);
    }
    f32x4 dx[QT][DT];
    clear_rows(dx);
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
        if (p.hidden - c * 32 < 32) clear_padding(dg, p.hidden - c * 32), clear_padding(du, p.hidden - c * 32);
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
    store_rows<T>(dx, p.y, p.dim, (const T*)nullptr, (const T*)nullptr, 0, row0, p.rows);
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

template <class T>
struct NarrowWeightArgs {
    const T *x, *dy;
    int64_t x_ld, dy_ld;
    const u16* chunks;
    float *gate, *up, *down, *b_gate, *b_up, *b_down;   // [splits] of each gradient
    int64_t rows, each;                                 // rows of a split: a whole number of 32
    int64_t dim, hidden, out;
};

// The gradients of the weights over a share of the rows: a wavefront has 16 hidden units, their weights and their sums in
// registers, and a block's wavefronts go through the rows together, 32 at a time: gate, up and dh of those rows and units (rows down
// this time, a lane has 4 rows of a unit), and the products of what comes of them with the columns of x and dy.
// Bound by vector instructions, as the others: 131 072 rows of 64 -> 256 -> 64 in bfloat16 54 us, 477 TFLOP/s of products.  Hidden
// numbers' gradients that narrow_backward_kernel stored would be 201 MB written and read, 80 us.
// Four wavefronts to a block and three to a SIMD where their registers allow it (131 072 rows of 64 -> 256 -> 64 in bfloat16: 64 us
// with eight and two, 53 with four and three); where they do not, two, and eight to a block where four would have too many of
// the rows' numbers on their way.  In float32 the planes of the weights and the sums do not fit two wavefronts' registers where features or
// numbers of the result are more than 32: 20 to 32 bytes of a lane wait in memory, 120 to 176 where both are.  (A step of 131 072 rows
// of 64 -> 256 -> 64: 505 us.)
template <class T, int KD, int KO>
constexpr int kNarrowWeightWaves = (Form<T>::planes == 1 ? KD + KO > 6 : KD + KO > 2) ? 8 : 4;
template <class T, int KD, int KO>
constexpr int kNarrowWeightPerSimd = Form<T>::planes == 1 && KD + KO <= 4 ? 3 : 2;
template <class T, int KD, int KO, int activation>
__global__ __launch_bounds__((kNarrowWeightWaves<T, KD, KO> * kWave), (kNarrowWeightPerSimd<T, KD, KO>)) void narrow_weight_kernel(NarrowWeightArgs<T> p) {
    using C = Chunk<KD, KO, true>;
    constexpr int planes = Form<T>::planes, DT = 2 * KD, OT = 2 * KO, waves = kNarrowWeightWaves<T, KD, KO>, threads = waves * kWave;
    using X = RowTile<KD, planes>;
    using Y = RowTile<KO, planes>;
    constexpr int nx = (X::pieces + threads - 1) / threads, ny = (Y::pieces + threads - 1) / threads;
    __shared__ __align__(16) u16 lds[2][X::numbers + Y::numbers];
    const int thread = threadIdx.x, lane = thread % kWave, l = lane & 15, g = lane >> 4, wave = thread / kWave;
    const int64_t tile = (int64_t)blockIdx.y * waves + wave, split = blockIdx.x;
    const int64_t first = split * p.each, end = least(first + p.each, p.rows);
    const bool works = tile * 16 < p.hidden;
    u16x8 wg[KD][planes], wu[KD][planes], wd[KO][planes];
    float bg = 0.0f, bu = 0.0f;
    if (works) {
        const int half = (int)(tile % 2);
        const u16* const at = p.chunks + tile / 2 * C::numbers(planes);
#pragma unroll
        for (int s = 0; s < KD; ++s) fragment_of<planes>(at, C::gate + half * KD + s, wg[s]), fragment_of<planes>(at, C::up + half * KD + s, wu[s]);
#pragma unroll
        for (int s = 0; s < KO; ++s) fragment_of<planes>(at, C::down + half * KO + s, wd[s]);
        const float* const bias = reinterpret_cast<const float*>(at + C::fragments * planes * 512);
        bg = bias[half * 16 + l];
        bu = bias[32 + half * 16 + l];
    }
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    f32x4 gate_sum[DT], up_sum[DT], down_sum[OT];
    float bg_sum = 0.0f, bu_sum = 0.0f, bd_sum[ny][8];
#pragma unroll
    for (int d = 0; d < DT; ++d) gate_sum[d] = up_sum[d] = zero;
#pragma unroll
    for (int o = 0; o < OT; ++o) down_sum[o] = zero;
#pragma unroll
    for (int i = 0; i < ny; ++i)
        for (int j = 0; j < 8; ++j) bd_sum[i][j] = 0.0f;
    Raw<T> rx[nx], ry[ny];
    // (the rows of this split: what lies behind them is not theirs)
    const Matrix<T> mx{p.x, p.x_ld, end, p.dim}, my{p.dy, p.dy_ld, end, p.out};
    auto read = [&](int64_t row0) {
#pragma unroll
        for (int i = 0; i < nx; ++i) {
            const int piece = i * threads + thread, row = piece / (KD * 4);
            if (X::pieces % threads == 0 || piece < X::pieces) mx.read(rx[i], row0 + row, piece % (KD * 4) * 8);
        }
#pragma unroll
        for (int i = 0; i < ny; ++i) {
            const int piece = i * threads + thread, row = piece / (KO * 4);
            if (Y::pieces % threads == 0 || piece < Y::pieces) my.read(ry[i], row0 + row, piece % (KO * 4) * 8);
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
            rx[i].lay(laid, p.dim - piece % (KD * 4) * 8, mx.ragged());
            for (int q = 0; q < planes; ++q) *reinterpret_cast<u16x8*>(X::at(x + q * X::plane, piece / (KD * 4), piece % (KD * 4))) = laid[q];
        }
#pragma unroll
        for (int i = 0; i < ny; ++i) {
            const int piece = i * threads + thread;
            if (Y::pieces % threads != 0 && piece >= Y::pieces) continue;
            u16x8 laid[planes];
            ry[i].lay(laid, p.out - piece % (KO * 4) * 8, my.ragged());
            for (int q = 0; q < planes; ++q) *reinterpret_cast<u16x8*>(Y::at(dy + q * Y::plane, piece / (KO * 4), piece % (KO * 4))) = laid[q];
            for (int j = 0; j < 8; ++j) bd_sum[i][j] += (float)ry[i].v[j];
        }
        __syncthreads();
        if (row0 + 32 < end) read(row0 + 32);
        if (!works) continue;
        u16x4 h[2][planes], dg[2][planes], du[2][planes];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            f32x4 gate = zero + bg, up = zero + bu, dh = zero;
#pragma unroll
            for (int s = 0; s < KD; ++s) {
                u16x8 a[planes];
                X::along(x, q, s, a);
                gate = multiply<T>(a, wg[s], gate);
                up = multiply<T>(a, wu[s], up);
            }
#pragma unroll
            for (int s = 0; s < KO; ++s) {
                u16x8 a[planes];
                Y::along(dy, q, s, a);
                if (planes == 3 && q == 1)   // (half of the rows turned around: what the biases' gradients are sums of)
                    dh = multiply_turned<T>(a, wd[s], dh);
                else
                    dh = multiply<T>(a, wd[s], dh);
            }
            f32x4 vh, vg, vu;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float slope;
                const float a = activate<planes == 3, activation>(gate[i], &slope);
                vh[i] = a * up[i];
                vg[i] = dh[i] * up[i] * slope;
                vu[i] = dh[i] * a;
                bg_sum += vg[i];
                bu_sum += vu[i];
            }
            Form<T>::split(vh, h[q]);
            Form<T>::split(vg, dg[q]);
            Form<T>::split(vu, du[q]);
        }
        u16x8 th[planes], tg[planes], tu[planes];
        turn<T>(h, th);
        turn<T>(dg, tg);
        turn<T>(du, tu);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            u16x8 a[planes];
            X::across(x, d, a);
            gate_sum[d] = multiply<T>(a, tg, gate_sum[d]);
            up_sum[d] = multiply<T>(a, tu, up_sum[d]);
        }
#pragma unroll
        for (int o = 0; o < OT; ++o) {
            u16x8 a[planes];
            Y::across(dy, o, a);
            down_sum[o] = multiply<T>(th, a, down_sum[o]);
        }
    }
    if (works) {
        const int64_t h = tile * 16 + l, h4 = tile * 16 + g * 4;
        if (h < p.hidden) {   // (a lane has 4 features of a unit)
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const int64_t col = d * 16 + g * 4;
                if (col >= p.dim) continue;
                store_four(p.gate + (split * p.hidden + h) * p.dim, gate_sum[d], col, p.dim);
                store_four(p.up + (split * p.hidden + h) * p.dim, up_sum[d], col, p.dim);
            }
        }
#pragma unroll
        for (int o = 0; o < OT; ++o)   // (4 units of a number of the result)
            if (o * 16 + l < p.out && h4 < p.hidden) store_four(p.down + (split * p.out + o * 16 + l) * p.hidden, down_sum[o], h4, p.hidden);
        bg_sum += __shfl_xor(bg_sum, 16, kWave), bu_sum += __shfl_xor(bu_sum, 16, kWave);
        bg_sum += __shfl_xor(bg_sum, 32, kWave), bu_sum += __shfl_xor(bu_sum, 32, kWave);
        if (g == 0 && h < p.hidden) p.b_gate[split * p.hidden + h] = bg_sum, p.b_up[split * p.hidden + h] = bu_sum;
    }
    if (blockIdx.y != 0) return;
    // the sums of dy: a thread has those of its pieces, 8 columns of a row in 32
    float* const sums = reinterpret_cast<float*>(lds);
    static_assert(sizeof(lds) >= 32 * KO * 32 * sizeof(float), "room");
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ny; ++i) {
        const int piece = i * threads + thread;
        if (Y::pieces % threads == 0 || piece < Y::pieces)
#pragma unroll
            for (int j = 0; j < 8; ++j) sums[piece * 8 + j] = bd_sum[i][j];
    }
    __syncthreads();
    for (int c = thread; c < p.out; c += threads) {
        float sum = 0.0f;
#pragma unroll
        for (int row = 0; row < 32; ++row) sum += sums[row * KO * 32 + c];
        p.b_down[split * p.out + c] = sum;
    }
}

}  // namespace svox_decoder
