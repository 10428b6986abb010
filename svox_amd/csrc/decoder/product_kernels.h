// product_kernels.h -- the gated feed-forward block as products of whole matrices, for rows enough to fill tiles.
//
// forward   hidden_kernel   h = act(x Wg' + bg) * (x Wu' + bu)            both products of a tile side by side, h alone is stored
//           output_kernel   y = h Wd' + bd + residual
// backward  hidden_kernel   gate and up again, dh = dy Wd, then h, dgate = dh up act'(gate), dup = dh act(gate)
//           output_kernel   dx = dgate Wg + dup Wu
//           weight_kernel   dWg = dgate' x, dWu = dup' x, dWd = dy' h, the biases' gradients as products with ones; the rows
//                           are shared out where the tiles are few, and join_kernel adds the parts in their order
#pragma once
#include "tile.h"

#include <utility>

namespace svox_decoder {

// NB products of one left operand with NB right ones, a block's tile of each.
template <class T, class S, bool along_a, bool along_b, int NB>
struct Product {
    static constexpr int planes = Form<T>::planes;
    using A = TileOf<along_a, S::BM, S::KT, S::threads>;
    using B = TileOf<along_b, S::BN, S::KT, S::threads>;
    static constexpr int stage = planes * (A::numbers + NB * B::numbers);   // 16-bit numbers

    static constexpr int loads = planes * (A::loads + NB * B::loads);       // of a lane

    struct Operands {
        A a;
        B b[NB];
        int64_t plane_a, plane_b[NB];
    };
    static __device__ __forceinline__ void load(Operands& o, u16* lds) {
#pragma unroll
        for (int p = 0; p < planes; ++p) {
            o.a.load(p * o.plane_a, lds + p * A::numbers);
#pragma unroll
            for (int i = 0; i < NB; ++i) o.b[i].load(p * o.plane_b[i], lds + planes * A::numbers + (p * NB + i) * B::numbers);
        }
        o.a.advance();
#pragma unroll
        for (int i = 0; i < NB; ++i) o.b[i].advance();
    }
    // What a wavefront multiplies at a time: `part` of its rows and all of its columns over 32 of the reduction.
    static constexpr int parts = S::TM * planes > 6 ? 2 : 1, PM = S::TM / parts;
    static_assert(PM * parts == S::TM, "equal parts");
    struct Rows {
        u16x8 a[PM][planes];
    };
    struct Columns {
        u16x8 b[NB][S::TN][planes];
    };
    static __device__ __forceinline__ void read(const u16* lds, int step, int part, int wm, Rows& f) {
#pragma unroll
        for (int m = 0; m < PM; ++m)
#pragma unroll
            for (int p = 0; p < planes; ++p) f.a[m][p] = A::fragment(lds + p * A::numbers, (wm * S::TM + part * PM + m) * 16, step);
    }
    static __device__ __forceinline__ void read(const u16* lds, int step, int wn, Columns& f) {
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int n = 0; n < S::TN; ++n)
#pragma unroll
                for (int p = 0; p < planes; ++p)
                    f.b[i][n][p] = B::fragment(lds + planes * A::numbers + (p * NB + i) * B::numbers, (wn * S::TN + n) * 16, step);
    }
    // ones: also the sums of the left operand's columns (over the reduction), in `sums`; those of float32 as the products are, this unit's
    // by themselves and added to the others in 32 bits, and every other time with minus ones.  odd: of the steps of the reduction; turning:
    // see run
    template <bool ones, bool odd, bool turning>
    static __device__ __forceinline__ void multiply_all(const Rows& rows, const Columns& columns, int part, f32x4 (&acc)[NB][S::TM][S::TN], f32x4* sums) {
        if constexpr (ones) {
            u16x8 one;
            for (int i = 0; i < 8; ++i) one[i] = Form<T>::one() ^ (planes == 3 && odd ? 0x8000 : 0);
#pragma unroll
            for (int m = 0; m < PM; ++m) {
                f32x4& all = sums[part * PM + m];
                f32x4 sum = planes == 3 ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : all;
#pragma unroll
                for (int p = planes; p-- > 0;) sum = Form<T>::mma(one, rows.a[m][p], sum);
                if constexpr (planes == 3)
                    all = odd ? all - sum : all + sum;
                else
                    all = sum;
            }
        }
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int n = 0; n < S::TN; ++n)
#pragma unroll
                for (int m = 0; m < PM; ++m) {
                    f32x4& c = acc[i][part * PM + m][n];
                    if (turning && ((part * PM + m) & 1) == odd)
                        c = multiply_turned<T>(columns.b[i][n], rows.a[m], c);
                    else
                        c = multiply<T>(columns.b[i][n], rows.a[m], c);
                }
    }
    // Adds the products over [k, k_end) of a and b to acc, with two `pairs` also those of a[1] and b[1], which are as large.  LDS holds
    // S::stages tiles of the reduction, registers the fragments of two units (a step of 32, or half of the rows of one): while
    // one is multiplied the next one is read, also from tile to tile.  At the barrier between two tiles every wavefront has read
    // all of the first, whose place the loads of a later one take, and all lanes' loads of the second have arrived (a lane's
    // loads arrive in their order, so that waiting for some leaves the later ones on their way).
    // turning: every other 32 of the reduction by multiply_turned, for float32 numbers that are summed up over the rows afterwards; of two
    // neighbouring tiles of rows it is not the same ones, so that a reduction of one step has turned rows too
    template <bool ones, int pairs = 1, bool turning = false>
    static __device__ __forceinline__ void run(const Planes* a, const Planes* b, int64_t m0, int64_t n0, int64_t k, int64_t k_end, u16* lds,
                                               f32x4 (&acc)[NB][S::TM][S::TN], f32x4* sums) {
        if (k >= k_end) return;
        constexpr int steps = S::KT / 32;
        const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave), wm = wave % S::WM, wn = wave / S::WM;
        static_assert(pairs == 1 || NB == 1, "");
        const int each = (int)((k_end - k + S::KT - 1) / S::KT), tiles = pairs * each;
        Operands o = operands(a[0], b, m0, n0, k, std::make_integer_sequence<int, NB>());
        int loaded = 0;
        auto load_next = [&] {
            if (pairs == 2 && loaded == each) o = operands(a[1], b + 1, m0, n0, k, std::make_integer_sequence<int, NB>());
            const int of_pair = pairs == 2 && loaded >= each ? loaded - each : loaded;
            if (of_pair == each - 1) {   // (an operand's own end may come a little before k_end, which is a whole number of 8)
                const int64_t at = k + (int64_t)of_pair * S::KT;
                o.a.last(least(k_end, along_a ? a[0].cols : a[0].rows) - at);
#pragma unroll
                for (int i = 0; i < NB; ++i) o.b[i].last(least(k_end, along_b ? b[i].cols : b[i].rows) - at);
            }
            load(o, lds + loaded % S::stages * stage);
            ++loaded;
        };
        // `later`: whole tiles that may still be on their way
        auto wait = [&](bool later) {
            if (later)
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((S::stages - 2) * loads) : "memory");
            else
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        };
        __syncthreads();   // (another product's last tile may still be read)
#pragma unroll
        for (int i = 0; i < S::stages - 1; ++i)
            if (i < tiles) load_next();
        wait(loaded == S::stages - 1);
        if (loaded < tiles) load_next();
        Rows rows[2];
        Columns columns[2];
        read(lds, 0, 0, wm, rows[0]);
        read(lds, 0, wn, columns[0]);
        constexpr int units = steps * parts;
        auto tile = [&](int t, auto odd) {   // its first fragments are in rows[odd * units mod 2], columns[odd * steps mod 2]
            constexpr int row = decltype(odd)::value * units, column = decltype(odd)::value * steps;
            const u16 *at = lds + t % S::stages * stage;
#pragma unroll
            for (int u = 0; u < units; ++u) {
                const int next = (u + 1) % units;
                if (u + 1 == units) {
                    if (t + 1 < tiles) {
                        wait(loaded - t - 2 >= S::stages - 2);
                        if (loaded < tiles) load_next();
                        at = lds + (t + 1) % S::stages * stage;
                        read(at, 0, 0, wm, rows[(row + units) & 1]);
                        read(at, 0, wn, columns[(column + steps) & 1]);
                    }
                } else {
                    read(at, next / parts, next % parts, wm, rows[(row + u + 1) & 1]);
                    if (next % parts == 0) read(at, next / parts, wn, columns[(column + next / parts) & 1]);
                }
                const Rows& r = rows[(row + u) & 1];
                const Columns& c = columns[(column + u / parts) & 1];
                if ((column + u / parts) & 1)
                    multiply_all<ones, true, turning>(r, c, u % parts, acc, sums);
                else
                    multiply_all<ones, false, turning>(r, c, u % parts, acc, sums);
            }
        };
        if constexpr (steps % 2 == 0) {
            for (int t = 0; t < tiles; ++t) tile(t, std::integral_constant<int, 0>());
        } else {
            for (int t = 0; t < tiles; t += 2) {
                tile(t, std::integral_constant<int, 0>());
                if (t + 1 < tiles) tile(t + 1, std::integral_constant<int, 1>());
            }
        }
    }
    template <int... i>
    static __device__ __forceinline__ Operands operands(const Planes& a, const Planes* b, int64_t m0, int64_t n0, int64_t k,
                                                        std::integer_sequence<int, i...>) {
        return Operands{A(a, m0, k), {B(b[i], n0, k)...}, a.plane, {b[i].plane...}};
    }
};

template <int NB, int TM, int TN>
__device__ __forceinline__ void clear(f32x4 (&acc)[NB][TM][TN]) {
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int m = 0; m < TM; ++m)
#pragma unroll
            for (int n = 0; n < TN; ++n) acc[i][m][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
}

// Where a lane's four numbers of a tile lie: row m, columns n..n+3.
template <class S>
struct Place {
    int64_t m0, n0;
    __device__ Place(int64_t tile_m, int64_t tile_n) {
        const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
        m0 = tile_m + (wave % S::WM) * S::TM * 16 + (lane & 15);
        n0 = tile_n + (wave / S::WM) * S::TN * 16 + (lane >> 4) * 4;
    }
    __device__ int64_t row(int m) const { return m0 + m * 16; }
    __device__ int64_t col(int n) const { return n0 + n * 16; }
};

// numbers n..n+3 of `count`, of which `room` from n on can be read; what is read beyond `count` is of no meaning
template <class T>
__device__ __forceinline__ f32x4 four_of(const T* from, int64_t n, int64_t room) {
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (!from) return v;
    const auto f = load_some<T, 4>(from + n, room);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (float)f[i];
    return v;
}
template <class T>
__device__ __forceinline__ void store_four(T* to, f32x4 v, int64_t n, int64_t count) {
    if (n + 4 <= count) {
        typename Few<T, 4>::vector f;
        for (int i = 0; i < 4; ++i) f[i] = (T)v[i];
        store_few<T, 4>(to + n, f);
    } else {
        for (int i = 0; i < 4; ++i)
            if (n + i < count) to[n + i] = (T)v[i];
    }
}

// Results go to memory through LDS, whole rows of a block's tile at a time.  From a lane's own four numbers a store writes 16 pieces of
// 32 bytes, each to a row of its own, and that is slow: the hidden numbers' gradients of 16 384 rows of 1024 -> 4096, in bfloat16 on
// tiles of 256 x 128, take 775 us so and 497 through LDS (387 with nothing stored).  `of` tiles of rows of each wavefront have
// room at a time; pieces of 16 bytes lie in an order that depends on the row, as the operands' tiles do.
constexpr int fitting(int tiles, int bytes, int room) {
    int of = tiles;
    while (tiles % of != 0 || of * bytes > room) --of;
    return of;
}
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
template <class S, class N, int of>
struct Staged {
    static constexpr int per = 16 / (int)sizeof(N), pieces = S::BN / per, rows = S::WM * of * 16, numbers = rows * S::BN;
    static constexpr int turn = pieces < 8 ? pieces - 1 : 7;
    static __device__ __forceinline__ int at(int row, int col) { return row * S::BN + ((col / per) ^ (row & turn)) * per + col % per; }
    // where a lane's four numbers of tile (m, n) lie
    static __device__ __forceinline__ int at_tile(int m, int n) {
        const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
        return at((wave % S::WM * of + m % of) * 16 + (lane & 15), (wave / S::WM * S::TN + n) * 16 + (lane >> 4) * 4);
    }
    // f(where it lies, its row, its first column) of every piece, `m` the first of the tiles
    template <class F>
    static __device__ __forceinline__ void each(int64_t m0, int64_t n0, int m, F f) {
#pragma unroll 4
        for (int i = threadIdx.x; i < rows * pieces; i += S::threads) {
            const int row = i / pieces, col = i % pieces * per;
            f(at(row, col), m0 + (row / (of * 16) * S::TM + m) * 16 + row % (of * 16), n0 + col);
        }
    }
};
// A tile of results, rounded to N, to rows of `cols` numbers
template <class S, int room, class N, class V>
__device__ __forceinline__ void store_tile(u16* lds, N* to, int64_t m0, int64_t n0, int64_t rows, int64_t cols, V value) {
    constexpr int of = fitting(S::TM, S::WM * 16 * S::BN * (int)sizeof(N), room * 2);
    using Tile = Staged<S, N, of>;
    N* const staged = reinterpret_cast<N*>(lds);
    typedef typename Few<N, 4>::vector four;
    typedef typename Few<N, Tile::per>::vector piece;
#pragma unroll
    for (int m = 0; m < S::TM; m += of) {
        lds_barrier();
#pragma unroll
        for (int n = 0; n < S::TN; ++n)
#pragma unroll
            for (int i = 0; i < of; ++i)
                *reinterpret_cast<four*>(staged + Tile::at_tile(m + i, n)) = __builtin_convertvector(value(m + i, n), four);
        lds_barrier();
        Tile::each(m0, n0, m, [&](int at, int64_t row, int64_t col) {
            if (row >= rows) return;
            const piece v = *reinterpret_cast<const piece*>(staged + at);
            N* const out = to + row * cols + col;
            if (col + Tile::per <= cols) {
                store_few<N, Tile::per>(out, v);
            } else {
#pragma unroll
                for (int i = 0; i < Tile::per; ++i)
                    if (col + i < cols) out[i] = v[i];
            }
        });
    }
}

template <class T>
struct HiddenArgs {
    Planes x, w_gate, w_up;      // (rows, dim), (hidden, dim) twice
    Planes dy, w_down;           // backward: (rows, out), (out, hidden)
    const T *b_gate, *b_up;      // or NULL
    u16 *h, *dgate, *dup;        // planes of (rows, ldh)
    float *b_gate_part, *b_up_part;   // backward: sums over rows of dgate and dup, (tiles_m WM, hidden), or NULL
    int64_t ldh, plane;
    int64_t rows, dim, hidden, out;
    int64_t tiles_m, tiles_n;
    int activation;
};

// The sums over 16 lanes (16 rows) of the biases' gradients, before they are rounded, at `row` of the parts.
__device__ __forceinline__ void keep_bias_sums(f32x4 gate, f32x4 up, float* gate_part, float* up_part, int64_t row, int64_t col, int64_t hidden) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 1; d < 16; d *= 2) {
            gate[i] += __shfl_xor(gate[i], d, kWave);
            up[i] += __shfl_xor(up[i], d, kWave);
        }
    if ((threadIdx.x & 15) != 0) return;
    if (gate_part) store_four(gate_part + row * hidden, gate, col, hidden);
    if (up_part) store_four(up_part + row * hidden, up, col, hidden);
}

// Measured, 16 384 rows of 1024 -> 4096 -> 1024 in bfloat16: forward 281 us, 979 TFLOP/s, of which storing 134 MB is some 50 us that nothing
// else covers; gradients 481 us, 857 TFLOP/s, with 403 MB to store (a library's product of 4096^3 1403), and five registers of a lane that
// wait in memory, once a tile.  8192 rows of 256 -> 1024 -> 256 in float32: 78 and 132 us, 110 and 98 TFLOP/s of float32, six times that of
// the matrix cores'.
template <class T, class S, bool backward>
__global__ __launch_bounds__(S::threads, 2) void hidden_kernel(HiddenArgs<T> p) {
    using Forward = Product<T, S, true, true, 2>;
    using Back = Product<T, S, true, false, 1>;
    constexpr int planes = Form<T>::planes;
    static_assert(Back::stage <= Forward::stage, "room");
    __shared__ __align__(16) u16 lds[S::stages * Forward::stage];
    int64_t tm, tn;
    tile_at(position_of_block(blockIdx.x, gridDim.x), p.tiles_m, p.tiles_n, tm, tn);
    const int64_t m0 = tm * S::BM, n0 = tn * S::BN;
    f32x4 acc[2][S::TM][S::TN], dh[1][S::TM][S::TN];
    clear(acc);
    const Planes w[2] = {p.w_gate, p.w_up};
    Forward::template run<false>(&p.x, w, m0, n0, 0, p.x.cols, lds, acc, nullptr);
    if constexpr (backward) {
        clear(dh);
        Back::template run<false, 1, planes == 3>(&p.dy, &p.w_down, m0, n0, 0, p.dy.cols, lds, dh, nullptr);
    }
    const Place<S> place(m0, n0);
    constexpr int results = backward ? 3 : 1;
    // (half of LDS at a time where that is enough: the gradients of large tiles 482 us so, 495 with all of it, which is stored later)
    constexpr int row_tile = results * planes * S::WM * 16 * S::BN * 2, room = S::stages * Forward::stage * 2;
    constexpr int of = fitting(S::TM, row_tile, row_tile * 2 <= room ? room / 2 : room);
    using Tile = Staged<S, u16, of>;
    with_activation(p.activation, [&](auto activation) {
        f32x4 gate_sum[S::TN], up_sum[S::TN];
#pragma unroll
        for (int m = 0; m < S::TM; m += of) {
            lds_barrier();
#pragma unroll
            for (int n = 0; n < S::TN; ++n) {
                if (m == 0) gate_sum[n] = up_sum[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                const int64_t col = place.col(n);
                if (col >= p.ldh) continue;
                const f32x4 bg = four_of(p.b_gate, col, p.hidden - col), bu = four_of(p.b_up, col, p.hidden - col);
#pragma unroll
                for (int j = 0; j < of; ++j) {
                    f32x4 result[3];   // h, dgate, dup
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float g = acc[0][m + j][n][i] + bg[i], u = acc[1][m + j][n][i] + bu[i];
                        float slope;
                        const float a = activate<planes == 3, decltype(activation)::value>(g, backward ? &slope : nullptr);
                        result[0][i] = a * u;
                        if constexpr (backward) {
                            result[1][i] = dh[0][m + j][n][i] * u * slope;
                            result[2][i] = dh[0][m + j][n][i] * a;
                        }
                    }
                    const int at = Tile::at_tile(m + j, n);
#pragma unroll
                    for (int r = 0; r < results; ++r) {
                        u16x4 part[planes];
                        Form<T>::split(result[r], part);
#pragma unroll
                        for (int q = 0; q < planes; ++q) *reinterpret_cast<u16x4*>(lds + (r * planes + q) * Tile::numbers + at) = part[q];
                    }
                    if constexpr (backward)
                        if (place.row(m + j) < p.rows) {
                            gate_sum[n] += result[1];
                            up_sum[n] += result[2];
                        }
                }
            }
            lds_barrier();
            Tile::each(m0, n0, m, [&](int at, int64_t row, int64_t col) {
                if (row >= p.rows || col >= p.ldh) return;
                u16* const to[3] = {p.h, p.dgate, p.dup};
                auto keep = [&](auto ends) {
#pragma unroll
                    for (int r = 0; r < results; ++r)
#pragma unroll
                        for (int q = 0; q < planes; ++q) {
                            u16x8 v = *reinterpret_cast<const u16x8*>(lds + (r * planes + q) * Tile::numbers + at);
                            if constexpr (decltype(ends)::value)
#pragma unroll
                                for (int i = 0; i < 8; ++i) v[i] = col + i < p.hidden ? v[i] : (u16)0;
                            *reinterpret_cast<u16x8*>(to[r] + q * p.plane + row * p.ldh + col) = v;
                        }
                };
                // (zeros beyond the last hidden unit: a row of infinities has made NaN of those that pad it)
                if (col + 8 > p.hidden) keep(std::true_type());
                else keep(std::false_type());
            });
        }
        if constexpr (backward)
            if (p.b_gate_part || p.b_up_part)
#pragma unroll
                for (int n = 0; n < S::TN; ++n)
                    if (place.col(n) < p.ldh)
                        keep_bias_sums(gate_sum[n], up_sum[n], p.b_gate_part, p.b_up_part, tm * S::WM + threadIdx.x / kWave % S::WM, place.col(n),
                                       p.hidden);
    });
}

template <class T>
struct OutputArgs {
    Planes a[2], b[2];     // y = a[0] b[0] + a[1] b[1]; one product where b is used along its rows
    const T *bias, *residual;
    int64_t residual_ld;
    T* y;                  // (rows, cols), dense
    int64_t rows, cols;
    int64_t tiles_m, tiles_n;
};

// along_b: b is (cols, reduction), else (reduction, cols).  Measured, as above: bfloat16 124 us, 1112 TFLOP/s, and 244 us, 1126 TFLOP/s (x's
// gradient); float32 35 and 61 us, 121 and 141 TFLOP/s.
template <class T, class S, bool along_b>
__global__ __launch_bounds__(S::threads, 2) void output_kernel(OutputArgs<T> p) {
    using P = Product<T, S, true, along_b, 1>;
    __shared__ __align__(16) u16 lds[S::stages * P::stage];
    int64_t tm, tn;
    tile_at(position_of_block(blockIdx.x, gridDim.x), p.tiles_m, p.tiles_n, tm, tn);
    const int64_t m0 = tm * S::BM, n0 = tn * S::BN;
    f32x4 acc[1][S::TM][S::TN];
    clear(acc);
    P::template run<false, along_b ? 1 : 2>(p.a, p.b, m0, n0, 0, p.a[0].cols, lds, acc, nullptr);
    const Place<S> place(m0, n0);
#pragma unroll
    for (int n = 0; n < S::TN; ++n) {
        const int64_t col = place.col(n);
        if (col >= p.cols) continue;
        const f32x4 bias = four_of(p.bias, col, p.cols - col);
#pragma unroll
        for (int m = 0; m < S::TM; ++m) {
            const int64_t row = place.row(m);
            if (row >= p.rows) continue;
            acc[0][m][n] += bias;
            if (p.residual) acc[0][m][n] += four_of(p.residual + row * p.residual_ld, col, (p.rows - 1 - row) * p.residual_ld + p.cols - col);
        }
    }
    store_tile<S, S::stages * P::stage>(lds, p.y, m0, n0, p.rows, p.cols, [&](int m, int n) { return acc[0][m][n]; });
}

// One weight's gradient: a' b over the rows, (m, n), and the sums of a's columns.
template <class T>
struct WeightJob {
    Planes a, b;
    int64_t m, n, tiles_m, tiles_n;
    float *part, *sums_part;   // [splits][m][n], [splits][m]; unused with one split
    T *out, *sums_out;         // sums_out NULL: no bias
};
template <class T>
struct WeightArgs {
    WeightJob<T> job[3];
    int64_t rows, each;        // rows of a split: a whole number of KT
    int splits;
};

// Measured, as above: bfloat16 441 us, 935 TFLOP/s, on 192 tiles and as many of 256 compute units (four splits would fill them, and
// leave 201 MB of parts to write and read); float32 105 us, 122 TFLOP/s.
template <class T, class S>
__global__ __launch_bounds__(S::threads, 2) void weight_kernel(WeightArgs<T> p) {
    using P = Product<T, S, false, false, 1>;
    __shared__ __align__(16) u16 lds[S::stages * P::stage];
    const int64_t position = position_of_block(blockIdx.x, gridDim.x), tiles = gridDim.x / p.splits, split = position / tiles;
    int64_t t = position % tiles, tm, tn;
    int j = 0;
    while (j < 2 && t >= p.job[j].tiles_m * p.job[j].tiles_n) {
        t -= p.job[j].tiles_m * p.job[j].tiles_n;
        ++j;
    }
    const WeightJob<T> job = p.job[j];
    tile_at(t, job.tiles_m, job.tiles_n, tm, tn);
    const int64_t m0 = tm * S::BM, n0 = tn * S::BN;
    const int64_t k = split * p.each, k_end = k + p.each < p.rows ? k + p.each : p.rows;
    f32x4 acc[1][S::TM][S::TN], sums[S::TM];
    clear(acc);
    for (int m = 0; m < S::TM; ++m) sums[m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const bool with_sums = job.sums_out && n0 == 0;
    if (with_sums)
        P::template run<true>(&job.a, &job.b, m0, n0, k, k_end, lds, acc, sums);
    else
        P::template run<false>(&job.a, &job.b, m0, n0, k, k_end, lds, acc, sums);
    const Place<S> place(m0, n0);
    if (with_sums && place.n0 == 0)   // (every column of the product with ones is the sum)
#pragma unroll
        for (int m = 0; m < S::TM; ++m) {
            const int64_t row = place.row(m);
            if (row >= job.m) continue;
            if (p.splits > 1)
                job.sums_part[split * job.m + row] = sums[m][0];
            else
                job.sums_out[row] = (T)sums[m][0];
        }
    if (!job.out) return;
    const auto value = [&](int m, int n) { return acc[0][m][n]; };
    if (p.splits > 1)
        store_tile<S, S::stages * P::stage>(lds, job.part + split * job.m * job.n, m0, n0, job.m, job.n, value);
    else
        store_tile<S, S::stages * P::stage>(lds, job.out, m0, n0, job.m, job.n, value);
}

// out = the sum of the parts, always in the same order: a block's lanes in 1 to 32 groups, four numbers to a lane, the parts over the
// groups.  Bound by the bytes of the parts.
template <class T>
struct JoinArgs {
    struct Job {
        const float* part;
        T* out;
        int64_t count;
        int splits, groups;
    } job[6];
    int64_t blocks[6];   // of every job
};
constexpr int kJoinThreads = 1024;
// (Up to four parts to a lane.  Three weights of 2048 x 768 and two parts: 13 us so, 117 with 32 groups whatever the parts are.)
inline int join_groups(int64_t splits) {
    int groups = 1;
    while (groups < 32 && groups * 4 < splits) groups *= 2;
    return groups;
}
template <class T>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(JoinArgs<T> p) {
    __shared__ f32x4 shared[kJoinThreads];
    int64_t block = blockIdx.x;
    int j = 0;
    while (j < 5 && block >= p.blocks[j]) block -= p.blocks[j++];
    const auto job = p.job[j];
    const int lanes = kJoinThreads / job.groups, lane = threadIdx.x % lanes, group = threadIdx.x / lanes;
    const int64_t i = (block * lanes + lane) * 4;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    if (i < job.count)
#pragma unroll 4
        for (int s = group; s < job.splits; s += job.groups) sum += four_of(job.part + s * job.count, i, job.count - i);
    if (job.groups > 1) {
        shared[threadIdx.x] = sum;
        __syncthreads();
        if (group == 0)
#pragma unroll 4
            for (int g = 1; g < job.groups; ++g) sum += shared[g * lanes + lane];
    }
    if (group == 0 && i < job.count) store_four(job.out, sum, i, job.count);
}

// Matrices laid out for TileOf: rows of whole 8 numbers, zeros beyond the columns, planes for float32.  A lane has 8 numbers; a
// block goes through rows with 256, 64 or 16 lanes to each.
template <class T>
struct LayJob {
    const T* from;
    int64_t ld;          // of `from`
    Planes to;
    int64_t cols;        // of `from`
    int64_t blocks, each;   // blocks, and rows of one
    int lanes;
};
template <class T>
struct LayArgs {
    LayJob<T> job[5];
};
// Bound by the bytes: 8192 x 256 and 3 x 1024 x 256 in float32, 11.4 us (12 MB read, 18 MB written).
constexpr int kLayThreads = 256;
template <class T>
__global__ __launch_bounds__(kLayThreads) void lay_kernel(LayArgs<T> p) {
    int64_t block = blockIdx.x;
    int j = 0;
    while (j < 4 && block >= p.job[j].blocks) block -= p.job[j++].blocks;
    const LayJob<T> job = p.job[j];
    const int rows = kLayThreads / job.lanes, lane = threadIdx.x % job.lanes;
    const int64_t first = block * job.each, end = least(first + job.each, job.to.rows);
#pragma unroll 4
    for (int64_t row = first + threadIdx.x / job.lanes; row < end; row += rows)
        for (int64_t col = lane * 8; col < job.to.cols; col += job.lanes * 8) {
            // (what can be read reaches to the end of the matrix, what is read beyond the row is taken for zeros)
            auto v = load_some<T, 8>(job.from + row * job.ld + col, (job.to.rows - 1 - row) * job.ld + job.cols - col);
            if (job.cols % 8 != 0)
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = col + i < job.cols ? v[i] : (T)0.0f;
            u16* const to = const_cast<u16*>(job.to.at) + row * job.to.ld + col;
            u16x8 out[Form<T>::planes];
            planes_of<T>(v, out);
#pragma unroll
            for (int q = 0; q < Form<T>::planes; ++q) *reinterpret_cast<u16x8*>(to + q * job.to.plane) = out[q];
        }
}

}  // namespace svox_decoder
