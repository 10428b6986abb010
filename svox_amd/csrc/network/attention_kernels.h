// attention_kernels.h -- attention within packed sequences, and its gradients.
//
//   s_ij = scale q_i . k_j,  o_i = sum_j p_ij v_j,  p_ij = exp(s_ij - m_i) / l_i,  m_i = max_j s_ij,  l_i = sum_j exp(s_ij - m_i)
//   delta_i = do_i . o_i,  dv_j = sum_i p_ij do_i,  ds_ij = p_ij (do_i . v_j - delta_i),  dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i
//
// over the keys j that query i sees.  Heads that share keys are taken together: a "row" is a query's token and one of the `group` heads of
// a head of keys, rows of a token side by side, so that a tile of keys is read once for all of them and the gradients of keys are sums
// over rows in registers.  A block takes a tile of rows and goes through the union of the keys that they see, which is one piece as
// sequences are packed in order: short sequences share a tile, and no launch depends on their lengths, which only the GPU knows.
//
// The backward pass computes scores twice, once for dq and once for dk and dv: seven products where one pass with atomic sums of dq
// would do with five, but sums in a fixed order, the same call the same bits.
//
// Scores and their exponentials, sums, maxima and results are in 32 bits.  p and ds are rounded to 16-bit operands where the type has 16 bits, as the matrix
// cores take them (in 32 bits they take seven times as long): a sum of many is off by what one rounding is, in the mean.
#pragma once
#include "attention_rules.h"
#include "attention_tile.h"

namespace svox_network {

template <class T>
struct AttendArgs {
    const T *q, *k, *v, *out, *grad;   // out (tokens, heads, dim) dense
    T* y;                              // forward: the result
    T* rest;                           // what rounding took from the result, times kLeft, as `out`, or NULL
    T *dq, *dk, *dv;                   // dense
    float *lse, *delta;                // [kv head][row]: log2 of the sum of exponentials, and its sum of do o
    float* part;                       // where the work of a tile is split: [kv head][split][row][DP] (keys and values: two of them)
    f32x2* stats;                      // [kv head][split][row]: maximum (of base 2), less kForwardRaised, and sum
    int64_t q_stride, q_head, k_stride, k_head, v_stride, v_head, grad_stride, grad_head;
    Sequences seq;
    int rows, keys;                    // of a kv head
    int group, kv_heads, dim;
    int tiles;
    int splits, steps;                 // blocks that may share a tile's other axis, and how many steps along it each is to have at least
    int* used;                         // [kv head][tile]: how many of them did
    const int* order;                  // tiles, those with the most to do first, or NULL
    int runs, last_first;              // blocks of an XCD take a few tiles side by side, else heads go round the XCDs; the last tiles come first
    float scale;
};

constexpr float kLog2E = 1.4426950408889634f, kNoSum = 3.0e38f;   // (the lse of a row that sees no key)

// Powers of two that keep the operands of products away from where float16's numbers run out (bfloat16 has float32's): from 2^-14 down they have fewer
// bits, from 2^-25 down none.  p of a row of n keys is some 1 / n: dv takes it times 2^14, of 65 536 at most four times what p can be (dv of 20
// rows of 8 heads over 262 144 keys: 10.4 times the error of one rounding without it, 1.4 with it).
template <class T>
constexpr int kRaised = std::is_same_v<T, F16> ? 14 : 0;
// The forward pass takes exponentials times 2^8, relative to a maximum that may lag behind by 2^4 (other types: 2^8): one that is 2^-22 of the largest has
// all of its bits still.  (8192 keys, all but the first 13 below it and their values 100 times its: 6.5 to 20 times the error of one rounding without it, at
// most 1.8 with it; the time is the same.)
template <class T>
constexpr int kForwardRaised = std::is_same_v<T, F16> ? 8 : 0;
template <class T>
constexpr int kLag = std::is_same_v<T, F16> ? 4 : 8;
template <class T>
constexpr float kLowered = std::is_same_v<T, F16> ? 0x1p-14f : 1.0f;
// ds, which may be anything, each row of dq and each key of dk takes times a power of two of its own, `up`: from kMostUp on, with which no number of
// float16 leaves float32's range, down to where the largest so far lies below 2^15, each time by as much as brings it to 2^14; the sum goes along.
// (Gradients of some 1e-3, 200 rows over 32 768 keys: dq 22.6 times the error of one rounding without it, 1.01 with it.  61 sequences' dq takes
// 85 -> 93 us for it, dk and dv 143 -> 161.)
template <class T>
constexpr bool kOwnScale = std::is_same_v<T, F16>;
constexpr float kMostUp = 0x1p80f;
template <int DB>
__device__ __forceinline__ float fit(float (&ds)[16], float& up, f32x16 (&acc)[DB]) {
    float most = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) most = fmaxf(most, __builtin_fabsf(ds[r]));
    if (!__any(most > 0x1p15f)) return 1.0f;
    most = most_of_halves(most);      // (the halves share the sum)
    const float less = most > 0x1p15f && most < __builtin_inff() ? __builtin_ldexpf(1.0f, 14 - __builtin_amdgcn_frexp_expf(most)) : 1.0f;
    up *= less;
#pragma unroll
    for (int r = 0; r < 16; ++r) ds[r] *= less;
#pragma unroll
    for (int db = 0; db < DB; ++db) acc[db] *= less;
    return less;
}

// The work of a block: a tile, a kv head, a part of the tile's other axis.
struct Place {
    int tile, head, split;   // no tile: tile < 0
};
template <class T>
__device__ __forceinline__ Place place_of_block(const AttendArgs<T>& p) {
    // (a tile's first blocks before all others: most tiles may need no more, and blocks go round the eight XCDs)
    const unsigned units = gridDim.x / p.splits, unit = blockIdx.x % units;
    Place at;
    at.split = blockIdx.x / units;
    if (p.order) {
        const unsigned i = unit / p.kv_heads;
        return {p.order[i], (int)(unit - i * p.kv_heads), at.split};
    }
    if (p.runs) {
        // (each time round the XCDs one further: sequences of a power of two would otherwise give one XCD all of their last tiles)
        const unsigned i = unit / 8, round = i / kAttendRun, xcd = (unit + round) % 8, position = (round * 8 + xcd) * kAttendRun + i % kAttendRun;
        at.head = position / p.tiles;
        at.tile = position - at.head * p.tiles;
        if (at.head >= p.kv_heads) return {-1, 0, 0};
    } else {
        at.tile = unit / p.kv_heads;
        at.head = unit - at.tile * p.kv_heads;
    }
    if (p.last_first) at.tile = p.tiles - 1 - at.tile;
    return at;
}
// A split's part of the tiles of `size` of a span.  How many blocks share it goes by its length, which only the GPU knows: as many as get
// p.steps tiles each.
struct Part {
    Span span;
    int used;
};
template <class T>
__device__ __forceinline__ Part part_of(const AttendArgs<T>& p, const Spans& all, int size, const Place& place) {
    if (all.low >= all.high) return {{0, 0}, 1};
    const int tiles = (all.high - all.low + size - 1) / size, most = (tiles + p.steps - 1) / p.steps, used = most < p.splits ? most : p.splits;
    if (used == 1) return {{all.low, all.high}, 1};
    const int each = (tiles + used - 1) / used;
    const int64_t low = all.low + (int64_t)place.split * each * size, high = low + (int64_t)each * size;
    return {{(int)(low < all.high ? low : all.high), (int)(high < all.high ? high : all.high)}, used};
}

__device__ __forceinline__ void clip(Span& see, const Span& part) { see.high = min(see.high, part.high); }

// rows r of `x`, (tokens, heads, dim) with strides
template <class T>
__device__ __forceinline__ const T* row_at(const T* x, int r, int group, int head, int64_t stride, int64_t head_stride) {
    const unsigned token = group == 1 ? (unsigned)r : (unsigned)r / (unsigned)group;
    return x + (int64_t)token * stride + ((int64_t)head * group + (r - (int)token * group)) * head_stride;
}

// What the rows of a wavefront's lanes (row `mine` + lane % 32) see, all of them together, and those of its block together, rows
// r0 .. r0 + rows - 1; of rows where `keys` is not set.  Rows that are not there see everything, so that they never make a mask necessary.
__device__ __forceinline__ Spans spans_of(const Sequences& s, bool keys, int mine, int count, int r0, int rows, int group, Span& see, Spans& block) {
    const int lane = (int)threadIdx.x % kWave, last = min(r0 + rows, count) - 1, here = min(mine + 32, count) - mine;
    const int per_token = keys ? group : 1, per_other = keys ? 1 : group;
    // (the upper lanes look at the block's first and last row)
    const int r = mine + lane % 32, looked = lane < 32 ? min(r, last) : lane == 32 ? r0 : last;
    Span v = per_token == 1 ? span_of(s, keys, looked, r0, last) : span_of(s, keys, looked / per_token, r0 / per_token, last / per_token);
    v.low *= per_other, v.high *= per_other;
    block = {__builtin_amdgcn_readlane(v.low, 32), __builtin_amdgcn_readlane(v.high, 33), __builtin_amdgcn_readlane(v.low, 33),
             __builtin_amdgcn_readlane(v.high, 32)};
    Spans all{0, 0, INT32_MIN, INT32_MAX};
    if (here > 0)
        all = {__builtin_amdgcn_readlane(v.low, 0), __builtin_amdgcn_readlane(v.high, here - 1), __builtin_amdgcn_readlane(v.low, here - 1),
               __builtin_amdgcn_readlane(v.high, 0)};
    v.low = __shfl(v.low, lane % 32, kWave), v.high = __shfl(v.high, lane % 32, kWave);
    see = r < count ? v : Span{INT32_MIN, INT32_MAX};
    return all;
}

// `place`, an end of what a lane sees, counted from `from`: modulo 2^32, as the ends of rows that are not there are those of the integers, and what it
// then is does not matter.
__device__ __forceinline__ int from_place(int place, int from) { return (int)((unsigned)place - (unsigned)from); }

// A lane's 16 scores whose rows lie below `low`, or from `high` on (counted from the first of them), become `v`.
template <class Scores>
__device__ __forceinline__ void hide_below(Scores& s, int low, float v) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = row_of(r) < low ? v : s[r];
}
template <class Scores>
__device__ __forceinline__ void hide_from(Scores& s, int high, float v) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = row_of(r) < high ? s[r] : v;
}

// What is left of a number that is rounded to T.  The backward pass takes delta from both: with the rounded result alone delta was off by a
// part in 2^11 (f16), for all of a row's keys alike, and dq and dk with it (1659 causal rows of 64: 1.54 times the error of one rounding, 1.42 so).
// float16's times 2^11, which makes it the result at most, as float16 has few bits for what a small result leaves (values of some 1e-4, gradients of some
// 2000, 4000 keys: dq 4.3 times the error of one rounding as it is, 1.4 so).
template <class T>
constexpr float kLeft = std::is_same_v<T, F16> ? 0x1p11f : 1.0f;
template <class T>
__device__ __forceinline__ float left_of(float v) {
    return (v - (float)(T)v) * kLeft<T>;
}

// ---- forward.  Four wavefronts, of which `across` share rows and take a part of every tile's keys each.
template <class T, int DP, int across, bool narrow>
struct ForwardShape {
    static constexpr int down = 4 / across, rows = down * 32;
    static constexpr int keys = across == 4 ? 128 : (narrow ? 32 : 64), mine = keys / across, blocks = mine / 32;
    static constexpr int stages = across == 4 && sizeof(T) == 4 && DP == 128 ? 1 : 2;   // tiles in LDS
    static constexpr int tile = keys * DP;
};

// (float32, heads of 32: registers for four wavefronts a SIMD rather than three: 512 windows of 64 cells, 4 heads of 16, 36 -> 30 us; 8 of 4096 644 -> 625.)
template <class T, int DP, int across, bool direct, bool far>
__global__ __launch_bounds__(kAttendThreads, sizeof(T) == 4 && DP > 64 ? 1 : sizeof(T) == 4 && DP == 32 && across == 1 && direct ? (far ? 3 : 4) : 2)
void attend_kernel(AttendArgs<T> p) {
    using S = ForwardShape<T, DP, across, sizeof(T) == 4 && (DP == 128 || (far && DP == 64 && !direct))>;
    using F = Frag<T>;
    using Eight = typename F::Eight;
    constexpr int DB = DP / 32, KB = S::blocks;
    constexpr int join_numbers = across > 1 ? 4 * 32 * (DP + 2) : 0;   // floats
    constexpr int tile_bytes = 2 * S::stages * S::tile * (int)sizeof(T), join_bytes = join_numbers * 4;
    __shared__ __attribute__((aligned(16))) char lds[tile_bytes > join_bytes ? tile_bytes : join_bytes];
    __shared__ int found[2];                     // the tile of a stage that holds infinite numbers or NaN (or chance: it is looked at once more)
    __shared__ unsigned kinds[3][S::keys][DB];   // NaN, inf and -inf that were taken out of a tile of v
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave), h = half_of();
    const Place place = place_of_block(p);
    if (place.tile < 0) return;
    const int r0 = place.tile * S::rows, mine = r0 + wave / across * 32;

    Eight q[DP / 16];
    load_row<T, DP, direct>(row_at(p.q, min(mine + (int)threadIdx.x % 32, p.rows - 1), p.group, place.head, p.q_stride, p.q_head), p.dim, q);
    Span see;
    Spans block;
    const Spans spans = spans_of(p.seq, true, mine, p.rows, r0, S::rows, p.group, see, block);
    const Part share = part_of(p, block, S::keys, place);
    if (place.split >= share.used) return;
    if (p.splits > 1 && place.split == 0 && threadIdx.x == 0) p.used[place.head * p.tiles + place.tile] = share.used;
    const Span part = share.span;
    clip(see, part);

    const float to2 = p.scale * kLog2E;
    // Narrow heads: vector instructions are what bounds them (32 rows, 64 keys of 32 numbers: 115 of them, of which 32 are exponentials at half the rate,
    // some 590 cycles; 8 products of 32 cycles): the exponentials' sum is one more product, with ones, of which a lane's first number is kept
    // (512 windows of 512 cells, 4 heads of 32: 154 -> 149 us).
    constexpr bool by_product = sizeof(T) == 2 && DP <= 64;
    f32x16 acc[DB], ones_acc = {};
    float m = -__builtin_inff(), l = 0.0f;
    Eight ones;
    if constexpr (by_product) {
        const float one[8] = {1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f};
        ones = F::pack(one);
    }
    T* const tiles = reinterpret_cast<T*>(lds);
#pragma unroll
    for (int db = 0; db < DB; ++db) acc[db] = f32x16{};
    Loader<T, DP, S::keys, direct> ks(p.k + place.head * p.k_head, p.k_stride, 0, 1, p.dim), vs(p.v + place.head * p.v_head, p.v_stride, 0, 1, p.dim);
    const auto load = [&](int k0, int stage) {
        ks.load(k0, part.high - k0, tiles + stage * 2 * S::tile);
        vs.load(k0, part.high - k0, tiles + (stage * 2 + 1) * S::tile);
    };
    const auto finish = [&](int stage, int k0) {
        ks.finish(tiles + stage * 2 * S::tile);
        vs.finish(tiles + (stage * 2 + 1) * S::tile);
        if (block.masks(k0, S::keys) && holds_odd<T, DP, S::keys>(tiles + (stage * 2 + 1) * S::tile)) found[stage] = k0;
        __syncthreads();
    };
    if (part.low < part.high) {
        load(part.low, 0);
        finish(0, part.low);
    }
    // vmcnt(0).  What stays in registers has arrived; the compiler, which does not see the tiles' loads, would else wait for it where it is first
    // used in the loop, and for the next tile with it.
    __builtin_amdgcn_s_waitcnt(0x0f70);
    int stage = 0;
    for (int k0 = part.low; k0 < part.high; k0 += S::keys) {
        const bool more = k0 + S::keys < part.high;
        if (more && S::stages == 2) load(k0 + S::keys, stage ^ 1);
        const T* const kt = tiles + stage * 2 * S::tile;
        const T* const vt = kt + S::tile;
        const bool odd = block.masks(k0, S::keys) && found[stage] == k0;
        if (odd) {
            for (int i = (int)threadIdx.x; i < 3 * S::keys * DB; i += kAttendThreads) (&kinds[0][0][0])[i] = 0;
            take_out_odd<T, DP, S::keys>(tiles + (stage * 2 + 1) * S::tile, [&](int row, int column, float x) {
                atomicOr(&kinds[x != x ? 0 : x > 0.0f ? 1 : 2][row][column / 32], 1u << column % 32);
            });
        }
        const int kw = k0 + wave % across * S::mine;   // this wavefront's keys
        if (kw < spans.high && kw + S::mine > spans.low && kw < part.high) {
            if constexpr (DP == 128) __builtin_amdgcn_s_setprio(1);   // (the other wavefront of the SIMD has exponentials to compute meanwhile: 633 -> 600 us)
            f32x16 s[KB];
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                s[b] = f32x16{};
#pragma unroll
                for (int t = 0; t < DP / 16; ++t) {
                    if (sizeof(T) == 4 && 16 * t >= p.dim) break;   // (float32's products are dear)
                    s[b] = F::mma(Tile<T, DP>::along(kt, wave % across * S::mine + 32 * b, t), q[t], s[b]);
                }
            }
            if constexpr (DP == 128) __builtin_amdgcn_s_setprio(0);
            // (the tile's end lies beyond what some lane sees, if it lies beyond the part)
            if (kw < spans.all_low) {
#pragma unroll
                for (int b = 0; b < KB; ++b) hide_below(s[b], from_place(see.low, kw + 32 * b + 4 * h), -__builtin_inff());
            }
            if (kw + S::mine > min(spans.all_high, part.high)) {
#pragma unroll
                for (int b = 0; b < KB; ++b) hide_from(s[b], from_place(see.high, kw + 32 * b + 4 * h), -__builtin_inff());
            }
            Eight e[KB][2];
            float most = m;
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) most = fmaxf(most, s[b][r]);
            most = most_of_halves(most);
            // The maximum that exponentials are relative to need not be the largest score: any will do whose exponentials stay in range.  It is moved, and
            // the sums with it, where a row's has grown by more than 2^kLag (a wavefront's 32 rows find new maxima in two tiles of three of a
            // long sequence: 16 384 causal rows, 8 heads of 128 581 -> 550 us).
            const bool grown = (most - m) * to2 > (float)kLag<T>;      // (not where both are infinite: exponentials of -inf are 0, and the row of an inf is NaN)
            if (__any(grown)) {
                const float less = grown ? __builtin_amdgcn_exp2f((m - most) * to2) : 1.0f;
                if constexpr (by_product) ones_acc[0] *= less;
                else l *= less;
#pragma unroll
                for (int db = 0; db < DB; ++db) acc[db] *= less;
                m = grown ? most : m;      // (each row by itself: no row has other bits for what its neighbours hold)
            }
            const float from = m == -__builtin_inff() ? 0.0f : m * to2 - (float)kForwardRaised<T>;   // (nothing seen yet: exponentials of -inf are 0)
            float sum = 0.0f;      // (of this step alone: one addition a step to what may be the sum of very many)
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                float x[16];
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    x[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][r], to2, -from));
                    if constexpr (!by_product) sum += x[r];
                }
                e[b][0] = F::pack(x);
                e[b][1] = F::pack(x + 8);
            }
            if constexpr (!by_product) l += sum;
            if constexpr (far) {
                accumulate_apart<DP>(acc, vt, wave % across * S::mine, e);
            } else {
#pragma unroll
                for (int b = 0; b < KB; ++b)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int at = wave % across * S::mine + 32 * b + 16 * c;
                        accumulate<T, DP>(acc, vt, at, e[b][c]);
                        if constexpr (by_product) ones_acc = F::mma(ones, e[b][c], ones_acc);
                    }
            }
            if (odd) {
                // (v's numbers that were taken out, for the lanes that see them: p is positive)
#pragma unroll
                for (int kind = 0; kind < 3; ++kind) {
                    unsigned which[DB] = {};
#pragma unroll 1
                    for (int i = wave % across * S::mine; i < (wave % across + 1) * S::mine; ++i)
                        if (k0 + i >= see.low && k0 + i < see.high)
#pragma unroll
                            for (int db = 0; db < DB; ++db) which[db] |= kinds[kind][i][db];
                    const float odd_one = kind == 0 ? __builtin_nanf("") : kind == 1 ? __builtin_inff() : -__builtin_inff();
#pragma unroll
                    for (int db = 0; db < DB; ++db)
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (which[db] >> (row_of(r) + 4 * h) & 1) acc[db][r] += odd_one;
                }
            }
        }
        if constexpr (S::stages == 2) {
            stage ^= 1;
            if (more) finish(stage, k0 + S::keys);
        } else {
            __syncthreads();
            if (more) load(k0 + S::keys, 0), finish(0, k0 + S::keys);
        }
    }

    l = by_product ? ones_acc[0] : sum_of_halves(l);
    if constexpr (across > 1) {
        // the wavefronts' sums, joined by the first: every lane finds its own numbers of the others
        static_assert(across == 4, "all wavefronts share rows");
        __syncthreads();
        float* const shared = reinterpret_cast<float*>(lds);
        const int lane = (int)threadIdx.x % kWave;
        constexpr int each = DB * 16 * kWave;   // numbers of a wavefront, then its maxima and sums
        static_assert(4 * (each + 64) <= join_numbers, "room");
        float* const own = shared + wave * (each + 64);
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) own[(db * 16 + r) * kWave + lane] = acc[db][r];
        if (lane < 32) own[each + lane] = m, own[each + 32 + lane] = l;
        __syncthreads();
        if (wave != 0) return;
        float most = m;
        for (int w = 1; w < 4; ++w) most = fmaxf(most, shared[w * (each + 64) + each + lane % 32]);
        const float from = most == -__builtin_inff() ? 0.0f : most;
        l = 0.0f;
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[db] = f32x16{};
        for (int w = 0; w < 4; ++w) {
            const float* const other = shared + w * (each + 64);
            if (other[each + lane % 32] == -__builtin_inff() && other[each + 32 + lane % 32] == 0.0f) continue;
            const float less = __builtin_amdgcn_exp2f((other[each + lane % 32] - from) * to2);
            l = __builtin_fmaf(other[each + 32 + lane % 32], less, l);
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[db][r] = __builtin_fmaf(other[(db * 16 + r) * kWave + lane], less, acc[db][r]);
        }
        m = most;
    }
    const int thread = thread_again(), half = thread / 32 % 2, r = mine + thread % 32;
    if (r >= p.rows) return;
    // (what a row that sees keys has, though all of its scores are -inf, is not what one that sees none has)
    const bool some = max(see.low, part.low) < see.high;
    if (share.used > 1) {
        const int64_t at = ((int64_t)place.head * p.splits + place.split) * p.rows + r;
        if (half == 0) p.stats[at] = f32x2{some ? fmaxf(m * to2 - (float)kForwardRaised<T>, -3.0e38f) : -__builtin_inff(), some ? l : 0.0f};
        if (some) store_row<float, DB>(p.part + at * DP, DP, acc, 1.0f, half);
    } else {
        const unsigned token = (unsigned)r / again(p.group);
        const int64_t to = (((int64_t)token * p.kv_heads + place.head) * p.group + (r - (int)token * p.group)) * p.dim;
        const float factor = some ? 1.0f / l : 0.0f;
        store_row<T, DB>(p.y + to, p.dim, acc, factor, half);
        if (p.rest) {
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[db][i] = left_of<T>(acc[db][i] * factor);
            store_row<T, DB>(p.rest + to, p.dim, acc, 1.0f, half);
        }
        if (p.lse && half == 0) p.lse[(int64_t)place.head * p.rows + r] = some ? __builtin_fmaf(m, to2, __builtin_amdgcn_logf(l) - (float)kForwardRaised<T>) : kNoSum;
    }
}

template <class T>
__device__ __forceinline__ void store_joined(const AttendArgs<T>& p, int64_t i, int head, int r, int lane, float most, float l, f32x4 sum) {
    const bool some = most != -__builtin_inff();
    const float factor = some ? 1.0f / l : 0.0f;
    const int token = r / p.group;
    const int64_t to = (((int64_t)token * p.kv_heads + head) * p.group + (r - token * p.group)) * p.dim + 4 * lane;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (4 * lane + j < p.dim) {
            p.y[to + j] = (T)(sum[j] * factor);
            if (p.rest) p.rest[to + j] = (T)left_of<T>(sum[j] * factor);
        }
    if (p.lse && lane == 0) p.lse[i] = some ? most + __builtin_amdgcn_logf(l) : kNoSum;
}

// The splits' sums of a row, where there are several: a row by as many lanes as its numbers are fours, one split after another.
template <class T, int DP>
__global__ __launch_bounds__(kAttendThreads) void attend_join_kernel(AttendArgs<T> p, int rows) {
    constexpr int lanes = DP / 4;
    const int lane = (int)threadIdx.x % lanes;
    const int64_t all = (int64_t)p.kv_heads * p.rows, step = (int64_t)gridDim.x * (kAttendThreads / lanes);
    for (int64_t i = (int64_t)blockIdx.x * (kAttendThreads / lanes) + threadIdx.x / lanes; i < all; i += step) {
        const int head = (int)(i / p.rows), r = (int)(i - (int64_t)head * p.rows);
        const int used = p.used[head * p.tiles + r / rows];
        if (used == 1) continue;
        const int64_t first = (int64_t)head * p.splits * p.rows + r;
        float most = -__builtin_inff(), l = 0.0f;
        for (int s = 0; s < used; ++s) most = fmaxf(most, p.stats[first + (int64_t)s * p.rows][0]);
        f32x4 sum = {};
        for (int s = 0; s < used; ++s) {
            const int64_t at = first + (int64_t)s * p.rows;
            const f32x2 stat = p.stats[at];
            if (stat[0] == -__builtin_inff()) continue;   // (nothing seen, nothing stored)
            const float less = __builtin_amdgcn_exp2f(stat[0] - most);
            l = __builtin_fmaf(stat[1], less, l);
            sum += *reinterpret_cast<const f32x4*>(p.part + at * DP + 4 * lane) * less;
        }
        store_joined<T>(p, i, head, r, lane, most, l, sum);
    }
}
// Of many splits: a row a block, as many splits at once as there are lanes for.
template <class T, int DP>
__global__ __launch_bounds__(kAttendThreads) void attend_join_many_kernel(AttendArgs<T> p, int rows) {
    constexpr int lanes = DP / 4, groups = kAttendThreads / lanes;
    __shared__ f32x4 room[kAttendThreads];
    __shared__ float sums[kAttendThreads];
    const int lane = (int)threadIdx.x % lanes, group = (int)threadIdx.x / lanes;
    const int64_t all = (int64_t)p.kv_heads * p.rows, each = (all + gridDim.x - 1) / gridDim.x;
    for (int64_t i = blockIdx.x * each; i < least((blockIdx.x + 1) * each, all); ++i) {
        const int head = (int)(i / p.rows), r = (int)(i - (int64_t)head * p.rows);
        const int used = p.used[head * p.tiles + r / rows];
        if (used == 1) continue;
        const int64_t first = (int64_t)head * p.splits * p.rows + r;
        float most = -__builtin_inff();
        for (int s = (int)threadIdx.x % kWave; s < used; s += kWave) most = fmaxf(most, p.stats[first + (int64_t)s * p.rows][0]);
#pragma unroll
        for (int d = 1; d < kWave; d *= 2) most = fmaxf(most, __shfl_xor(most, d, kWave));
        f32x4 sum = {};
        float l = 0.0f;
#pragma unroll 4
        for (int s = group; s < used; s += groups) {
            const int64_t at = first + (int64_t)s * p.rows;
            const f32x2 stat = p.stats[at];
            const f32x4 part = *reinterpret_cast<const f32x4*>(p.part + at * DP + 4 * lane);
            const bool some = stat[0] != -__builtin_inff();   // (else nothing was seen, and nothing stored)
            const float less = __builtin_amdgcn_exp2f(stat[0] - most);
            l += some ? stat[1] * less : 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[j] += some ? part[j] * less : 0.0f;
        }
        __syncthreads();
        room[threadIdx.x] = sum;
        if (lane == 0) sums[group] = l;
        __syncthreads();
        if (group != 0) continue;
        l = 0.0f;
        for (int g = 0; g < groups; ++g) l += sums[g];
        for (int g = 1; g < groups; ++g) sum += room[g * lanes + lane];
        store_joined<T>(p, i, head, r, lane, most, l, sum);
    }
}

// delta of row `row`, whose gradient is g: its sum of do o, by two lanes
template <class T, int DP, bool direct>
__device__ __forceinline__ float delta_of(const AttendArgs<T>& p, int row, int head, const typename Frag<T>::Eight (&g)[DP / 16]) {
    typename Frag<T>::Eight o[DP / 16];
    const unsigned token = (unsigned)row / (unsigned)p.group;
    const int64_t at = (((int64_t)token * p.kv_heads + head) * p.group + (row - (int)token * p.group)) * p.dim;
    load_row<T, DP, direct>(p.out + at, p.dim, o);
    float delta = 0.0f;
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) delta += dot<T>(o[t], g[t]);
    if (p.rest) {
        load_row<T, DP, direct>(p.rest + at, p.dim, o);
        float left = 0.0f;
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) left += dot<T>(o[t], g[t]);
        delta = __builtin_fmaf(left, 1.0f / kLeft<T>, delta);
    }
    return sum_of_halves(delta);
}
// Where dq, whose kernel computes it too, is not asked for.
template <class T, int DP>
__global__ __launch_bounds__(kAttendThreads) void attend_delta_kernel(AttendArgs<T> p) {
    const int64_t tiles = ((int64_t)p.rows + 127) / 128;
    for (int64_t i = blockIdx.x; i < tiles * p.kv_heads; i += gridDim.x) {
        const int head = (int)(i / tiles), mine = (int)(i - head * tiles) * 128 + (int)threadIdx.x / kWave * 32 + (int)threadIdx.x % 32, row = min(mine, p.rows - 1);
        typename Frag<T>::Eight g[DP / 16];
        load_row<T, DP, false>(row_at(p.grad, row, p.group, head, p.grad_stride, p.grad_head), p.dim, g);
        const float delta = delta_of<T, DP, false>(p, row, head, g);
        if (half_of() == 0 && mine < p.rows) p.delta[(int64_t)head * p.rows + row] = delta;
    }
}

// ---- dq: rows as forward, through the keys they see.  (float32, heads of 32: tiles of 32 keys leave registers for four wavefronts a SIMD, 64 for
// three: 512 windows of 64 cells, 4 heads of 16, 34 -> 28 us; heads of 64 lose as much as they gain, those of 128 have room for no more.)
// (Heads of 64 in 16 bits: registers for three wavefronts a SIMD rather than two, 536 -> 472 us for 16 384 causal rows, 8 heads; with two of the four
// fragments of g in LDS as good.)
template <class T, int DP, bool direct, bool far>
__global__ __launch_bounds__(kAttendThreads, sizeof(T) == 4 && DP > 64 ? 1 : sizeof(T) == 2 && DP == 64 && direct ? 3 : 2)
void attend_query_grad_kernel(AttendArgs<T> p) {
    using F = Frag<T>;
    using Eight = typename F::Eight;
    constexpr int DB = DP / 32, rows = 128, keys = sizeof(T) == 4 && (DP != 64 || (far && !direct)) ? 32 : 64, tile = keys * DP, KB = keys / 32;
    __shared__ __attribute__((aligned(16))) T tiles[4 * tile];
    __shared__ int found[2];              // the tile of a stage that holds infinite numbers or NaN, or none
    __shared__ unsigned bad[keys / 32];   // keys that are not finite
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave), h = half_of();
    const Place place = place_of_block(p);
    if (place.tile < 0) return;
    const int r0 = place.tile * rows, mine = r0 + wave * 32, row = min(mine + (int)threadIdx.x % 32, p.rows - 1);

    Eight q[DP / 16], g[DP / 16];
    load_row<T, DP, direct>(row_at(p.q, row, p.group, place.head, p.q_stride, p.q_head), p.dim, q);
    load_row<T, DP, direct>(row_at(p.grad, row, p.group, place.head, p.grad_stride, p.grad_head), p.dim, g);
    Span see;
    Spans block;
    const Spans spans = spans_of(p.seq, true, mine, p.rows, r0, rows, p.group, see, block);
    const Part share = part_of(p, block, keys, place);
    if (place.split >= share.used) return;
    if (p.splits > 1 && place.split == 0 && threadIdx.x == 0) p.used[place.head * p.tiles + place.tile] = share.used;
    const Span part = share.span;
    clip(see, part);

    const float lse = p.lse[(int64_t)place.head * p.rows + row];
    float delta = delta_of<T, DP, direct>(p, row, place.head, g);
    if (place.split == 0 && h == 0 && mine + (int)threadIdx.x % 32 < p.rows) p.delta[(int64_t)place.head * p.rows + row] = delta;
    // (registers for float16's `fit`: 32 keys at a time, or a fragment of g in LDS)
    constexpr bool one_by_one = kOwnScale<T> && DP == 64;
    constexpr int kept = kOwnScale<T> && DP == 128 && !direct ? DP / 16 - 1 : DP / 16;
    __shared__ Eight rest[kept < DP / 16 ? DP / 16 - kept : 1][kept < DP / 16 ? kAttendThreads : 1];
#pragma unroll
    for (int t = kept; t < DP / 16; ++t) rest[t - kept][threadIdx.x] = g[t];
    const float to2 = p.scale * kLog2E;
    f32x16 acc[DB];
    float none = 0.0f, up = kOwnScale<T> ? kMostUp : 1.0f;
    delta *= up;
#pragma unroll
    for (int db = 0; db < DB; ++db) acc[db] = f32x16{};
    Loader<T, DP, keys, direct> ks(p.k + place.head * p.k_head, p.k_stride, 0, 1, p.dim), vs(p.v + place.head * p.v_head, p.v_stride, 0, 1, p.dim);
    const auto load = [&](int k0, int stage) {
        ks.load(k0, part.high - k0, tiles + stage * 2 * tile);
        vs.load(k0, part.high - k0, tiles + (stage * 2 + 1) * tile);
    };
    const auto finish = [&](int stage, int k0) {
        ks.finish(tiles + stage * 2 * tile);
        vs.finish(tiles + (stage * 2 + 1) * tile);
        if (block.masks(k0, keys) && holds_odd<T, DP, keys>(tiles + stage * 2 * tile)) found[stage] = k0;
        __syncthreads();
    };
    if (part.low < part.high) {
        load(part.low, 0);
        finish(0, part.low);
    }
    // vmcnt(0).  What stays in registers has arrived; the compiler, which does not see the tiles' loads, would else wait for it where it is first
    // used in the loop, and for the next tile with it.
    __builtin_amdgcn_s_waitcnt(0x0f70);
    int stage = 0;
    for (int k0 = part.low; k0 < part.high; k0 += keys) {
        const bool more = k0 + keys < part.high;
        if (more) load(k0 + keys, stage ^ 1);
        const T* const kt = tiles + stage * 2 * tile;
        const T* const vt = kt + tile;
        const bool odd = block.masks(k0, keys) && found[stage] == k0;
        if (odd) {
            if (threadIdx.x < keys / 32) bad[threadIdx.x] = 0;
            take_out_odd<T, DP, keys>(tiles + stage * 2 * tile, [&](int row, int, float) { atomicOr(&bad[row / 32], 1u << row % 32); });
        }
        if (k0 < spans.high && k0 + keys > spans.low) {
#pragma unroll one_by_one ? 1 : KB
            for (int b = 0; b < KB; ++b) {
                f32x16 s = {}, dp = {};
#pragma unroll
                for (int t = 0; t < DP / 16; ++t) {
                    if (sizeof(T) == 4 && 16 * t >= p.dim) break;
                    s = F::mma(Tile<T, DP>::along(kt, 32 * b, t), q[t], s);
                    dp = F::mma(Tile<T, DP>::along(vt, 32 * b, t), t < kept ? g[t] : rest[t < kept ? 0 : t - kept][threadIdx.x], dp);
                }
                float ds[16];
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float p_r = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], to2, -lse));
                    if constexpr (kOwnScale<T>) ds[r] = p_r * __builtin_fmaf(dp[r], up, -delta);
                    else ds[r] = p_r * (dp[r] - delta);
                }
                if (k0 < spans.all_low) hide_below(ds, from_place(see.low, k0 + 32 * b + 4 * h), 0.0f);
                if (k0 + keys > min(spans.all_high, part.high)) hide_from(ds, from_place(see.high, k0 + 32 * b + 4 * h), 0.0f);
                if constexpr (kOwnScale<T>) delta *= fit(ds, up, acc);
                if constexpr (far) {
                    const Eight e[1][2] = {{F::pack(ds), F::pack(ds + 8)}};
                    accumulate_apart<DP>(acc, kt, 32 * b, e);
                } else {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        accumulate<T, DP>(acc, kt, 32 * b + 16 * c, F::pack(ds + 8 * c));
                    }
                }
            }
        }
        if (odd)      // (whoever sees a key that is not finite has no gradient that is)
            for (int i = 0; i < keys; ++i)
                if ((bad[i / 32] >> i % 32 & 1) && k0 + i >= see.low && k0 + i < see.high) none = __builtin_nanf("");
        stage ^= 1;
        if (more) finish(stage, k0 + keys);
    }
#pragma unroll
    for (int db = 0; db < DB; ++db) acc[db] += none;
    const int thread = thread_again(), half = thread / 32 % 2, r = mine + thread % 32;
    if (r >= p.rows) return;
    if (share.used > 1) {
        store_row<float, DB>(p.part + (((int64_t)place.head * p.splits + place.split) * p.rows + r) * DP, DP, acc, 1.0f / up, half);
    } else {
        const unsigned token = (unsigned)r / again(p.group);
        store_row<T, DB>(p.dq + (((int64_t)token * p.kv_heads + place.head) * p.group + (r - (int)token * p.group)) * p.dim, p.dim, acc, p.scale / up, half);
    }
}

// ---- dk and dv: a tile of keys, 32 to a wavefront, through the rows that see them.  (Rows of a tile, 32 or 64: float32 with heads of 32 437 -> 400 us
// by 32, with heads of 64 2600 -> 2820; heads of 128 have registers for 32.)
// How many wavefronts share a SIMD: four with heads of 32, three with heads of 64 in 16 bits, and some of v's fragments in LDS for it (`kept`), where
// registers alone left three and two: float32 512 windows of 64 cells, 4 heads of 16, 42 -> 30 us, 8 of 4096, heads of 32, 1330 -> 1220 (16 384 causal
// rows 2650 -> 2840: all blocks start at once, the long with the short); bfloat16 windows of 1024, 4 heads of 32, 72 -> 62; heads of 64, 16 384 causal rows
// 786 -> 752, 61 sequences of f16 154 -> 140 (with `fit` 161).
template <class T, int DP, bool direct, bool far>
__global__ __launch_bounds__(kAttendThreads, DP == 32 ? (direct ? (far ? 3 : 4) : 2) : sizeof(T) == 4 ? 1 : DP == 64 ? (direct ? 3 : 2) : direct ? 2 : 1)
void attend_key_grad_kernel(AttendArgs<T> p) {
    using F = Frag<T>;
    using Eight = typename F::Eight;
    constexpr int DB = DP / 32, keys = 128, rows = (sizeof(T) == 4 && DP == 32) || DP == 128 ? 32 : 64, tile = rows * DP, RB = rows / 32;
    __shared__ __attribute__((aligned(16))) T tiles[4 * tile];
    __shared__ int found[2];   // the tile of a stage that holds infinite numbers or NaN, or none
    __shared__ __attribute__((aligned(16))) float shared[2][2][rows];   // lse and -delta of a tile's rows
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave), h = half_of();
    const Place place = place_of_block(p);
    if (place.tile < 0) return;
    const int j0 = place.tile * keys, mine = j0 + wave * 32, key = min(mine + (int)threadIdx.x % 32, p.keys - 1);

    Span see;
    Spans block;
    const Spans spans = spans_of(p.seq, false, mine, p.keys, j0, keys, p.group, see, block);
    const Part share = part_of(p, block, rows, place);
    if (place.split >= share.used) return;
    if (p.splits > 1 && place.split == 0 && threadIdx.x == 0) p.used[place.head * p.tiles + place.tile] = share.used;
    const Span part = share.span;
    clip(see, part);

    // (Fragments of v that stay in registers; the others stay in LDS.  Heads of 128: registers that were missing lay in memory, and to load them again was to
    // wait for the next tile too: 1460 -> 1380 us for 16 384 causal rows, 8 heads, by that alone; 1228 with all that came since.)
    constexpr int kept = DP == 32 ? 1 : sizeof(T) == 4 ? DP / 16 : DP == 64 ? (kOwnScale<T> ? 0 : 1) : kOwnScale<T> ? 2 : 4;
    // (float16: `fit` needs some as well, and has them by 32 rows at a time and more of v in LDS)
    constexpr bool one_by_one = kOwnScale<T> && DP <= 64;
    __shared__ Eight rest[kept < DP / 16 ? DP / 16 - kept : 1][kept < DP / 16 ? kAttendThreads : 1];
    Eight k[DP / 16], v[DP / 16];
    load_row<T, DP, direct>(p.k + (int64_t)key * p.k_stride + place.head * p.k_head, p.dim, k);
    load_row<T, DP, direct>(p.v + (int64_t)key * p.v_stride + place.head * p.v_head, p.dim, v);
#pragma unroll
    for (int t = kept; t < DP / 16; ++t) rest[t - kept][threadIdx.x] = v[t];
    const float to2 = p.scale * kLog2E;
    const float* const lse = p.lse + (int64_t)place.head * p.rows;
    const float* const delta = p.delta + (int64_t)place.head * p.rows;
    f32x16 dk[DB], dv[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) dk[db] = dv[db] = f32x16{};
    Loader<T, DP, rows, direct> qs(p.q + (int64_t)place.head * p.group * p.q_head, p.q_stride, p.q_head, p.group, p.dim),
        gs(p.grad + (int64_t)place.head * p.group * p.grad_head, p.grad_stride, p.grad_head, p.group, p.dim);
    float stat = 0.0f, up = kOwnScale<T> ? kMostUp * kLowered<T> : 1.0f;
    const auto load = [&](int i0, int stage) {
        if ((int)threadIdx.x < 2 * rows) {
            const int at = min(i0 + (int)threadIdx.x % rows, part.high - 1);
            stat = (int)threadIdx.x < rows ? lse[at] - (float)kRaised<T> : -delta[at];
        }
        qs.load(i0, part.high - i0, tiles + stage * 2 * tile);
        gs.load(i0, part.high - i0, tiles + (stage * 2 + 1) * tile);
    };
    const auto finish = [&](int stage, int i0) {
        qs.finish(tiles + stage * 2 * tile);
        gs.finish(tiles + (stage * 2 + 1) * tile);
        // (where q or the gradient of a row is not finite, one of these is not, or the row sees no key)
        if ((int)threadIdx.x < 2 * rows) {
            shared[stage][threadIdx.x / rows][threadIdx.x % rows] = stat;
            if (!(__builtin_fabsf(stat) < kNoSum)) found[stage] = i0;
        }
        __syncthreads();
    };
    if (part.low < part.high) {
        load(part.low, 0);
        finish(0, part.low);
    }
    // vmcnt(0).  What stays in registers has arrived; the compiler, which does not see the tiles' loads, would else wait for it where it is first
    // used in the loop, and for the next tile with it.
    __builtin_amdgcn_s_waitcnt(0x0f70);
    int stage = 0;
    for (int i0 = part.low; i0 < part.high; i0 += rows) {
        const bool more = i0 + rows < part.high;
        if (more) load(i0 + rows, stage ^ 1);
        const T* const qt = tiles + stage * 2 * tile;
        const T* const gt = qt + tile;
        if (block.masks(i0, rows) && found[stage] == i0) {
            // (keys that see a row that is not finite have no gradient that is)
            take_out_odd<T, DP, 2 * rows>(tiles + stage * 2 * tile, [&](int row, int, float) { shared[stage][0][row % rows] = __builtin_nanf(""); });
        }
        if (i0 < spans.high && i0 + rows > spans.low) {
#pragma unroll one_by_one ? 1 : RB
            for (int b = 0; b < RB; ++b) {
                // (heads of 128: one product's fragments at a time, as the sums and the fragments that stay take most of the registers)
                f32x16 s = {}, dp;
#pragma unroll
                for (int t = 0; t < DP / 16; ++t) {
                    if (sizeof(T) == 4 && 16 * t >= p.dim) break;
                    s = F::mma(Tile<T, DP>::along(qt, 32 * b, t), k[t], s);
                }
                if constexpr (DP == 128 || one_by_one) __builtin_amdgcn_sched_barrier(0);
                float e[16], ds[16];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4 from = *reinterpret_cast<const f32x4*>(&shared[stage][0][32 * b + 8 * i + 4 * h]);
                    const f32x4 less = *reinterpret_cast<const f32x4*>(&shared[stage][1][32 * b + 8 * i + 4 * h]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        e[4 * i + j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * i + j], to2, -from[j]));
                        dp[4 * i + j] = less[j];
                    }
                }
                const bool below = i0 < spans.all_low, beyond = i0 + rows > min(spans.all_high, part.high);
                const int low = from_place(see.low, i0 + 32 * b + 4 * h), high = from_place(see.high, i0 + 32 * b + 4 * h);
                if (below) hide_below(e, low, 0.0f);
                if (beyond) hide_from(e, high, 0.0f);
#pragma unroll
                for (int t = 0; t < DP / 16; ++t) {
                    if (sizeof(T) == 4 && 16 * t >= p.dim) break;
                    dp = F::mma(Tile<T, DP>::along(gt, 32 * b, t), t < kept ? v[t] : rest[t < kept ? 0 : t - kept][one_by_one ? thread_again() : (int)threadIdx.x], dp);
                }
                if constexpr (DP == 128 || one_by_one) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int r = 0; r < 16; ++r) ds[r] = kOwnScale<T> ? e[r] * dp[r] * up : e[r] * dp[r];
                if (below) hide_below(ds, low, 0.0f);
                if (beyond) hide_from(ds, high, 0.0f);
                if constexpr (kOwnScale<T>) (void)fit(ds, up, dk);
                if constexpr (far) {
                    const Eight pe[1][2] = {{F::pack(e), F::pack(e + 8)}}, pd[1][2] = {{F::pack(ds), F::pack(ds + 8)}};
                    accumulate_apart<DP>(dv, gt, 32 * b, pe);
                    if constexpr (DP == 32) __builtin_amdgcn_sched_barrier(0);
                    accumulate_apart<DP>(dk, qt, 32 * b, pd);
                } else {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int at = 32 * b + 16 * c;
                        const Eight pe = F::pack(e + 8 * c), pd = F::pack(ds + 8 * c);
                        accumulate<T, DP>(dv, gt, at, pe);
                        accumulate<T, DP>(dk, qt, at, pd);
                    }
                }
            }
        }
        stage ^= 1;
        if (more) finish(stage, i0 + rows);
    }
    const int thread = thread_again(), half = thread / 32 % 2, j = mine + thread % 32;
    if (j >= p.keys) return;
    if (share.used > 1) {
        float* const at = p.part + (((int64_t)place.head * p.splits + place.split) * p.keys + j) * DP;
        store_row<float, DB>(at, DP, dk, kLowered<T> / up, half);
        store_row<float, DB>(at + (int64_t)p.kv_heads * p.splits * p.keys * DP, DP, dv, kLowered<T>, half);
    } else {
        const int64_t at = ((int64_t)j * p.kv_heads + place.head) * p.dim;
        if (p.dk) store_row<T, DB>(p.dk + at, p.dim, dk, p.scale * kLowered<T> / up, half);
        if (p.dv) store_row<T, DB>(p.dv + at, p.dim, dv, kLowered<T>, half);
    }
}

// The splits' sums of a gradient, where there are several: [kv head][split][row][DP] to (tokens, kv heads, group, dim)
template <class T, int DP>
__global__ __launch_bounds__(kAttendThreads) void attend_sum_kernel(AttendArgs<T> p, const float* part, int64_t rows, int tile, int group, float factor, T* to) {
    constexpr int lanes = DP / 4;
    const int lane = (int)threadIdx.x % lanes;
    const int64_t all = rows * p.kv_heads, step = (int64_t)gridDim.x * (kAttendThreads / lanes);
    for (int64_t i = (int64_t)blockIdx.x * (kAttendThreads / lanes) + threadIdx.x / lanes; i < all; i += step) {
        const int64_t head = i / rows, r = i - head * rows, token = r / group;
        const int used = p.used[head * p.tiles + r / tile];
        if (used == 1) continue;
        f32x4 sum = {};
        for (int s = 0; s < used; ++s) sum += *reinterpret_cast<const f32x4*>(part + ((head * p.splits + s) * rows + r) * DP + 4 * lane);
        T* const at = to + ((token * p.kv_heads + head) * group + (r - token * group)) * p.dim;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (4 * lane + j < p.dim) at[4 * lane + j] = (T)(sum[j] * factor);
    }
}

}  // namespace svox_network
