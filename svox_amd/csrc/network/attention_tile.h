// attention_tile.h -- what the attention kernels are made of: products of 32 x 32 on the matrix cores, tiles of rows in LDS and the two
// ways to read them, and which keys a query sees.
//
// All kernels compute scores the way round that leaves a lane with one query (or one key: backward, for keys and values) and 16 of the
// others, in the order in which the matrix cores hand results out: number r of a lane is row (r mod 4) + 8 (r / 4) + 4 half, half = lane / 32.
// As the order of a reduction is free as long as both operands have the same, those 16 numbers go into the next product as they lie in
// the registers, eight to a fragment, and only the other operand is read in that order: no score passes through LDS.
#pragma once
#include "../decoder/tile.h"

namespace svox_network {

using namespace svox_decoder;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s16x4 LdsFour;

constexpr int kAttendThreads = 256;

// A fragment is 16 of the reduction, eight of them in each half of a wavefront.  float32 goes through the matrix cores as it is, two of the
// reduction at a time.
template <class T>
struct Frag {
    typedef u16x8 Eight;
    typedef typename Few<T, 8>::vector Numbers;
    static __device__ __forceinline__ f32x16 mma(Eight a, Eight b, f32x16 c) {
        if constexpr (std::is_same_v<T, Bf16>)
            return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ Eight pack(const float* v) {
        return __builtin_bit_cast(Eight, __builtin_convertvector((f32x8){v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]}, Numbers));
    }
};
template <>
struct Frag<float> {
    typedef f32x8 Eight;
    typedef f32x8 Numbers;
    static __device__ __forceinline__ f32x16 mma(Eight a, Eight b, f32x16 c) {
#pragma unroll
        for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ Eight pack(const float* v) { return (Eight){v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]}; }
};

// the sum of the products of two fragments' numbers
template <class T>
__device__ __forceinline__ float dot(typename Frag<T>::Eight a, typename Frag<T>::Eight b) {
    const auto x = __builtin_bit_cast(typename Frag<T>::Numbers, a), y = __builtin_bit_cast(typename Frag<T>::Numbers, b);
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = __builtin_fmaf((float)x[e], (float)y[e], sum);
    return sum;
}

// row of a result's number r, and of a fragment's number e that holds results
__device__ __forceinline__ constexpr int row_of(int r) { return (r & 3) + 8 * (r >> 2); }

__device__ __forceinline__ int half_of() { return (int)threadIdx.x / 32 % 2; }

// A tile of rows of DP numbers in LDS.  The 16-byte pieces of a row lie in an order that depends on the row, so that lanes that read a piece of
// different rows, and those that read four rows across, find them in different banks.  Rows of 256 bytes fill the banks: sixteen pieces change places, for
// sixteen rows, and reads take half as long as with eight (16 384 causal rows of bfloat16, 8 heads, by that alone: forward 586 -> 576 us, dq 864 -> 848, dk and dv,
// which wait for one product after another, as before; with all that came since, under the profiler, 531, 776 and 1228).  Narrower rows and float32's: eight, as what sixteen save in LDS they cost in registers (heads
// of 64: dk and dv 84 -> 86 us).
template <class T, int DP>
struct Tile {
    static constexpr int V = 16 / (int)sizeof(T), pieces = DP / V;   // numbers of a piece, pieces of a row
    static constexpr bool sixteen = sizeof(T) == 2 && DP == 128;
    static constexpr int most = sixteen ? 16 : 8, ring = pieces < most ? pieces : most;   // pieces that change places
    static __device__ __forceinline__ int turn(int row) {
        if constexpr (sixteen) return (row & 3) << 2 | (row >> 1 & 2) | (row >> 3 & 1);   // (eight rows on, the lowest bit is another)
        else if constexpr (pieces == 4) return (row & 2) | (row >> 2 & 1);
        else return (row & 3) << 1 | (row >> 2 & 1);
    }
    // (what is the same for all lanes stands by itself: it goes into the instructions' own offsets)
    static __device__ __forceinline__ int at(int row, int piece) { return row * DP + piece / ring * ring * V + ((piece % ring) ^ turn(row)) * V; }

    // numbers 16 t + 8 half .. of row r0 + lane % 32; r0 a whole number of 16
    static __device__ __forceinline__ typename Frag<T>::Eight along(const T* lds, int r0, int t) {
        const int row = (int)threadIdx.x % 32, h = half_of(), turned = turn(row);
        const T* const from = lds + row * DP;
        if constexpr (sizeof(T) == 2) {
            return *reinterpret_cast<const u16x8*>(from + r0 * DP + 2 * t / ring * ring * V + ((2 * t % ring) ^ (h ^ turned)) * V);
        } else {
            const int even = 4 * t % ring, beyond = r0 * DP + 4 * t / ring * ring * V;
            const f32x4 a = *reinterpret_cast<const f32x4*>(from + beyond + (even ^ (2 * h ^ turned)) * V);
            const f32x4 b = *reinterpret_cast<const f32x4*>(from + beyond + ((even + 1) ^ (2 * h ^ turned)) * V);
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
    // number 32 db + lane % 32 of rows r0 + row_of(0 .. 7) + 4 half; r0 a whole number of 16
    static __device__ __forceinline__ typename Frag<T>::Eight across(const T* lds, int r0, int db) {
        const int lane = (int)threadIdx.x % kWave, h = half_of();
        if constexpr (sizeof(T) == 2) {
            const int l = lane & 15, row = 4 * h + (l >> 2), piece = (lane >> 3 & 2) + (l >> 1 & 1);   // of the first 32 columns
            const T* const from = lds + row * DP + (l & 1) * 4;
            const int turned = piece ^ turn(row);
            u16x8 both;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const s16x4 four = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsFour*)(from + (r0 + 8 * half) * DP + 4 * db / ring * ring * V + ((4 * db % ring ^ (sixteen ? half : 0)) ^ turned) * V));
#pragma unroll
                for (int i = 0; i < 4; ++i) both[half * 4 + i] = (u16)four[i];
            }
            return both;
        } else {
            const int c = lane % 32;
            typename Frag<T>::Eight v;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int row = row_of(e) + 4 * h;   // (the eight pieces of a row's 32 columns)
                v[e] = lds[(r0 + row) * DP + 32 * db + ((c / 4) ^ turn(row)) * 4 + c % 4];
            }
            return v;
        }
    }
};

// `rows` rows of heads in memory on their way to a tile.  Row r of the tile is row `first` + r of what `group` heads of a token make up, the
// token's rows side by side.  Rows from `left` on and numbers from `dim` on arrive as zeros.
//
// `direct`: from memory to LDS without a register, 16 bytes a lane, whose places follow one another there, so that it is the lane that takes
// another piece of memory where pieces change places.  Everything lies at whole numbers of 16 bytes then.
template <class T, int DP, int rows, bool direct>
struct Loader;

template <class T, int DP, int rows>
struct Loader<T, DP, rows, true> {
    using Shape = Tile<T, DP>;
    static constexpr int V = Shape::V, each = rows * Shape::pieces / kAttendThreads;
    static_assert(rows * Shape::pieces % kAttendThreads == 0, "as many pieces for every thread");
    static constexpr unsigned range = 0x80000000u, outside = 0x80000000u;   // bytes: beyond the range the hardware delivers zeros
    unsigned at[each];
    const T* base;
    int64_t stride, head_stride;
    int group, dim;

    __device__ __forceinline__ Loader(const T* x, int64_t stride_, int64_t head_stride_, int group_, int dim_)
        : base(x), stride(stride_), head_stride(head_stride_), group(group_), dim(dim_) {
        places(0);
    }
    __device__ __forceinline__ int row_of_load(int i) const { return (i * kAttendThreads + (int)threadIdx.x) / Shape::pieces; }
    __device__ __forceinline__ void places(int first) {
        const int begin = first % group;   // (0 but where a tile begins within a token)
#pragma unroll
        for (int i = 0; i < each; ++i) {
            const int row = row_of_load(i), slot = (i * kAttendThreads + (int)threadIdx.x) % Shape::pieces;
            const int column = (slot / Shape::ring * Shape::ring + ((slot % Shape::ring) ^ Shape::turn(row))) * V;
            const int token = group == 1 ? row : (begin + row) / group, head = group == 1 ? 0 : (begin + row) % group;
            at[i] = column < dim ? (unsigned)((token * stride + head * head_stride + column) * (int)sizeof(T)) : outside;
        }
    }
    __device__ __forceinline__ void load(int first, int left, T* lds) {
        if (rows % group != 0) places(first);
        const uint64_t from = (uint64_t)(base + first / group * stride);
        const u32x4 buffer = {(unsigned)from, (unsigned)(from >> 32) & 0xffffu, range, 0x00020000u};
        const int wave_first = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave * kWave);
#pragma unroll
        for (int i = 0; i < each; ++i)
            load_to_lds(buffer, left >= rows || row_of_load(i) < left ? at[i] : outside, reinterpret_cast<u16*>(lds + (i * kAttendThreads + wave_first) * V));
    }
    // before the barrier behind which a tile is read
    __device__ __forceinline__ void finish(T*) const { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
};

// Through registers: any alignment of the type's own.  The next tile's loads are in flight while this one is multiplied.
template <class T, int DP, int rows>
struct Loader<T, DP, rows, false> {
    using Shape = Tile<T, DP>;
    static constexpr int V = Shape::V, each = rows * Shape::pieces / kAttendThreads;
    typename Few<T, V>::vector v[each];
    const T* base;
    int64_t stride, head_stride;
    int group, dim;

    __device__ __forceinline__ Loader(const T* x, int64_t stride_, int64_t head_stride_, int group_, int dim_)
        : base(x), stride(stride_), head_stride(head_stride_), group(group_), dim(dim_) {}
    __device__ __forceinline__ void load(int first, int left, T*) {
#pragma unroll
        for (int i = 0; i < each; ++i) {
            const int piece = i * kAttendThreads + (int)threadIdx.x, row = piece / Shape::pieces, column = piece % Shape::pieces * V;
            const unsigned r = (unsigned)(first + row), token = r / (unsigned)group;
            v[i] = load_some<T, V>(base + token * stride + (r - token * group) * head_stride + column, row < left ? dim - column : 0);
        }
    }
    __device__ __forceinline__ void finish(T* lds) const {
#pragma unroll
        for (int i = 0; i < each; ++i) {
            const int piece = i * kAttendThreads + (int)threadIdx.x;
            *reinterpret_cast<typename Few<T, V>::vector*>(lds + Shape::at(piece / Shape::pieces, piece % Shape::pieces)) = v[i];
        }
    }
};

// Infinite numbers and NaN in a tile of which not every row is seen by every lane.  A score that is masked is 0, and 0 times what its row
// holds is 0, unless that is one of these: they are taken out of the tile, and those who do see them are told otherwise.
//
// Whether the pieces of a tile that this wavefront's threads have loaded hold any; before the barrier behind which the tile is read.
template <class T, int DP, int rows>
__device__ __forceinline__ bool holds_odd(const T* lds) {
    typedef unsigned Words __attribute__((ext_vector_type(4)));
    // (an exponent of ones becomes a carry into the sign's place)
    constexpr unsigned low = sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu, one = sizeof(T) == 4 ? 0x00800000u : std::is_same_v<T, Bf16> ? 0x00800080u : 0x04000400u;
    unsigned found = 0;
#pragma unroll
    for (int i = 0; i < rows * Tile<T, DP>::pieces / kAttendThreads; ++i) {
        const int place = i * kAttendThreads + (int)threadIdx.x;
        const Words w = (*reinterpret_cast<const Words*>(lds + Tile<T, DP>::at(place / Tile<T, DP>::pieces, place % Tile<T, DP>::pieces)) & low) + one;
        found |= w[0] | w[1] | w[2] | w[3];
    }
    return __any((found & ~low) != 0);
}

// threadIdx.x, and a number that is the same for all, from which what is needed behind a loop, or seldom within, is found once more: the
// compiler would else keep it in registers throughout.
__device__ __forceinline__ int thread_again() {
    int t = (int)threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
}
__device__ __forceinline__ unsigned again(unsigned v) {
    asm volatile("" : "+s"(v));
    return v;
}

// Takes them out, all threads together; f(row, column, number) for each, by one thread.  The tile can be read when this returns.
template <class T, int DP, int rows, class F>
__device__ __forceinline__ void take_out_odd(T* lds, F f) {
    __syncthreads();
#pragma unroll 1
    for (int i = thread_again(); i < rows * DP; i += kAttendThreads) {
        const int row = i / DP, column = i % DP;
        T* const at = lds + Tile<T, DP>::at(row, column / Tile<T, DP>::V) + column % Tile<T, DP>::V;
        const float v = (float)*at;
        if (__builtin_fabsf(v) < __builtin_inff()) continue;
        f(row, column, v);
        *at = (T)0.0f;
    }
    __syncthreads();
}

// Fragments of a row in memory, as an operand that stays in registers: numbers 16 t + 8 half .. of `row`, zeros from `dim` on.
template <class T, int DP, bool direct>
__device__ __forceinline__ void load_row(const T* row, int dim, typename Frag<T>::Eight (&out)[DP / 16]) {
    constexpr int V = 16 / (int)sizeof(T);
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) {
        const int at = 16 * t + 8 * half_of();
        typename Few<T, 8>::vector v = {};
        if constexpr (direct) {     // (pieces are there as a whole or not at all)
            if (V == 8 ? at < dim : at + V < dim) v = load_few<T, 8>(row + at);
            else if (V < 8 && at < dim)
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] = row[at + i];
        } else {
            v = load_some<T, 8>(row + at, dim - at);
        }
        out[t] = __builtin_bit_cast(typename Frag<T>::Eight, v);
    }
}

// ---- packed sequences
// Where they begin and end, n + 1 places, as they come from the caller's memory: whatever stands there is brought within 0 .. total.
struct Offsets {
    const void* at;   // or NULL: one sequence, 0 .. total
    int wide, n;
    int total;
    float each;       // sequences to a token, in the mean
    __device__ __forceinline__ int operator()(int i) const {
        if (!at) return i == 0 ? 0 : total;
        const int64_t v = wide ? ((const int64_t*)at)[i] : (int64_t)((const int32_t*)at)[i];
        return v < 0 ? 0 : v > total ? total : (int)v;
    }
};
// The last i with offsets(i) <= t, or 0: by the whole wavefront, 64 places at a time.  (At most n whatever the places hold.)
__device__ __forceinline__ int last_not_beyond(const Offsets& o, int t) {
    if (!o.at) return 0;
    const int lane = (int)threadIdx.x % kWave;
    int low = 0, size = o.n + 1;
    while (true) {
        const int step = (size + kWave - 1) / kWave, at = lane * step;
        const int found = __popcll(__ballot(at < size && o(low + at) <= t));
        if (found == 0) return low;
        low += (found - 1) * step;
        if (step == 1) return low;
        size = min(step, size - (found - 1) * step);
    }
}

struct Span {
    int low, high;   // none: low == high
};
struct Sequences {
    Offsets q, k;
    int causal;
};
// What every lane's token `t` sees of the other axis; `keys`: t is a query, else a key.  A lane's tokens are none before `first` and none beyond
// `last`.  Where sequences are in order, spans do not go back from token to token, also those that are empty.
__device__ __forceinline__ Span span_of(const Sequences& s, bool keys, int t, int first, int last) {
    const Offsets &mine = keys ? s.q : s.k, &other = keys ? s.k : s.q;
    const int lane = (int)threadIdx.x % kWave;
    // 64 places, one a lane, about where sequences of one length would have the first token's, or all of them: it is among them as a rule, and nothing
    // has to be looked for first
    const int guess = (int)((float)first * mine.each) - kWave / 2;
    int a = max(0, min(guess, mine.n + 1 - kWave));
    int place = min(a + lane, mine.n), mine_at = mine(place), other_at = other(place);
    int found = __popcll(__ballot(mine_at <= first)) - 1;
    if (found < 0 ? a > 0 : (found == kWave - 1 && a + found < mine.n) || (__builtin_amdgcn_readlane(mine_at, kWave - 1) <= last && a + kWave - 1 < mine.n)) {
        a = last_not_beyond(mine, first);
        place = min(a + lane, mine.n), mine_at = mine(place), other_at = other(place);
        found = 0;
    }
    found = max(found, 0);
    int m0, m1, o0, o1;
    const int next = min(found + 1, kWave - 1);
    if (__builtin_amdgcn_readlane(mine_at, next) > last) {
        m0 = __builtin_amdgcn_readlane(mine_at, found), m1 = __builtin_amdgcn_readlane(mine_at, next);
        o0 = __builtin_amdgcn_readlane(other_at, found), o1 = __builtin_amdgcn_readlane(other_at, next);
    } else if (a + kWave - 1 >= mine.n || __builtin_amdgcn_readlane(mine_at, kWave - 1) > last) {
        int i = 0;
#pragma unroll
        for (int d = kWave / 2; d > 0; d /= 2) {
            const int there = __shfl(mine_at, i + d, kWave);   // (by all lanes)
            if (i + d < kWave - 1 && there <= t) i += d;
        }
        m0 = __shfl(mine_at, i, kWave), m1 = __shfl(mine_at, i + 1, kWave);
        o0 = __shfl(other_at, i, kWave), o1 = __shfl(other_at, i + 1, kWave);
    } else {
        int low = a, high = mine.n;
        while (low < high) {
            const int middle = low + (high - low + 1) / 2;      // (there may be more than 2^30 sequences)
            if (mine(middle) <= t) low = middle;
            else high = middle - 1;
        }
        const int after = min(low + 1, mine.n);
        m0 = mine(low), m1 = mine(after), o0 = other(low), o1 = other(after);
    }
    o1 = max(o0, o1);
    if (t < m0) return {o0, o0};
    if (t >= m1) return {o1, o1};
    if (!s.causal) return {o0, o1};
    const int ends = (o1 - o0) - (m1 - m0);   // (the places are counted from the sequences' ends)
    if (keys) {
        const int64_t seen = (int64_t)(t - m0) + ends + 1;
        return {o0, o0 + (int)(seen < 0 ? 0 : seen > o1 - o0 ? o1 - o0 : seen)};
    }
    const int64_t hidden = (int64_t)(t - m0) + ends;   // (mine are keys: ends is of queries less keys)
    return {o0 + (int)(hidden < 0 ? 0 : hidden > o1 - o0 ? o1 - o0 : hidden), o1};
}

// What a wavefront's lanes, or a block's, see: the span of all, and the one that every lane sees whole.
struct Spans {
    int low, high;            // of all; none: low >= high
    int all_low, all_high;
    // whether some lane does not see all of the `n` from `first` on
    __device__ __forceinline__ bool masks(int first, int n) const { return first < all_low || first + n > all_high; }
};

// acc += across rows r0 .. r0 + 15 of a tile times `b`
template <class T, int DP>
__device__ __forceinline__ void accumulate(f32x16 (&acc)[DP / 32], const T* lds, int r0, typename Frag<T>::Eight b) {
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) acc[db] = Frag<T>::mma(Tile<T, DP>::across(lds, r0, db), b, acc[db]);
}

// The same of 32 KB rows from r0 on for float32, whose sums have no fewer bits than the result: these products are added up by themselves and then to acc, so
// that a sum over very many rows is not one addition after another.
template <int DP, int KB>
__device__ __forceinline__ void accumulate_apart(f32x16 (&acc)[DP / 32], const float* lds, int r0, const Frag<float>::Eight (&e)[KB][2]) {
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) {
        f32x16 sum = {};
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int c = 0; c < 2; ++c) sum = Frag<float>::mma(Tile<float, DP>::across(lds, r0 + 32 * b + 16 * c, db), e[b][c], sum);
        acc[db] += sum;
    }
}

// the sum, and the larger, of a lane's number and that of the lane 32 away
__device__ __forceinline__ float sum_of_halves(float v) {
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(both[0]) + __uint_as_float(both[1]);
}
__device__ __forceinline__ float most_of_halves(float v) {
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
}

// A row of a result, a lane's 16 numbers of every 32: to memory as `V`, times `factor`.
template <class V, int DB>
__device__ __forceinline__ void store_row(V* row, int dim, const f32x16 (&acc)[DB], float factor, int half) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = db * 32 + 8 * i + 4 * half;
            const f32x4 v = {acc[db][4 * i] * factor, acc[db][4 * i + 1] * factor, acc[db][4 * i + 2] * factor, acc[db][4 * i + 3] * factor};
            if (at + 4 <= dim) {
                store_few<V, 4>(row + at, __builtin_convertvector(v, typename Few<V, 4>::vector));
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (at + j < dim) row[at + j] = (V)v[j];
            }
        }
}

}  // namespace svox_network
