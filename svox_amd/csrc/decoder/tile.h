// tile.h -- products of matrices on the matrix cores: operands in memory, their tiles in LDS, the fragments read from there.
//
// An operand is a matrix of 16-bit numbers (Planes: one, or three for float32) whose row length is a whole number of 8.  It
// is used along its rows (the reduction runs along a row: `along`) or across them (the reduction runs down a column).  Its
// tiles go to LDS by buffer loads, 16 bytes a lane, without passing through registers; what lies outside the matrix arrives as
// zeros, so that no edge needs a branch later.
//
// LDS holds a tile as it lies in memory, but for an order of the 16-byte pieces that depends on the row, chosen so that the
// eight lanes a clock serves fall on different banks:
//   along:  [rows][KT] numbers; piece i of row r lies at i ^ (r mod 8) (KT = 64), at i ^ (r/2 mod 4) (KT = 32).
//           A lane reads its 8 numbers of a row by one ds_read_b128.
//   across: [KT][columns]; pieces of 16 numbers, piece i of row k lies at i ^ (k mod 4 + 4 (k/8 mod 2)).
//           ds_read_b64_tr_b16 turns 4 rows x 16 columns around on their way out: lane l of 16 gets column l.
#pragma once
#include "common.h"

namespace svox_decoder {

struct Planes {
    const u16* at;
    int64_t ld;      // numbers from row to row: a whole number of 8
    int64_t plane;   // numbers from plane to plane
    int64_t rows;
    int64_t cols;    // readable numbers of a row: a whole number of 8, zeros beyond the matrix
};

typedef __attribute__((address_space(3))) void Lds;
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// 16 bytes of every lane to LDS, where a wavefront's lie one lane's after another.  Written out because the compiler, where it knows of
// such a load, lets every transposing read of LDS wait for all of them, the next tiles' too (a step of 16 384 rows of 1024 -> 4096 ->
// 1024 in bfloat16: 1845 us so, 2011 from the builtin).  No register is loaded.  Who reads waits for vmcnt and a barrier first.
// (The address of the buffer may come from a vector instruction just before: five wait states.  Where the compiler cannot tell that it
// is the same for all lanes the build fails; to make it so by readfirstlane costs the weights' kernel registers it does not have.)
__device__ __forceinline__ void load_to_lds(u32x4 buffer, unsigned at, u16* lds) {
    const unsigned to = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(Lds*)lds);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(at), "s"(buffer) : "m0", "memory");
}

// One plane's tile of an operand: R rows (along) or columns (across) of the result, KT of the reduction.
//
// A lane's pieces lie at offsets from the tile's first number that do not change from tile to tile of the reduction: the loads
// take them from registers, and the address that moves is scalar.  What lies outside the matrix gets an offset beyond the
// buffer's range, for which the hardware delivers zeros.
template <bool along, int R, int KT, int threads>
struct TileOf {
    static constexpr int numbers = R * KT;
    static constexpr int pieces = numbers / 8;                                   // of 16 bytes, one a lane and load
    static constexpr int loads = pieces < threads ? 1 : pieces / threads;
    static_assert(pieces < threads ? threads % pieces == 0 : pieces % threads == 0, "every wavefront has as many loads");
    static constexpr unsigned range = 0x80000000u, outside = 0x80000000u;   // bytes
    static constexpr int64_t most_ld = (int64_t)1 << 22;                    // 256 rows of it stay within the range

    static __device__ __forceinline__ int turn_along(int row) { return KT == 64 ? (row & 7) : ((row >> 1) & 3); }
    static __device__ __forceinline__ int turn_across(int k) { return ((k & 3) | ((k >> 1) & 4)) & (R / 16 - 1); }

    // (where there are more lanes than pieces, several wavefronts load the same ones to the same place)
    static __device__ __forceinline__ int piece_of(int load, int thread) { return load * threads + (pieces < threads ? thread % pieces : thread); }

    const u16* next;          // plane 0's first number of the next tile to load
    int64_t step;             // numbers from tile to tile
    unsigned at[loads];

    // tiles of rows (columns) r0.. from reduction index k0 on
    __device__ __forceinline__ TileOf(const Planes& m, int64_t r0, int64_t k0) {
        next = m.at + (along ? r0 * m.ld + k0 : k0 * m.ld + r0);
        step = along ? KT : KT * m.ld;
#pragma unroll
        for (int i = 0; i < loads; ++i) {
            const int piece = piece_of(i, threadIdx.x);
            if constexpr (along) {
                const int row = piece / (KT / 8), slot = piece % (KT / 8);
                at[i] = r0 + row < m.rows ? (unsigned)((row * m.ld + (slot ^ turn_along(row)) * 8) * 2) : outside;
            } else {
                const int row = piece / (R / 8), slot = piece % (R / 8);
                const int c = (((slot >> 1) ^ turn_across(row)) * 2 + (slot & 1)) * 8;
                at[i] = r0 + c < m.cols ? (unsigned)((row * m.ld + c) * 2) : outside;
            }
        }
    }
    // before the last tile: `left` indices of the reduction are left of it
    __device__ __forceinline__ void last(int64_t left) {
        if (left >= KT) return;
#pragma unroll
        for (int i = 0; i < loads; ++i) {
            const int piece = piece_of(i, threadIdx.x);
            int k;
            if constexpr (along) {
                const int row = piece / (KT / 8), slot = piece % (KT / 8);
                k = (slot ^ turn_along(row)) * 8;
            } else {
                k = piece / (R / 8);
            }
            if (k >= left) at[i] = outside;
        }
    }
    __device__ __forceinline__ void load(int64_t plane, u16* lds) const {
        const int wave_first = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave * kWave);
        const uint64_t from = (uint64_t)(next + plane);
        const u32x4 buffer = {(unsigned)from, (unsigned)(from >> 32) & 0xffffu, range, 0x00020000u};
#pragma unroll
        for (int i = 0; i < loads; ++i) load_to_lds(buffer, at[i], lds + piece_of(i, wave_first) * 8);
    }
    __device__ __forceinline__ void advance() { next += step; }

    // the fragment of rows (columns) r..r+15 and reduction indices 32 step..32 step + 31
    static __device__ __forceinline__ u16x8 fragment(const u16* lds, int r, int step) {
        const int lane = threadIdx.x % kWave, group = lane >> 4, l = lane & 15;
        if constexpr (along) {
            const int row = r + l;
            return *reinterpret_cast<const u16x8*>(lds + row * KT + ((step * 4 + group) ^ turn_along(row)) * 8);
        } else {
            u16x8 both;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int k = step * 32 + group * 8 + half * 4 + (l >> 2);
                const u16* const from = lds + k * R + ((r / 16) ^ turn_across(k)) * 16 + (l & 3) * 4;
                const s16x4 four = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)from);
                for (int i = 0; i < 4; ++i) both[half * 4 + i] = (u16)four[i];
            }
            return both;
        }
    }
};

// Blocks go round the eight XCDs, each with an L2 of its own: block b of n as the position of its work, so that every XCD gets a run
// of neighbouring work.
__device__ __forceinline__ int64_t position_of_block(int64_t b, int64_t n) {
    const int64_t xcd = b % 8, each = n / 8, left = n % 8;
    return xcd * each + (xcd < left ? xcd : left) + b / 8;
}
// The tile of `tiles_m` x `tiles_n` at position t: `down` tiles down before the next to the right, so that what the blocks of an XCD
// read at a time is a few rows of tiles and a few columns.
__device__ __forceinline__ void tile_at(int64_t t, int64_t tiles_m, int64_t tiles_n, int64_t& m, int64_t& n) {
    constexpr int64_t down = 4;   // (a step of 16 384 rows of 1024 -> 4096 -> 1024 in bfloat16: 2 1580, 4 1556, 8 1557, 16 1591 us)
    const int64_t group = t / (down * tiles_n), first = group * down;
    const int64_t high = tiles_m - first < down ? tiles_m - first : down;
    const int64_t within = t - group * down * tiles_n;
    m = first + within % high;
    n = within / high;
}

}  // namespace svox_decoder
