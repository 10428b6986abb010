// tile.h -- products of matrices on the matrix cores: operands in memory, their tiles in LDS, the fragments read from there.
//
// An operand is a matrix of 16-bit numbers (Planes: one, or three for float32) whose row length is a whole number of 8.  It
// is used along its rows (the reduction runs along a row: `along`) or across them (the reduction runs down a column).  Its
// tiles go to LDS by global_load_lds, 16 bytes a lane, without passing through registers; what lies outside the matrix is
// read from 16 bytes of zeros, so that no edge needs a branch later.
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

static __device__ __align__(16) const u16 kZeros[8] = {0, 0, 0, 0, 0, 0, 0, 0};

typedef __attribute__((address_space(3))) void Lds;
typedef const __attribute__((address_space(1))) void Global;

__device__ __forceinline__ void to_lds(const u16* from, u16* lds) {
    __builtin_amdgcn_global_load_lds((Global*)from, (Lds*)lds, 16, 0, 0);
}

// One plane's tile of an operand: R rows (along) or columns (across) of the result, KT of the reduction.
template <bool along, int R, int KT, int threads>
struct TileOf {
    static constexpr int numbers = R * KT;
    static constexpr int loads = numbers / 8 / threads;
    static_assert(numbers % (8 * threads) == 0, "whole rounds of 16 bytes a lane");

    static __device__ __forceinline__ int turn_along(int row) { return KT == 64 ? (row & 7) : ((row >> 1) & 3); }
    static __device__ __forceinline__ int turn_across(int k) { return ((k & 3) | ((k >> 1) & 4)) & (R / 16 - 1); }

    // the tile at row (column) r0 and reduction index k0 of `m`, up to k_end
    static __device__ __forceinline__ void load(const Planes& m, const u16* plane, int64_t r0, int64_t k0, int64_t k_end, u16* lds) {
        const int t = threadIdx.x, wave = t / kWave;
#pragma unroll
        for (int i = 0; i < loads; ++i) {
            const int piece = i * threads + t;
            const u16* from;
            bool there;
            if constexpr (along) {
                const int row = piece / (KT / 8), slot = piece % (KT / 8);
                const int64_t k = k0 + ((slot ^ turn_along(row)) * 8), r = r0 + row;
                there = r < m.rows && k < k_end;
                from = plane + r * m.ld + k;
            } else {
                const int row = piece / (R / 8), slot = piece % (R / 8);
                const int64_t k = k0 + row, c = r0 + (((slot >> 1) ^ turn_across(row)) * 2 + (slot & 1)) * 8;
                there = k < k_end && k < m.rows && c < m.cols;
                from = plane + k * m.ld + c;
            }
            to_lds(there ? from : kZeros, lds + (size_t)(i * threads + wave * kWave) * 8);
        }
    }

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

// Which tile of `tiles_m` x `tiles_n` a block works on.  Blocks go round the eight XCDs, each with an L2 of its own: every XCD
// gets a run of neighbouring tiles, and a run goes through 8 tiles down before the next to the right, so that what its blocks
// read at a time is a few rows of tiles and a few columns.
__device__ __forceinline__ void tile_of_block(int64_t block, int64_t blocks, int64_t tiles_m, int64_t tiles_n, int64_t& m, int64_t& n) {
    const int64_t xcd = block % 8, each = blocks / 8, left = blocks % 8;
    const int64_t t = xcd * each + (xcd < left ? xcd : left) + block / 8;
    constexpr int64_t down = 8;
    const int64_t group = t / (down * tiles_n), first = group * down;
    const int64_t high = tiles_m - first < down ? tiles_m - first : down;
    const int64_t within = t - group * down * tiles_n;
    m = first + within % high;
    n = within / high;
}

}  // namespace svox_decoder
