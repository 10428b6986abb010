// rules.h -- which of its kernels a call of the gated feed-forward block runs on, by its sizes: host code alone, of no GPU's headers.
#pragma once
#include <cstdint>
#include <type_traits>

#include "../../../include/svox_decoder.h"

namespace svox_decoder {

constexpr int kWave = 64;
inline int64_t up_to(int64_t n, int64_t whole) { return (n + whole - 1) / whole * whole; }
inline int64_t pieces(int64_t n, int64_t size) { return (n + size - 1) / size; }

// The shape of a block's work: BM x BN numbers of the result, KT of the reduction at a time, WM x WN wavefronts, and how many
// tiles of the reduction LDS holds (one that is multiplied, the others on their way).
template <int BM_, int BN_, int KT_, int WM_, int WN_, int stages_>
struct Shape {
    static constexpr int BM = BM_, BN = BN_, KT = KT_, WM = WM_, WN = WN_, threads = WM * WN * kWave, stages = stages_;
    static constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
};

enum Size { kSmall, kDeep, kMedium, kLarge };

// the 32s of features, and of numbers of the result, that the kernels of narrow layers are made for
inline int narrow_steps(int n) { return n <= 32 ? 1 : n <= 64 ? 2 : 4; }

// planes: 1 for the 16-bit types, 3 for float32.  A call of few rows goes to few_kernels.h, else one of narrow layers to narrow_kernels.h,
// else to product_kernels.h.
template <int planes>
struct Rules {
    // ---- few rows
    // Up to 64 rows always; up to 2048 while the products stay small, where the other kernels wait more than they multiply.  (Forward
    // pass of 256 -> 1024 -> 256, bfloat16, 512 rows 18.7 us here and 19.3 on tiles, 1024 rows 24.1 and 18.9; float32, 1024 rows 44 and
    // 53, 2048 rows 68 and 56.  Gradients, 1024 rows 40 and 45, 2048 rows 70 and 60; float32, 103 and 135, 181 and 168.)
    static bool few_rows(const SvoxGatedFfn& s, bool backward) {
        const double most = planes == 1 ? (backward ? 0.9e9 : 0.4e9) : (backward ? 1.5e9 : 1.2e9);
        return s.rows <= 64 || (s.rows <= 2048 && (double)s.rows * s.hidden * (2.0 * s.dim + s.out) <= most);
    }

    // ---- narrow layers
    static constexpr int kNarrowMost = planes == 1 ? 128 : 64;   // features, and numbers of the result
    // Where rows enough fill the compute units with blocks that go through all hidden numbers; with fewer the products of whole matrices have
    // more blocks.  (Forward pass in bfloat16 of 64 -> 2048 -> 64, 4500 rows 45.7 us here and 32.6 there, 14 000 rows 46.9 and 54.5; of
    // 112 -> 1024 -> 128, 8000 rows 36.4 and 26.1, 20 000 rows 41.4 and 49.8; of 32 -> 1000 -> 28, 4500 rows 25.0 and 23.3, 14 000
    // rows 25.5 and 33.0; in float32, 4500 rows 47.9 and 54.9; of 64 -> 2048 -> 64, 4500 rows 122 and 89, 14 000 rows 124 and 168.
    // Gradients in bfloat16 of 64 -> 2048 -> 64, 3000 rows 74 and 66, 8000 rows 87 and 118; of 112 -> 1024 -> 128, 8000 rows 94 and 72,
    // 20 000 rows 150 and 131; of 32 -> 1000 -> 28, 3000 rows 37 and 47; in float32 of 64 -> 2048 -> 64, 3000 rows 235 and 178, 8000
    // rows 282 and 303.)  The rule does not ask for the hidden units, of which the rows it was measured on have 1000 and more, and is wrong
    // where the figures say so: gradients of 112 -> 1024 -> 128 from 11 520 rows to 20 000 and more.
    static bool narrow(const SvoxGatedFfn& s, bool backward) {
        const int64_t wide = (int64_t)s.dim + s.out, most = backward ? 48 * wide : planes == 1 ? 8192 : 64 * wide;
        return s.dim <= kNarrowMost && s.out <= kNarrowMost && s.rows >= most;
    }
    // 16 or 32 rows to a wavefront: 32 halve what it reads of LDS, 16 fill the GPU sooner and are all that float32's planes leave room
    // for.  (Rows of 64 -> 256 -> 64, bfloat16, forward and dx: 131 072 rows 27.5, 37.2 us with 16, 25.4, 34.5 with 32; 10 007 rows of
    // 76 -> 203 -> 49, float16: 10.8, 13.1 and 14.1, 17.2.  65 537 rows of 32 -> 128 -> 28, float32, forward: 20.7 and 22.8.)  Where
    // between the two the line is best was not measured: 98 304 rows fill the compute units three times with blocks of 128.
    static int narrow_tiles(int64_t rows) { return planes == 1 && rows >= 98304 ? 2 : 1; }

    // ---- products of whole matrices
    static constexpr int kKT = planes == 1 ? 64 : 32;
    // Medium tiles, two blocks of them to a compute unit, where there are enough; small ones with more of the reduction on its way, where
    // a block waits for memory more than it multiplies; and for 16 bits large ones, of which each block has a compute unit's LDS for
    // itself, where these fill the compute units as well: a tile of 256 x 256 takes half as many bytes from the L2 for a product as one
    // of 128 x 128 does, and two thirds as many from LDS.
    // (The step of 16 384 rows of 1024 -> 4096 -> 1024 in bfloat16 takes 1553 us with large tiles, 1799 with medium ones; its hidden
    // numbers 281 and 315, result 125 and 145, their gradients 499 and 575, x's 241 and 295, the weights' 447 and 500.  Medium tiles
    // take it 2021 us with eight wavefronts to a block, 2090 with four.  The step of 8192 rows of 256 -> 1024 -> 256 in float32, whose planes
    // make tiles three times as large, 537 us with tiles of 128 x 128 and one block to a compute unit, 500 with half as large ones and
    // two.)
    struct Medium {
        using Hidden = std::conditional_t<planes == 1, Shape<128, 64, kKT, 2, 4, 2>, Shape<64, 64, kKT, 2, 2, 2>>;
        using Output = std::conditional_t<planes == 1, Shape<128, 128, kKT, 2, 4, 2>, Shape<64, 128, kKT, 2, 2, 2>>;
        using Weight = Output;
    };
    struct Small {
        using Hidden = Shape<64, 32, kKT, 2, 2, 4>;
        using Output = Shape<64, 64, kKT, 2, 2, 4>;
        using Weight = Output;
    };
    struct Large {
        using Hidden = std::conditional_t<planes == 1, Shape<256, 128, kKT, 2, 4, 2>, typename Medium::Hidden>;
        using Output = std::conditional_t<planes == 1, Shape<256, 256, kKT, 2, 4, 2>, typename Medium::Output>;
        using Weight = Output;
    };
    // Tiles of float32 that get a compute unit each: 64 of the reduction at a time, for twice as many wavefronts.  (Medium tiles, deep ones
    // and small ones, y and x's gradient: 8192 rows of 256 -> 1024 -> 256, 256 tiles, 43 and 75, 34 and 62, 52 and 102 us; 9000 rows, 282
    // tiles, 52 and 78, 55 and 104, 72 and 144; 4096 rows, 128 tiles, 36 and 65, 28 and 53, 28 and 54.  Hidden numbers and their gradients
    // of 2300 rows of 256 -> 440, 252 tiles, 16 and 24, 13 and 20, 20 and 30.)
    struct Deep {
        using Hidden = std::conditional_t<planes == 1, typename Medium::Hidden, Shape<64, 64, 64, 2, 4, 2>>;
        using Output = std::conditional_t<planes == 1, typename Medium::Output, Shape<64, 128, 64, 2, 4, 2>>;
        using Weight = typename Medium::Weight;
    };
    static constexpr int64_t kMediumTiles = 192, kUnits = 256;
    static constexpr double kMediumSlower = 1.15;
    template <class S>
    static int64_t tiles_of(int64_t m, int64_t n) {
        return pieces(m, S::BM) * pieces(n, S::BN);
    }
    // the time that `tiles` take, `at_once` of them to a compute unit and the reduction in `splits`: in rounds of the compute units, by
    // the numbers of a tile
    template <class S>
    static double time_of(int64_t tiles, int at_once, int64_t splits) {
        return (double)(pieces(tiles * splits, at_once * kUnits) * at_once * S::BM * S::BN) / (double)splits;
    }
    static bool large_pays(double medium, double large) { return planes == 1 && large <= kMediumSlower * medium; }
    template <class M, class L>
    static Size size_of(int64_t m, int64_t n) {
        const int64_t medium = tiles_of<M>(m, n);
        if (planes == 3 && medium <= kUnits) return medium <= kUnits / 2 ? kSmall : kDeep;
        return medium < kMediumTiles ? kSmall : large_pays(time_of<M>(medium, 2, 1), time_of<L>(tiles_of<L>(m, n), 1, 1)) ? kLarge : kMedium;
    }

    static Size hidden_size(int64_t rows, int64_t ldh) { return size_of<typename Medium::Hidden, typename Large::Hidden>(rows, ldh); }
    static Size output_size(int64_t rows, int64_t cols) { return size_of<typename Medium::Output, typename Large::Output>(rows, cols); }

    // The tiles of the weights' gradients, and the rows of a split.
    struct Split {
        int64_t each;
        int splits;
        Size size;
    };
    template <class S>
    static int64_t weight_tiles(const SvoxGatedFfn& s) {
        return 2 * tiles_of<S>(s.hidden, s.dim) + tiles_of<S>(s.out, s.hidden);
    }
    static Split weight_split(const SvoxGatedFfn& s) {
        Split w;
        const int64_t small = weight_tiles<typename Small::Weight>(s), medium = weight_tiles<typename Medium::Weight>(s), large = weight_tiles<typename Large::Weight>(s);
        const int64_t steps = pieces(s.rows, kKT);
        const int64_t large_splits = large < kUnits ? kUnits / large : 1, medium_splits = pieces(2 * kUnits, medium);
        // (rows enough for two blocks a compute unit of eight steps each make up for few tiles)
        w.size = kMedium;
        if (medium * steps < 2 * kUnits * 8) w.size = kSmall;
        else if (large_pays(time_of<typename Medium::Weight>(medium, 2, medium_splits), time_of<typename Large::Weight>(large, 1, large_splits))) w.size = kLarge;
        int64_t splits = w.size == kLarge ? large_splits : w.size == kMedium ? medium_splits : pieces(2 * kUnits, small);
        if (splits > pieces(steps, 8)) splits = pieces(steps, 8);
        w.each = up_to(pieces(s.rows, splits), kKT);
        w.splits = (int)pieces(s.rows, w.each);
        return w;
    }
};

}  // namespace svox_decoder
