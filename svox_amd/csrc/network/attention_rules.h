// attention_rules.h -- which of its kernels a call of attention runs on and into how many parts its work is split, by its sizes: host code
// alone, of no GPU's headers.
#pragma once
#include <cstdint>

#include "../../../include/svox_network.h"
#include "../decoder/rules.h"

namespace svox_network {

using svox_decoder::pieces;

inline int attend_width(int dim) { return dim <= 32 ? 32 : dim <= 64 ? 64 : 128; }

struct AttendPlan {
    int rows;            // of a block's tile
    int splits, steps;   // blocks that may share a tile's other axis, and the least steps of each
    bool few;
    bool ordered;        // tiles in the order of what they have to do, which a launch of its own finds out
    bool far;            // float32: the other axis is so long that sums along it are made of parts
};

constexpr int64_t kAttendBlocks = 512;   // two for each compute unit

// How a tile's other axis is split, `size` at a time.  What a tile sees of it only the GPU knows; in all likelihood it is `length`, and where
// there are several sequences, or a causal one, it differs from tile to tile.  A block gets as many steps as leave two blocks for every
// place on the GPU, two at least; as many blocks may share a tile as a tile of the whole axis would need, in launches of up to 2048 blocks (one that
// finds nothing left to do costs two microseconds of its place).
inline AttendPlan split(AttendPlan plan, int64_t blocks, int64_t length, int64_t whole, int64_t size) {
    // (float32, 8 heads of 32, steps: sequences of 4096 4840 us without parts, 5040 with; 16 384 causal rows 6020, 5600; heads of 64 and 128 within 1 %.  Rows of 65 536
    // keys are 196 times the error of one rounding off without, 29 to 41 with.)
    plan.far = !plan.few && length >= 2048;
    plan.splits = plan.steps = 1;
    if (blocks < 1 || blocks >= 2 * kAttendBlocks) return plan;
    const int64_t steps = pieces(length, size) * blocks / (2 * kAttendBlocks);
    plan.steps = (int)(steps < 2 ? 2 : steps);
    const int64_t wanted = pieces(pieces(whole, size), plan.steps), most = 4 * kAttendBlocks / blocks;
    const int64_t splits = wanted < most ? wanted : most;
    plan.splits = (int)(splits < 1 ? 1 : splits > 512 ? 512 : splits);
    return plan;
}
// Whether tiles are to be put in order: where sequences may differ in length, the blocks are more than the GPU has places for but not so many that the
// last ones matter little, and each has enough to do for the launch, some six microseconds, to pay.  (Its places are in LDS: up to 4095 sequences.)
inline AttendPlan ordered(AttendPlan plan, const SvoxAttention& s, int64_t tiles, int64_t length) {
    const int64_t blocks = tiles * s.kv_heads;
    plan.ordered = s.sequences >= 2 && s.sequences < 4096 && blocks >= kAttendBlocks / 2 && blocks < 8 * kAttendBlocks && length >= 256;
    return plan;
}
// The part of `other` that a tile of `rows` out of `all` sees where sequences are of one length.
inline int64_t likely_length(int64_t other, int64_t sequences, int64_t rows, int64_t all) {
    const int64_t sequences_of_tile = all > 0 ? 1 + (rows * sequences - 1) / all : 1;
    const int64_t length = pieces(other, sequences < 1 ? 1 : sequences) * sequences_of_tile;
    return length < other ? length : other;
}

// Tiles of 128 rows where there are enough of them for the GPU, or where keys are read so often that rows of a tile matter more than places: from
// some number of scores on, which are dearest where heads are wide, and in float32.  (Tiles of 32 rows and of 128, us, bfloat16: 8192 rows of one head of
// 128, 1024 keys 48, 32; 4096 rows, 512 keys 21, 22; 4096 rows of 8 heads of 64, 4096 keys 81, 68; 2048 rows, 2048 keys 36, 37; 16 384 rows of 2 heads of
// 32, 4096 keys 49, 49; 8192 rows, 2048 keys 24, 30.  float32: 1024 rows of 8 heads of 64, 1024 keys 52, 41; 512 rows, 512 keys 21, 25.)
inline AttendPlan forward_plan(const SvoxAttention& s) {
    const int64_t rows = s.queries * (s.heads / s.kv_heads), tiles = pieces(rows, 128), length = likely_length(s.keys, s.sequences, 128, rows);
    const int width = attend_width(s.dim), dear = s.dtype == SVOX_DECODER_F32 || width == 128 ? 22 : width == 64 ? 26 : 27;
    const bool many = rows >= 256 && length >= ((int64_t)1 << dear) / (rows * s.kv_heads);
    if (tiles * s.kv_heads >= kAttendBlocks || many)
        return ordered(split({128, 1, 1, false, false, false}, tiles * s.kv_heads, length, s.keys, 64), s, tiles, length);
    return split({32, 1, 1, true, false, false}, pieces(rows, 32) * s.kv_heads, likely_length(s.keys, s.sequences, 32, rows), s.keys, 128);
}
inline AttendPlan query_grad_plan(const SvoxAttention& s) {
    const int64_t rows = s.queries * (s.heads / s.kv_heads), tiles = pieces(rows, 128), length = likely_length(s.keys, s.sequences, 128, rows);
    return ordered(split({128, 1, 1, false, false, false}, tiles * s.kv_heads, length, s.keys, 64), s, tiles, length);
}
inline AttendPlan key_grad_plan(const SvoxAttention& s) {
    const int64_t rows = s.queries * (s.heads / s.kv_heads), tiles = pieces(s.keys, 128), length = likely_length(rows, s.sequences, 128, s.keys);
    return ordered(split({128, 1, 1, false, false, false}, tiles * s.kv_heads, length, rows, 64), s, tiles, length);
}

// Whether tiles go from memory to LDS 16 bytes at a time: everything lies at whole numbers of 16 bytes, and no tile of up to 128 rows reaches
// further than 32 bits count.
inline bool direct_heads(const SvoxAttention& s, const void* x, int64_t stride, int64_t head, int64_t group) {
    const int64_t size = s.dtype == SVOX_DECODER_F32 ? 4 : 2;
    return (uintptr_t)x % 16 == 0 && s.dim * size % 16 == 0 && stride * size % 16 == 0 && head * size % 16 == 0 && 130 * stride + group * head < (int64_t)1 << 28;
}
inline bool direct_loads(const SvoxAttention& s) {
    return direct_heads(s, s.q, s.q_stride, s.q_head, s.heads / s.kv_heads) && direct_heads(s, s.k, s.k_stride, s.k_head, 1) &&
           direct_heads(s, s.v, s.v_stride, s.v_head, 1);
}
inline bool direct_loads(const SvoxAttention& s, const SvoxAttentionGrads& g) {
    return direct_heads(s, g.grad, g.grad_stride, g.grad_head, s.heads / s.kv_heads);
}

// Whether the blocks of an XCD take a few tiles side by side: where many sequences share the keys out, so that one's stay in an XCD's cache, and
// there are tiles for all XCDs.  Heads of few long sequences go round the XCDs instead.
inline bool in_runs(const SvoxAttention& s, int64_t tiles) { return s.sequences >= 16 && tiles * s.kv_heads >= kAttendBlocks; }

// Tiles that blocks of an XCD take side by side, and the blocks of `units` tiles of heads in such runs for all eight XCDs.
constexpr int kAttendRun = 8;
inline int64_t in_whole_runs(int64_t units) { return svox_decoder::up_to(units, 8 * kAttendRun); }

inline int64_t attention_space(const SvoxAttention& s, bool backward) {
    const int64_t rows = s.queries * (s.heads / s.kv_heads), width = attend_width(s.dim);
    const auto whole = [](int64_t bytes) { return (bytes + 255) / 256 * 256; };
    const auto space = [&](const AttendPlan& plan, int64_t count, int64_t numbers) {
        return plan.splits > 1 ? whole(s.kv_heads * plan.splits * count * numbers * 4) + whole(s.kv_heads * pieces(count, plan.rows) * 4) : 0;
    };
    const auto order = [&](const AttendPlan& plan, int64_t count) { return plan.ordered ? whole(pieces(count, plan.rows) * 4) : 0; };
    if (!backward) {
        const AttendPlan plan = forward_plan(s);
        return order(plan, rows) + space(plan, rows, width) + (plan.splits > 1 ? whole(s.kv_heads * plan.splits * rows * 8) : 0);
    }
    const AttendPlan of_q = query_grad_plan(s), of_k = key_grad_plan(s);
    const int64_t q = space(of_q, rows, width), k = space(of_k, s.keys, 2 * width);
    return whole(s.kv_heads * rows * 4) + order(of_q, rows) + order(of_k, s.keys) + (q > k ? q : k);
}

}  // namespace svox_network
