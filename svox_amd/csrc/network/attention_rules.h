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
};

constexpr int64_t kAttendBlocks = 512;   // two for each compute unit

// How a tile's other axis is split, `size` at a time.  What a tile sees of it only the GPU knows; in all likelihood it is `length`, and where
// there are several sequences, or a causal one, it differs from tile to tile.  A block gets as many steps as leave two blocks for every
// place on the GPU, two at least; as many blocks may share a tile as a tile of the whole axis would need, in launches of up to 2048 blocks (one that
// finds nothing left to do costs two microseconds of its place).
inline AttendPlan split(AttendPlan plan, int64_t blocks, int64_t length, int64_t whole, int64_t size) {
    plan.splits = plan.steps = 1;
    if (blocks < 1 || blocks >= 2 * kAttendBlocks) return plan;
    const int64_t steps = pieces(length, size) * blocks / (2 * kAttendBlocks);
    plan.steps = (int)(steps < 2 ? 2 : steps);
    const int64_t wanted = pieces(pieces(whole, size), plan.steps), most = 4 * kAttendBlocks / blocks;
    const int64_t splits = wanted < most ? wanted : most;
    plan.splits = (int)(splits < 1 ? 1 : splits > 512 ? 512 : splits);
    return plan;
}
// The part of `other` that a tile of `rows` out of `all` sees where sequences are of one length.
inline int64_t likely_length(int64_t other, int64_t sequences, int64_t rows, int64_t all) {
    const int64_t sequences_of_tile = all > 0 ? 1 + (rows * sequences - 1) / all : 1;
    const int64_t length = pieces(other, sequences < 1 ? 1 : sequences) * sequences_of_tile;
    return length < other ? length : other;
}

inline AttendPlan forward_plan(const SvoxAttention& s) {
    const int64_t rows = s.queries * (s.heads / s.kv_heads), blocks = pieces(rows, 128) * s.kv_heads;
    if (blocks >= kAttendBlocks) return split({128, 1, 1, false}, blocks, likely_length(s.keys, s.sequences, 128, rows), s.keys, 64);
    return split({32, 1, 1, true}, pieces(rows, 32) * s.kv_heads, likely_length(s.keys, s.sequences, 32, rows), s.keys, 128);
}
inline AttendPlan query_grad_plan(const SvoxAttention& s) {
    const int64_t rows = s.queries * (s.heads / s.kv_heads);
    return split({128, 1, 1, false}, pieces(rows, 128) * s.kv_heads, likely_length(s.keys, s.sequences, 128, rows), s.keys, 64);
}
inline AttendPlan key_grad_plan(const SvoxAttention& s) {
    const int64_t rows = s.queries * (s.heads / s.kv_heads);
    return split({128, 1, 1, false}, pieces(s.keys, 128) * s.kv_heads, likely_length(rows, s.sequences, 128, s.keys), rows, 64);
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

inline int64_t attention_space(const SvoxAttention& s, bool backward) {
    const int64_t rows = s.queries * (s.heads / s.kv_heads), width = attend_width(s.dim);
    const auto whole = [](int64_t bytes) { return (bytes + 255) / 256 * 256; };
    const auto space = [&](const AttendPlan& plan, int64_t count, int64_t numbers) {
        return plan.splits > 1 ? whole(s.kv_heads * plan.splits * count * numbers * 4) + whole(s.kv_heads * pieces(count, plan.rows) * 4) : 0;
    };
    if (!backward) {
        const AttendPlan plan = forward_plan(s);
        return space(plan, rows, width) + (plan.splits > 1 ? whole(s.kv_heads * plan.splits * rows * 8) : 0);
    }
    const int64_t q = space(query_grad_plan(s), rows, width), k = space(key_grad_plan(s), s.keys, 2 * width);
    return whole(s.kv_heads * rows * 4) + (q > k ? q : k);
}

}  // namespace svox_network
