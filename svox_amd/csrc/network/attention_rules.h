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
    int rows;      // of a block's tile
    int splits;    // blocks that share a tile's other axis
    bool few;
};

constexpr int64_t kAttendBlocks = 512;   // two for each compute unit

// Blocks for a tile's other axis, of which a tile sees `length` in all likelihood, `size` at a time: as many as fill the GPU, each with
// two steps at least.
inline int splits_for(int64_t blocks, int64_t length, int64_t size) {
    if (blocks >= kAttendBlocks || blocks < 1) return 1;
    const int64_t wanted = kAttendBlocks / blocks, most = length / (2 * size);
    const int64_t splits = wanted < most ? wanted : most;
    return (int)(splits < 1 ? 1 : splits > 256 ? 256 : splits);
}
// The part of `other` that a tile of `rows` out of `all` sees where sequences are of one length.
inline int64_t likely_length(int64_t other, int64_t sequences, int64_t rows, int64_t all) {
    const int64_t sequences_of_tile = all > 0 ? 1 + (rows * sequences - 1) / all : 1;
    const int64_t length = pieces(other, sequences < 1 ? 1 : sequences) * sequences_of_tile;
    return length < other ? length : other;
}

inline AttendPlan forward_plan(const SvoxAttention& s) {
    const int64_t rows = s.queries * (s.heads / s.kv_heads), blocks = pieces(rows, 128) * s.kv_heads;
    if (blocks >= kAttendBlocks) return {128, 1, false};
    const int64_t small = pieces(rows, 32) * s.kv_heads;
    return {32, splits_for(small, likely_length(s.keys, s.sequences, 32, rows), 128), true};
}
inline AttendPlan query_grad_plan(const SvoxAttention& s) {
    const int64_t rows = s.queries * (s.heads / s.kv_heads), blocks = pieces(rows, 128) * s.kv_heads;
    return {128, splits_for(blocks, likely_length(s.keys, s.sequences, 128, rows), 64), false};
}
inline AttendPlan key_grad_plan(const SvoxAttention& s) {
    const int64_t rows = s.queries * (s.heads / s.kv_heads), blocks = pieces(s.keys, 128) * s.kv_heads;
    return {128, splits_for(blocks, likely_length(rows, s.sequences, 128, s.keys), 64), false};
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

// Whether the blocks of an XCD take tiles side by side: where many sequences share the keys out, so that one's stay in an XCD's cache.  The
// tiles of few long ones differ in work where they are causal, and go round.
inline bool in_runs(const SvoxAttention& s) { return s.sequences >= 16; }

inline int64_t attention_space(const SvoxAttention& s, bool backward) {
    const int64_t rows = s.queries * (s.heads / s.kv_heads), width = attend_width(s.dim);
    const auto whole = [](int64_t bytes) { return (bytes + 255) / 256 * 256; };
    if (!backward) {
        const int64_t parts = forward_plan(s).splits;
        return parts > 1 ? whole(s.kv_heads * parts * rows * width * 4) + whole(s.kv_heads * parts * rows * 8) : 0;
    }
    const int64_t of_q = query_grad_plan(s).splits, of_k = key_grad_plan(s).splits;
    const int64_t q = of_q > 1 ? s.kv_heads * of_q * rows * width * 4 : 0, k = of_k > 1 ? 2 * s.kv_heads * of_k * s.keys * width * 4 : 0;
    return whole(s.kv_heads * rows * 4) + (q > k ? q : k);
}

}  // namespace svox_network
