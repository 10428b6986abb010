// ffn_plan.h -- what the launches of the gated feed-forward block share on the host: the sizes of its narrow layers' workspaces, and
// the joining of gradients that were computed in parts.
#pragma once
#include "entry.h"
#include "narrow_kernels.h"

namespace svox_decoder {

inline int64_t gradient_numbers(const SvoxGatedFfn& s) {
    return 2 * (int64_t)s.hidden * s.dim + (int64_t)s.hidden * s.out + 2 * (int64_t)s.hidden + s.out;
}

// The parts of the weights' gradients, those of one after those of another, and the launch that adds them up.
template <class T>
struct Parts {
    JoinArgs<T> join{};
    int64_t blocks = 0;
    int jobs = 0;
    float* at;
    explicit Parts(float* part) : at(part) {}
    float* take(int64_t count, int64_t splits, void* out) {
        float* const part = at;
        at += splits * count;
        if (out) {
            const int groups = join_groups(splits);
            join.job[jobs] = {part, (T*)out, count, (int)splits, groups};
            join.blocks[jobs] = pieces(count, kJoinThreads / groups * 4);
            blocks += join.blocks[jobs++];
        }
        return part;
    }
    void launch(hipStream_t stream) const {
        if (blocks > 0) hipLaunchKernelGGL((join_kernel<T>), grid_of(blocks, kJoinThreads), dim3(kJoinThreads), 0, stream, join);
    }
};

// ---- narrow layers
// KD and KO, the 32s of features and of numbers of the result: 1, 2 or 4
#define SVOX_NARROW_STEPS(n, K, ...)                                    \
    if ((n) <= 32) { constexpr int K = 1; __VA_ARGS__; }                \
    else if ((n) <= 64) { constexpr int K = 2; __VA_ARGS__; }           \
    else if constexpr (Form<T>::planes == 1) { constexpr int K = 4; __VA_ARGS__; }
template <class T>
int64_t narrow_numbers(const SvoxGatedFfn& s, bool backward) {   // of the chunks, 16-bit
    const int64_t kd = narrow_steps(s.dim), ko = narrow_steps(s.out);
    return pieces(s.hidden, 32) * ((4 * kd + 2 * ko + (backward ? 4 * kd : 0)) * Form<T>::planes + 1) * 512;
}
// the rows of narrow_weight_kernel's splits
struct NarrowSplit {
    int64_t down, each;   // blocks over the hidden units
    int splits;
};
template <class T>
int narrow_weight_waves(const SvoxGatedFfn& s) {
    SVOX_NARROW_STEPS(s.dim, KD, SVOX_NARROW_STEPS(s.out, KO, { return (kNarrowWeightWaves<T, KD, KO>); }));
    return 1;
}
template <class T>
NarrowSplit narrow_split(const SvoxGatedFfn& s) {
    NarrowSplit n;
    n.down = pieces(s.hidden, 16 * narrow_weight_waves<T>(s));
    int64_t splits = pieces(512, n.down);
    if (splits > pieces(s.rows, 128)) splits = pieces(s.rows, 128);
    n.each = up_to(pieces(s.rows, splits), 32);
    n.splits = (int)pieces(s.rows, n.each);
    return n;
}
template <class T>
struct NarrowBackward {
    u16* chunks;
    float* part;
    NarrowSplit split;
    int64_t bytes;
    NarrowBackward(const SvoxGatedFfn& s, void* workspace) {
        Room room(workspace);
        split = narrow_split<T>(s);
        chunks = room.take<u16>(narrow_numbers<T>(s, true));
        part = room.take<float>(split.splits * gradient_numbers(s));
        bytes = room.used;
    }
};
// The launches for narrow layers, a unit of its own (narrow_type.hip) for every type and activation.
template <class T, int activation>
struct Narrow {
    static int forward(const SvoxGatedFfn& s, void* y, void* workspace, hipStream_t stream);
    static int backward(const SvoxGatedFfn& s, const void* grad_output, int64_t grad_stride, const SvoxGatedFfnGrads& grads, void* workspace,
                        hipStream_t stream);
};

}  // namespace svox_decoder
