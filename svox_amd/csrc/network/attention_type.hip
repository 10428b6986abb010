// attention_type.hip -- the attention kernels of one type (SVOX_DECODER_TYPE) for heads of up to SVOX_ATTEND_WIDTH numbers, and their launches.
#include "attention_kernels.h"
#include "attention_rules.h"
#include "entry.h"

namespace svox_network {

using T = SVOX_DECODER_TYPE;
constexpr int DP = SVOX_ATTEND_WIDTH;

namespace {

AttendArgs<T> args(const SvoxAttention& s) {
    AttendArgs<T> p{};
    p.q = (const T*)s.q, p.k = (const T*)s.k, p.v = (const T*)s.v;
    p.q_stride = s.q_stride, p.q_head = s.q_head;
    p.k_stride = s.k_stride, p.k_head = s.k_head;
    p.v_stride = s.v_stride, p.v_head = s.v_head;
    const void* const keys = s.key_offsets ? s.key_offsets : s.offsets;
    p.seq.q = {s.offsets, s.wide_offsets, s.offsets ? (int)s.sequences : 1, (int)s.queries};
    p.seq.k = {keys, s.wide_offsets, keys ? (int)s.sequences : 1, (int)s.keys};
    p.seq.causal = s.causal;
    p.group = s.heads / s.kv_heads;
    p.kv_heads = s.kv_heads;
    p.rows = (int)(s.queries * p.group);
    p.keys = (int)s.keys;
    p.dim = s.dim;
    p.scale = s.scale;
    return p;
}
template <class K>
void launch(K kernel, AttendArgs<T> p, int64_t count, int size, int splits, bool runs, hipStream_t stream) {
    p.tiles = (int)pieces(count, size);
    p.splits = splits;
    p.runs = runs;
    hipLaunchKernelGGL(kernel, grid_of((int64_t)p.tiles * p.kv_heads * splits, kAttendThreads), dim3(kAttendThreads), 0, stream, p);
}
template <bool direct>
void forward(const AttendArgs<T>& p, const AttendPlan& plan, bool runs, hipStream_t stream) {
    if (plan.few) launch(attend_kernel<T, DP, 1, 4, direct>, p, p.rows, plan.rows, plan.splits, runs, stream);
    else launch(attend_kernel<T, DP, 1, 1, direct>, p, p.rows, plan.rows, plan.splits, runs, stream);
}

}  // namespace

template <>
int launch_attention<T, DP>(const SvoxAttention& s, void* out, float* lse, void* workspace, hipStream_t stream) {
    AttendArgs<T> p = args(s);
    p.y = (T*)out;
    p.lse = lse;
    const AttendPlan plan = forward_plan(s);
    Room room(workspace);
    if (plan.splits > 1) {
        p.part = room.take<float>((int64_t)p.kv_heads * plan.splits * p.rows * DP);
        p.stats = room.take<f32x2>((int64_t)p.kv_heads * plan.splits * p.rows);
    }
    if (direct_loads(s)) forward<true>(p, plan, in_runs(s), stream);
    else forward<false>(p, plan, in_runs(s), stream);
    if (plan.splits > 1) {
        p.splits = plan.splits;
        hipLaunchKernelGGL((attend_join_kernel<T, DP>), dim3((unsigned)least((int64_t)p.kv_heads * p.rows, 1 << 16)), dim3(kAttendThreads), 0, stream, p);
    }
    return check_launch("attention");
}

template <>
int launch_attention_backward<T, DP>(const SvoxAttention& s, const SvoxAttentionGrads& g, void* workspace, hipStream_t stream) {
    AttendArgs<T> p = args(s);
    p.out = (const T*)g.out;
    p.grad = (const T*)g.grad;
    p.grad_stride = g.grad_stride, p.grad_head = g.grad_head;
    p.lse = const_cast<float*>(g.lse);
    p.dq = (T*)g.q, p.dk = (T*)g.k, p.dv = (T*)g.v;
    Room room(workspace);
    p.delta = room.take<float>((int64_t)p.kv_heads * p.rows);
    const AttendPlan of_q = query_grad_plan(s), of_k = key_grad_plan(s);
    const bool direct = s.dim == DP, runs = in_runs(s);
    if (p.rows > 0)
        hipLaunchKernelGGL((attend_delta_kernel<T>), dim3((unsigned)least(pieces((int64_t)p.rows * p.kv_heads, 16), 1 << 14)), dim3(kAttendThreads), 0, stream, p);
    char* const rest = room.at + room.used;
    const auto sum = [&](const float* part, int64_t rows, int group, int splits, float factor, T* to) {
        if (to)
            hipLaunchKernelGGL((attend_sum_kernel<T, DP>), dim3((unsigned)least(pieces(rows * p.kv_heads, kAttendThreads / (DP / 4)), 1 << 14)), dim3(kAttendThreads),
                               0, stream, part, rows, p.kv_heads, group, p.dim, splits, factor, to);
    };
    if (p.dq && p.rows > 0) {
        p.part = (float*)rest;
        if (direct) launch(attend_query_grad_kernel<T, DP, true>, p, p.rows, of_q.rows, of_q.splits, runs, stream);
        else launch(attend_query_grad_kernel<T, DP, false>, p, p.rows, of_q.rows, of_q.splits, runs, stream);
        if (of_q.splits > 1) sum(p.part, p.rows, p.group, of_q.splits, p.scale, p.dq);
    }
    if ((p.dk || p.dv) && p.keys > 0) {
        p.part = (float*)rest;
        if (direct) launch(attend_key_grad_kernel<T, DP, true>, p, p.keys, of_k.rows, of_k.splits, runs, stream);
        else launch(attend_key_grad_kernel<T, DP, false>, p, p.keys, of_k.rows, of_k.splits, runs, stream);
        if (of_k.splits > 1) {
            sum(p.part, p.keys, 1, of_k.splits, p.scale, p.dk);
            sum(p.part + (int64_t)p.kv_heads * of_k.splits * p.keys * DP, p.keys, 1, of_k.splits, 1.0f, p.dv);
        }
    }
    return check_launch("attention_backward");
}

}  // namespace svox_network
