// attention_type.hip -- the attention kernels of one type (SVOX_DECODER_TYPE) for heads of up to SVOX_ATTEND_WIDTH numbers, and their launches.
#include "attention_kernels.h"
#include "attention_order.h"
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
    const auto offsets = [&](const void* at, int64_t total) {
        const int n = at ? (int)s.sequences : 1;
        return Offsets{at, s.wide_offsets, n, (int)total, total > 0 ? (float)n / (float)total : 0.0f};
    };
    p.seq.q = offsets(s.offsets, s.queries);
    p.seq.k = offsets(keys, s.keys);
    p.seq.causal = s.causal;
    p.group = s.heads / s.kv_heads;
    p.kv_heads = s.kv_heads;
    p.rows = (int)(s.queries * p.group);
    p.keys = (int)s.keys;
    p.dim = s.dim;
    p.scale = s.scale;
    p.last_first = s.causal;   // (the last queries see most, as the first keys are seen by most)
    return p;
}
template <class K>
void launch(K kernel, AttendArgs<T>& p, const SvoxAttention& s, int64_t count, const AttendPlan& plan, hipStream_t stream) {
    p.tiles = (int)pieces(count, plan.rows);
    p.splits = plan.splits;
    p.steps = plan.steps;
    p.runs = !p.order && in_runs(s, p.tiles);
    const int64_t units = (int64_t)p.tiles * p.kv_heads;
    hipLaunchKernelGGL(kernel, grid_of((p.runs ? in_whole_runs(units) : units) * plan.splits, kAttendThreads), dim3(kAttendThreads), 0, stream, p);
}
// One axis of the launch that puts tiles in order.
OrderArgs::Axis order_axis(const AttendArgs<T>& p, const AttendPlan& plan, bool keys, int* to) {
    const int count = keys ? p.rows : p.keys;
    return {to, (int)pieces(count, plan.rows), count, plan.rows, p.group, keys};
}
// f(std::bool_constant of `direct`, of plan.far), of which 16-bit types have no kernels
template <class F>
void with_kind(bool direct, const AttendPlan& plan, F f) {
    if constexpr (sizeof(T) == 4)
        if (plan.far) return direct ? f(std::true_type(), std::true_type()) : f(std::false_type(), std::true_type());
    direct ? f(std::true_type(), std::false_type()) : f(std::false_type(), std::false_type());
}

}  // namespace

template <>
int launch_attention<T, DP>(const SvoxAttention& s, void* out, float* lse, void* rest, void* workspace, hipStream_t stream) {
    AttendArgs<T> p = args(s);
    p.y = (T*)out;
    p.lse = lse;
    p.rest = (T*)rest;
    const AttendPlan plan = forward_plan(s);
    Room room(workspace);
    if (plan.splits > 1) {
        p.part = room.take<float>((int64_t)p.kv_heads * plan.splits * p.rows * DP);
        p.stats = room.take<f32x2>((int64_t)p.kv_heads * plan.splits * p.rows);
        p.used = room.take<int>(p.kv_heads * pieces(p.rows, plan.rows));
    }
    if (plan.ordered) {
        OrderArgs o{p.seq, {}};
        o.axis[0] = order_axis(p, plan, true, room.take<int>(pieces(p.rows, plan.rows)));
        p.order = o.axis[0].to;
        launch_order(o, 1, stream);
    }
    if (plan.few) {
        if (direct_loads(s)) launch(attend_kernel<T, DP, 4, true, false>, p, s, p.rows, plan, stream);
        else launch(attend_kernel<T, DP, 4, false, false>, p, s, p.rows, plan, stream);
    } else {
        with_kind(direct_loads(s), plan, [&](auto direct, auto far) {
            launch(attend_kernel<T, DP, 1, decltype(direct)::value, decltype(far)::value>, p, s, p.rows, plan, stream);
        });
    }
    // (240 000 rows of up to 2 splits: 180 us by blocks, 13 by lanes; 32 rows of 12 splits: 5 us by blocks, 12 by lanes)
    const int64_t joined = (int64_t)p.kv_heads * p.rows;
    if (plan.splits > 16 || (plan.splits > 1 && joined <= 4096))
        hipLaunchKernelGGL((attend_join_many_kernel<T, DP>), dim3((unsigned)least(joined, 4096)), dim3(kAttendThreads), 0, stream, p, plan.rows);
    else if (plan.splits > 1)
        hipLaunchKernelGGL((attend_join_kernel<T, DP>), dim3((unsigned)least(pieces(joined, kAttendThreads / (DP / 4)), 1 << 14)), dim3(kAttendThreads), 0, stream, p,
                           plan.rows);
    return check_launch("attention");
}

template <>
int launch_attention_backward<T, DP>(const SvoxAttention& s, const SvoxAttentionGrads& g, void* workspace, hipStream_t stream) {
    AttendArgs<T> p = args(s);
    p.out = (const T*)g.out;
    p.grad = (const T*)g.grad;
    p.grad_stride = g.grad_stride, p.grad_head = g.grad_head;
    p.lse = const_cast<float*>(g.lse);
    p.rest = (T*)const_cast<void*>(g.rest);
    p.dq = (T*)g.q, p.dk = (T*)g.k, p.dv = (T*)g.v;
    Room room(workspace);
    p.delta = room.take<float>((int64_t)p.kv_heads * p.rows);
    const AttendPlan of_q = query_grad_plan(s), of_k = key_grad_plan(s);
    const bool direct = direct_loads(s) && direct_loads(s, g);
    if (p.rows > 0 && !p.dq)
        hipLaunchKernelGGL((attend_delta_kernel<T, DP>), dim3((unsigned)least(pieces(p.rows, 128) * p.kv_heads, 1 << 14)), dim3(kAttendThreads), 0, stream, p);
    const int* order[2] = {};
    {
        OrderArgs o{p.seq, {}};
        int n = 0;
        if (of_q.ordered && p.dq && p.rows > 0) order[0] = (o.axis[n++] = order_axis(p, of_q, true, room.take<int>(pieces(p.rows, of_q.rows)))).to;
        if (of_k.ordered && (p.dk || p.dv) && p.keys > 0) order[1] = (o.axis[n++] = order_axis(p, of_k, false, room.take<int>(pieces(p.keys, of_k.rows)))).to;
        if (n > 0) launch_order(o, n, stream);
    }
    const auto sum = [&](const float* part, int64_t rows, const AttendPlan& plan, int group, float factor, T* to) {
        if (to)
            hipLaunchKernelGGL((attend_sum_kernel<T, DP>), dim3((unsigned)least(pieces(rows * p.kv_heads, kAttendThreads / (DP / 4)), 1 << 14)), dim3(kAttendThreads),
                               0, stream, p, part, rows, plan.rows, group, factor, to);
    };
    if (p.dq && p.rows > 0) {
        Room mine = room;
        if (of_q.splits > 1) {
            p.used = mine.take<int>(p.kv_heads * pieces(p.rows, of_q.rows));
            p.part = mine.take<float>((int64_t)p.kv_heads * of_q.splits * p.rows * DP);
        }
        p.order = order[0];
        with_kind(direct, of_q, [&](auto d, auto far) { launch(attend_query_grad_kernel<T, DP, decltype(d)::value, decltype(far)::value>, p, s, p.rows, of_q, stream); });
        if (of_q.splits > 1) sum(p.part, p.rows, of_q, p.group, p.scale, p.dq);
    }
    if ((p.dk || p.dv) && p.keys > 0) {
        Room mine = room;
        p.last_first = 0;
        if (of_k.splits > 1) {
            p.used = mine.take<int>(p.kv_heads * pieces(p.keys, of_k.rows));
            p.part = mine.take<float>(2 * (int64_t)p.kv_heads * of_k.splits * p.keys * DP);
        }
        p.order = order[1];
        with_kind(direct, of_k, [&](auto d, auto far) { launch(attend_key_grad_kernel<T, DP, decltype(d)::value, decltype(far)::value>, p, s, p.keys, of_k, stream); });
        if (of_k.splits > 1) {
            sum(p.part, p.keys, of_k, 1, p.scale, p.dk);
            sum(p.part + (int64_t)p.kv_heads * of_k.splits * p.keys * DP, p.keys, of_k, 1, 1.0f, p.dv);
        }
    }
    return check_launch("attention_backward");
}

}  // namespace svox_network
