// attention_order.hip -- the tiles of an attention by what they have to do.
#include "attention_order.h"

namespace svox_network {

// The tiles of rows (queries') or keys by what they have to do, most first: blocks that start late then have little to do.  (61 causal sequences of
// up to 1659 rows, 8 heads of 64: forward 86 -> 71 us, dq 113 -> 93, dk and dv 175 -> 157, this launch 6 to 7 for each pass.)  One block for each of
// both; the places are in LDS.  Tiles that have as much to do come in any order, which changes nothing but when they are computed.
constexpr int kOrderThreads = 1024, kOrderPlaces = 4096, kOrderBuckets = 1024;

__global__ __launch_bounds__(kOrderThreads) void attend_order_kernel(OrderArgs p) {
    __shared__ int places[2][kOrderPlaces], buckets[kOrderBuckets];
    const OrderArgs::Axis x = p.axis[blockIdx.x];
    const Offsets &mine = x.keys ? p.seq.q : p.seq.k, &other = x.keys ? p.seq.k : p.seq.q;
    const int n = min(mine.n, kOrderPlaces - 1);
    for (int i = (int)threadIdx.x; i <= n; i += kOrderThreads) places[0][i] = mine(i), places[1][i] = other(i);
    buckets[threadIdx.x] = 0;
    __syncthreads();
    const auto edge = [&](int t, bool low) {      // where what token t sees begins, or ends
        int s = 0, last = n - 1;
        while (s < last) {
            const int middle = (s + last + 1) / 2;
            if (places[0][middle] <= t) s = middle;
            else last = middle - 1;
        }
        const int m0 = places[0][s], m1 = places[0][s + 1], o0 = places[1][s], o1 = max(o0, places[1][s + 1]), ends = (o1 - o0) - (m1 - m0);
        if (!p.seq.causal || low == (x.keys != 0)) return low ? o0 : o1;
        return min(max(o0 + (t - m0) + ends + (low ? 0 : 1), o0), o1);
    };
    const int per_token = x.keys ? x.group : 1;
    const auto bucket_of = [&](int tile) {
        const int first = tile * x.rows / per_token, last = (min((tile + 1) * x.rows, x.count) - 1) / per_token;
        const int length = (edge(last, false) - edge(first, true)) * (x.keys ? 1 : x.group);
        return kOrderBuckets - 1 - min(max(length, 0) / 64, kOrderBuckets - 1);
    };
    for (int i = (int)threadIdx.x; i < x.tiles; i += kOrderThreads) atomicAdd(&buckets[bucket_of(i)], 1);
    __syncthreads();
    // (where each bucket begins)
    const int own = buckets[threadIdx.x];
    for (int d = 1; d < kOrderBuckets; d *= 2) {
        const int before = (int)threadIdx.x >= d ? buckets[threadIdx.x - d] : 0;
        __syncthreads();
        buckets[threadIdx.x] += before;
        __syncthreads();
    }
    const int begin = buckets[threadIdx.x] - own;
    __syncthreads();
    buckets[threadIdx.x] = begin;
    __syncthreads();
    for (int i = (int)threadIdx.x; i < x.tiles; i += kOrderThreads) x.to[atomicAdd(&buckets[bucket_of(i)], 1)] = i;
}

void launch_order(const OrderArgs& p, int axes, hipStream_t stream) {
    hipLaunchKernelGGL(attend_order_kernel, dim3(axes), dim3(kOrderThreads), 0, stream, p);
}

}  // namespace svox_network
