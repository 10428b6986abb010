// clip.hip -- the norm of all numbers of many tensors together, and the tensors scaled where it exceeds a bound.
//
//   norm = sqrt(sum x^2),  y = x min(1, max_norm / norm)
//
// Two passes: squares_kernel sums squares, scale_kernel adds up the blocks' sums and scales.  Both are bound by memory, the tensors
// read twice and written once (the norm has to be known before the first number is written).  A tensor's address, size and type
// travel in the launch's arguments, up to kClipTable of them in one, so that a list of small tensors costs two launches and no copy to
// the GPU.  A block takes chunks of 16 KB, every gridDim-th of the launch's; the second pass takes them from the last to the first, so
// that it begins with what the first pass left in the last cache.
//
// Squares and their sums are in 64 bits: float32's largest numbers and a sum of 2^40 of them stay finite, so that a norm that is not finite
// says that a number is not.  So is the factor, which may be below float32's smallest numbers, and its product with a number.
#include "../decoder/common.h"
#include "entry.h"

namespace svox_network {

using namespace svox_decoder;

namespace {

constexpr int kClipThreads = 256, kClipTable = 96, kClipChunkBytes = 16384, kClipBlocks = 2048;

struct ClipEntry {
    const void* from;
    void* to;
    int64_t count;
    int64_t first_and_type;   // the first chunk of the launch that is this tensor's, times four, and its type
};
struct ClipTable {
    ClipEntry at[kClipTable];
    int64_t chunks;
    int n;
};
static_assert(sizeof(ClipTable) + 64 <= 4096, "a launch's arguments");

__device__ __forceinline__ int entry_of(const ClipTable& t, int64_t chunk) {
    int low = 0, high = t.n;   // the last entry whose first chunk is not beyond
    while (high - low > 1) {
        const int middle = (low + high) / 2;
        if (t.at[middle].first_and_type / 4 <= chunk) low = middle;
        else high = middle;
    }
    return low;
}

__device__ __forceinline__ double sum_of_wave(double v) {
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) v += __shfl_xor(v, d, kWave);
    return v;
}
// known to all threads of the block
__device__ __forceinline__ double sum_of_block(double v, double* room) {
    v = sum_of_wave(v);
    if (threadIdx.x % kWave == 0) room[threadIdx.x / kWave] = v;
    __syncthreads();
    v = room[0];
#pragma unroll
    for (int w = 1; w < kClipThreads / kWave; ++w) v += room[w];
    return v;
}

// A chunk: 4 pieces of 16 bytes a thread, all on their way before the first is used.
template <class T>
struct Chunk {
    static constexpr int V = 16 / (int)sizeof(T), numbers = kClipChunkBytes / (int)sizeof(T), loads = numbers / V / kClipThreads;
    typename Few<T, V>::vector v[loads];
    static __device__ __forceinline__ int64_t at(int64_t chunk, int i) { return chunk * numbers + ((int64_t)i * kClipThreads + threadIdx.x) * V; }
    __device__ __forceinline__ void load(const T* from, int64_t chunk, int64_t count) {
#pragma unroll
        for (int i = 0; i < loads; ++i) v[i] = load_some<T, V>(from + at(chunk, i), count - at(chunk, i));
    }
};

template <class T>
__device__ __forceinline__ double squares_of(const ClipEntry& e, int64_t chunk) {
    Chunk<T> c;
    c.load((const T*)e.from, chunk, e.count);
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < Chunk<T>::loads; ++i)
#pragma unroll
        for (int j = 0; j < Chunk<T>::V; ++j) {
            const double x = (double)(float)c.v[i][j];
            sum = __builtin_fma(x, x, sum);
        }
    return sum;
}

__global__ __launch_bounds__(kClipThreads) void squares_kernel(ClipTable t, double* part) {
    __shared__ double room[kClipThreads / kWave];
    double sum = 0.0;
    for (int64_t c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const ClipEntry& e = t.at[entry_of(t, c)];
        const int64_t chunk = c - e.first_and_type / 4;
        switch (e.first_and_type & 3) {
            case SVOX_DECODER_F32: sum += squares_of<float>(e, chunk); break;
            case SVOX_DECODER_F16: sum += squares_of<F16>(e, chunk); break;
            default: sum += squares_of<Bf16>(e, chunk);
        }
    }
    sum = sum_of_block(sum, room);
    if (threadIdx.x == 0) part[blockIdx.x] = sum;
}

template <class T>
__device__ __forceinline__ void scale(const ClipEntry& e, int64_t chunk, double factor) {
    Chunk<T> c;
    c.load((const T*)e.from, chunk, e.count);
#pragma unroll
    for (int i = 0; i < Chunk<T>::loads; ++i) {
        const int64_t at = Chunk<T>::at(chunk, i);
        typename Few<T, Chunk<T>::V>::vector v = c.v[i];
        if (factor != 1.0)     // (a copy keeps every bit)
#pragma unroll
            for (int j = 0; j < Chunk<T>::V; ++j) v[j] = (T)(float)((double)(float)v[j] * factor);
        if (at + Chunk<T>::V <= e.count) {
            store_few<T, Chunk<T>::V>((T*)e.to + at, v);
        } else {
#pragma unroll
            for (int j = 0; j < Chunk<T>::V; ++j)
                if (at + j < e.count) ((T*)e.to)[at + j] = v[j];
        }
    }
}

// `parts` sums of all launches of the first pass.  Every block adds them up for itself: at most kClipBlocks a launch, from the cache.
__global__ __launch_bounds__(kClipThreads) void scale_kernel(ClipTable t, const double* part, int parts, double max_norm, float* norm) {
    __shared__ double room[kClipThreads / kWave];
    double sum = 0.0;
    for (int i = threadIdx.x; i < parts; i += kClipThreads) sum += part[i];
    const double total = sqrt(sum_of_block(sum, room));
    const bool clipped = total > max_norm && total < __builtin_inf();
    const double factor = clipped ? max_norm / total : 1.0;
    if (blockIdx.x == 0 && threadIdx.x == 0 && norm) *norm = (float)total;
    for (int64_t c = t.chunks - 1 - blockIdx.x; c >= 0; c -= gridDim.x) {
        const ClipEntry& e = t.at[entry_of(t, c)];
        if (!clipped && e.to == e.from) continue;
        const int64_t chunk = c - e.first_and_type / 4;
        switch (e.first_and_type & 3) {
            case SVOX_DECODER_F32: scale<float>(e, chunk, factor); break;
            case SVOX_DECODER_F16: scale<F16>(e, chunk, factor); break;
            default: scale<Bf16>(e, chunk, factor);
        }
    }
}

int64_t chunks_of(const SvoxClipTensor& x) { return pieces(x.count, kClipChunkBytes / (x.dtype == SVOX_DECODER_F32 ? 4 : 2)); }

// f(table, blocks) for every launch of a pass
template <class F>
void for_tables(const SvoxClipTensor* tensors, int64_t n, F f) {
    ClipTable t{};
    for (int64_t i = 0; i < n; ++i) {
        const int64_t chunks = chunks_of(tensors[i]);
        if (chunks > 0) {
            t.at[t.n++] = {tensors[i].from, tensors[i].to, tensors[i].count, t.chunks * 4 + tensors[i].dtype};
            t.chunks += chunks;
        }
        if (t.n > 0 && (t.n == kClipTable || i + 1 == n)) {
            f(t, (int)least(t.chunks, kClipBlocks));
            t.n = 0, t.chunks = 0;
        }
    }
    if (t.n > 0) f(t, (int)least(t.chunks, kClipBlocks));
}

}  // namespace

int64_t clip_blocks(const SvoxClipTensor* tensors, int64_t n) {
    int64_t blocks = 0;
    for_tables(tensors, n, [&](const ClipTable&, int b) { blocks += b; });
    return blocks;
}

int launch_clip(const SvoxClipTensor* tensors, int64_t n, double max_norm, float* norm, double* part, hipStream_t stream) {
    int parts = 0;
    for_tables(tensors, n, [&](const ClipTable& t, int blocks) {
        hipLaunchKernelGGL(squares_kernel, dim3(blocks), dim3(kClipThreads), 0, stream, t, part + parts);
        parts += blocks;
    });
    if (parts == 0) hipLaunchKernelGGL(scale_kernel, dim3(1), dim3(kClipThreads), 0, stream, ClipTable{}, part, 0, max_norm, norm);
    for_tables(tensors, n, [&](const ClipTable& t, int blocks) {
        hipLaunchKernelGGL(scale_kernel, dim3(blocks), dim3(kClipThreads), 0, stream, t, part, parts, max_norm, norm);
        norm = nullptr;
    });
    return check_launch("clip_norm");
}

}  // namespace svox_network
