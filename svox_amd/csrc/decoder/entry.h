// entry.h -- what the units of libsvox_decoder.so share on the host: errors, and the launches of each type.
#pragma once
#include <hip/hip_runtime.h>

#include "../../../include/svox_decoder.h"

namespace svox_decoder {

__attribute__((format(printf, 2, 3))) int fail(int code, const char* fmt, ...);
int check_launch(const char* what);

// `blocks` blocks of a launch.  The runtime counts a launch's threads along each axis in 32 bits and runs what is left of a larger number,
// without an error (of the 16 777 218 blocks of 256 that 2^30 + 77 rows came to it ran two): such a launch gets no blocks here, which is
// an error that check_launch sees.
inline dim3 grid_of(int64_t blocks, int threads) { return dim3(blocks < ((int64_t)1 << 32) / threads ? (unsigned)blocks : 0); }

// A caller's workspace, given out in pieces of whole 256 bytes; with no address, only counted.
struct Room {
    char* at;
    int64_t used = 0;
    explicit Room(void* base) : at((char*)base) {}
    template <class T>
    T* take(int64_t count) {
        T* const p = at ? (T*)(at + used) : nullptr;
        used += (count * (int64_t)sizeof(T) + 255) / 256 * 256;
        return p;
    }
};

// (defined for every type in norm_type.hip and ffn_type.hip; arguments are checked before)
template <class T>
int launch_norm(const SvoxLayerNorm& s, void* y, float* stats, hipStream_t stream);
template <class T>
int launch_norm_backward(const SvoxLayerNorm& s, const float* stats, const void* grad_output, int64_t grad_stride, void* grad_x,
                         void* grad_weight, void* grad_bias, float* part, hipStream_t stream);
int norm_backward_blocks(int64_t rows, int dim, int piece);

template <class T>
int64_t ffn_workspace(const SvoxGatedFfn& s, bool backward);
template <class T>
int launch_ffn(const SvoxGatedFfn& s, void* y, void* workspace, hipStream_t stream);
template <class T>
int launch_ffn_backward(const SvoxGatedFfn& s, const void* grad_output, int64_t grad_stride, const SvoxGatedFfnGrads& grads, void* workspace,
                        hipStream_t stream);

}  // namespace svox_decoder
