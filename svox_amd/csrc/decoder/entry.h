// entry.h -- what the units of libsvox_decoder.so share on the host: the launches of each type.
#pragma once
#include "../../../include/svox_decoder.h"
#include "launch.h"

namespace svox_decoder {

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
