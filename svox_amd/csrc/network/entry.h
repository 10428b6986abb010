// entry.h -- what the units of libsvox_network.so share on the host: the launches of each type (arguments are checked before).
#pragma once
#include "../../../include/svox_network.h"
#include "../decoder/launch.h"

namespace svox_network {

using svox_decoder::check_launch;
using svox_decoder::fail;
using svox_decoder::grid_of;
using svox_decoder::Room;

// clip.hip
int64_t clip_blocks(const SvoxClipTensor* tensors, int64_t n);
int launch_clip(const SvoxClipTensor* tensors, int64_t n, double max_norm, float* norm, double* part, hipStream_t stream);

// (defined for every type in rotate_type.hip)
template <class T>
int launch_rotate(const SvoxRotateHeads& s, void* y_q, void* y_k, hipStream_t stream);
template <class T>
int launch_rotate_backward(const SvoxRotateHeads& s, const void* grad_q, const void* grad_k, const int64_t* grad, void* out_q, void* out_k,
                           void* out_q_weight, void* out_k_weight, float* part, hipStream_t stream);
template <class T>
int rotate_backward_blocks(const SvoxRotateHeads& s);   // each with a row of partial sums

// (defined for every type and width in attention_type.hip)
template <class T, int width>
int launch_attention(const SvoxAttention& s, void* out, float* lse, void* rest, void* workspace, hipStream_t stream);
template <class T, int width>
int launch_attention_backward(const SvoxAttention& s, const SvoxAttentionGrads& grads, void* workspace, hipStream_t stream);

}  // namespace svox_network
