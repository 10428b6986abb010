/*
 * svox_decoder.h -- C ABI of libsvox_decoder.so: the operators of a leaf decoder on AMD gfx950 (MI355X), layer norm
 * and the gated feed-forward block with their gradients.  (A leaf decoder is a small network that turns features kept
 * in the leaves of an N^3-tree into the records svox_hip.h's renderer reads.  The reference has no such operators.)
 *
 * Conventions, as in svox_hip.h
 *   - all pointers are device pointers valid on the current HIP device unless stated otherwise; `stream` is a
 *     hipStream_t carried as void* (NULL = the null stream); launches are asynchronous on it;
 *   - matrices are row-major; where a row stride is given it counts numbers, everything else is dense;
 *   - `dtype` is the type of every `void*` array of a call.  Sums, means and deviations are held in 32 bits;
 *   - workspaces are the caller's, at any address that is a whole number of 16; their contents need not outlive the call;
 *   - every function returns SVOX_OK (0) or a negative SvoxStatus; svox_decoder_last_error() returns a per-thread message
 *     for the last failing call; the library never allocates or frees device memory and keeps no state between calls;
 *   - arguments are checked before anything is launched.  Results do not depend on the order in which blocks run.
 */
#ifndef SVOX_DECODER_H_
#define SVOX_DECODER_H_

#include "svox_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define SVOX_DECODER_ABI_VERSION 1

typedef enum SvoxDecoderDType { SVOX_DECODER_F32 = 0, SVOX_DECODER_F16 = 1, SVOX_DECODER_BF16 = 2 } SvoxDecoderDType;

/* act(g): silu g / (1 + exp(-g)), gelu g Phi(g) with the normal distribution's Phi, relu max(g, 0), sigmoid 1 / (1 + exp(-g)) */
typedef enum SvoxActivation {
    SVOX_ACTIVATION_SILU = 0, SVOX_ACTIVATION_GELU = 1, SVOX_ACTIVATION_RELU = 2, SVOX_ACTIVATION_SIGMOID = 3
} SvoxActivation;

int svox_decoder_abi_version(void);
const char* svox_decoder_last_error(void);

/* y = (x - mean) / sqrt(variance + eps) * weight + bias, mean and variance (over dim, not dim - 1) of every row of x. */
typedef struct SvoxLayerNorm {
    const void* x;        /* (rows, dim), rows x_stride numbers apart */
    const void* weight;   /* (dim), or NULL: 1 */
    const void* bias;     /* (dim), or NULL: 0 */
    int64_t rows;         /* >= 0 */
    int64_t x_stride;     /* >= dim */
    int32_t dim;          /* >= 1 */
    int32_t dtype;
    float eps;
} SvoxLayerNorm;

/* y (rows, dim); stats (rows, 2), mean and 1 / sqrt(variance + eps) of every row, or NULL. */
int svox_layer_norm(const SvoxLayerNorm* spec, void* y, float* stats, void* stream);

/* The gradients of x (rows, dim), weight and bias (dim each), every one of them or NULL, from that of y (rows, dim), rows
 * grad_stride numbers apart, and the stats svox_layer_norm left.  spec->bias is not read. */
int svox_layer_norm_backward(const SvoxLayerNorm* spec, const float* stats, const void* grad_output, int64_t grad_stride,
                             void* grad_x, void* grad_weight, void* grad_bias, void* workspace, int64_t workspace_bytes,
                             void* stream);
/* The least workspace of svox_layer_norm_backward: 0 where neither weight's nor bias's gradient is asked for (`affine` 0). */
int64_t svox_layer_norm_workspace_bytes(const SvoxLayerNorm* spec, int32_t affine);

/* y = (act(x w_gate' + b_gate) * (x w_up' + b_up)) w_down' + b_down + residual
 * The products of float16 and bfloat16 take the hidden numbers, and their gradients, rounded to that type: in float16 those beyond 65504
 * become infinite and those below 2^-25 zero.  The products of float32 hold 24 bits throughout; an infinite number, or a finite one from
 * 3.396e38 on, makes NaN of the sums it is part of. */
typedef struct SvoxGatedFfn {
    const void* x;          /* (rows, dim), rows x_stride numbers apart */
    const void* w_gate;     /* (hidden, dim) */
    const void* w_up;       /* (hidden, dim) */
    const void* w_down;     /* (out, hidden) */
    const void* b_gate;     /* (hidden) or NULL: 0 */
    const void* b_up;       /* (hidden) or NULL: 0 */
    const void* b_down;     /* (out) or NULL: 0 */
    const void* residual;   /* (rows, out), rows residual_stride numbers apart, or NULL: 0 */
    int64_t rows;           /* >= 0 */
    int64_t x_stride, residual_stride;
    int32_t dim, hidden, out;   /* 1 .. 2^22 */
    int32_t dtype;
    int32_t activation;
} SvoxGatedFfn;

/* y (rows, out) */
int svox_gated_ffn(const SvoxGatedFfn* spec, void* y, void* workspace, int64_t workspace_bytes, void* stream);

/* Where the gradients go; NULL where one is not wanted.  (That of the residual is grad_output itself.) */
typedef struct SvoxGatedFfnGrads {
    void *x, *w_gate, *w_up, *w_down, *b_gate, *b_up, *b_down;   /* shaped like the inputs, dense */
} SvoxGatedFfnGrads;

/* grad_output (rows, out), rows grad_stride numbers apart.  The hidden numbers are computed again from x; spec->residual and
 * spec->b_down are not read. */
int svox_gated_ffn_backward(const SvoxGatedFfn* spec, const void* grad_output, int64_t grad_stride, const SvoxGatedFfnGrads* grads,
                            void* workspace, int64_t workspace_bytes, void* stream);

/* The least workspace of svox_gated_ffn (backward 0) or svox_gated_ffn_backward (1), or a negative SvoxStatus. */
int64_t svox_gated_ffn_workspace_bytes(const SvoxGatedFfn* spec, int32_t backward);

#ifdef __cplusplus
}
#endif
#endif /* SVOX_DECODER_H_ */
