/*
 * svox_network.h -- C ABI of libsvox_network.so: operators of networks over the cells of an N^3-tree on AMD gfx950 (MI355X):
 * attention within packed sequences of cells, the norms of queries and keys with the rotation by their positions, and the norm
 * of many gradients with its clipping.  (The reference has no such operators.)
 *
 * Conventions, as in svox_decoder.h
 *   - all pointers are device pointers valid on the current HIP device unless stated otherwise; `stream` is a
 *     hipStream_t carried as void* (NULL = the null stream); launches are asynchronous on it;
 *   - strides count numbers; everything without one is dense and row-major;
 *   - `dtype` is an SvoxDecoderDType, the type of every `void*` array of a call.  Sums and statistics are held in 32 bits or more;
 *   - workspaces are the caller's, at any address that is a whole number of 16; their contents need not outlive the call;
 *   - every function returns SVOX_OK (0) or a negative SvoxStatus; svox_network_last_error() returns a per-thread message
 *     for the last failing call; the library never allocates or frees device memory and keeps no state between calls;
 *   - arguments are checked before anything is launched.  Results do not depend on the order in which blocks run.
 */
#ifndef SVOX_NETWORK_H_
#define SVOX_NETWORK_H_

#include "svox_decoder.h"

#ifdef __cplusplus
extern "C" {
#endif

#define SVOX_NETWORK_ABI_VERSION 1

int svox_network_abi_version(void);
const char* svox_network_last_error(void);

/* One of the tensors of svox_clip_norm: `count` numbers, from `from` to `to` (which may be `from`). */
typedef struct SvoxClipTensor {
    const void* from;
    void* to;
    int64_t count;   /* >= 0 */
    int32_t dtype;
} SvoxClipTensor;

/* norm (one float) = the square root of the sum of the squares of all numbers, summed in 64 bits;
 * to = from * (max_norm / norm) where max_norm < norm < infinity, else from as it is.
 * `tensors` is an array in host memory; it is read before the call returns.  Tensors may not overlap others' `to`. */
int svox_clip_norm(const SvoxClipTensor* tensors, int64_t n, double max_norm, float* norm, void* workspace, int64_t workspace_bytes,
                   void* stream);
int64_t svox_clip_norm_workspace_bytes(const SvoxClipTensor* tensors, int64_t n);

/* Heads x of queries and keys, each divided by the root of the mean of its squares and then rotated by the row's positions:
 *   n = x / sqrt(mean(x^2) + eps) * weight
 *   angle_i = sum over axes of positions[row, axis] * frequencies[axis, i]     (in 64 bits),  i < rotated / 2
 *   y_a = n_a cos(angle_i) - n_b sin(angle_i),  y_b = n_b cos(angle_i) + n_a sin(angle_i)
 * with (a, b) = (i, i + rotated / 2), or (2 i, 2 i + 1) where `interleaved`; y = n from number `rotated` on. */
typedef enum SvoxPositionType { SVOX_POSITIONS_F32 = 0, SVOX_POSITIONS_F64 = 1, SVOX_POSITIONS_I32 = 2, SVOX_POSITIONS_I64 = 3 } SvoxPositionType;

typedef struct SvoxRotateHeads {
    const void *q, *k;                  /* (rows, heads, dim) and (rows, kv_heads, dim); a head's numbers lie side by side */
    const void *q_weight, *k_weight;    /* (dim), or NULL: 1 */
    const void* positions;              /* (rows, axes) */
    const float* frequencies;           /* (axes, rotated / 2) */
    int64_t rows;                       /* >= 0 */
    int64_t q_stride, q_head, k_stride, k_head;   /* from row to row and from head to head */
    int32_t heads, kv_heads;            /* >= 1 */
    int32_t dim;                        /* 1 .. 256 */
    int32_t rotated;                    /* even, 0 .. dim */
    int32_t axes;                       /* 1 .. 4 */
    int32_t interleaved, dtype, position_type;
    float eps;
} SvoxRotateHeads;

/* y_q (rows, heads, dim) and y_k (rows, kv_heads, dim) */
int svox_rotate_heads(const SvoxRotateHeads* spec, void* y_q, void* y_k, void* stream);

/* The gradients of q, k and their weights, each of them or NULL, from those of y_q and y_k, whose strides are `grad`'s: from row to row
 * and from head to head of y_q, then of y_k. */
int svox_rotate_heads_backward(const SvoxRotateHeads* spec, const void* grad_q, const void* grad_k, const int64_t grad[4], void* out_q,
                               void* out_k, void* out_q_weight, void* out_k_weight, void* workspace, int64_t workspace_bytes,
                               void* stream);
/* The least workspace of svox_rotate_heads_backward: 0 where no weight's gradient is asked for (`weights` 0). */
int64_t svox_rotate_heads_workspace_bytes(const SvoxRotateHeads* spec, int32_t weights);

/* Attention within packed sequences: sequence s holds queries offsets[s] .. offsets[s + 1] - 1 and keys key_offsets[s] ..
 * key_offsets[s + 1] - 1; a query sees the keys of its own sequence, all of them, or where `causal` those up to its own place counted from
 * the sequences' ends (query i of a sees keys up to i + b - a of b).  Query head h goes with kv head h / (heads / kv_heads).
 *   out = sum over keys of softmax(scale q . k) v;  0 where a query sees no key or belongs to no sequence
 * What the offsets hold is read on the GPU and not checked: places outside of 0 .. queries (keys) count as the nearest inside, and what
 * sequences that are not in order give is unspecified, but nothing outside of the arrays is read or written. */
typedef struct SvoxAttention {
    const void *q, *k, *v;       /* (queries, heads, dim), (keys, kv_heads, dim) twice; a head's numbers lie side by side */
    const void* offsets;         /* (sequences + 1) int32, or int64 where wide_offsets; NULL: one sequence of all */
    const void* key_offsets;     /* the same of the keys; NULL: as offsets */
    int64_t queries, keys;       /* >= 0; queries * heads / kv_heads and keys < 2^31 - 2^10, queries * heads and keys * kv_heads < 2^31 - 2^13 where
                                  * the rows, or keys, of a kv head count in whole 128s */
    int64_t sequences;           /* >= 1 (1 without offsets) */
    int64_t q_stride, q_head, k_stride, k_head, v_stride, v_head;   /* from row to row and from head to head */
    int32_t heads, kv_heads;     /* heads a multiple of kv_heads */
    int32_t dim;                 /* 1 .. 128 */
    int32_t dtype, wide_offsets, causal;
    float scale;                 /* > 0 */
} SvoxAttention;

/* out (queries, heads, dim).  What svox_attention_backward needs besides, or NULL: lse (queries * heads floats), of the scores' sums; rest
 * (queries, heads, dim), what rounding to 16 bits took from out (of float16 times 2^11). */
int svox_attention(const SvoxAttention* spec, void* out, float* lse, void* rest, void* workspace, int64_t workspace_bytes, void* stream);

typedef struct SvoxAttentionGrads {
    const void* out;                      /* what svox_attention left */
    const float* lse;
    const void* rest;                     /* or NULL: 0 */
    const void* grad;                     /* of out, (queries, heads, dim) */
    int64_t grad_stride, grad_head;       /* from row to row and from head to head */
    void *q, *k, *v;                      /* where the gradients go, dense; NULL where one is not wanted */
} SvoxAttentionGrads;

int svox_attention_backward(const SvoxAttention* spec, const SvoxAttentionGrads* grads, void* workspace, int64_t workspace_bytes, void* stream);

/* The least workspace of svox_attention (backward 0) or svox_attention_backward (1), or a negative SvoxStatus. */
int64_t svox_attention_workspace_bytes(const SvoxAttention* spec, int32_t backward);

#ifdef __cplusplus
}
#endif
#endif /* SVOX_NETWORK_H_ */
