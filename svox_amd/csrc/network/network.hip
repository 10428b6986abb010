// network.hip -- the extern "C" entry points of libsvox_network.so (declared in include/svox_network.h): argument checks and the
// choice of a type's kernels.
#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "../decoder/common.h"
#include "attention_rules.h"
#include "entry.h"
#include "rotate_kernels.h"

namespace svox_decoder {

static thread_local char g_error[512] = "";

int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_error, sizeof(g_error), fmt, ap);
    va_end(ap);
    return code;
}
int check_launch(const char* what) {
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return fail(SVOX_ERR_LAUNCH, "%s: %s", what, hipGetErrorString(err));
    return SVOX_OK;
}

}  // namespace svox_decoder

namespace svox_network {
namespace {

#define SVOX_TRY(call)                  \
    do {                                \
        const int rc_ = (call);         \
        if (rc_ != SVOX_OK) return rc_; \
    } while (0)

#define SVOX_BY_TYPE(dtype, ...)                                                   \
    switch (dtype) {                                                               \
        case SVOX_DECODER_F32: { using T = float; __VA_ARGS__; }                   \
        case SVOX_DECODER_F16: { using T = svox_decoder::F16; __VA_ARGS__; }       \
        default: { using T = svox_decoder::Bf16; __VA_ARGS__; }                    \
    }

// (2^46 numbers of a tensor: far more than a GPU holds, and products of sizes and strides stay below 2^63)
constexpr int64_t kMost = (int64_t)1 << 46;
constexpr int kMostHeads = 1 << 20;

int check_dtype(int dtype) {
    if (dtype < SVOX_DECODER_F32 || dtype > SVOX_DECODER_BF16) return fail(SVOX_ERR_BAD_DTYPE, "dtype must be 0, 1 or 2, got %d", dtype);
    return SVOX_OK;
}
int check_space(const void* workspace, int64_t bytes, int64_t least) {
    if (least <= 0) return SVOX_OK;
    if (!workspace) return fail(SVOX_ERR_NULL_POINTER, "the workspace is NULL");
    if ((uintptr_t)workspace % 16) return fail(SVOX_ERR_BAD_SHAPE, "the workspace does not begin at a whole number of 16 bytes");
    if (bytes < least) return fail(SVOX_ERR_BAD_SHAPE, "the workspace has %lld bytes, the call needs %lld", (long long)bytes, (long long)least);
    return SVOX_OK;
}
// (rows, heads, dim) with the last dimension dense.  Rows and heads may lie any distance apart, also none: they are read only.
int check_heads(const char* name, const void* at, int64_t rows, int64_t heads, int64_t row_stride, int64_t head_stride) {
    if (!at && rows > 0) return fail(SVOX_ERR_NULL_POINTER, "%s is NULL", name);
    if (row_stride < 0 || head_stride < 0) return fail(SVOX_ERR_BAD_SHAPE, "%s: strides must be >= 0", name);
    if (row_stride > kMost || head_stride > kMost || (rows > 0 && row_stride > kMost / rows) || head_stride > kMost / heads)
        return fail(SVOX_ERR_BAD_SHAPE, "%s is too large to index", name);
    return SVOX_OK;
}

int check_clip(const SvoxClipTensor* tensors, int64_t n) {
    if (n < 0) return fail(SVOX_ERR_BAD_SHAPE, "the number of tensors must be >= 0, got %lld", (long long)n);
    if (n > 0 && !tensors) return fail(SVOX_ERR_NULL_POINTER, "tensors is NULL");
    int64_t total = 0;
    for (int64_t i = 0; i < n; ++i) {
        SVOX_TRY(check_dtype(tensors[i].dtype));
        if (tensors[i].count < 0) return fail(SVOX_ERR_BAD_SHAPE, "count must be >= 0, got %lld", (long long)tensors[i].count);
        if (tensors[i].count > kMost || (total += tensors[i].count) > kMost) return fail(SVOX_ERR_BAD_SHAPE, "tensors are too large to index");
        if (tensors[i].count > 0 && (!tensors[i].from || !tensors[i].to)) return fail(SVOX_ERR_NULL_POINTER, "tensor %lld is NULL", (long long)i);
    }
    return SVOX_OK;
}

int check_rotate(const SvoxRotateHeads* s) {
    if (!s) return fail(SVOX_ERR_NULL_POINTER, "the spec is NULL");
    SVOX_TRY(check_dtype(s->dtype));
    if (s->rows < 0) return fail(SVOX_ERR_BAD_SHAPE, "rows must be >= 0, got %lld", (long long)s->rows);
    if (s->heads < 1 || s->kv_heads < 1 || s->heads > kMostHeads || s->kv_heads > kMostHeads)
        return fail(SVOX_ERR_BAD_SHAPE, "heads and kv_heads must be between 1 and %d, got %d and %d", kMostHeads, s->heads, s->kv_heads);
    if (s->dim < 1) return fail(SVOX_ERR_BAD_SHAPE, "dim must be >= 1, got %d", s->dim);
    if (s->dim > kRotateMostDim) return fail(SVOX_ERR_UNSUPPORTED, "dim must be <= %d, got %d", kRotateMostDim, s->dim);
    if (s->rotated < 0 || s->rotated > s->dim || s->rotated % 2)
        return fail(SVOX_ERR_BAD_SHAPE, "rotated must be an even number up to dim, got %d of %d", s->rotated, s->dim);
    if (s->axes < 1 || s->axes > 4) return fail(SVOX_ERR_BAD_SHAPE, "axes must be between 1 and 4, got %d", s->axes);
    if (s->position_type < SVOX_POSITIONS_F32 || s->position_type > SVOX_POSITIONS_I64)
        return fail(SVOX_ERR_BAD_DTYPE, "position_type must be 0, 1, 2 or 3, got %d", s->position_type);
    if (s->rows > kMost / ((int64_t)s->dim * (s->heads > s->kv_heads ? s->heads : s->kv_heads))) return fail(SVOX_ERR_BAD_SHAPE, "q or k is too large to index");
    SVOX_TRY(check_heads("q", s->q, s->rows, s->heads, s->q_stride, s->q_head));
    SVOX_TRY(check_heads("k", s->k, s->rows, s->kv_heads, s->k_stride, s->k_head));
    if (s->rows > 0 && s->rotated > 0 && (!s->positions || !s->frequencies)) return fail(SVOX_ERR_NULL_POINTER, "positions or frequencies are NULL");
    return SVOX_OK;
}
int64_t rotate_space(const SvoxRotateHeads& s, bool weights) {
    if (!weights || s.rows == 0) return 0;
    int64_t blocks = 0;
    const auto count = [&]() -> int64_t { SVOX_BY_TYPE(s.dtype, return rotate_backward_blocks<T>(s)); };
    blocks = count();
    return blocks * 2 * s.dim * (int64_t)sizeof(float);
}

int check_attention(const SvoxAttention* s) {
    if (!s) return fail(SVOX_ERR_NULL_POINTER, "the spec is NULL");
    SVOX_TRY(check_dtype(s->dtype));
    if (s->queries < 0 || s->keys < 0) return fail(SVOX_ERR_BAD_SHAPE, "queries and keys must be >= 0, got %lld and %lld", (long long)s->queries, (long long)s->keys);
    if (s->heads < 1 || s->kv_heads < 1 || s->heads > kMostHeads || s->heads % s->kv_heads)
        return fail(SVOX_ERR_BAD_SHAPE, "heads must be a multiple of kv_heads and between 1 and %d, got %d and %d", kMostHeads, s->heads, s->kv_heads);
    if (s->dim < 1) return fail(SVOX_ERR_BAD_SHAPE, "dim must be >= 1, got %d", s->dim);
    if (s->dim > 128) return fail(SVOX_ERR_UNSUPPORTED, "dim must be <= 128, got %d", s->dim);
    if (!(s->scale > 0.0f) || std::isinf(s->scale)) return fail(SVOX_ERR_BAD_SHAPE, "scale must be > 0 and finite, got %g", (double)s->scale);
    if (s->sequences < 1 || s->sequences > INT32_MAX - 1024) return fail(SVOX_ERR_BAD_SHAPE, "sequences must be between 1 and 2^31 - 2^10, got %lld", (long long)s->sequences);
    if (!s->offsets && (s->key_offsets || s->sequences != 1)) return fail(SVOX_ERR_NULL_POINTER, "offsets is NULL");
    if (s->offsets && !s->key_offsets && s->queries != s->keys)
        return fail(SVOX_ERR_BAD_SHAPE, "without key_offsets there must be as many keys as queries, got %lld and %lld", (long long)s->keys, (long long)s->queries);
    // (rows of a kv head are counted in 32 bits, and a launch has fewer than 2^24 blocks of 128 of them, also where their number is made a whole one of runs)
    const int64_t most = INT32_MAX - 1024, rows = s->heads / s->kv_heads;
    if (s->keys > most || s->queries > most / rows) return fail(SVOX_ERR_UNSUPPORTED, "queries * heads / kv_heads and keys must be < 2^31 - 2^10");
    for (const int64_t tiles : {svox_decoder::pieces(s->queries * rows, 128), svox_decoder::pieces(s->keys, 128)})
        if ((tiles + 1) * s->kv_heads >= 1 << 24 || (in_runs(*s, tiles) && in_whole_runs(tiles * s->kv_heads) >= 1 << 24))
            return fail(SVOX_ERR_UNSUPPORTED, "queries * heads and keys * kv_heads must be < 2^31 - 2^13");
    SVOX_TRY(check_heads("q", s->q, s->queries, s->heads, s->q_stride, s->q_head));
    SVOX_TRY(check_heads("k", s->k, s->keys, s->kv_heads, s->k_stride, s->k_head));
    return check_heads("v", s->v, s->keys, s->kv_heads, s->v_stride, s->v_head);
}
// the kernels of a call's type and width
#define SVOX_BY_TYPE_AND_WIDTH(s, ...)                              \
    SVOX_BY_TYPE((s).dtype, switch (attend_width((s).dim)) {        \
        case 32: { constexpr int width = 32; __VA_ARGS__; }         \
        case 64: { constexpr int width = 64; __VA_ARGS__; }         \
        default: { constexpr int width = 128; __VA_ARGS__; }        \
    })

// a gradient summed over no rows
__global__ void zero_kernel(uint16_t* at, int64_t count) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) at[i] = 0;
}
int zero(void* at, int64_t count, int dtype, hipStream_t stream) {
    if (!at || count == 0) return SVOX_OK;
    count *= dtype == SVOX_DECODER_F32 ? 2 : 1;
    hipLaunchKernelGGL(zero_kernel, grid_of(svox_decoder::least(svox_decoder::pieces(count, 256), 1 << 16), 256), dim3(256), 0, stream, (uint16_t*)at, count);
    return check_launch("zero");
}

}  // namespace
}  // namespace svox_network

using namespace svox_network;

#define SVOX_API extern "C" __attribute__((visibility("default")))

SVOX_API int svox_network_abi_version(void) { return SVOX_NETWORK_ABI_VERSION; }
SVOX_API const char* svox_network_last_error(void) { return svox_decoder::g_error; }

SVOX_API int64_t svox_clip_norm_workspace_bytes(const SvoxClipTensor* tensors, int64_t n) {
    SVOX_TRY(check_clip(tensors, n));
    return clip_blocks(tensors, n) * (int64_t)sizeof(double);
}

SVOX_API int svox_clip_norm(const SvoxClipTensor* tensors, int64_t n, double max_norm, float* norm, void* workspace, int64_t workspace_bytes,
                            void* stream) {
    SVOX_TRY(check_clip(tensors, n));
    if (!(max_norm >= 0.0)) return fail(SVOX_ERR_BAD_SHAPE, "max_norm must be >= 0, got %g", max_norm);
    if (!norm) return fail(SVOX_ERR_NULL_POINTER, "norm is NULL");
    SVOX_TRY(check_space(workspace, workspace_bytes, clip_blocks(tensors, n) * (int64_t)sizeof(double)));
    return launch_clip(tensors, n, max_norm, norm, (double*)workspace, (hipStream_t)stream);
}

SVOX_API int svox_rotate_heads(const SvoxRotateHeads* spec, void* y_q, void* y_k, void* stream) {
    SVOX_TRY(check_rotate(spec));
    if (spec->rows == 0) return SVOX_OK;
    if (!y_q || !y_k) return fail(SVOX_ERR_NULL_POINTER, "y_q or y_k is NULL");
    SVOX_BY_TYPE(spec->dtype, return launch_rotate<T>(*spec, y_q, y_k, (hipStream_t)stream));
}

SVOX_API int64_t svox_rotate_heads_workspace_bytes(const SvoxRotateHeads* spec, int32_t weights) {
    SVOX_TRY(check_rotate(spec));
    return rotate_space(*spec, weights != 0);
}

SVOX_API int svox_rotate_heads_backward(const SvoxRotateHeads* spec, const void* grad_q, const void* grad_k, const int64_t grad[4], void* out_q,
                                        void* out_k, void* out_q_weight, void* out_k_weight, void* workspace, int64_t workspace_bytes,
                                        void* stream) {
    SVOX_TRY(check_rotate(spec));
    if (!grad) return fail(SVOX_ERR_NULL_POINTER, "the strides of grad_q and grad_k are NULL");
    if (spec->rows == 0) {
        SVOX_TRY(zero(out_q_weight, spec->dim, spec->dtype, (hipStream_t)stream));
        return zero(out_k_weight, spec->dim, spec->dtype, (hipStream_t)stream);
    }
    SVOX_TRY(check_heads("grad_q", grad_q, spec->rows, spec->heads, grad[0], grad[1]));
    SVOX_TRY(check_heads("grad_k", grad_k, spec->rows, spec->kv_heads, grad[2], grad[3]));
    const bool weights = out_q_weight || out_k_weight;
    if (!weights && !out_q && !out_k) return SVOX_OK;
    SVOX_TRY(check_space(workspace, workspace_bytes, rotate_space(*spec, weights)));
    SVOX_BY_TYPE(spec->dtype, return launch_rotate_backward<T>(*spec, grad_q, grad_k, grad, out_q, out_k, out_q_weight, out_k_weight,
                                                               weights ? (float*)workspace : nullptr, (hipStream_t)stream));
}

SVOX_API int64_t svox_attention_workspace_bytes(const SvoxAttention* spec, int32_t backward) {
    SVOX_TRY(check_attention(spec));
    return attention_space(*spec, backward != 0);
}

SVOX_API int svox_attention(const SvoxAttention* spec, void* out, float* lse, void* rest, void* workspace, int64_t workspace_bytes, void* stream) {
    SVOX_TRY(check_attention(spec));
    if (spec->queries == 0) return SVOX_OK;
    if (!out) return fail(SVOX_ERR_NULL_POINTER, "out is NULL");
    SVOX_TRY(check_space(workspace, workspace_bytes, attention_space(*spec, false)));
    SVOX_BY_TYPE_AND_WIDTH(*spec, return (launch_attention<T, width>(*spec, out, lse, rest, workspace, (hipStream_t)stream)));
}

SVOX_API int svox_attention_backward(const SvoxAttention* spec, const SvoxAttentionGrads* grads, void* workspace, int64_t workspace_bytes, void* stream) {
    SVOX_TRY(check_attention(spec));
    if (!grads) return fail(SVOX_ERR_NULL_POINTER, "grads is NULL");
    if (!grads->q && !grads->k && !grads->v) return SVOX_OK;
    SVOX_TRY(check_heads("grad", grads->grad, spec->queries, spec->heads, grads->grad_stride, grads->grad_head));
    if (spec->queries > 0 && (!grads->out || !grads->lse)) return fail(SVOX_ERR_NULL_POINTER, "out or lse is NULL");
    SVOX_TRY(check_space(workspace, workspace_bytes, attention_space(*spec, true)));
    SVOX_BY_TYPE_AND_WIDTH(*spec, return (launch_attention_backward<T, width>(*spec, *grads, workspace, (hipStream_t)stream)));
}
