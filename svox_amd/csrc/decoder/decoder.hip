// decoder.hip -- the extern "C" entry points of libsvox_decoder.so (declared in include/svox_decoder.h): argument checks and
// the choice of a type's kernels.
#include <cstdarg>
#include <cstdio>

#include "common.h"
#include "entry.h"

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

// The blocks of a backward pass of layer norm, each with a row of partial sums: as many as the GPU runs at once, where there are
// rows for them.
int norm_backward_blocks(int64_t rows, int dim, int piece) {
    const int64_t row_pieces = pieces(dim, piece);
    int lanes = 4;
    while (lanes < 64 && lanes < row_pieces) lanes *= 2;
    if (row_pieces > 256) lanes = 256;
    const int64_t blocks = pieces(rows, 256 / lanes);
    return (int)(blocks < 1024 ? blocks : 1024);
}

namespace {

// (2^46 numbers of a matrix: far more than a GPU holds, and products of sizes and strides stay below 2^63)
constexpr int64_t kMost = (int64_t)1 << 46;
int check_matrix(const char* name, const void* at, int64_t rows, int64_t cols, int64_t stride) {
    if (!at && rows > 0) return fail(SVOX_ERR_NULL_POINTER, "%s is NULL", name);
    if (stride < cols) return fail(SVOX_ERR_BAD_SHAPE, "%s: a row of %lld numbers does not fit a stride of %lld", name, (long long)cols, (long long)stride);
    if (stride > kMost || (rows > 0 && stride > kMost / rows)) return fail(SVOX_ERR_BAD_SHAPE, "%s is too large to index", name);
    return SVOX_OK;
}
int check_dtype(int dtype) {
    if (dtype < SVOX_DECODER_F32 || dtype > SVOX_DECODER_BF16) return fail(SVOX_ERR_BAD_DTYPE, "dtype must be 0, 1 or 2, got %d", dtype);
    return SVOX_OK;
}
#define SVOX_TRY(call)                  \
    do {                                \
        const int rc_ = (call);         \
        if (rc_ != SVOX_OK) return rc_; \
    } while (0)

int check_norm(const SvoxLayerNorm* s) {
    if (!s) return fail(SVOX_ERR_NULL_POINTER, "the spec is NULL");
    SVOX_TRY(check_dtype(s->dtype));
    if (s->rows < 0) return fail(SVOX_ERR_BAD_SHAPE, "rows must be >= 0, got %lld", (long long)s->rows);
    if (s->dim < 1) return fail(SVOX_ERR_BAD_SHAPE, "dim must be >= 1, got %d", s->dim);
    return check_matrix("x", s->x, s->rows, s->dim, s->x_stride);
}

constexpr int kMostWidth = 1 << 22;   // (tiles of longer rows would leave the range of 32-bit offsets)
int check_ffn(const SvoxGatedFfn* s) {
    if (!s) return fail(SVOX_ERR_NULL_POINTER, "the spec is NULL");
    SVOX_TRY(check_dtype(s->dtype));
    if (s->rows < 0) return fail(SVOX_ERR_BAD_SHAPE, "rows must be >= 0, got %lld", (long long)s->rows);
    if (s->dim < 1 || s->hidden < 1 || s->out < 1)
        return fail(SVOX_ERR_BAD_SHAPE, "dim, hidden and out must be >= 1, got %d, %d, %d", s->dim, s->hidden, s->out);
    if (s->dim > kMostWidth || s->hidden > kMostWidth || s->out > kMostWidth)
        return fail(SVOX_ERR_UNSUPPORTED, "dim, hidden and out must be <= %d, got %d, %d, %d", kMostWidth, s->dim, s->hidden, s->out);
    if (s->activation < SVOX_ACTIVATION_SILU || s->activation > SVOX_ACTIVATION_SIGMOID)
        return fail(SVOX_ERR_UNSUPPORTED, "unknown activation %d", s->activation);
    SVOX_TRY(check_matrix("x", s->x, s->rows, s->dim, s->x_stride));
    SVOX_TRY(check_matrix("w_gate", s->w_gate, s->hidden, s->dim, s->dim));
    SVOX_TRY(check_matrix("w_up", s->w_up, s->hidden, s->dim, s->dim));
    SVOX_TRY(check_matrix("w_down", s->w_down, s->out, s->hidden, s->hidden));
    SVOX_TRY(check_matrix("the hidden numbers", s, s->rows, s->hidden, (int64_t)s->hidden + 8));
    SVOX_TRY(check_matrix("y", s, s->rows, s->out, s->out));
    if (s->residual) SVOX_TRY(check_matrix("residual", s->residual, s->rows, s->out, s->residual_stride));
    return SVOX_OK;
}
int check_space(const void* workspace, int64_t bytes, int64_t least) {
    if (least <= 0) return SVOX_OK;
    if (!workspace) return fail(SVOX_ERR_NULL_POINTER, "the workspace is NULL");
    if ((uintptr_t)workspace % 16) return fail(SVOX_ERR_BAD_SHAPE, "the workspace does not begin at a whole number of 16 bytes");
    if (bytes < least) return fail(SVOX_ERR_BAD_SHAPE, "the workspace has %lld bytes, the call needs %lld", (long long)bytes, (long long)least);
    return SVOX_OK;
}

#define SVOX_BY_TYPE(dtype, ...)                                                   \
    switch (dtype) {                                                               \
        case SVOX_DECODER_F32: { using T = float; __VA_ARGS__; }                   \
        case SVOX_DECODER_F16: { using T = svox_decoder::F16; __VA_ARGS__; }       \
        default: { using T = svox_decoder::Bf16; __VA_ARGS__; }                    \
    }

int64_t norm_space(const SvoxLayerNorm& s, bool affine) {
    if (!affine || s.rows == 0) return 0;
    return (int64_t)norm_backward_blocks(s.rows, s.dim, s.dtype == SVOX_DECODER_F32 ? 4 : 8) * 2 * s.dim * (int64_t)sizeof(float);
}

// a gradient summed over no rows
__global__ void zero_kernel(u16* at, int64_t count) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) at[i] = 0;
}
int zero(void* at, int64_t count, int dtype, hipStream_t stream) {
    if (!at) return SVOX_OK;
    count *= dtype == SVOX_DECODER_F32 ? 2 : 1;
    hipLaunchKernelGGL(zero_kernel, grid_of(least(pieces(count, 256), 1 << 16), 256), dim3(256), 0, stream, (u16*)at, count);
    return check_launch("zero");
}

}  // namespace
}  // namespace svox_decoder

using namespace svox_decoder;

#define SVOX_API extern "C" __attribute__((visibility("default")))

SVOX_API int svox_decoder_abi_version(void) { return SVOX_DECODER_ABI_VERSION; }
SVOX_API const char* svox_decoder_last_error(void) { return g_error; }

SVOX_API int svox_layer_norm(const SvoxLayerNorm* spec, void* y, float* stats, void* stream) {
    SVOX_TRY(check_norm(spec));
    if (spec->rows == 0) return SVOX_OK;
    if (!y) return fail(SVOX_ERR_NULL_POINTER, "y is NULL");
    SVOX_BY_TYPE(spec->dtype, return launch_norm<T>(*spec, y, stats, (hipStream_t)stream));
}

SVOX_API int64_t svox_layer_norm_workspace_bytes(const SvoxLayerNorm* spec, int32_t affine) {
    SVOX_TRY(check_norm(spec));
    return norm_space(*spec, affine != 0);
}

SVOX_API int svox_layer_norm_backward(const SvoxLayerNorm* spec, const float* stats, const void* grad_output, int64_t grad_stride,
                                      void* grad_x, void* grad_weight, void* grad_bias, void* workspace, int64_t workspace_bytes,
                                      void* stream) {
    SVOX_TRY(check_norm(spec));
    if (spec->rows == 0) {
        SVOX_TRY(zero(grad_weight, spec->dim, spec->dtype, (hipStream_t)stream));
        return zero(grad_bias, spec->dim, spec->dtype, (hipStream_t)stream);
    }
    SVOX_TRY(check_matrix("grad_output", grad_output, spec->rows, spec->dim, grad_stride));
    if (!stats) return fail(SVOX_ERR_NULL_POINTER, "stats is NULL");
    const bool affine = grad_weight || grad_bias;
    if (!affine && !grad_x) return SVOX_OK;
    SVOX_TRY(check_space(workspace, workspace_bytes, norm_space(*spec, affine)));
    SVOX_BY_TYPE(spec->dtype, return launch_norm_backward<T>(*spec, stats, grad_output, grad_stride, grad_x, grad_weight, grad_bias,
                                                             affine ? (float*)workspace : nullptr, (hipStream_t)stream));
}

SVOX_API int64_t svox_gated_ffn_workspace_bytes(const SvoxGatedFfn* spec, int32_t backward) {
    SVOX_TRY(check_ffn(spec));
    if (spec->rows == 0) return 0;
    SVOX_BY_TYPE(spec->dtype, return ffn_workspace<T>(*spec, backward != 0));
}

SVOX_API int svox_gated_ffn(const SvoxGatedFfn* spec, void* y, void* workspace, int64_t workspace_bytes, void* stream) {
    SVOX_TRY(check_ffn(spec));
    if (spec->rows == 0) return SVOX_OK;
    if (!y) return fail(SVOX_ERR_NULL_POINTER, "y is NULL");
    SVOX_BY_TYPE(spec->dtype, {
        SVOX_TRY(check_space(workspace, workspace_bytes, ffn_workspace<T>(*spec, false)));
        return launch_ffn<T>(*spec, y, workspace, (hipStream_t)stream);
    });
}

SVOX_API int svox_gated_ffn_backward(const SvoxGatedFfn* spec, const void* grad_output, int64_t grad_stride, const SvoxGatedFfnGrads* grads,
                                     void* workspace, int64_t workspace_bytes, void* stream) {
    SVOX_TRY(check_ffn(spec));
    if (!grads) return fail(SVOX_ERR_NULL_POINTER, "grads is NULL");
    if (spec->rows == 0) {
        const int64_t wide = (int64_t)spec->hidden * spec->dim, down = (int64_t)spec->hidden * spec->out;
        void* const at[6] = {grads->w_gate, grads->w_up, grads->w_down, grads->b_gate, grads->b_up, grads->b_down};
        const int64_t count[6] = {wide, wide, down, spec->hidden, spec->hidden, spec->out};
        for (int i = 0; i < 6; ++i) SVOX_TRY(zero(at[i], count[i], spec->dtype, (hipStream_t)stream));
        return SVOX_OK;
    }
    SVOX_TRY(check_matrix("grad_output", grad_output, spec->rows, spec->out, grad_stride));
    SVOX_BY_TYPE(spec->dtype, {
        SVOX_TRY(check_space(workspace, workspace_bytes, ffn_workspace<T>(*spec, true)));
        return launch_ffn_backward<T>(*spec, grad_output, grad_stride, *grads, workspace, (hipStream_t)stream);
    });
}
