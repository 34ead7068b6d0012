// extern "C" boundary of the row operators: argument checks and workspace carving.  Declarations: include/yolohead.h.
#include <algorithm>
#include "yh_rows.h"

namespace {

size_t round_up(size_t v, size_t a) { return (v + a - 1) / a * a; }
size_t element_size(int32_t type) { return type == YH_FLOAT32 ? 4 : type == YH_INT8 ? 1 : 2; }

int check_float_type(int32_t type, const char *what)
{
    if (type != YH_FLOAT32 && type != YH_BFLOAT16 && type != YH_FLOAT16)
        return yh::report(YH_ERR_INVALID_ARG, "%s %d is not YH_FLOAT32, YH_BFLOAT16 or YH_FLOAT16", what, type);
    return YH_OK;
}

int check_sizes(int64_t rows, int32_t a, int32_t b)
{
    if (rows < 0) return yh::report(YH_ERR_INVALID_ARG, "rows %lld is negative", (long long)rows);
    if (a < 1 || b < 1) return yh::report(YH_ERR_INVALID_ARG, "%d channels: at least one is needed", std::min(a, b));
    if (rows >= YH_MAX_ROWS) return yh::report(YH_ERR_LIMIT, "rows %lld is not below %d", (long long)rows, YH_MAX_ROWS);
    if (a > YH_MAX_ROW_CHANNELS || b > YH_MAX_ROW_CHANNELS)
        return yh::report(YH_ERR_LIMIT, "%d channels exceed %d", std::max(a, b), YH_MAX_ROW_CHANNELS);
    if (rows * std::max(a, b) >= (int64_t)1 << 36) return yh::report(YH_ERR_LIMIT, "rows * channels is not below 2^36");
    if ((int64_t)a * b >= (int64_t)1 << 31) return yh::report(YH_ERR_LIMIT, "%d x %d weights are not below 2^31", a, b);
    return YH_OK;
}

// A matrix of rows: not null (unless there is nothing in it), aligned to its elements, rows that do not overlap if written.
int check_rows(const void *p, int64_t ld, int64_t cols, int64_t rows, size_t element, bool written, const char *name)
{
    if (!p && rows > 0) return yh::report(YH_ERR_INVALID_ARG, "%s is null", name);
    if (ld < (written ? cols : 0))
        return yh::report(YH_ERR_INVALID_ARG, "%s: %lld elements from row to row, %lld channels", name, (long long)ld, (long long)cols);
    if (ld >= (int64_t)1 << 36) return yh::report(YH_ERR_LIMIT, "%s: %lld elements from row to row are not below 2^36", name, (long long)ld);
    if (reinterpret_cast<uintptr_t>(p) % element) return yh::report(YH_ERR_ALIGN, "%s is not aligned to its %zu-byte elements", name, element);
    return YH_OK;
}

int check_vector(const void *p, bool needed, const char *name)
{
    if (!p && needed) return yh::report(YH_ERR_INVALID_ARG, "%s is null", name);
    if (reinterpret_cast<uintptr_t>(p) & 3u) return yh::report(YH_ERR_ALIGN, "%s is not aligned to its 4-byte elements", name);
    return YH_OK;
}

int check_workspace(const void *p, size_t have, size_t need)
{
    if (need == 0) return YH_OK;
    if (!p || have < need) return yh::report(YH_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", p ? have : (size_t)0, need);
    if (reinterpret_cast<uintptr_t>(p) & 15u) return yh::report(YH_ERR_ALIGN, "workspace is not 16-byte aligned");
    return YH_OK;
}

int launched(hipError_t e, const char *what) { return e == hipSuccess ? YH_OK : yh::report_hip(e, what); }

#define YH_TRY(call)                       \
    do {                                   \
        const int rc_ = (call);            \
        if (rc_ != YH_OK) return rc_;      \
    } while (0)

}  // namespace

extern "C" {

int yh_quantize_rows(const void *x, int32_t dtype, int64_t ldx, int64_t rows, int32_t k,
                     int8_t *codes, int64_t ldc, float *scale, void *stream)
{
    YH_TRY(check_float_type(dtype, "dtype"));
    YH_TRY(check_sizes(rows, k, 1));
    YH_TRY(check_rows(x, ldx, k, rows, element_size(dtype), false, "x"));
    YH_TRY(check_rows(codes, ldc, k, rows, 1, true, "codes"));
    YH_TRY(check_vector(scale, rows > 0, "scale"));
    if (rows == 0) return YH_OK;
    YH_TRY(yh::require_device());
    return launched(yh::launch_quantize({x, ldx, dtype}, rows, k, codes, ldc, scale, static_cast<hipStream_t>(stream)), "quantize launch");
}

int yh_dequantize_rows(const int8_t *codes, int64_t ldc, const float *scale, int64_t rows, int32_t k,
                       void *x, int32_t dtype, int64_t ldx, void *stream)
{
    YH_TRY(check_float_type(dtype, "dtype"));
    YH_TRY(check_sizes(rows, k, 1));
    YH_TRY(check_rows(codes, ldc, k, rows, 1, false, "codes"));
    YH_TRY(check_vector(scale, rows > 0, "scale"));
    YH_TRY(check_rows(x, ldx, k, rows, element_size(dtype), true, "x"));
    if (rows == 0) return YH_OK;
    YH_TRY(yh::require_device());
    return launched(yh::launch_dequantize(codes, ldc, scale, rows, k, x, ldx, dtype, static_cast<hipStream_t>(stream)), "dequantize launch");
}

// The codes of x inside the workspace: rows of a multiple of 16 bytes, the scales behind them.
static size_t codes_pitch(int32_t k) { return round_up((size_t)k, 16); }

int yh_matmul_int8_workspace_bytes(int64_t rows, int32_t k, int32_t n, int32_t x_dtype, int32_t want_codes, size_t *bytes)
{
    if (!bytes) return yh::report(YH_ERR_INVALID_ARG, "bytes is null");
    if (x_dtype != YH_INT8) YH_TRY(check_float_type(x_dtype, "x_dtype"));
    YH_TRY(check_sizes(rows, k, n));
    *bytes = want_codes || !yh::product_needs_codes(rows, k, n, x_dtype) ? 0 : (size_t)rows * (codes_pitch(k) + 4);
    return YH_OK;
}

int yh_matmul_int8(const void *x, int32_t x_dtype, int64_t ldx, const float *x_scale, int64_t rows, int32_t k,
                   const int8_t *w, int64_t ldw, const float *w_scale, int32_t n, const float *bias,
                   void *y, int32_t y_dtype, int64_t ldy, int8_t *codes, int64_t ldc, float *scale,
                   void *workspace, size_t workspace_bytes, void *stream)
{
    const bool want = codes || scale, whole = x_dtype == YH_INT8;
    size_t need = 0;
    YH_TRY(yh_matmul_int8_workspace_bytes(rows, k, n, x_dtype, want, &need));
    YH_TRY(check_float_type(y_dtype, "y_dtype"));
    YH_TRY(check_rows(x, ldx, k, rows, element_size(x_dtype), false, "x"));
    YH_TRY(check_vector(x_scale, whole && rows > 0, "x_scale"));
    if (!whole && x_scale) return yh::report(YH_ERR_INVALID_ARG, "x_scale belongs to an x of YH_INT8");
    if (whole && want) return yh::report(YH_ERR_INVALID_ARG, "x is given as codes: there are none to leave");
    YH_TRY(check_rows(w, ldw, k, n, 1, false, "w"));
    YH_TRY(check_vector(w_scale, true, "w_scale"));
    YH_TRY(check_vector(bias, false, "bias"));
    YH_TRY(check_rows(y, ldy, n, rows, element_size(y_dtype), true, "y"));
    if (want) {
        YH_TRY(check_rows(codes, ldc, k, rows, 1, true, "codes"));
        YH_TRY(check_vector(scale, rows > 0, "scale"));
    }
    YH_TRY(check_workspace(workspace, workspace_bytes, need));
    if (rows == 0) return YH_OK;
    YH_TRY(yh::require_device());
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (!want && need) {
        ldc = (int64_t)codes_pitch(k);
        codes = static_cast<int8_t *>(workspace);
        scale = reinterpret_cast<float *>(codes + rows * ldc);
    }
    return launched(yh::launch_int8_product({x, ldx, x_dtype}, x_scale, rows, k, w, ldw, w_scale, n, bias, y, ldy, y_dtype, codes, ldc, scale, st),
                    "product launch");
}

int yh_weight_grad_workspace_bytes(int64_t rows, int32_t n, int32_t k, size_t *bytes)
{
    if (!bytes) return yh::report(YH_ERR_INVALID_ARG, "bytes is null");
    YH_TRY(check_sizes(rows, n, k));
    *bytes = yh::weight_grad_workspace(rows, n, k);
    return YH_OK;
}

int yh_weight_grad(const void *dy, int32_t dtype, int64_t lddy, const int8_t *codes, int64_t ldc, const float *scale,
                   int64_t rows, int32_t n, int32_t k, float *dw, float *db,
                   void *workspace, size_t workspace_bytes, void *stream)
{
    size_t need = 0;
    YH_TRY(yh_weight_grad_workspace_bytes(rows, n, k, &need));
    YH_TRY(check_float_type(dtype, "dtype"));
    YH_TRY(check_rows(dy, lddy, n, rows, element_size(dtype), false, "dy"));
    YH_TRY(check_rows(codes, ldc, k, rows, 1, false, "codes"));
    YH_TRY(check_vector(scale, rows > 0, "scale"));
    YH_TRY(check_vector(dw, true, "dw"));
    YH_TRY(check_vector(db, false, "db"));
    YH_TRY(check_workspace(workspace, workspace_bytes, need));
    YH_TRY(yh::require_device());
    return launched(yh::launch_weight_grad({dy, lddy, dtype}, codes, ldc, scale, rows, n, k, dw, db, workspace, static_cast<hipStream_t>(stream)),
                    "weight gradient launch");
}

int yh_input_grad(const void *dy, int32_t dtype, int64_t lddy, const int8_t *w, int64_t ldw, const float *w_scale,
                  int64_t rows, int32_t n, int32_t k, void *dx, int64_t lddx, void *stream)
{
    YH_TRY(check_float_type(dtype, "dtype"));
    YH_TRY(check_sizes(rows, n, k));
    YH_TRY(check_rows(dy, lddy, n, rows, element_size(dtype), false, "dy"));
    YH_TRY(check_rows(w, ldw, k, n, 1, false, "w"));
    YH_TRY(check_vector(w_scale, true, "w_scale"));
    YH_TRY(check_rows(dx, lddx, k, rows, element_size(dtype), true, "dx"));
    if (rows == 0) return YH_OK;
    YH_TRY(yh::require_device());
    return launched(yh::launch_input_grad({dy, lddy, dtype}, w, ldw, w_scale, rows, n, k, dx, lddx, static_cast<hipStream_t>(stream)),
                    "input gradient launch");
}

int yh_norm_act_workspace_bytes(int64_t rows, int32_t c, int32_t dtype, size_t *bytes)
{
    if (!bytes) return yh::report(YH_ERR_INVALID_ARG, "bytes is null");
    YH_TRY(check_float_type(dtype, "dtype"));
    YH_TRY(check_sizes(rows, c, 1));
    if (rows < 1) return yh::report(YH_ERR_INVALID_ARG, "statistics of no rows");
    const int blocks = yh::norm_blocks(rows, c, dtype);
    *bytes = blocks > 1 ? (size_t)c * 2 * sizeof(double) * blocks : 0;
    return YH_OK;
}

int yh_norm_act_forward(const void *z, int64_t ldz, const void *residual, int64_t ldr, int32_t dtype, int64_t rows, int32_t c,
                        const float *gamma, const float *beta, double eps, float slope,
                        void *a, int64_t lda, int8_t *kept, int64_t ldk, float *scale, float *mean, float *invstd,
                        float *running_mean, float *running_var, double momentum,
                        void *workspace, size_t workspace_bytes, void *stream)
{
    size_t need = 0;
    YH_TRY(yh_norm_act_workspace_bytes(rows, c, dtype, &need));
    if (!(eps >= 0.0)) return yh::report(YH_ERR_INVALID_ARG, "eps %g is negative", eps);
    const size_t e = element_size(dtype);
    YH_TRY(check_rows(z, ldz, c, rows, e, false, "z"));
    if (residual) YH_TRY(check_rows(residual, ldr, c, rows, e, false, "residual"));
    YH_TRY(check_rows(a, lda, c, rows, e, true, "a"));
    if (!kept != !scale) return yh::report(YH_ERR_INVALID_ARG, "kept and scale come together");
    if (kept) YH_TRY(check_rows(kept, ldk, c, rows, 1, true, "kept"));
    if (!running_mean != !running_var) return yh::report(YH_ERR_INVALID_ARG, "running_mean and running_var come together");
    YH_TRY(check_vector(gamma, true, "gamma"));
    YH_TRY(check_vector(beta, true, "beta"));
    YH_TRY(check_vector(scale, false, "scale"));
    YH_TRY(check_vector(mean, true, "mean"));
    YH_TRY(check_vector(invstd, true, "invstd"));
    YH_TRY(check_vector(running_mean, false, "running_mean"));
    YH_TRY(check_vector(running_var, false, "running_var"));
    YH_TRY(check_workspace(workspace, workspace_bytes, need));
    YH_TRY(yh::require_device());
    return launched(yh::launch_norm_forward({z, ldz, dtype}, {residual, ldr, dtype}, rows, c, gamma, beta, eps, slope, a, lda, kept, ldk, scale,
                                            mean, invstd, running_mean, running_var, momentum, workspace, static_cast<hipStream_t>(stream)),
                    "norm launch");
}

int yh_norm_act_backward(const void *da, int64_t ldda, int32_t dtype, int64_t rows, int32_t c,
                         const int8_t *kept, int64_t ldk, const float *scale, const float *gamma, const float *invstd, float slope,
                         void *dz, int64_t lddz, float *dgamma, float *dbeta,
                         void *workspace, size_t workspace_bytes, void *stream)
{
    size_t need = 0;
    YH_TRY(yh_norm_act_workspace_bytes(rows, c, dtype, &need));
    const size_t e = element_size(dtype);
    YH_TRY(check_rows(da, ldda, c, rows, e, false, "da"));
    YH_TRY(check_rows(kept, ldk, c, rows, 1, false, "kept"));
    YH_TRY(check_rows(dz, lddz, c, rows, e, true, "dz"));
    YH_TRY(check_vector(scale, true, "scale"));
    YH_TRY(check_vector(gamma, true, "gamma"));
    YH_TRY(check_vector(invstd, true, "invstd"));
    YH_TRY(check_vector(dgamma, true, "dgamma"));
    YH_TRY(check_vector(dbeta, true, "dbeta"));
    YH_TRY(check_workspace(workspace, workspace_bytes, need));
    YH_TRY(yh::require_device());
    return launched(yh::launch_norm_backward({da, ldda, dtype}, rows, c, kept, ldk, scale, gamma, invstd, slope, dz, lddz, dgamma, dbeta,
                                             workspace, static_cast<hipStream_t>(stream)), "norm gradient launch");
}

}  // extern "C"
