// moe_row_ops.cpp -- host side of the operators on rows (include/moe_ops.h): the norm with 8-bit results and its
// gradient, quantised rows, tokens sorted by expert and back.
//
// As moe_ops.cpp: nothing here allocates device memory, and every check runs before the first launch.

#include <hip/hip_runtime.h>

#include "moe_host.h"
#include "moe_launch.h"
#include "moe_ops.h"

using namespace moe::host;

namespace {

bool is_float(int32_t t) { return t == MOE_DT_FLOAT32 || t == MOE_DT_FLOAT16 || t == MOE_DT_BFLOAT16; }

moe_status check_rows(const char* op, int64_t T, int64_t H, int32_t dtype, bool int8 = false) {
    if (T < 0 || H <= 0)
        return fail(MOE_ERR_ARG, "%s: sizes must be rows >= 0, H > 0 (rows=%lld H=%lld)", op, (long long)T,
                    (long long)H);
    if (!is_float(dtype) && !(int8 && dtype == MOE_DT_INT8))
        return fail(MOE_ERR_ARG, "%s: type %d (float32, float16%s bfloat16 expected)", op, dtype,
                    int8 ? ", int8 or" : " or");
    if (H > kMaxDim)
        return fail(MOE_ERR_UNSUPPORTED, "%s: H=%lld exceeds %lld", op, (long long)H, (long long)kMaxDim);
    if (T > kInt32Max) return fail(MOE_ERR_UNSUPPORTED, "%s: %lld rows are too many", op, (long long)T);
    return ok();
}

moe_status check_stride(const char* op, const char* what, int64_t rows, int64_t width, int64_t ld) {
    if ((rows > 1 && ld < width) || ld < 0 || ld > int64_t{1} << 40)
        return fail(MOE_ERR_ARG, "%s: %s rows %lld elements apart hold %lld", op, what, (long long)ld,
                    (long long)width);
    return ok();
}

moe_status check_norm(const char* op, int64_t T, int64_t H, int32_t dtype, int32_t gamma_type, float eps) {
    const moe_status st = check_rows(op, T, H, dtype);
    if (st != MOE_OK) return st;
    if (gamma_type != dtype && gamma_type != MOE_DT_FLOAT32)
        return fail(MOE_ERR_ARG, "%s: gamma type %d (the rows' or float32 expected)", op, gamma_type);
    if (!(eps > 0.0f) || !(eps - eps == 0.0f)) return fail(MOE_ERR_ARG, "%s: eps must be positive and finite", op);
    return ok();
}

// A workspace of 32-bit words
moe_status check_words(const char* op, const void* workspace, size_t bytes, size_t need) {
    if (need == 0) return ok();
    if (!workspace || bytes < need)
        return fail(MOE_ERR_WORKSPACE, "%s: workspace %zu bytes at %p, need %zu", op, bytes, workspace, need);
    if (reinterpret_cast<uintptr_t>(workspace) % 4 != 0)
        return fail(MOE_ERR_UNSUPPORTED, "%s: workspace must be 4-byte aligned", op);
    return ok();
}

moe_status check_picks(const char* op, int64_t T, int64_t K) {
    if (K < 1) return fail(MOE_ERR_ARG, "%s: topK=%lld must be at least 1", op, (long long)K);
    if (product_exceeds(T, K, kInt32Max - 1))
        return fail(MOE_ERR_UNSUPPORTED, "%s: T=%lld K=%lld too large", op, (long long)T, (long long)K);
    return ok();
}

moe_status check_permute(const char* op, int64_t T, int64_t E, int64_t K) {
    if (T < 0 || E <= 0 || K < 1 || K > E)
        return fail(MOE_ERR_ARG, "%s: T >= 0 and 1 <= topK <= numExperts expected (T=%lld K=%lld E=%lld)", op,
                    (long long)T, (long long)K, (long long)E);
    if (E > kMaxExperts)
        return fail(MOE_ERR_UNSUPPORTED, "%s: numExperts=%lld exceeds %lld", op, (long long)E, (long long)kMaxExperts);
    return check_picks(op, T, K);
}

// moe_unpermute_grad and, with `any`, moe_unpermute_grad_any
moe_status unpermute_grad(const void* grad_y, int64_t grad_y_stride, const void* rows, const int32_t* position,
                          const void* weights, int32_t weights_type, void* grad_rows, void* grad_weights, bool any,
                          void* workspace, size_t workspace_bytes, int64_t T, int64_t H, int64_t K, int32_t dtype,
                          void* stream) {
    const char* op = "MoeUnpermuteGrad";
    moe_status st = check_rows(op, T, H, dtype);
    if (st == MOE_OK) st = check_picks(op, T, K);
    if (st == MOE_OK) st = check_stride(op, "grad_y", T, H, grad_y_stride);
    if (st != MOE_OK) return st;
    if (weights && !is_float(weights_type)) return fail(MOE_ERR_ARG, "%s: weights type %d", op, weights_type);
    if (T == 0) return ok();
    if (!grad_y || !position || !grad_rows || (weights && (!rows || !grad_weights)))
        return fail(MOE_ERR_NULL, "%s: null tensor pointer", op);
    if (any) st = check_words(op, workspace, workspace_bytes, static_cast<size_t>(T) * K * 2 * sizeof(int32_t));
    if (st != MOE_OK) return st;
    moe::UnsortArgs u{};
    u.rows = rows;
    u.R = T * K;
    u.position = position;
    u.weights = weights;
    u.weights_type = weights_type;
    u.grad_y = grad_y;
    u.ldy = grad_y_stride;
    u.y = grad_rows;
    u.grad_weights = grad_weights;
    if (any) {
        u.heads = static_cast<int32_t*>(workspace);
        u.links = u.heads + T * K;
    }
    u.T = T;
    u.H = static_cast<int>(H);
    u.K = static_cast<int>(K);
    u.type = dtype;
    const hipError_t err = moe::launch_unsort_grad(u, as_stream(stream));
    if (err != hipSuccess) return hip_fail(err, "MoeUnpermuteGrad launch");
    return ok();
}

}  // namespace

extern "C" {

moe_status moe_add_rms_norm(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                            const void* gamma, int32_t gamma_type, void* y, void* sum, int8_t* q, float* scale,
                            int64_t T, int64_t H, float eps, int32_t dtype, void* stream) {
    const char* op = "MoeAddRmsNorm";
    moe_status st = check_norm(op, T, H, dtype, gamma_type, eps);
    if (st == MOE_OK) st = check_stride(op, "x", T, H, x_stride);
    if (st == MOE_OK && residual) st = check_stride(op, "residual", T, H, residual_stride);
    if (st != MOE_OK) return st;
    if ((q == nullptr) != (scale == nullptr)) return fail(MOE_ERR_NULL, "%s: q and scale go together", op);
    if (T == 0 || (!y && !sum && !q)) return ok();
    if (!x || !gamma) return fail(MOE_ERR_NULL, "%s: null tensor pointer", op);
    moe::NormArgs n{};
    n.x = x;
    n.ldx = x_stride;
    n.residual = residual;
    n.ldr = residual_stride;
    n.gamma = gamma;
    n.gamma_f32 = gamma_type == MOE_DT_FLOAT32;
    n.y = y;
    n.sum = sum;
    n.q = q;
    n.scale = scale;
    n.rows = T;
    n.H = static_cast<int>(H);
    n.eps = eps;
    const hipError_t err = moe::launch_norm(n, dtype, true, as_stream(stream));
    if (err != hipSuccess) return hip_fail(err, "MoeAddRmsNorm launch");
    return ok();
}

size_t moe_add_rms_norm_grad_workspace_bytes(int64_t T, int64_t H) {
    if (check_rows("MoeAddRmsNormGrad", T, H, MOE_DT_FLOAT32) != MOE_OK || H > moe::kNormGradMost) return 0;
    return static_cast<size_t>(moe::norm_grad_blocks(T, static_cast<int>(H))) * H * sizeof(float);
}

moe_status moe_add_rms_norm_grad(const void* grad_y, int64_t grad_y_stride, const void* sum, int64_t sum_stride,
                                 const void* gamma, int32_t gamma_type, const void* grad_sum, int64_t grad_sum_stride,
                                 void* grad_x, void* grad_gamma, void* workspace, size_t workspace_bytes, int64_t T,
                                 int64_t H, float eps, int32_t dtype, void* stream) {
    const char* op = "MoeAddRmsNormGrad";
    moe_status st = check_norm(op, T, H, dtype, gamma_type, eps);
    if (st == MOE_OK) st = check_stride(op, "grad_y", T, H, grad_y_stride);
    if (st == MOE_OK) st = check_stride(op, "sum", T, H, sum_stride);
    if (st == MOE_OK && grad_sum) st = check_stride(op, "grad_sum", T, H, grad_sum_stride);
    if (st != MOE_OK) return st;
    if (H > moe::kNormGradMost)
        return fail(MOE_ERR_UNSUPPORTED, "%s: H=%lld exceeds %d", op, (long long)H, moe::kNormGradMost);
    if (!grad_gamma && (!grad_x || T == 0)) return ok();
    if (T > 0 && (!grad_y || !sum || !gamma)) return fail(MOE_ERR_NULL, "%s: null tensor pointer", op);
    if (grad_gamma) st = check_words(op, workspace, workspace_bytes, moe_add_rms_norm_grad_workspace_bytes(T, H));
    if (st != MOE_OK) return st;
    moe::NormArgs n{};
    n.x = sum;
    n.ldx = sum_stride;
    n.gamma = gamma;
    n.gamma_f32 = gamma_type == MOE_DT_FLOAT32;
    n.grad_y = grad_y;
    n.ldy = grad_y_stride;
    n.grad_sum = grad_sum;
    n.lds = grad_sum_stride;
    n.y = grad_x;
    n.part = grad_gamma ? static_cast<float*>(workspace) : nullptr;
    n.rows = T;
    n.H = static_cast<int>(H);
    n.eps = eps;
    const hipError_t err = moe::launch_norm_grad(n, dtype, grad_gamma, as_stream(stream));
    if (err != hipSuccess) return hip_fail(err, "MoeAddRmsNormGrad launch");
    return ok();
}

moe_status moe_quantize(const void* x, int64_t x_stride, int8_t* q, float* scale, int64_t rows, int64_t H,
                        int32_t dtype, void* stream) {
    const char* op = "MoeQuantize";
    moe_status st = check_rows(op, rows, H, dtype);
    if (st == MOE_OK) st = check_stride(op, "x", rows, H, x_stride);
    if (st != MOE_OK) return st;
    if (rows == 0) return ok();
    if (!x || !q || !scale) return fail(MOE_ERR_NULL, "%s: null tensor pointer", op);
    moe::NormArgs n{};
    n.x = x;
    n.ldx = x_stride;
    n.q = q;
    n.scale = scale;
    n.rows = rows;
    n.H = static_cast<int>(H);
    const hipError_t err = moe::launch_norm(n, dtype, false, as_stream(stream));
    if (err != hipSuccess) return hip_fail(err, "MoeQuantize launch");
    return ok();
}

size_t moe_permute_workspace_bytes(int64_t T, int64_t E, int64_t K) {
    if (check_permute("MoePermute", T, E, K) != MOE_OK) return 0;
    return moe::sort_scratch_bytes(T, static_cast<int>(E), static_cast<int>(K));
}

moe_status moe_permute(const void* x, int64_t x_stride, const float* x_scale, const int32_t* expert_ids, void* rows,
                       float* row_scale, int32_t* offsets, int32_t* position, void* workspace, size_t workspace_bytes,
                       int64_t T, int64_t H, int64_t E, int64_t K, int32_t dtype, void* stream) {
    const char* op = "MoePermute";
    moe_status st = check_rows(op, T, H, dtype, true);
    if (st == MOE_OK) st = check_permute(op, T, E, K);
    if (st == MOE_OK) st = check_stride(op, "x", T, H, x_stride);
    if (st != MOE_OK) return st;
    if ((x_scale == nullptr) != (row_scale == nullptr) && T > 0)
        return fail(MOE_ERR_NULL, "%s: x_scale and row_scale go together", op);
    if (!offsets || (T > 0 && (!x || !expert_ids || !rows || !position)))
        return fail(MOE_ERR_NULL, "%s: null tensor pointer", op);
    st = check_words(op, workspace, workspace_bytes,
                     moe::sort_scratch_bytes(T, static_cast<int>(E), static_cast<int>(K)));
    if (st != MOE_OK) return st;
    moe::SortArgs s{};
    s.ids = expert_ids;
    s.x = x;
    s.scale = x_scale;
    s.rows = rows;
    s.row_scale = row_scale;
    s.offsets = offsets;
    s.position = position;
    s.scratch = static_cast<int32_t*>(workspace);
    s.T = T;
    s.ldx = x_stride;
    s.H = static_cast<int>(H);
    s.E = static_cast<int>(E);
    s.K = static_cast<int>(K);
    s.bytes = dtype == MOE_DT_INT8 ? 1 : dtype == MOE_DT_FLOAT32 ? 4 : 2;
    const hipError_t err = moe::launch_sort(s, as_stream(stream));
    if (err != hipSuccess) return hip_fail(err, "MoePermute launch");
    return ok();
}

moe_status moe_unpermute(const void* rows, int64_t num_rows, const int32_t* position, const void* weights,
                         int32_t weights_type, void* y, int64_t T, int64_t H, int64_t K, int32_t dtype, void* stream) {
    const char* op = "MoeUnpermute";
    moe_status st = check_rows(op, T, H, dtype);
    if (st == MOE_OK) st = check_picks(op, T, K);
    if (st != MOE_OK) return st;
    if (num_rows < 0 || num_rows > kInt32Max)
        return fail(MOE_ERR_ARG, "%s: %lld rows", op, (long long)num_rows);
    if (weights && !is_float(weights_type)) return fail(MOE_ERR_ARG, "%s: weights type %d", op, weights_type);
    if (T == 0) return ok();
    if (!position || !y || (num_rows > 0 && !rows)) return fail(MOE_ERR_NULL, "%s: null tensor pointer", op);
    moe::UnsortArgs u{};
    u.rows = rows;
    u.R = num_rows;
    u.position = position;
    u.weights = weights;
    u.weights_type = weights_type;
    u.y = y;
    u.T = T;
    u.H = static_cast<int>(H);
    u.K = static_cast<int>(K);
    u.type = dtype;
    const hipError_t err = moe::launch_unsort(u, as_stream(stream));
    if (err != hipSuccess) return hip_fail(err, "MoeUnpermute launch");
    return ok();
}

moe_status moe_unpermute_grad(const void* grad_y, int64_t grad_y_stride, const void* rows, const int32_t* position,
                              const void* weights, int32_t weights_type, void* grad_rows, void* grad_weights,
                              int64_t T, int64_t H, int64_t K, int32_t dtype, void* stream) {
    return unpermute_grad(grad_y, grad_y_stride, rows, position, weights, weights_type, grad_rows, grad_weights, false,
                          nullptr, 0, T, H, K, dtype, stream);
}

size_t moe_unpermute_grad_any_workspace_bytes(int64_t T, int64_t K) {
    const char* op = "MoeUnpermuteGrad";
    if (check_rows(op, T, 1, MOE_DT_FLOAT32) != MOE_OK || check_picks(op, T, K) != MOE_OK) return 0;
    return static_cast<size_t>(T) * K * 2 * sizeof(int32_t);
}

moe_status moe_unpermute_grad_any(const void* grad_y, int64_t grad_y_stride, const void* rows, const int32_t* position,
                                  const void* weights, int32_t weights_type, void* grad_rows, void* grad_weights,
                                  void* workspace, size_t workspace_bytes, int64_t T, int64_t H, int64_t K,
                                  int32_t dtype, void* stream) {
    return unpermute_grad(grad_y, grad_y_stride, rows, position, weights, weights_type, grad_rows, grad_weights, true,
                          workspace, workspace_bytes, T, H, K, dtype, stream);
}

}  // extern "C"
