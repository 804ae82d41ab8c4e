// moe_linear.hip -- MoeLinear and MoeLinearGrad for gfx950: y = act(x W^T + b) + r and its gradients.
//
// No counterpart in the reference, whose products are the expert FFN's (op_kernel/moe_expert_ffn.cpp:265-394).
// Every product here is C[m][n] = sum_k P[m][k] Q[n][k] with fp16 or bf16 operands and fp32 sums (MFMA):
//   forward    P = x  (by rows), Q = W (by rows, or by k when W is a transposed view)
//   grad_x     P = dz (by rows), Q = W read the other way round
//   grad_W     P = dz (by k: its T rows are the reduction), Q = x (by k)
// The tiles here, 32 to 256 rows by 128, are for products that do not fill the GPU with 256 x 256 ones; where even
// these leave CUs idle the product is split over k and a second launch adds the pieces in order. What bounds them is
// the copies into LDS: 24 KB a stage and two workgroups a CU, 0.65 us for both (64 rows), is 19 TB/s over the GPU, and
// 128 and 256 rows come to 18 and 13 TB/s. So the taller tile wins until the pieces' sums cost more than its reads
// save.
//   T = 4097, H = 7168, N = 256 (130 tiles of 64 rows in 3 pieces): 25.6 + 4.2 us, of which x from HBM alone is 11
//   both gradients' products at T = 1000, H = 1056, N = 733, one launch of 256 workgroups: 10.9 + 3.2 us
#include "moe_linear_mid.h"

namespace moe {

namespace {

// Both gradient products in one launch: neither needs the other, and small ones leave the GPU half empty. The first
// x_blocks workgroups have grad_x.
template <typename T, bool QK, int BM>
__global__ __launch_bounds__(mid_threads(BM)) __attribute__((amdgpu_waves_per_eu(2, 2))) void gemm_pair_kernel(
    GemmArgs x, GemmArgs w, int x_blocks) {
    extern __shared__ __align__(16) uint16_t lds[];
    const int block = static_cast<int>(blockIdx.x);
    if (block < x_blocks)
        gemm_mid<T, false, QK, BM, false, true>(x, (x.m + BM - 1) / BM, (x.n + kBN - 1) / kBN, block, x_blocks, lds);
    else
        gemm_mid<T, true, true, 128, false, true>(w, (w.m + 127) / 128, (w.n + kBN - 1) / kBN, block - x_blocks,
                                                  static_cast<int>(gridDim.x) - x_blocks, lds);
}

template <typename T, bool QK, int BM>
hipError_t run_pair(const GemmArgs& x, const GemmArgs& w, hipStream_t stream) {
    constexpr int kLds = mid_lds_bytes(BM) > mid_lds_bytes(128) ? mid_lds_bytes(BM) : mid_lds_bytes(128);
    const int x_blocks = mid_grid(x, BM, kBN);
    TraceScope trace("moe_linear_gemm", stream);
    gemm_pair_kernel<T, QK, BM><<<x_blocks + mid_grid(w, 128, kBN), mid_threads(BM), kLds, stream>>>(x, w, x_blocks);
    return hipGetLastError();
}
template <typename T>
hipError_t run_pair_any(const GemmArgs& x, const GemmArgs& w, bool q_by_k, int bm, hipStream_t stream) {
    if (bm == 32) return q_by_k ? run_pair<T, true, 32>(x, w, stream) : run_pair<T, false, 32>(x, w, stream);
    if (bm == 64) return q_by_k ? run_pair<T, true, 64>(x, w, stream) : run_pair<T, false, 64>(x, w, stream);
    return q_by_k ? run_pair<T, true, 128>(x, w, stream) : run_pair<T, false, 128>(x, w, stream);
}

template <typename T, bool PK, bool QK, int BM, bool SWIGLU>
hipError_t run_mid_direct(const GemmArgs& g, bool direct, hipStream_t stream) {
    return direct ? run_mid<T, PK, QK, BM, SWIGLU, true>(g, stream) : run_mid<T, PK, QK, BM, SWIGLU, false>(g, stream);
}

template <typename T>
hipError_t run_mid_any(const GemmArgs& g, bool p_by_k, bool q_by_k, bool direct, int bm, hipStream_t stream) {
    const bool swiglu = g.act == kActSwiglu;
    if (p_by_k) return bm == 256 ? run_mid<T, true, true, 256, false, true>(g, stream)
                                 : run_mid_direct<T, true, true, 128, false>(g, direct, stream);
    if (bm == 256) {  // direct operands only
        if (q_by_k) return swiglu ? run_mid<T, false, true, 256, true, true>(g, stream)
                                  : run_mid<T, false, true, 256, false, true>(g, stream);
        return swiglu ? run_mid<T, false, false, 256, true, true>(g, stream)
                      : run_mid<T, false, false, 256, false, true>(g, stream);
    }
    if (bm == 128) {
        if (q_by_k) return swiglu ? run_mid_direct<T, false, true, 128, true>(g, direct, stream)
                                  : run_mid_direct<T, false, true, 128, false>(g, direct, stream);
        return swiglu ? run_mid_direct<T, false, false, 128, true>(g, direct, stream)
                      : run_mid_direct<T, false, false, 128, false>(g, direct, stream);
    }
    if (bm == 64) {
        if (q_by_k) return swiglu ? run_mid_direct<T, false, true, 64, true>(g, direct, stream)
                                  : run_mid_direct<T, false, true, 64, false>(g, direct, stream);
        return swiglu ? run_mid_direct<T, false, false, 64, true>(g, direct, stream)
                      : run_mid_direct<T, false, false, 64, false>(g, direct, stream);
    }
    if (q_by_k) return swiglu ? run_mid_direct<T, false, true, 32, true>(g, direct, stream)
                              : run_mid_direct<T, false, true, 32, false>(g, direct, stream);
    return swiglu ? run_mid_direct<T, false, false, 32, true>(g, direct, stream)
                  : run_mid_direct<T, false, false, 32, false>(g, direct, stream);
}

// What is left of a training step's gradients in one launch: the split products' sums and the bias's column sums
template <typename T>
__global__ __launch_bounds__(kReduceThreads) void grad_tail_kernel(GradTail t) {
    int block = static_cast<int>(blockIdx.x);
    if (block < t.x_blocks) return gemm_reduce<T, false>(t.x, block);
    block -= t.x_blocks;
    if (block < t.w_blocks) return gemm_reduce<T, false>(t.w, block);
    column_sums<T>(t.sums, t.bias_grad, t.Z, t.sum_rows, block - t.w_blocks);
}

template <typename T>
hipError_t prepare_256() {
    for (const void* fn : {reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, false, 256, false, true>),
                           reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, false, 256, true, true>),
                           reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, true, 256, false, true>),
                           reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, true, 256, true, true>),
                           reinterpret_cast<const void*>(&gemm_mid_kernel<T, true, true, 256, false, true>)}) {
        const hipError_t err = ensure_lds_limit(fn, mid_lds_bytes(256));
        if (err != hipSuccess) return err;
    }
    return hipSuccess;
}

template <typename T, int BM>
hipError_t prepare_bm() {
    const int lds = mid_lds_bytes(BM);
    for (const void* fn : {reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, false, BM, false, true>),
                           reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, false, BM, true, true>),
                           reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, true, BM, false, true>),
                           reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, true, BM, true, true>),
                           reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, false, BM, false, false>),
                           reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, false, BM, true, false>),
                           reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, true, BM, false, false>),
                           reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, true, BM, true, false>),
                           reinterpret_cast<const void*>(&gemm_pair_kernel<T, false, BM>),
                           reinterpret_cast<const void*>(&gemm_pair_kernel<T, true, BM>)}) {
        const hipError_t err = ensure_lds_limit(fn, lds);
        if (err != hipSuccess) return err;
    }
    return hipSuccess;
}

}  // namespace

hipError_t launch_gemm_mid(const GemmArgs& g, bool p_by_k, bool q_by_k, bool bf16, bool direct, int bm,
                           hipStream_t stream) {
    return bf16 ? run_mid_any<Bf16>(g, p_by_k, q_by_k, direct, bm, stream)
                : run_mid_any<Half>(g, p_by_k, q_by_k, direct, bm, stream);
}

hipError_t launch_gemm_reduce(const GemmArgs& g, bool bf16, hipStream_t stream) {
    const bool swiglu = g.act == kActSwiglu;
    const int64_t work = part_cols(g.n) / 4 * g.m;
    const int grid = static_cast<int>((work + kReduceThreads - 1) / kReduceThreads);
    TraceScope trace("moe_linear_reduce", stream);
    if (bf16) {
        if (swiglu) gemm_reduce_kernel<Bf16, true><<<grid, kReduceThreads, 0, stream>>>(g);
        else gemm_reduce_kernel<Bf16, false><<<grid, kReduceThreads, 0, stream>>>(g);
    } else {
        if (swiglu) gemm_reduce_kernel<Half, true><<<grid, kReduceThreads, 0, stream>>>(g);
        else gemm_reduce_kernel<Half, false><<<grid, kReduceThreads, 0, stream>>>(g);
    }
    return hipGetLastError();
}

hipError_t launch_gemm_pair(const GemmArgs& x, const GemmArgs& w, bool q_by_k, bool bf16, int bm, hipStream_t stream) {
    return bf16 ? run_pair_any<Bf16>(x, w, q_by_k, bm, stream) : run_pair_any<Half>(x, w, q_by_k, bm, stream);
}

hipError_t launch_grad_tail(GradTail t, bool bf16, hipStream_t stream) {
    t.x_blocks = t.x.splits > 1 ? static_cast<int>(reduce_blocks(t.x)) : 0;
    t.w_blocks = t.w.splits > 1 ? static_cast<int>(reduce_blocks(t.w)) : 0;
    const int grid = t.x_blocks + t.w_blocks + (t.bias_grad ? (t.Z + kSumColumns - 1) / kSumColumns : 0);
    if (grid == 0) return hipSuccess;
    TraceScope trace("moe_linear_reduce", stream);
    if (bf16) grad_tail_kernel<Bf16><<<grid, kReduceThreads, 0, stream>>>(t);
    else grad_tail_kernel<Half><<<grid, kReduceThreads, 0, stream>>>(t);
    return hipGetLastError();
}

hipError_t prepare_gemm_mid() {  // 128-row tiles keep within 64 KB
    hipError_t err = prepare_256<Half>();
    if (err == hipSuccess) err = prepare_256<Bf16>();
    if (err == hipSuccess) err = prepare_bm<Half, 32>();
    if (err == hipSuccess) err = prepare_bm<Half, 64>();
    if (err == hipSuccess) err = prepare_bm<Bf16, 32>();
    if (err == hipSuccess) err = prepare_bm<Bf16, 64>();
    return err;
}

}  // namespace moe
