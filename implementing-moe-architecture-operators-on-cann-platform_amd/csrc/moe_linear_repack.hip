// moe_linear_repack.hip -- operands whose rows are no multiple of 16 bytes, laid out anew for the dense products.
//
// The products copy 16 bytes at a time straight into LDS, so a row of 8 n + r elements cannot be read in place from any
// row but the first. One pass copies such operands into the workspace with their rows padded with zeros to whole
// granules; the fast kernels then run as for any other size. The pass moves each byte twice and the launch takes about
// 3 us.
#include "moe_gemm.h"

namespace moe {

namespace {

constexpr int kThreads = 256;

__global__ __launch_bounds__(kThreads) void repack_kernel(RepackArgs a, int64_t granules) {
    const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < granules; i += step) {
        int64_t first = 0;
#pragma unroll
        for (int m = 0; m < kRepackMost; ++m) {
            const Repack& r = a.m[m];
            const int per = r.dst_cols / 8;
            const int64_t count = r.rows * per, at = i - first;
            if (at >= 0 && at < count) {
                const int64_t row = at / per;
                const int col = static_cast<int>(at - row * per) * 8;
                *reinterpret_cast<s16x8*>(r.dst + row * r.dst_ld + col) =
                    load8(r.src + row * r.src_ld + col, r.cols - col, col);
            }
            first += count;
        }
    }
}

}  // namespace

hipError_t launch_repack(const RepackArgs& a, hipStream_t stream) {
    int64_t granules = 0;
    for (const Repack& r : a.m) granules += r.rows * (r.dst_cols / 8);
    if (granules == 0) return hipSuccess;
    TraceScope trace("moe_linear_repack", stream);
    const int64_t blocks = (granules + kThreads - 1) / kThreads;
    repack_kernel<<<static_cast<unsigned>(blocks < (1 << 20) ? blocks : 1 << 20), kThreads, 0, stream>>>(a, granules);
    return hipGetLastError();
}

}  // namespace moe
