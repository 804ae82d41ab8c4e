// moe_linear_grad.hip -- the elementwise part of MoeLinearGrad: dz = dy * act'(z) and the bias's gradient, the column
// sums of dz.
//
// dz is rounded to the operands' 16-bit type, once, because the two products that take it run on the matrix cores; the
// column sums take it before that rounding. Rows of dz are padded to a multiple of 8 with zeros, so that the products
// read it with 16-byte copies whatever the width.
// One workgroup has 64 threads x 8 columns of a block of rows (the 4 waves take rows in turn), so a wave's access is
// 1 KB of one row. Its column sums go through LDS in wave order to one row of `part`; colsum_kernel adds those in order:
// no atomics, so the result does not depend on timing.
#include "moe_gemm.h"

namespace moe {

namespace {

constexpr int kThreads = 256;
constexpr int kCols = 512;  // columns of a workgroup

__device__ __forceinline__ float slope(float z, int act) {
    switch (act) {
        case kActRelu: return z > 0.0f ? 1.0f : 0.0f;
        case kActGelu:
            return 0.5f * erfcf(z * -0.70710678118654752f) + z * 0.39894228040143268f * expf(-0.5f * z * z);
        case kActGeluTanh: {
            const float a = 0.79788456080286536f, b = 0.044715f;
            const float t = tanhf(a * (z + b * z * z * z));
            return 0.5f * (1.0f + t) + 0.5f * z * (1.0f - t * t) * a * (1.0f + 3.0f * b * z * z);
        }
        case kActSilu: {
            const float s = 1.0f / (1.0f + expf(-z));
            return s * (1.0f + z * (1.0f - s));
        }
        default: return 1.0f;
    }
}

struct ActGradArgs {
    const uint16_t* dy;   // [T, N], rows ldy apart
    const uint16_t* pre;  // [T, N] (SwiGLU: [T, 2N]) contiguous, or null (no activation)
    uint16_t* dz;         // [T, ldz] or null (the column sums alone)
    float* part;          // [row blocks, Z] column sums or null
    int64_t ldy, ldz;
    int64_t rows_per_block;
    int64_t T;
    int N, Z;
    int act;
};

// 8 columns of one dz row from column c on: SwiGLU columns below N are the gate's, the others up's
template <typename T>
__device__ __forceinline__ void dz8(const ActGradArgs& a, int64_t t, int c, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int col = c + e;
        v[e] = 0.0f;
        if (col >= a.Z) continue;
        if (a.act == kActSwiglu) {
            const bool up = col >= a.N;
            const int n = up ? col - a.N : col;
            const float dy = T::load(a.dy[t * a.ldy + n]);
            const float zg = T::load(a.pre[t * a.Z + n]);
            const float s = 1.0f / (1.0f + expf(-zg));
            v[e] = up ? dy * zg * s : dy * T::load(a.pre[t * a.Z + a.N + n]) * s * (1.0f + zg * (1.0f - s));
        } else {
            const float dy = T::load(a.dy[t * a.ldy + col]);
            v[e] = a.pre ? dy * slope(T::load(a.pre[t * a.Z + col]), a.act) : dy;
        }
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void act_grad_kernel(ActGradArgs a) {
    __shared__ float sums[kThreads / kWave][kCols];
    const int lane = lane_id(), wave = static_cast<int>(threadIdx.x) / kWave;
    const int c0 = static_cast<int>(blockIdx.x) * kCols, c = c0 + lane * 8;
    const int64_t t0 = static_cast<int64_t>(blockIdx.y) * a.rows_per_block;
    const int64_t t1 = t0 + a.rows_per_block < a.T ? t0 + a.rows_per_block : a.T;
    float total[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const int64_t width = a.dz ? a.ldz : a.Z;
    if (c < width) {
        for (int64_t t = t0 + wave; t < t1; t += kThreads / kWave) {
            float v[8];
            dz8<T>(a, t, c, v);
            s16x8 o;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                total[e] += v[e];
                o[e] = static_cast<short>(T::store(v[e]));
            }
            if (a.dz) *reinterpret_cast<s16x8*>(a.dz + t * a.ldz + c) = o;
        }
    }
    if (!a.part) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[wave][lane * 8 + e] = total[e];
    __syncthreads();
    for (int i = static_cast<int>(threadIdx.x); i < kCols && c0 + i < a.Z; i += kThreads) {
        float s = sums[0][i];
#pragma unroll
        for (int w = 1; w < kThreads / kWave; ++w) s += sums[w][i];
        a.part[static_cast<int64_t>(blockIdx.y) * a.Z + c0 + i] = s;
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void colsum_kernel(const float* __restrict__ part, uint16_t* __restrict__ out,
                                                          int Z, int blocks) {
    const int c = static_cast<int>(blockIdx.x) * kThreads + static_cast<int>(threadIdx.x);
    if (c >= Z) return;
    float s = 0.0f;
    for (int b = 0; b < blocks; ++b) s += part[static_cast<int64_t>(b) * Z + c];
    out[c] = T::store(s);
}

}  // namespace

int act_grad_row_blocks(int64_t T, int Z) {
    // about 2048 workgroups over rows and columns, at least 16 rows each (the partial sums stay small beside dz)
    const int64_t cols = (Z + kCols - 1) / kCols;
    const int64_t want = cols > 2048 ? 1 : 2048 / cols;
    const int64_t most = (T + 15) / 16;
    const int64_t n = want < most ? want : most;
    return static_cast<int>(n < 1 ? 1 : n);
}

hipError_t launch_act_grad(const uint16_t* dy, int64_t ldy, const uint16_t* pre, uint16_t* dz, int64_t ldz, float* part,
                           uint16_t* bias_grad, int64_t T, int N, int act, bool bf16, hipStream_t stream) {
    ActGradArgs a{};
    a.dy = dy;
    a.pre = pre;
    a.dz = dz;
    a.part = bias_grad ? part : nullptr;
    a.ldy = ldy;
    a.ldz = ldz;
    a.T = T;
    a.N = N;
    a.Z = act == kActSwiglu ? 2 * N : N;
    a.act = act;
    const int blocks = act_grad_row_blocks(T, a.Z);
    a.rows_per_block = (T + blocks - 1) / blocks;
    const int64_t width = dz ? ldz : a.Z;
    const dim3 grid(static_cast<unsigned>((width + kCols - 1) / kCols), static_cast<unsigned>(blocks));
    {
        TraceScope trace("moe_linear_act_grad", stream);
        if (bf16) act_grad_kernel<Bf16><<<grid, kThreads, 0, stream>>>(a);
        else act_grad_kernel<Half><<<grid, kThreads, 0, stream>>>(a);
    }
    hipError_t err = hipGetLastError();
    if (err != hipSuccess || !bias_grad) return err;
    {
        TraceScope trace("moe_linear_bias_grad", stream);
        const int cgrid = (a.Z + kThreads - 1) / kThreads;
        if (bf16) colsum_kernel<Bf16><<<cgrid, kThreads, 0, stream>>>(part, bias_grad, a.Z, blocks);
        else colsum_kernel<Half><<<cgrid, kThreads, 0, stream>>>(part, bias_grad, a.Z, blocks);
    }
    return hipGetLastError();
}

}  // namespace moe
