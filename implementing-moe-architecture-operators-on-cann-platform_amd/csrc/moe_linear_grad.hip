// moe_linear_grad.hip -- the elementwise part of MoeLinearGrad: dz = dy * act'(z) and the bias's gradient, the column
// sums of dz.
//
// dz is rounded to the operands' 16-bit type, once, because the two products that take it run on the matrix cores; the
// column sums take it before that rounding. Rows of dz are padded to a multiple of 8 with zeros, so that the products
// read it with 16-byte copies whatever the width.
// Memory bound: dy and z read once, dz written once (SwiGLU: 5 values per output). One workgroup has 64 lanes x 8 columns
// of a block of rows (the 4 waves take rows in turn), so a wave's access is 1 KB of one row; a SwiGLU lane does the gate
// and the up column together. Rows off 16 bytes are read element by element. Column sums go through LDS in wave order to
// one row of `part`; colsum_kernel adds those in a fixed order: no atomics, so the result does not depend on timing.
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

// How the columns of a workgroup are read and computed
enum Mode {
    kScalar = 0,  // any width and alignment, dz's columns
    kVector = 1,  // 16-byte loads
    kPairs = 2    // 16-byte loads, SwiGLU: y's columns, gate and up together
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
__device__ __forceinline__ s16x8 round8(const float (&v)[8]) {
    s16x8 o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = static_cast<short>(T::store(v[e]));
    return o;
}

template <typename T, int MODE>
__global__ __launch_bounds__(kThreads) void act_grad_kernel(ActGradArgs a) {
    constexpr int kSums = MODE == kPairs ? 2 : 1;
    __shared__ float sums[kThreads / kWave][kSums][kCols];
    const int lane = lane_id(), wave = static_cast<int>(threadIdx.x) / kWave;
    const int c0 = static_cast<int>(blockIdx.x) * kCols, c = c0 + lane * 8;
    const int64_t t0 = static_cast<int64_t>(blockIdx.y) * a.rows_per_block;
    const int64_t t1 = t0 + a.rows_per_block < a.T ? t0 + a.rows_per_block : a.T;
    float total[kSums][8] = {};
    const int64_t width = MODE == kPairs ? a.N : a.dz ? a.ldz : a.Z;
    if (c < width) {
#pragma unroll 2
        for (int64_t t = t0 + wave; t < t1; t += kThreads / kWave) {
            float v[kSums][8];
            if constexpr (MODE == kScalar) {
                dz8<T>(a, t, c, v[0]);
            } else {
                const s16x8 d = *reinterpret_cast<const s16x8*>(a.dy + t * a.ldy + c);
                s16x8 z = {}, u = {};
                if (a.pre) z = *reinterpret_cast<const s16x8*>(a.pre + t * a.Z + c);
                if (MODE == kPairs) u = *reinterpret_cast<const s16x8*>(a.pre + t * a.Z + a.N + c);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float dy = T::load(static_cast<uint16_t>(d[e])), zg = T::load(static_cast<uint16_t>(z[e]));
                    if (MODE == kPairs) {
                        const float s = 1.0f / (1.0f + expf(-zg));
                        v[0][e] = dy * T::load(static_cast<uint16_t>(u[e])) * s * (1.0f + zg * (1.0f - s));
                        v[kSums - 1][e] = dy * zg * s;
                    } else {
                        v[0][e] = a.pre ? dy * slope(zg, a.act) : dy;
                    }
                }
            }
#pragma unroll
            for (int q = 0; q < kSums; ++q) {
#pragma unroll
                for (int e = 0; e < 8; ++e) total[q][e] += v[q][e];
                if (a.dz) *reinterpret_cast<s16x8*>(a.dz + t * a.ldz + q * a.N + c) = round8<T>(v[q]);
            }
        }
    }
    if (!a.part) return;
#pragma unroll
    for (int q = 0; q < kSums; ++q)
#pragma unroll
        for (int e = 0; e < 8; ++e) sums[wave][q][lane * 8 + e] = total[q][e];
    __syncthreads();
    const int valid = MODE == kPairs ? a.N : a.Z;
    for (int i = static_cast<int>(threadIdx.x); i < kCols && c0 + i < valid; i += kThreads) {
#pragma unroll
        for (int q = 0; q < kSums; ++q) {
            float s = sums[0][q][i];
#pragma unroll
            for (int w = 1; w < kThreads / kWave; ++w) s += sums[w][q][i];
            a.part[static_cast<int64_t>(blockIdx.y) * a.Z + q * a.N + c0 + i] = s;
        }
    }
}

// 16 columns a workgroup; its 16 groups of threads add every 16th row of `part`, then the groups' sums in order
constexpr int kGroups = 16, kColsSum = kThreads / kGroups;
template <typename T>
__global__ __launch_bounds__(kThreads) void colsum_kernel(const float* __restrict__ part, uint16_t* __restrict__ out,
                                                          int Z, int blocks) {
    __shared__ float sums[kGroups][kColsSum];
    const int i = static_cast<int>(threadIdx.x) % kColsSum, q = static_cast<int>(threadIdx.x) / kColsSum;
    const int c = static_cast<int>(blockIdx.x) * kColsSum + i;
    float s = 0.0f;
    if (c < Z) {
#pragma unroll 4
        for (int b = q; b < blocks; b += kGroups) s += part[static_cast<int64_t>(b) * Z + c];
    }
    sums[q][i] = s;
    __syncthreads();
    if (q != 0 || c >= Z) return;
#pragma unroll
    for (int g = 1; g < kGroups; ++g) s += sums[g][i];
    out[c] = T::store(s);
}

template <typename T>
hipError_t run_act_grad(const ActGradArgs& a, int blocks, hipStream_t stream) {
    const bool aligned = a.N % 8 == 0 && a.ldy % 8 == 0 &&
                         ((reinterpret_cast<uintptr_t>(a.dy) | reinterpret_cast<uintptr_t>(a.pre)) & 15) == 0;
    const bool pairs = aligned && a.act == kActSwiglu;
    const int64_t width = pairs ? a.N : a.dz ? a.ldz : a.Z;
    const dim3 grid(static_cast<unsigned>((width + kCols - 1) / kCols), static_cast<unsigned>(blocks));
    TraceScope trace("moe_linear_act_grad", stream);
    if (pairs) act_grad_kernel<T, kPairs><<<grid, kThreads, 0, stream>>>(a);
    else if (aligned) act_grad_kernel<T, kVector><<<grid, kThreads, 0, stream>>>(a);
    else act_grad_kernel<T, kScalar><<<grid, kThreads, 0, stream>>>(a);
    return hipGetLastError();
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
    hipError_t err = bf16 ? run_act_grad<Bf16>(a, blocks, stream) : run_act_grad<Half>(a, blocks, stream);
    if (err != hipSuccess || !bias_grad) return err;
    {
        TraceScope trace("moe_linear_bias_grad", stream);
        const int cgrid = (a.Z + kColsSum - 1) / kColsSum;
        if (bf16) colsum_kernel<Bf16><<<cgrid, kThreads, 0, stream>>>(part, bias_grad, a.Z, blocks);
        else colsum_kernel<Half><<<cgrid, kThreads, 0, stream>>>(part, bias_grad, a.Z, blocks);
    }
    return hipGetLastError();
}

}  // namespace moe
