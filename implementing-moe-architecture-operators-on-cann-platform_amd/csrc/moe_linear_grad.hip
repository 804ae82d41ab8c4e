// moe_linear_grad.hip -- the elementwise part of MoeLinearGrad: dz = dy * act'(z) and the bias's gradient, the column
// sums of dz.
//
// dz is rounded to the operands' 16-bit type, once, because the two products that take it run on the matrix cores; the
// column sums take it before that rounding. Rows of dz are padded to a multiple of 8 with zeros, so that the products
// read it with 16-byte copies whatever the width.
// Memory bound: dy and z read once, dz written once (SwiGLU: 5 values per output). One workgroup has 64 lanes x 8 columns
// of a block of rows (the 4 waves take rows in turn), so a wave's access is 1 KB of one row; a SwiGLU lane does the gate
// and the up column together. Rows off 16 bytes take loads of any alignment. Column sums go through LDS in wave order to
// one row of `part`; column_sums adds those in a fixed order: no atomics, so the result does not depend on timing.
#include "moe_gemm.h"

namespace moe {

namespace {

constexpr int kThreads = 256;
constexpr int kCols = 512;  // columns of a workgroup

__device__ __forceinline__ float slope(float z, int act) {
    switch (act) {
        case kActRelu: return z > 0.0f ? 1.0f : 0.0f;
        case kActGelu: {
            float e;
            const float c = normal_cdf(z, e);
            return c + z * 0.39894228040143268f * e;
        }
        case kActGeluTanh: {
            const float s = sigmoid_fast(kTanhA * (z + kTanhB * z * z * z));
            return s * (1.0f + z * (1.0f - s) * kTanhA * (1.0f + 3.0f * kTanhB * z * z));
        }
        case kActSilu: {
            const float s = sigmoid_fast(z);
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
    kAny = 0,     // any width and alignment, dz's columns
    kVector = 1,  // aligned 16-byte loads
    kPairs = 2    // aligned 16-byte loads, SwiGLU: y's columns, gate and up together
};

template <typename T>
__device__ __forceinline__ float at(const s16x8& v, int e) {
    return T::load(static_cast<uint16_t>(v[e]));
}

// 8 columns of one dz row from column c on, zeros from Z on: SwiGLU columns below N are the gate's, the others up's
template <typename T>
__device__ __forceinline__ void dz8(const ActGradArgs& a, int64_t t, int c, float (&v)[8]) {
    const uint16_t *dy = a.dy + t * a.ldy, *pre = a.pre + t * a.Z;
    if (a.act == kActSwiglu) {
        const bool up = c >= a.N;
        const int n = up ? c - a.N : c, valid = a.N - n;
        if (valid >= 8 || (up && valid > 0)) {  // all gate or all up
            const s16x8 d = load8(dy + n, valid, n), zg = load8(pre + n, valid, n), zu = load8(pre + a.N + n, valid, n);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float g = at<T>(zg, e), s = sigmoid_fast(g);
                v[e] = e >= valid ? 0.0f : at<T>(d, e) * (up ? g * s : at<T>(zu, e) * s * (1.0f + g * (1.0f - s)));
            }
            return;
        }
#pragma unroll 1
        for (int e = 0; e < 8; ++e) {  // the last gate columns and the first up columns
            const int col = c + e, m = col < a.N ? col : col - a.N;
            float x = 0.0f;
            if (col < a.Z) {
                const float d = T::load(dy[m]), g = T::load(pre[m]), s = sigmoid_fast(g);
                x = d * (col < a.N ? T::load(pre[a.N + m]) * s * (1.0f + g * (1.0f - s)) : g * s);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i == e) v[i] = x;
        }
        return;
    }
    const s16x8 d = load8(dy + c, a.Z - c, c), z = a.pre ? load8(pre + c, a.Z - c, c) : s16x8{};
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = a.pre ? at<T>(d, e) * slope(at<T>(z, e), a.act) : at<T>(d, e);
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
            if constexpr (MODE == kAny) {
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
                        const float s = sigmoid_fast(zg);
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
    else act_grad_kernel<T, kAny><<<grid, kThreads, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace

int act_grad_row_blocks(int64_t T, int Z) {
    // about 2048 workgroups over rows and columns, at least 8 rows each (two a wave)
    const int64_t cols = (Z + kCols - 1) / kCols;
    const int64_t want = cols > 2048 ? 1 : 2048 / cols;
    const int64_t most = (T + 7) / 8;
    const int64_t n = want < most ? want : most;
    return static_cast<int>(n < 1 ? 1 : n);
}

hipError_t launch_act_grad(const uint16_t* dy, int64_t ldy, const uint16_t* pre, uint16_t* dz, int64_t ldz, float* part,
                           int64_t T, int N, int act, bool bf16, hipStream_t stream) {
    ActGradArgs a{};
    a.dy = dy;
    a.pre = pre;
    a.dz = dz;
    a.part = part;
    a.ldy = ldy;
    a.ldz = ldz;
    a.T = T;
    a.N = N;
    a.Z = act == kActSwiglu ? 2 * N : N;
    a.act = act;
    const int blocks = act_grad_row_blocks(T, a.Z);
    a.rows_per_block = (T + blocks - 1) / blocks;
    return bf16 ? run_act_grad<Bf16>(a, blocks, stream) : run_act_grad<Half>(a, blocks, stream);
}

}  // namespace moe
