// moe_linear_grad.hip -- the elementwise part of MoeLinearGrad: dz = dy * act'(z) and the bias's gradient, the column
// sums of dz.
//
// dz is rounded to the operands' 16-bit type, once, because the two products that take it run on the matrix cores; the
// column sums take it before that rounding. dy may be fp32, the gradient of an fp32 result: fp16 would lose what is
// below 6e-8 of it and overflow above 65504, so dz is then multiplied by the power of two that takes its largest finite
// value to [2^14, 2^15). A first launch finds that value (its maxima of workgroups, which every workgroup of the second
// reads), and the products' epilogue multiplies by the inverse before it rounds. bf16 has fp32's range and needs none.
// T = 4096, Z = 256: 4.7 us for the value, 4.9 for dz.
// Rows of dz are padded to a multiple of 8 with zeros, so that the products read it with 16-byte copies whatever the
// width. Memory bound: dy and z read once, dz written once (SwiGLU: 5 values per output). One workgroup has 64 lanes x
// 8 columns of a block of rows (the 4 waves take rows in turn), so a wave's access is 1 KB of one row; a SwiGLU lane
// does the gate and the up column together. Rows off 16 bytes take loads of any alignment. Column sums go through LDS
// in wave order to one row of `part`; column_sums adds those in a fixed order: no atomics, so the result does not
// depend on timing.
#include "moe_gemm.h"

#include <type_traits>

namespace moe {

namespace {

constexpr int kThreads = 256;
constexpr int kCols = 512;  // columns of a workgroup

// pre may hold infinities and values whose powers overflow: a sum that is finite in fp32 rounds to them. From +-128 on
// every slope below is at its limit in fp32, where the formulas would give 0 * infinity. NaN stays.
__device__ __forceinline__ float bounded(float z) { return fabsf(z) > 128.0f ? copysignf(128.0f, z) : z; }

__device__ __forceinline__ float slope(float v, int act) {
    const float z = bounded(v);
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
// silu's slope at a SwiGLU's gate g, and silu itself, which grows with g
__device__ __forceinline__ float silu_slope(float g, float& silu) {
    const float z = bounded(g), s = sigmoid_fast(z);
    silu = (g < -128.0f ? z : g) * s;
    return s * (1.0f + z * (1.0f - s));
}

struct ActGradArgs {
    const void* dy;       // [T, N], rows ldy apart
    const uint16_t* pre;  // [T, N] (SwiGLU: [T, 2N]) contiguous, or null (no activation)
    uint16_t* dz;         // [T, ldz] or null (the column sums alone)
    float* part;          // [row blocks, Z] column sums or null
    float* peaks;         // the largest |dz| of npeaks workgroups, the scale's inverse at kGradPeaks; or null
    int npeaks;
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

// dy's values: D is uint16_t (the operands' type T) or float
template <typename T>
__device__ __forceinline__ float dy_value(const uint16_t* p) {
    return T::load(*p);
}
template <typename T>
__device__ __forceinline__ float dy_value(const float* p) {
    return *p;
}
template <typename T>
__device__ __forceinline__ void load_dy8(const uint16_t* p, int valid, int before, float (&d)[8]) {
    const s16x8 x = load8(p, valid, before);
#pragma unroll
    for (int e = 0; e < 8; ++e) d[e] = at<T>(x, e);
}
template <typename T>
__device__ __forceinline__ void load_dy8(const float* p, int valid, int, float (&d)[8]) {
    typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
    if (valid >= 8) {
        const f32x4 x = *reinterpret_cast<const f32x4_any*>(p), y = *reinterpret_cast<const f32x4_any*>(p + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) d[e] = x[e], d[e + 4] = y[e];
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) d[e] = e < valid ? p[e] : 0.0f;
}

// 8 columns of one dz row from column c on, zeros from Z on: SwiGLU columns below N are the gate's, the others up's
template <typename T, typename D>
__device__ __forceinline__ void dz8(const ActGradArgs& a, int64_t t, int c, float (&v)[8]) {
    const D* dy = static_cast<const D*>(a.dy) + t * a.ldy;
    const uint16_t* pre = a.pre + t * a.Z;
    float d[8];
    if (a.act == kActSwiglu) {
        const bool up = c >= a.N;
        const int n = up ? c - a.N : c, valid = a.N - n;
        if (valid >= 8 || (up && valid > 0)) {  // all gate or all up
            load_dy8<T>(dy + n, valid, n, d);
            const s16x8 zg = load8(pre + n, valid, n), zu = load8(pre + a.N + n, valid, n);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float silu;
                const float s = silu_slope(at<T>(zg, e), silu);
                v[e] = e >= valid ? 0.0f : d[e] * (up ? silu : at<T>(zu, e) * s);
            }
            return;
        }
#pragma unroll 1
        for (int e = 0; e < 8; ++e) {  // the last gate columns and the first up columns
            const int col = c + e, m = col < a.N ? col : col - a.N;
            float x = 0.0f;
            if (col < a.Z) {
                float silu;
                const float s = silu_slope(T::load(pre[m]), silu);
                x = dy_value<T>(dy + m) * (col < a.N ? T::load(pre[a.N + m]) * s : silu);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i == e) v[i] = x;
        }
        return;
    }
    load_dy8<T>(dy + c, a.Z - c, c, d);
    const s16x8 z = a.pre ? load8(pre + c, a.Z - c, c) : s16x8{};
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = a.pre ? d[e] * slope(at<T>(z, e), a.act) : d[e];
}

// The largest of v over the workgroup, in every thread
__device__ __forceinline__ float workgroup_max(float v) {
    __shared__ float tops[kThreads / kWave];
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, kWave));
    if (lane_id() == 0) tops[threadIdx.x / kWave] = v;
    __syncthreads();
    v = tops[0];
#pragma unroll
    for (int w = 1; w < kThreads / kWave; ++w) v = fmaxf(v, tops[w]);
    return v;
}

// The largest finite |dz| of a workgroup's granules
template <typename T>
__global__ __launch_bounds__(kThreads) void grad_peak_kernel(ActGradArgs a) {
    const int per = (a.Z + 7) / 8;
    const int64_t granules = a.T * per, step = static_cast<int64_t>(gridDim.x) * kThreads;
    float most = 0.0f;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < granules; i += step) {
        float v[8];
        const int64_t t = i / per;
        dz8<T, float>(a, t, static_cast<int>(i - t * per) * 8, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float x = fabsf(v[e]);
            most = x > most && x < __builtin_huge_valf() ? x : most;  // not NaN
        }
    }
    most = workgroup_max(most);
    if (threadIdx.x == 0) a.peaks[blockIdx.x] = most;
}

// log2 of dz's scale: every finite |dz| times that is below 2^15, and both it and its inverse are normal numbers
__device__ __forceinline__ int scale_log2(const ActGradArgs& a) {
    const int i = static_cast<int>(threadIdx.x);
    const float most = workgroup_max(i < a.npeaks ? a.peaks[i] : 0.0f);
    return most > 0.0f ? min(14 - ilogbf(most), 126) : 0;
}

template <typename T>
__device__ __forceinline__ s16x8 round8(const float (&v)[8], float scale) {
    s16x8 o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = static_cast<short>(T::store(v[e] * scale));
    return o;
}

template <typename T, int MODE, typename D>
__global__ __launch_bounds__(kThreads) void act_grad_kernel(ActGradArgs a) {
    constexpr int kSums = MODE == kPairs ? 2 : 1;
    __shared__ float sums[kThreads / kWave][kSums][kCols];
    const int lane = lane_id(), wave = static_cast<int>(threadIdx.x) / kWave;
    const int c0 = static_cast<int>(blockIdx.x) * kCols, c = c0 + lane * 8;
    const int64_t t0 = static_cast<int64_t>(blockIdx.y) * a.rows_per_block;
    const int64_t t1 = t0 + a.rows_per_block < a.T ? t0 + a.rows_per_block : a.T;
    float total[kSums][8] = {}, scale = 1.0f;
    if constexpr (std::is_same_v<D, float>) {
        if (a.peaks) {
            const int log2 = scale_log2(a);
            scale = ldexpf(1.0f, log2);
            if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) a.peaks[kGradPeaks] = ldexpf(1.0f, -log2);
        }
    }
    const int64_t width = MODE == kPairs ? a.N : a.dz ? a.ldz : a.Z;
    if (c < width) {
#pragma unroll 2
        for (int64_t t = t0 + wave; t < t1; t += kThreads / kWave) {
            float v[kSums][8];
            if constexpr (MODE == kAny) {
                dz8<T, D>(a, t, c, v[0]);
            } else {
                const s16x8 d = *reinterpret_cast<const s16x8*>(static_cast<const uint16_t*>(a.dy) + t * a.ldy + c);
                s16x8 z = {}, u = {};
                if (a.pre) z = *reinterpret_cast<const s16x8*>(a.pre + t * a.Z + c);
                if (MODE == kPairs) u = *reinterpret_cast<const s16x8*>(a.pre + t * a.Z + a.N + c);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float dy = T::load(static_cast<uint16_t>(d[e])), zg = T::load(static_cast<uint16_t>(z[e]));
                    if (MODE == kPairs) {
                        float silu;
                        const float s = silu_slope(zg, silu);
                        v[0][e] = dy * T::load(static_cast<uint16_t>(u[e])) * s;
                        v[kSums - 1][e] = dy * silu;
                    } else {
                        v[0][e] = a.pre ? dy * slope(zg, a.act) : dy;
                    }
                }
            }
#pragma unroll
            for (int q = 0; q < kSums; ++q) {
#pragma unroll
                for (int e = 0; e < 8; ++e) total[q][e] += v[q][e];
                if (a.dz) *reinterpret_cast<s16x8*>(a.dz + t * a.ldz + q * a.N + c) = round8<T>(v[q], scale);
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
    if (pairs) act_grad_kernel<T, kPairs, uint16_t><<<grid, kThreads, 0, stream>>>(a);
    else if (aligned) act_grad_kernel<T, kVector, uint16_t><<<grid, kThreads, 0, stream>>>(a);
    else act_grad_kernel<T, kAny, uint16_t><<<grid, kThreads, 0, stream>>>(a);
    return hipGetLastError();
}

// fp32 dy: one path for every width and alignment
template <typename T>
hipError_t run_act_grad_f32(ActGradArgs a, int blocks, hipStream_t stream) {
    TraceScope trace("moe_linear_act_grad", stream);
    if (a.peaks) {
        const int64_t groups = (a.T * ((a.Z + 7) / 8) + kThreads - 1) / kThreads;
        a.npeaks = static_cast<int>(groups < kGradPeaks ? groups : kGradPeaks);
        grad_peak_kernel<T><<<static_cast<unsigned>(a.npeaks), kThreads, 0, stream>>>(a);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return err;
    }
    const int64_t width = a.dz ? a.ldz : a.Z;
    const dim3 grid(static_cast<unsigned>((width + kCols - 1) / kCols), static_cast<unsigned>(blocks));
    act_grad_kernel<T, kAny, float><<<grid, kThreads, 0, stream>>>(a);
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

hipError_t launch_act_grad(const ActGrad& g, hipStream_t stream) {
    ActGradArgs a{};
    a.dy = g.dy;
    a.pre = g.pre;
    a.dz = g.dz;
    a.part = g.part;
    a.peaks = g.peaks;
    a.ldy = g.ldy;
    a.ldz = g.ldz;
    a.T = g.T;
    a.N = g.N;
    a.Z = g.act == kActSwiglu ? 2 * g.N : g.N;
    a.act = g.act;
    const int blocks = act_grad_row_blocks(a.T, a.Z);
    a.rows_per_block = (a.T + blocks - 1) / blocks;
    if (g.dy_f32)
        return g.bf16 ? run_act_grad_f32<Bf16>(a, blocks, stream) : run_act_grad_f32<Half>(a, blocks, stream);
    return g.bf16 ? run_act_grad<Bf16>(a, blocks, stream) : run_act_grad<Half>(a, blocks, stream);
}

}  // namespace moe
