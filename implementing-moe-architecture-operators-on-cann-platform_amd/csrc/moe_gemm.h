// moe_gemm.h -- pieces shared by the dense product kernels (moe_linear*.hip): element types, operand layouts, the
// fused epilogue and the arguments of a product.
#pragma once

#include "moe_device.h"
#include "moe_launch.h"

namespace moe {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

// 16-bit element types of the products; storage is uint16_t bits everywhere
struct Half {
    static __device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    }
    static __device__ __forceinline__ float load(uint16_t b) { return f16_bits_to_f32(b); }
    static __device__ __forceinline__ uint16_t store(float v) { return f32_to_f16_bits(v); }
};
struct Bf16 {
    static __device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    }
    static __device__ __forceinline__ float load(uint16_t b) {
        return __builtin_bit_cast(float, static_cast<uint32_t>(b) << 16);
    }
    // round to nearest even (v_cvt_pk_bf16_f32), NaN kept
    static __device__ __forceinline__ uint16_t store(float v) {
        return __builtin_bit_cast(uint16_t, static_cast<__bf16>(v));
    }
};

// A product C[m][n] = sum_k P[m][k] Q[n][k]. An operand is stored by rows (its k contiguous, rows `ld` elements apart)
// or by k (its rows contiguous, the k `ld` elements apart).
struct GemmArgs {
    const uint16_t* p;
    const uint16_t* q;
    int64_t ldp, ldq;
    int m, n, k;          // n: output columns; with SwiGLU Q has 2 n rows, the n gate rows first
    void* out;            // [m, n], contiguous
    uint16_t* pre;        // [m, n or 2 n] sums before the activation, rounded to the operands' type; may be null
    const uint16_t* bias; // [n or 2 n] or null
    const void* residual; // [m, n] of out's type or null
    int act;              // moe_activation
    int out_f32;          // out (and residual) fp32, else the operands' type
    float* partial;       // [splits, m, part_ld] fp32 sums of a product split over k
    int splits;           // 1: the whole k in one workgroup, through the epilogue
    int split_k;          // k of one split, a multiple of the kernels' stage
};

// Row pitch of the partial sums: columns (SwiGLU: gate and up apart) rounded up to whole 16-byte stores
__host__ __device__ constexpr int64_t part_cols(int n) { return (static_cast<int64_t>(n) + 3) / 4 * 4; }
__host__ __device__ constexpr int64_t part_ld(int n, bool swiglu) { return part_cols(n) * (swiglu ? 2 : 1); }

// Activations in fp32. gelu through erfc: 1 + erf(z / sqrt 2) loses every digit for large negative z.
__device__ __forceinline__ float activate(float z, int act) {
    switch (act) {
        case kActRelu: return z > 0.0f ? z : (z != z ? z : 0.0f);
        case kActGelu: return 0.5f * z * erfcf(z * -0.70710678118654752f);
        case kActGeluTanh: return 0.5f * z * (1.0f + tanhf(0.79788456080286536f * (z + 0.044715f * z * z * z)));
        case kActSilu: return z / (1.0f + expf(-z));
        default: return z;
    }
}

// 4 consecutive columns col .. col + 3 of one output row (those below n; `vec`: rows start on whole vectors, so four
// valid columns are one access), from the sums z (SwiGLU: of the gate) and u (of the up rows).
template <typename T, bool SWIGLU>
__device__ __forceinline__ void store4(const GemmArgs& g, int64_t row, int col, f32x4 z, f32x4 u, bool vec) {
    if (col >= g.n) return;
    const int valid = min(4, g.n - col);
    const bool whole = vec && valid == 4;
    if (g.bias) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (r < valid) {
                z[r] += T::load(g.bias[col + r]);
                if (SWIGLU) u[r] += T::load(g.bias[g.n + col + r]);
            }
        }
    }
    if (g.pre) {
        uint16_t* pz = g.pre + row * (SWIGLU ? 2 * static_cast<int64_t>(g.n) : g.n) + col;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (r < valid) {
                pz[r] = T::store(z[r]);
                if (SWIGLU) pz[g.n + r] = T::store(u[r]);
            }
        }
    }
    float y[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) y[r] = SWIGLU ? swiglu_f32(z[r], u[r]) : activate(z[r], g.act);
    const int64_t at = row * g.n + col;
    if (g.out_f32) {
        const float* res = static_cast<const float*>(g.residual);
        float* out = static_cast<float*>(g.out) + at;
        if (whole) {
            f32x4 v = {y[0], y[1], y[2], y[3]};
            if (res) v += *reinterpret_cast<const f32x4*>(res + at);
            *reinterpret_cast<f32x4*>(out) = v;
        } else {
            for (int r = 0; r < valid; ++r) out[r] = res ? y[r] + res[at + r] : y[r];
        }
    } else {
        const uint16_t* res = static_cast<const uint16_t*>(g.residual);
        uint16_t* out = static_cast<uint16_t*>(g.out) + at;
        if (whole) {
            if (res) {
                const uint2 v = *reinterpret_cast<const uint2*>(res + at);
                y[0] += T::load(static_cast<uint16_t>(v.x));
                y[1] += T::load(static_cast<uint16_t>(v.x >> 16));
                y[2] += T::load(static_cast<uint16_t>(v.y));
                y[3] += T::load(static_cast<uint16_t>(v.y >> 16));
            }
            *reinterpret_cast<uint2*>(out) =
                make_uint2(T::store(y[0]) | (static_cast<uint32_t>(T::store(y[1])) << 16),
                           T::store(y[2]) | (static_cast<uint32_t>(T::store(y[3])) << 16));
        } else {
            for (int r = 0; r < valid; ++r) out[r] = T::store(res ? y[r] + T::load(res[at + r]) : y[r]);
        }
    }
}

// Whether store4 may use whole vectors: 4 columns are 8 or 16 bytes, aligned in every row
__host__ __device__ __forceinline__ bool vector_rows(const GemmArgs& g) {
    const uintptr_t mask = g.out_f32 ? 15 : 7;
    return g.n % 4 == 0 && ((reinterpret_cast<uintptr_t>(g.out) | reinterpret_cast<uintptr_t>(g.residual)) & mask) == 0;
}

// ds_read_b64_tr_b16: 8 bytes per lane, handed out transposed within each 16-lane group (lane i gets element i % 4 of
// the 8 bytes addressed by lanes 4 j + i / 4, j = 0 .. 3)
__device__ __forceinline__ s16x4 lds_read_transposed(const uint16_t* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p));
}

// kernels' launches
hipError_t launch_gemm_mid(const GemmArgs& g, bool p_by_k, bool q_by_k, bool bf16, bool direct, int bm,
                           hipStream_t stream);
hipError_t launch_gemm_reduce(const GemmArgs& g, bool bf16, hipStream_t stream);

}  // namespace moe
