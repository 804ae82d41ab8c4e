// moe_rows.h -- rows of fp16, bf16 or fp32 values, at any alignment, and their 8-bit form; shared by the
// kernels that work row by row (moe_norm.hip, moe_expert_rows.hip).
#pragma once

#include "moe_gemm.h"

namespace moe {

struct F32 {
    using Bits = float;
    static __device__ __forceinline__ float load(float v) { return v; }
    static __device__ __forceinline__ float store(float v) { return v; }
};

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
// Vectors at any address: the hardware takes them, only the compiler has to know
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));

// Rows are taken V values a lane and step: 8, or 1 of rows shorter than 8. The last step of a row whose length is no
// multiple of 8 begins 8 before the row's end, so it repeats values of the step before it (both lanes compute and write
// the same), which only sums have to leave out. at: the first column, <= that of the step; skip: values to leave out.
template <int V>
struct Step {
    int at, skip;
    bool live;  // false: past the row; `at` is a column that can be read all the same
};
template <int V>
__device__ __forceinline__ Step<V> step_at(int col, int H) {
    const bool live = col < H;
    const int at = min(col, H - V);
    return Step<V>{live ? at : 0, live ? col - at : V, live};
}
// The same for lanes that all read and write: those past the row repeat its last values
template <int V>
__device__ __forceinline__ Step<V> step_repeating(int col, int H) {
    const int at = min(col, H - V);
    return Step<V>{at, min(col - at, V), true};
}

// V values as they are stored
template <typename T, int V>
struct RawRow {
    static constexpr int kVectors = V * sizeof(typename T::Bits) / 16;
    u32x4 v[kVectors];
    template <bool NT = false>  // past the caches
    __device__ __forceinline__ void load(const typename T::Bits* p) {
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
            const u32x4_any* at = reinterpret_cast<const u32x4_any*>(p + i * (16 / sizeof(typename T::Bits)));
            v[i] = NT ? __builtin_nontemporal_load(at) : *at;
        }
    }
    __device__ __forceinline__ float get(int j) const {
        if constexpr (sizeof(typename T::Bits) == 4) {
            const uint32_t b = v[j / 4][j % 4];  // a value: of a vector's element the cast would take the first one
            return __builtin_bit_cast(float, b);
        } else {
            return T::load(static_cast<uint16_t>(v[0][j / 2] >> (j % 2 * 16)));
        }
    }
};
template <typename T>
struct RawRow<T, 1> {
    typename T::Bits v;
    template <bool NT = false>
    __device__ __forceinline__ void load(const typename T::Bits* p) { v = *p; }
    __device__ __forceinline__ float get(int) const { return T::load(v); }
};

template <typename T, int V>
__device__ __forceinline__ void load_row(const typename T::Bits* p, float (&v)[V]) {
    RawRow<T, V> raw;
    raw.load(p);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = raw.get(j);
}

// 16 bytes of a result, past the caches where it will not be read from them
template <bool NT>
__device__ __forceinline__ void store16(void* p, u32x4 v) {
    if (NT) __builtin_nontemporal_store(v, static_cast<u32x4_any*>(p));
    else *static_cast<u32x4_any*>(p) = v;
}

template <typename T, int V, bool NT = false>
__device__ __forceinline__ void store_row(typename T::Bits* p, const float (&v)[V]) {
    if constexpr (V == 1) {
        *p = T::store(v[0]);
    } else if constexpr (sizeof(typename T::Bits) == 2) {
        const uint2 a = pack4<T>(f32x4{v[0], v[1], v[2], v[3]}), b = pack4<T>(f32x4{v[4], v[5], v[6], v[7]});
        store16<NT>(p, u32x4{a.x, a.y, b.x, b.y});
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h)
            store16<NT>(p + 4 * h,
                        __builtin_bit_cast(u32x4, f32x4{v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]}));
    }
}

// All-reduce over a whole wave, every lane active: the lanes of a DPP row of 16 by rotations, then the four rows'
// results
template <int CTRL>
__device__ __forceinline__ uint32_t turned(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), CTRL, 0xf, 0xf, true));
}
template <int CTRL>
__device__ __forceinline__ float turned(float v) {
    return __builtin_bit_cast(float, turned<CTRL>(__builtin_bit_cast(uint32_t, v)));
}
template <int CTRL>
__device__ __forceinline__ double turned(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint64_t hi = turned<CTRL>(static_cast<uint32_t>(b >> 32)), lo = turned<CTRL>(static_cast<uint32_t>(b));
    return __builtin_bit_cast(double, hi << 32 | lo);
}
__device__ __forceinline__ uint32_t of_lane(uint32_t v, int lane) {
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane));
}
__device__ __forceinline__ float of_lane(float v, int lane) {
    return __builtin_bit_cast(float, of_lane(__builtin_bit_cast(uint32_t, v), lane));
}
__device__ __forceinline__ double of_lane(double v, int lane) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint64_t hi = of_lane(static_cast<uint32_t>(b >> 32), lane), lo = of_lane(static_cast<uint32_t>(b), lane);
    return __builtin_bit_cast(double, hi << 32 | lo);
}
template <typename V>
__device__ __forceinline__ V wave_sum(V v) {
    v += turned<0x128>(v);
    v += turned<0x124>(v);
    v += turned<0x122>(v);
    v += turned<0x121>(v);
    return (of_lane(v, 0) + of_lane(v, 16)) + (of_lane(v, 32) + of_lane(v, 48));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = max(v, turned<0x128>(v));
    v = max(v, turned<0x124>(v));
    v = max(v, turned<0x122>(v));
    v = max(v, turned<0x121>(v));
    return max(max(of_lane(v, 0), of_lane(v, 16)), max(of_lane(v, 32), of_lane(v, 48)));
}

// Rows as 8-bit integers: q = rint(p * (127 / top)), top the row's largest magnitude; the quotient and the products are
// rounded to fp32 (no contraction), so the integers depend on the values alone. A top below 2^-60, whose quotient could
// overflow, is taken with the values times 2^64. A row with an infinity or a NaN has zeros (and scale NaN).
struct RowQuant {
    float up, inverse;
    bool finite;
};
// top_bits: the largest of the magnitudes' bit patterns, which order as the magnitudes do, NaN above all
__device__ __forceinline__ RowQuant row_quant(uint32_t top_bits) {
#pragma clang fp contract(off)
    const float top = __builtin_bit_cast(float, top_bits);
    RowQuant r;
    r.finite = top_bits < 0x7f800000u;
    r.up = top < 0x1p-60f ? 0x1p64f : 1.0f;
    r.inverse = r.finite && top > 0.0f ? 127.0f / (top * r.up) : 0.0f;
    return r;
}
// One of them in the low byte: adding 1.5 * 2^23 rounds to the nearest integer (ties to even) and leaves it there
__device__ __forceinline__ uint32_t quantize(float p, const RowQuant& r) {
#pragma clang fp contract(off)
    return __builtin_bit_cast(uint32_t, (r.finite ? p * r.up : 0.0f) * r.inverse + 12582912.0f);
}
template <int V>
__device__ __forceinline__ void store_quant(int8_t* q, const float (&p)[V], const RowQuant& r) {
    if constexpr (V == 1) {
        *q = static_cast<int8_t>(quantize(p[0], r));
    } else {
        uint32_t b[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) b[j] = quantize(p[j], r) & 255u;
        *reinterpret_cast<u32x2_any*>(q) =
            u32x2{b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24, b[4] | b[5] << 8 | b[6] << 16 | b[7] << 24};
    }
}

}  // namespace moe
