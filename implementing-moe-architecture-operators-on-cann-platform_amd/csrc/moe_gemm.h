// moe_gemm.h -- pieces shared by the dense product kernels (moe_linear*.hip): element types, operand layouts, the
// fused epilogue and the arguments of a product.
#pragma once

#include "moe_device.h"
#include "moe_launch.h"

#include <type_traits>

namespace moe {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

// 16-bit element types of the products; storage is uint16_t bits everywhere
struct Half {
    using Bits = uint16_t;
    static constexpr bool kInt8 = false;
    static __device__ __forceinline__ f32x4 add(f32x4 a, f32x4 b) { return a + b; }
    static __device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    }
    static __device__ __forceinline__ float load(uint16_t b) { return f16_bits_to_f32(b); }
    static __device__ __forceinline__ uint16_t store(float v) { return f32_to_f16_bits(v); }
};
struct Bf16 {
    using Bits = uint16_t;
    static constexpr bool kInt8 = false;
    static __device__ __forceinline__ f32x4 add(f32x4 a, f32x4 b) { return a + b; }
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

// 8-bit integers with results of type O. A pair of them stands where the 16-bit types have one value, so the kernels
// move the same bytes: k, the strides and the stages count pairs (of operands that 16-byte copies cannot read, bytes).
// The fp32 registers of the sums hold int32 bits up to the epilogue, which applies the scales; k is short enough that
// no sum leaves 32 bits.
template <typename O>
struct Int8 {
    using Bits = uint16_t;
    static constexpr bool kInt8 = true;
    static __device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c) {
        return __builtin_bit_cast(
            f32x4, __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b),
                                                         __builtin_bit_cast(i32x4, c), 0, 0, 0));
    }
    static __device__ __forceinline__ f32x4 add(f32x4 a, f32x4 b) {
        return __builtin_bit_cast(f32x4, __builtin_bit_cast(i32x4, a) + __builtin_bit_cast(i32x4, b));
    }
    static __device__ __forceinline__ float load(uint16_t b) { return O::load(b); }
    // Of the fp32 value, in every kernel: where nothing stands between them the compiler makes one instruction of the
    // last product and its conversion to fp16, which leaves out the product's rounding and changes 1 value in 17000
    static __device__ __forceinline__ uint16_t store(float v) {
        if constexpr (std::is_same_v<O, Half>) asm("" : "+v"(v));
        return O::store(v);
    }
};

// A product C[m][n] = sum_k P[m][k] Q[n][k]. An operand is stored by rows (its k contiguous, rows `ld` elements apart)
// or by k (its rows contiguous, the k `ld` elements apart).
struct GemmArgs {
    const uint16_t* p;
    const uint16_t* q;
    int64_t ldp, ldq;
    int m, n, k;          // n: output columns; with SwiGLU Q has 2 n rows, the n gate rows first
    int up;               // Q row of the first up row: n, or past a repacked operand's padding
    void* out;            // [m, n], contiguous
    uint16_t* pre;        // [m, n or 2 n] sums before the activation, rounded to the operands' type; may be null
    const uint16_t* bias; // [n or 2 n] or null
    const void* residual; // [m, n] of out's type or null
    const float* factor;  // device: multiplies the sums first (an operand was scaled); null: 1. Not with SwiGLU
    int act;              // moe_activation
    int out_f32;          // out (and residual) fp32, else the operands' type
    float* partial;       // [splits, m, part_ld] fp32 sums of a product split over k
    int splits;           // 1: the whole k in one workgroup, through the epilogue
    int split_k;          // k of one split, a multiple of the kernels' stage
    const float* row_scale;  // 8-bit operands: [m], and [n or 2 n] of the columns; bias then is of out's type
    const float* col_scale;
    // Products of experts: P rows [offsets[e], offsets[e + 1]), of the first from 0 on, by Q + e q_expert (bytes), with
    // the columns' scales and bias from e (n or 2 n) on; rows from offsets[experts] on are zeros. 0: one product
    int experts;
    int64_t q_expert;
    const int32_t* offsets;
};

// An item of the experts' products: items are the tiles of bm rows x ntiles of one expert after another
struct GroupItem {
    int expert, row0, row1;  // of the expert
    int first;               // its first item
};
__device__ __forceinline__ const uint16_t* group_q(const GemmArgs& g, int e) {
    return reinterpret_cast<const uint16_t*>(reinterpret_cast<const char*>(g.q) + e * g.q_expert);
}
// The experts' items in a wave's registers: lane l has experts l, l + 64, ... An expert's rows end at its offset within
// [0, m], or where the last one's did if that is further, and begin there: whatever the offsets say, every row below
// `rows` is one expert's and the items are as many as the grids are made for.
constexpr int kGroupParts = 4;  // of 64 experts
struct GroupTable {
    int row0[kGroupParts], row1[kGroupParts], end[kGroupParts];  // rows, and the items up to the expert's last
    int total, rows;
};
__device__ __forceinline__ int group_items(int row0, int row1, int bm, int ntiles) {
    return (row1 - row0 + bm - 1) / bm * ntiles;
}
// v of the lane before, `first` in lane 0 (every lane active)
__device__ __forceinline__ int lane_before(int v, int first) {
    return __builtin_amdgcn_update_dpp(first, v, 0x138, 0xf, 0xf, false);
}
__device__ __forceinline__ GroupTable group_table(const GemmArgs& g, int bm, int ntiles) {
    const int lane = lane_id();
    GroupTable t;
    t.total = t.rows = 0;
#pragma unroll
    for (int s = 0; s < kGroupParts; ++s) {
        const int e = min(s * kWave + lane, g.experts - 1);  // lanes past the experts: without rows behind the last
        t.row1[s] = s * kWave < g.experts ? min(max(g.offsets[e + 1], 0), g.m) : 0;
    }
#pragma unroll
    for (int s = 0; s < kGroupParts; ++s) {
        int row0 = t.rows, row1 = max(t.row1[s], t.rows);
        if (s * kWave < g.experts) {
            row0 = lane_before(row1, t.rows);
            if (__ballot(row1 < row0) != 0) {  // they fall: the largest so far
#pragma unroll
                for (int d = 1; d < kWave; d <<= 1) row1 = max(row1, __shfl_up(row1, d, kWave));
                row0 = lane_before(row1, t.rows);
            }
            t.rows = __builtin_amdgcn_readlane(row1, kWave - 1);
        }
        t.row0[s] = row0;
        t.row1[s] = row1;
    }
#pragma unroll
    for (int s = 0; s < kGroupParts; ++s) {
        int end = group_items(t.row0[s], t.row1[s], bm, ntiles);
        if (s * kWave < g.experts) {
#pragma unroll
            for (int d = 1; d < kWave; d <<= 1) {
                const int v = __shfl_up(end, d, kWave);
                if (lane >= d) end += v;
            }
        }
        t.end[s] = t.total + end;
        t.total = __builtin_amdgcn_readlane(t.end[s], kWave - 1);
    }
    return t;
}
// The item `at`, below t.total: its expert is the first whose items end past it
__device__ __forceinline__ GroupItem group_find(const GroupTable& t, int bm, int ntiles, int at) {
    GroupItem item{};
    bool found = false;
#pragma unroll
    for (int s = 0; s < kGroupParts; ++s) {
        const uint64_t past = __ballot(t.end[s] > at);
        if (found || past == 0) continue;
        const int l = __builtin_ctzll(past);
        item.expert = s * kWave + l;
        item.row0 = __builtin_amdgcn_readlane(t.row0[s], l);
        item.row1 = __builtin_amdgcn_readlane(t.row1[s], l);
        item.first = __builtin_amdgcn_readlane(t.end[s], l) - group_items(item.row0, item.row1, bm, ntiles);
        found = true;
    }
    return item;
}
// The same for an item at or behind `item`, from one expert to the next: scalar loads, which leave the copies in flight
// alone, and no vector registers
__device__ __forceinline__ void group_advance(const GemmArgs& g, int bm, int ntiles, int at, GroupItem& item) {
    typedef const __attribute__((address_space(4))) int32_t* Constant;
    const Constant offsets = reinterpret_cast<Constant>(reinterpret_cast<uintptr_t>(g.offsets));
    int items = group_items(item.row0, item.row1, bm, ntiles);
    while (at >= item.first + items && item.expert + 1 < g.experts) {
        item.first += items;
        ++item.expert;
        item.row0 = item.row1;
        item.row1 = max(item.row0, min(offsets[item.expert + 1], g.m));
        items = group_items(item.row0, item.row1, bm, ntiles);
    }
}
// The rows behind the last expert's, over all workgroups
__device__ __forceinline__ void group_zero_rows(const GemmArgs& g, int rows, int block, int blocks) {
    const int64_t from = static_cast<int64_t>(rows) * g.n, to = static_cast<int64_t>(g.m) * g.n;
    for (int64_t i = from + static_cast<int64_t>(block) * blockDim.x + threadIdx.x; i < to;
         i += static_cast<int64_t>(blocks) * blockDim.x) {
        if (g.out_f32) static_cast<float*>(g.out)[i] = 0.0f;
        else static_cast<uint16_t*>(g.out)[i] = 0;
    }
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // the kernels count their copies from here on
}
// The product of one expert alone: P and the result keep the rows' numbers
template <bool SWIGLU>
__device__ __forceinline__ GemmArgs group_args(const GemmArgs& g, const GroupItem& item) {
    GemmArgs e = g;
    const int64_t cols = static_cast<int64_t>(item.expert) * (SWIGLU ? 2 * static_cast<int64_t>(g.n) : g.n);
    e.q = group_q(g, item.expert);
    e.m = item.row1;
    e.col_scale += cols;
    if (g.bias) e.bias += g.out_f32 ? 2 * cols : cols;
    return e;
}

// Row pitch of the partial sums: columns (SwiGLU: gate and up apart) rounded up to whole 16-byte stores
__host__ __device__ constexpr int64_t part_cols(int n) { return (static_cast<int64_t>(n) + 3) / 4 * 4; }
__host__ __device__ constexpr int64_t part_ld(int n, bool swiglu) { return part_cols(n) * (swiglu ? 2 : 1); }

// 1 / (1 + e^-z) with the hardware exp2 and reciprocal (about 1 ulp each; the exponent's rounding moves it by at most
// 0.34 * 2^-24)
__device__ __forceinline__ float sigmoid_fast(float z) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.4426950408889634f));
}

// The normal distribution function Phi(z) = 1/2 erfc(-z / sqrt 2) and e = e^(-z^2 / 2). From the tail's side, so that a
// large negative z keeps its digits: Phi(-x) = e^(-x^2 / 2) Q(x), where Q(x) = 1/2 erfcx(x / sqrt 2) falls from 1/2
// like 1 / x. Q is t P(t) with t = 1 / (1 + 0.35 x) and P of degree 8, fitted here for the least relative error over x
// = 0 .. 14 (2^-24.9; past that e is 0 in fp32). The exponent is taken in two parts, since its rounding alone would
// move e by x^2 2^-25. Together within 2^-21 of itself (rounded stepwise on the host over 400000 z).
__device__ __forceinline__ float normal_cdf(float z, float& e) {
    constexpr float kHalfLog2E = 0.72134752044448170f, kRest = static_cast<float>(0.72134752044448170368 - kHalfLog2E);
    const float x = fminf(fabsf(z), 15.0f);
    const float t = __builtin_amdgcn_rcpf(1.0f + 0.35f * x);
    const float h = x * x, l = fmaf(x, x, -h), y = h * -kHalfLog2E;
    const float rest = fmaf(h, -kHalfLog2E, -y) - (l * kHalfLog2E + h * kRest);
    const float whole = __builtin_amdgcn_exp2f(y);
    e = whole + whole * (rest * 0.69314718055994531f);
    float p = -0.02914593182504177f;
    p = fmaf(p, t, 0.14397171139717102f);
    p = fmaf(p, t, -0.2557142674922943f);
    p = fmaf(p, t, 0.15917418897151947f);
    p = fmaf(p, t, -0.023109864443540573f);
    p = fmaf(p, t, 0.10550802201032639f);
    p = fmaf(p, t, 0.11983286589384079f);
    p = fmaf(p, t, 0.13986186683177948f);
    p = fmaf(p, t, 0.13962140679359436f);
    const float tail = p * t * e;
    return z < 0.0f ? tail : 1.0f - tail;
}
constexpr float kTanhA = 2.0f * 0.79788456080286536f, kTanhB = 0.044715f;  // 1/2 (1 + tanh a) = sigmoid(2 a)

// Activations in fp32
__device__ __forceinline__ float activate(float z, int act) {
    switch (act) {
        case kActRelu: return z > 0.0f ? z : (z != z ? z : 0.0f);
        case kActGelu: {
            float e;
            return z * normal_cdf(z, e);
        }
        case kActGeluTanh: return z * sigmoid_fast(kTanhA * (z + kTanhB * z * z * z));
        case kActSilu: return z * sigmoid_fast(z);
        default: return z;
    }
}
__device__ __forceinline__ f32x4 activate4(f32x4 z, int act) {
    if (act == kActNone) return z;
    return f32x4{activate(z[0], act), activate(z[1], act), activate(z[2], act), activate(z[3], act)};
}

// Two fp32 pairs as 16-bit values, each rounded to nearest even
template <typename T>
__device__ __forceinline__ uint2 pack4(f32x4 y) {
    return make_uint2(T::store(y[0]) | (static_cast<uint32_t>(T::store(y[1])) << 16),
                      T::store(y[2]) | (static_cast<uint32_t>(T::store(y[3])) << 16));
}

// Sums of 8-bit products: int32 bits times the row's scale, times the columns'
__device__ __forceinline__ f32x4 scaled4(f32x4 bits, float row_scale, f32x4 col_scale) {
    const i32x4 v = __builtin_bit_cast(i32x4, bits);
#pragma unroll
    for (int r = 0; r < 4; ++r) col_scale[r] *= static_cast<float>(v[r]) * row_scale;
    return col_scale;
}
__device__ __forceinline__ f32x4 load_scales4(const float* p, int valid) {
    f32x4 c = {0.f, 0.f, 0.f, 0.f};
    if (valid >= 4) {
        c = *reinterpret_cast<const f32x4_any*>(p);
    } else {
#pragma unroll
        for (int r = 0; r < 3; ++r)
            if (r < valid) c[r] = p[r];
    }
    return c;
}

// The scales that a wave's epilogue needs, loaded before its blocks: at each block's own time their latency was most of
// the epilogue (256 x 256 tiles: 12.5 us of 25 at H = 2048). A lane has the same 8 columns in every block (SwiGLU: gate
// and up), and of each 64 rows the scale of one, which the block's lanes fetch from each other.
template <bool SWIGLU, int ROWS>
struct WaveScales {
    static constexpr int kParts = (ROWS + kWave - 1) / kWave;
    f32x4 z[2], u[2];
    float rows[kParts];
    __device__ __forceinline__ void load(const GemmArgs& g, int lane, int row0, int col) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int valid = g.n - col - 4 * e;
            z[e] = load_scales4(g.col_scale + col + 4 * e, valid);
            u[e] = SWIGLU ? load_scales4(g.col_scale + g.n + col + 4 * e, valid) : z[e];
        }
#pragma unroll
        for (int p = 0; p < kParts; ++p) rows[p] = g.row_scale[min(row0 + p * kWave + lane, g.m - 1)];
    }
    // of row r of the wave's
    __device__ __forceinline__ float row(int r) const {
        float v = __shfl(rows[0], r % kWave, kWave);
        if (kParts > 1) {
            const float w = __shfl(rows[kParts - 1], r % kWave, kWave);
            v = r < kWave ? v : w;
        }
        return v;
    }
};
struct NoScales {};

// The epilogue of 4 consecutive columns col .. col + 3 of one output row, the first `valid` of which exist: bias, the
// sums before the activation stored, activation, residual. z: the sums (SwiGLU: the gate's, u the up rows'). `whole`:
// all four are there and aligned, so they are one access.
template <typename T, bool SWIGLU>
__device__ __forceinline__ f32x4 finish4(const GemmArgs& g, int64_t row, int col, int valid, bool whole, f32x4 z,
                                         f32x4 u) {
    if (!SWIGLU && g.factor) z *= *g.factor;
    if (T::kInt8 && g.bias && g.out_f32) {
        const float* bias = reinterpret_cast<const float*>(g.bias);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (r < valid) {
                z[r] += bias[col + r];
                if (SWIGLU) u[r] += bias[g.n + col + r];
            }
        }
    } else if (g.bias) {
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
        if (whole && (reinterpret_cast<uintptr_t>(g.pre) & 7) == 0) {
            *reinterpret_cast<uint2*>(pz) = pack4<T>(z);
            if (SWIGLU) *reinterpret_cast<uint2*>(pz + g.n) = pack4<T>(u);
        } else {
            for (int r = 0; r < valid; ++r) {
                pz[r] = T::store(z[r]);
                if (SWIGLU) pz[g.n + r] = T::store(u[r]);
            }
        }
    }
    f32x4 y;
    if (SWIGLU) {
#pragma unroll
        for (int r = 0; r < 4; ++r) y[r] = z[r] * sigmoid_fast(z[r]) * u[r];
    } else {
        y = activate4(z, g.act);
    }
    if (!g.residual) return y;
    const int64_t at = row * g.n + col;
    if (g.out_f32) {
        const float* res = static_cast<const float*>(g.residual) + at;
        if (whole) return y + *reinterpret_cast<const f32x4*>(res);
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (r < valid) y[r] += res[r];
    } else {
        const uint16_t* res = static_cast<const uint16_t*>(g.residual) + at;
        if (whole) {
            const uint2 v = *reinterpret_cast<const uint2*>(res);
            return f32x4{y[0] + T::load(static_cast<uint16_t>(v.x)), y[1] + T::load(static_cast<uint16_t>(v.x >> 16)),
                         y[2] + T::load(static_cast<uint16_t>(v.y)), y[3] + T::load(static_cast<uint16_t>(v.y >> 16))};
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (r < valid) y[r] += T::load(res[r]);
    }
    return y;
}

// The same, written to out; columns from n on are left alone. `vec`: whole vectors are aligned (vector_rows). SCALED:
// sums of 8-bit products have their scales.
template <typename T, bool SWIGLU, bool SCALED = false>
__device__ __forceinline__ void store4(const GemmArgs& g, int64_t row, int col, f32x4 z, f32x4 u, bool vec) {
    if (col >= g.n) return;
    const int valid = min(4, g.n - col);
    const bool whole = vec && valid == 4;
    if (T::kInt8 && !SCALED) {
        const float rs = g.row_scale[row];
        z = scaled4(z, rs, load_scales4(g.col_scale + col, valid));
        if (SWIGLU) u = scaled4(u, rs, load_scales4(g.col_scale + g.n + col, valid));
    }
    const f32x4 y = finish4<T, SWIGLU>(g, row, col, valid, whole, z, u);
    const int64_t at = row * g.n + col;
    if (g.out_f32) {
        float* out = static_cast<float*>(g.out) + at;
        if (whole) *reinterpret_cast<f32x4*>(out) = y;
        else
            for (int r = 0; r < valid; ++r) out[r] = y[r];
    } else {
        uint16_t* out = static_cast<uint16_t*>(g.out) + at;
        if (whole) *reinterpret_cast<uint2*>(out) = pack4<T>(y);
        else
            for (int r = 0; r < valid; ++r) out[r] = T::store(y[r]);
    }
}

// Whether store4 may use whole vectors: 4 columns are 8 or 16 bytes, aligned in every row
__host__ __device__ __forceinline__ bool vector_rows(const GemmArgs& g) {
    const uintptr_t mask = g.out_f32 ? 15 : 7;
    return g.n % 4 == 0 && ((reinterpret_cast<uintptr_t>(g.out) | reinterpret_cast<uintptr_t>(g.residual)) & mask) == 0;
}

template <typename T, bool SWIGLU, int ROWS>
using EpilogueScales = std::conditional_t<T::kInt8, WaveScales<SWIGLU, ROWS>, NoScales>;

// Whether store_block may write 8 columns of the 16-bit result at once
__device__ __forceinline__ bool whole_lines(const GemmArgs& g, bool vec) {
    return vec && !g.out_f32 && g.n % 8 == 0 && (reinterpret_cast<uintptr_t>(g.out) & 15) == 0;
}

// 16 rows of a wave's sums on their way to memory. They pass through a piece of LDS that is the wave's own, 16 rows x
// NB blocks of 16 columns of fp32 (SwiGLU: the first half gate, the second up), so that a lane has 8 columns of one row
// and what the epilogue reads and writes is whole lines. Granule G (16 bytes) of row r stands at G ^ r.
template <int NB>
__device__ __forceinline__ void put_block(float* stg, int row16, int kg, int j, f32x4 v) {
    *reinterpret_cast<f32x4*>(stg + (row16 * NB * 4 + ((j * 4 + kg) ^ (NB == 4 ? row16 : row16 % (NB * 4)))) * 4) = v;
}
// scales: of 8-bit products (WaveScales), the block being the wave's rows from wave_row on.
template <typename T, bool SWIGLU, int NB, typename S>
__device__ __forceinline__ void store_block(const GemmArgs& g, const float* stg, int lane, int row0, int col0, bool vec,
                                            bool lines, const S& scales, int wave_row) {
    constexpr int kGranules = NB * 4, kPer = (SWIGLU ? NB / 2 : NB) * 2;  // lanes of a row
    auto get = [&](int r, int gr) __attribute__((always_inline)) {
        return *reinterpret_cast<const f32x4*>(stg + (r * kGranules + (gr ^ (NB == 4 ? r : r % kGranules))) * 4);
    };
    // the reads take what other lanes of this wave just wrote (LDS operations of one wave run in order)
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll 1
    for (int h = 0; h < (16 * kPer + kWave - 1) / kWave; ++h) {
        const int r = h * (kWave / kPer) + lane / kPer, c = lane % kPer;
        float rs = 1.0f;
        if constexpr (T::kInt8) rs = scales.row(wave_row + r % 16);  // every lane gives its rows' before some leave
        if (16 * kPer < kWave && r >= 16) continue;
        const int row = row0 + r, col = col0 + c * 8;
        f32x4 z[2], u[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            z[e] = get(r, 2 * c + e);
            u[e] = SWIGLU ? get(r, kGranules / 2 + 2 * c + e) : z[e];
        }
        if constexpr (T::kInt8) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                z[e] = scaled4(z[e], rs, scales.z[e]);
                if (SWIGLU) u[e] = scaled4(u[e], rs, scales.u[e]);
            }
        }
        if (row >= g.m || col >= g.n) continue;
        if (lines) {
            const uint2 a = pack4<T>(finish4<T, SWIGLU>(g, row, col, 4, true, z[0], u[0]));
            const uint2 b = pack4<T>(finish4<T, SWIGLU>(g, row, col + 4, 4, true, z[1], u[1]));
            *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(g.out) + static_cast<int64_t>(row) * g.n + col) =
                u32x4{a.x, a.y, b.x, b.y};
        } else {
            store4<T, SWIGLU, true>(g, row, col, z[0], u[0], vec);
            store4<T, SWIGLU, true>(g, row, col + 4, z[1], u[1], vec);
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");  // read before the next block's writes
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// ds_read_b64_tr_b16: 8 bytes per lane, handed out transposed within each 16-lane group (lane i gets element i % 4 of
// the 8 bytes addressed by lanes 4 j + i / 4, j = 0 .. 3). An operand tile stored by k (64 k x 128 rows, 256 bytes a k)
// gives a fragment of 16 rows and 32 k as two such reads, 4 k each. These read N fragments for both 32-k steps of a
// stage, addr[n] being the lane's address at its first k. Inline assembly, with the wait in the same block: at the
// builtin the compiler waits for every direct-to-LDS copy in flight (256 x 256 tiles, T = 8192: 1195 us with that
// wait).
__device__ __forceinline__ void read_transposed(const uint32_t (&addr)[4], s16x8 (&f)[2][4]) {
    s16x4 v[4][4];
    asm volatile(
        "ds_read_b64_tr_b16 %0, %16\n\tds_read_b64_tr_b16 %1, %16 offset:1024\n\t"
        "ds_read_b64_tr_b16 %4, %17\n\tds_read_b64_tr_b16 %5, %17 offset:1024\n\t"
        "ds_read_b64_tr_b16 %8, %18\n\tds_read_b64_tr_b16 %9, %18 offset:1024\n\t"
        "ds_read_b64_tr_b16 %12, %19\n\tds_read_b64_tr_b16 %13, %19 offset:1024\n\t"
        "ds_read_b64_tr_b16 %2, %16 offset:8192\n\tds_read_b64_tr_b16 %3, %16 offset:9216\n\t"
        "ds_read_b64_tr_b16 %6, %17 offset:8192\n\tds_read_b64_tr_b16 %7, %17 offset:9216\n\t"
        "ds_read_b64_tr_b16 %10, %18 offset:8192\n\tds_read_b64_tr_b16 %11, %18 offset:9216\n\t"
        "ds_read_b64_tr_b16 %14, %19 offset:8192\n\tds_read_b64_tr_b16 %15, %19 offset:9216\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(v[0][0]), "=&v"(v[0][1]), "=&v"(v[0][2]), "=&v"(v[0][3]), "=&v"(v[1][0]), "=&v"(v[1][1]),
          "=&v"(v[1][2]), "=&v"(v[1][3]), "=&v"(v[2][0]), "=&v"(v[2][1]), "=&v"(v[2][2]), "=&v"(v[2][3]),
          "=&v"(v[3][0]), "=&v"(v[3][1]), "=&v"(v[3][2]), "=&v"(v[3][3])
        : "v"(addr[0]), "v"(addr[1]), "v"(addr[2]), "v"(addr[3])
        : "memory");
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int n = 0; n < 4; ++n)
            f[kk][n] = __builtin_shufflevector(v[n][2 * kk], v[n][2 * kk + 1], 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ __forceinline__ void read_transposed(const uint32_t (&addr)[2], s16x8 (&f)[2][2]) {
    s16x4 v[2][4];
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:1024\n\t"
        "ds_read_b64_tr_b16 %4, %9\n\tds_read_b64_tr_b16 %5, %9 offset:1024\n\t"
        "ds_read_b64_tr_b16 %2, %8 offset:8192\n\tds_read_b64_tr_b16 %3, %8 offset:9216\n\t"
        "ds_read_b64_tr_b16 %6, %9 offset:8192\n\tds_read_b64_tr_b16 %7, %9 offset:9216\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(v[0][0]), "=&v"(v[0][1]), "=&v"(v[0][2]), "=&v"(v[0][3]), "=&v"(v[1][0]), "=&v"(v[1][1]),
          "=&v"(v[1][2]), "=&v"(v[1][3])
        : "v"(addr[0]), "v"(addr[1])
        : "memory");
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int n = 0; n < 2; ++n)
            f[kk][n] = __builtin_shufflevector(v[n][2 * kk], v[n][2 * kk + 1], 0, 1, 2, 3, 4, 5, 6, 7);
}
// The lane's address in such a tile of the fragment of rows r0 .. r0 + 15 (r0 a multiple of 16) at the first k. The
// 32-byte pairs of a k stand at pair ^ f(k), f(k) = (k & 3) | (k >> 3 & 1) << 2, which depends on the lane alone here.
__device__ __forceinline__ uint32_t transposed_address(const uint16_t* tile, int r0, int lane) {
    const int kg = lane >> 4, j = (lane & 15) >> 2, q = lane & 3, f = (j | ((kg & 1) << 2)) << 1;
    const uint16_t* p = tile + (kg * 8 + j) * 128 + (((r0 / 8 + (q >> 1)) ^ f) * 8) + (q & 1) * 4;
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const uint16_t*)p));
}

// 16 columns a workgroup of 256 threads; its 16 groups add every 16th row of `part`, then the groups' sums in order
constexpr int kSumColumns = 16;
template <typename T>
__device__ __forceinline__ void column_sums(const float* __restrict__ part, uint16_t* __restrict__ out, int Z, int rows,
                                            int block) {
    constexpr int kGroups = 16;
    __shared__ float sums[kGroups][kSumColumns];
    const int i = static_cast<int>(threadIdx.x) % kSumColumns, q = static_cast<int>(threadIdx.x) / kSumColumns;
    const int c = block * kSumColumns + i;
    float s = 0.0f;
    if (c < Z) {
#pragma unroll 4
        for (int b = q; b < rows; b += kGroups) s += part[static_cast<int64_t>(b) * Z + c];
    }
    sums[q][i] = s;
    __syncthreads();
    if (q != 0 || c >= Z) return;
#pragma unroll
    for (int g = 1; g < kGroups; ++g) s += sums[g][i];
    out[c] = T::store(s);
}

// 8 values of a row from p on, of which `valid` exist (zeros past them); any alignment. `before`: values of the row
// that stand before p. A row's end is the 8 values that end there, moved down: one load, where single ones wait for
// each other.
__device__ __forceinline__ s16x8 load8(const uint16_t* p, int valid, int before) {
    typedef short s16x8_any __attribute__((ext_vector_type(8), aligned(2)));
    typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
    if (valid >= 8) return *reinterpret_cast<const s16x8_any*>(p);
    s16x8 v = {0, 0, 0, 0, 0, 0, 0, 0};
    if (valid <= 0) return v;
    if (before + valid >= 8) {
        const u64x2 x = __builtin_bit_cast(u64x2, *reinterpret_cast<const s16x8_any*>(p + valid - 8));
        const int bits = 16 * (8 - valid), b = bits & 63;  // 16 .. 112
        const uint64_t high = x[1] >> b;
        return __builtin_bit_cast(s16x8, bits >= 64 ? u64x2{high, 0} : u64x2{x[0] >> b | x[1] << (64 - b), high});
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < valid) v[e] = static_cast<short>(p[e]);
    return v;
}

// 16 bytes of a row from p on, of which `valid` exist (zeros past them); any alignment
__device__ __forceinline__ s16x8 load16(const uint8_t* p, int valid, int before) {
    typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
    typedef uint64_t u64x2_any __attribute__((ext_vector_type(2), aligned(1)));
    u64x2 x = {0, 0};
    if (valid >= 16) {
        x = *reinterpret_cast<const u64x2_any*>(p);
    } else if (valid > 0 && before + valid >= 16) {  // the 16 that end at the row's end, moved down
        x = *reinterpret_cast<const u64x2_any*>(p + valid - 16);
        const int bits = 8 * (16 - valid), b = bits & 63;  // 8 .. 120
        const uint64_t high = x[1] >> b;
        x = bits >= 64 ? u64x2{high, 0} : u64x2{x[0] >> b | x[1] << (64 - b), high};
    } else {
        for (int e = 0; e < valid; ++e) x[e / 8] |= static_cast<uint64_t>(p[e]) << (e % 8 * 8);
    }
    return __builtin_bit_cast(s16x8, x);
}

// Copies of matrices with rows padded with zeros to dst_cols, a multiple of 8 (moe_linear_repack.hip)
struct Repack {
    const uint16_t* src;
    uint16_t* dst;
    int64_t src_ld, dst_ld, rows;
    int cols, dst_cols;
};
constexpr int kRepackMost = 3;
struct RepackArgs {
    Repack m[kRepackMost];
};
hipError_t launch_repack(const RepackArgs& a, hipStream_t stream);
// Of 8-bit rows, padded to whole 16 bytes: `rows` of cols bytes, src_ld apart, and group_ld from one group's to the
// next's
struct Repack8 {
    const uint8_t* src;
    uint8_t* dst;
    int64_t src_ld, group_ld, rows;
    int cols;
};
hipError_t launch_repack8(const Repack8& x, const Repack8& w, int64_t groups, hipStream_t stream);

// What follows the gradients' products: the reduction of those that were split (splits > 1), the bias's column sums
struct GradTail {
    GemmArgs x, w;
    int x_blocks, w_blocks;
    const float* sums;    // [sum_rows, Z]
    uint16_t* bias_grad;  // null: not wanted
    int Z, sum_rows;
};

// kernels' launches; prepare_*: their LDS limits on the current device, before the first launch of a call
hipError_t prepare_gemm_mid();
hipError_t prepare_gemm_stream();
hipError_t prepare_gemm_tiled();
hipError_t launch_gemm_mid(const GemmArgs& g, bool p_by_k, bool q_by_k, bool bf16, bool direct, int bm,
                           hipStream_t stream);
// grad_x (bm rows a tile) and grad_W (both operands by k) together; 16-byte copies
hipError_t launch_gemm_pair(const GemmArgs& x, const GemmArgs& w, bool q_by_k, bool bf16, int bm, hipStream_t stream);
hipError_t launch_grad_tail(GradTail t, bool bf16, hipStream_t stream);
// at most 64 rows, both operands by rows, 16-byte loads
hipError_t launch_gemm_stream(const GemmArgs& g, bool bf16, hipStream_t stream);
// 256 x 256 tiles; operands that 16-byte copies can read
hipError_t launch_gemm_tiled(const GemmArgs& g, bool p_by_k, bool q_by_k, bool bf16, hipStream_t stream);
hipError_t launch_gemm_reduce(const GemmArgs& g, bool bf16, hipStream_t stream);

// The same of 8-bit operands, both by rows; bf16: the results. With experts mid takes 64 or 128 rows a tile, and no
// product is split
hipError_t prepare_int8_mid();
hipError_t prepare_int8_stream();
hipError_t prepare_int8_tiled();
hipError_t launch_int8_mid(const GemmArgs& g, bool bf16, bool direct, int bm, hipStream_t stream);
hipError_t launch_int8_stream(const GemmArgs& g, bool bf16, hipStream_t stream);
hipError_t launch_int8_tiled(const GemmArgs& g, bool bf16, hipStream_t stream);
hipError_t launch_int8_reduce(const GemmArgs& g, bool bf16, hipStream_t stream);

}  // namespace moe
