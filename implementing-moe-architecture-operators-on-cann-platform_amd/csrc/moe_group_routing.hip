// moe_group_routing.hip -- MoeRoutingGroupTopK and its gradient for gfx950: from logits [T, E] to experts and weights.
//
// The reference routes by softmax and top-K alone (op_kernel/moe_routing.cpp:238-369). Here
//   s = sigmoid(l) or softmax(l),  c = s + bias
//   groups of E / G consecutive experts, each scored by its best c or the sum of its two best; the best topGroups stay
//   the K best c among them in descending order, ties to the lowest index; w = scale * s, over the K's sum if asked
// An expert whose logit or c is NaN or -inf is not available; picks with no expert left are id -1, weight 0.
//
// The choice is the definition's, not fp32's: without a bias experts are compared by their logits, which order the
// scores exactly; with one, c is computed in fp32 with a bound on its error (gap_limit). Where a group that stays and
// one that does not are nearer than theirs (group_error), the row's groups are scored again in float64; where two
// neighbours among its picks are, the picks go on past the K-th until a clear gap and are put in order by their float64
// values. That is some rows in a hundred, but a launch waits for its slowest wave: a float64 copy of the whole choice,
// whose code is never in the instruction cache when it is needed, cost 9 us. Where kMore picks more leave no gap (equal
// scores, biases that leave few bits for the scores), the K best of the row are taken by their float64 values, one
// maximum of the wave each: calls with 256 equal scores a row take 10.7 us at T = 1 and 43 at T = 16384, where picking
// and ordering all of them took 157 and 660 (with 8 groups 16.2 and 75, before 62 and 240).
//
// A wave has 4 tokens, 16 lanes (a DPP row) each, up to 16 experts a lane in registers as order-preserving integers;
// few tokens of many experts have a wave each. A pick is the maximum over the lane (max3) and over the row (4 DPP
// steps), and its removal: 16 compares and 16 selects. Where the key's low 8 bits can hold the expert, the maximum
// names the pick: ~50 instructions for 4 tokens. fp32 logits without a bias need all of their bits: the lowest index
// that has the maximum is searched, ~95 instructions. Group scores go through LDS, one lane per (token, group). Vector
// instructions bound the kernel (T = 16384, E = 256, K = 8, fp32 logits: 10.3 us without bias and groups, 17 us with a
// bias and 4 of 8 groups by their two best, of which a copy of the logits is 4 us; the search in place of the key's
// bits 21 us). At T = 1 the one wave's chain takes 6 us.
#include "moe_device.h"
#include "moe_launch.h"
#include "moe_ops.h"

#include <type_traits>

namespace moe {

namespace {

constexpr int kRow = 16;  // lanes of a DPP row
constexpr int kRowTokens = kWave / kRow;  // tokens of a wave with a DPP row each
constexpr int kMaxE = 256;
constexpr int kMore = 8;                     // picks past the K-th
constexpr int kNoPick = 0xffff;              // a pick with no expert left
constexpr int kGone = -2147483647 - 1;         // the key of an expert that is not available or was picked
constexpr float kLow = -__builtin_huge_valf();
constexpr double kNone = -__builtin_huge_val();

template <typename L>
__device__ __forceinline__ float logit(const void* p, int64_t i);
struct F32 {};
struct F16 {};
struct B16 {};
template <>
__device__ __forceinline__ float logit<F32>(const void* p, int64_t i) {
    return static_cast<const float*>(p)[i];
}
template <>
__device__ __forceinline__ float logit<F16>(const void* p, int64_t i) {
    return f16_bits_to_f32(static_cast<const uint16_t*>(p)[i]);
}
template <>
__device__ __forceinline__ float logit<B16>(const void* p, int64_t i) {
    return __builtin_bit_cast(float, static_cast<uint32_t>(static_cast<const uint16_t*>(p)[i]) << 16);
}
template <typename L>
__device__ __forceinline__ void put(void* p, int64_t i, float v);
template <>
__device__ __forceinline__ void put<F32>(void* p, int64_t i, float v) {
    static_cast<float*>(p)[i] = v;
}
template <>
__device__ __forceinline__ void put<F16>(void* p, int64_t i, float v) {
    static_cast<uint16_t*>(p)[i] = f32_to_f16_bits(v);
}
template <>
__device__ __forceinline__ void put<B16>(void* p, int64_t i, float v) {
    static_cast<uint16_t*>(p)[i] = __builtin_bit_cast(uint16_t, static_cast<__bf16>(v));
}

// 4 consecutive logits, aligned
template <typename L>
__device__ __forceinline__ void load4(const void* p, int64_t i, float* v) {
    if constexpr (std::is_same_v<L, F32>) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + i);
        v[0] = x[0], v[1] = x[1], v[2] = x[2], v[3] = x[3];
    } else {
        const uint2 x = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
        const uint16_t b[4] = {static_cast<uint16_t>(x.x), static_cast<uint16_t>(x.x >> 16), static_cast<uint16_t>(x.y),
                               static_cast<uint16_t>(x.y >> 16)};
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = logit<L>(b, j);
    }
}

// All-reduce over the LANES lanes of a token: a DPP row of 16 by rotations; of a whole wave the rows' four results
// after that
template <int CTRL>
__device__ __forceinline__ int dpp(int v) {
    return __builtin_amdgcn_mov_dpp(v, CTRL, 0xf, 0xf, true);
}
__device__ __forceinline__ int row_of(int v, int row) { return __builtin_amdgcn_readlane(v, row * kRow); }
template <int LANES>
__device__ __forceinline__ int row_max_i(int v) {
    v = max(v, dpp<0x128>(v));
    v = max(v, dpp<0x124>(v));
    v = max(v, dpp<0x122>(v));
    v = max(v, dpp<0x121>(v));
    return LANES == kRow ? v : max(max(row_of(v, 0), row_of(v, 1)), max(row_of(v, 2), row_of(v, 3)));
}
template <int LANES>
__device__ __forceinline__ int row_min_i(int v) {
    v = min(v, dpp<0x128>(v));
    v = min(v, dpp<0x124>(v));
    v = min(v, dpp<0x122>(v));
    v = min(v, dpp<0x121>(v));
    return LANES == kRow ? v : min(min(row_of(v, 0), row_of(v, 1)), min(row_of(v, 2), row_of(v, 3)));
}
template <int LANES>
__device__ __forceinline__ double row_sum(double v) {
#pragma unroll
    for (int d = LANES / 2; d > 0; d >>= 1) v += __shfl_xor(v, d, LANES);
    return v;
}
template <int LANES>
__device__ __forceinline__ float row_sum_f(float v) {
    auto turned = [](float x, auto ctrl) {
        return __builtin_bit_cast(float, dpp<decltype(ctrl)::value>(__builtin_bit_cast(int, x)));
    };
    v += turned(v, std::integral_constant<int, 0x128>());
    v += turned(v, std::integral_constant<int, 0x124>());
    v += turned(v, std::integral_constant<int, 0x122>());
    v += turned(v, std::integral_constant<int, 0x121>());
    if (LANES == kRow) return v;
    auto row = [&](int i) { return __builtin_bit_cast(float, row_of(__builtin_bit_cast(int, v), i)); };
    return (row(0) + row(1)) + (row(2) + row(3));
}

// A double as the lane that a DPP control names has it; as row `row`'s first lane has it
template <int CTRL>
__device__ __forceinline__ double dpp_d(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = dpp<CTRL>(static_cast<int>(b)), hi = dpp<CTRL>(static_cast<int>(b >> 32));
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ double row_of_d(double v, int row) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = row_of(static_cast<int>(b), row), hi = row_of(static_cast<int>(b >> 32), row);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
// Over a DPP row
__device__ __forceinline__ double row_sum_d(double v) {
    v += dpp_d<0x128>(v);
    v += dpp_d<0x124>(v);
    v += dpp_d<0x122>(v);
    v += dpp_d<0x121>(v);
    return v;
}
// Over the wave
__device__ __forceinline__ double wave_max_d(double v) {
    v = fmax(v, dpp_d<0x128>(v));
    v = fmax(v, dpp_d<0x124>(v));
    v = fmax(v, dpp_d<0x122>(v));
    v = fmax(v, dpp_d<0x121>(v));
    return fmax(fmax(row_of_d(v, 0), row_of_d(v, 1)), fmax(row_of_d(v, 2), row_of_d(v, 3)));
}

// Floats as integers in the same order (-0 as 0); key_value undoes it
__device__ __forceinline__ int key_of(float v) {
    const int b = __builtin_bit_cast(int, v + 0.0f);
    return b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float key_value(int k) { return __builtin_bit_cast(float, k ^ ((k >> 31) & 0x7fffffff)); }

// Two fp32 values of c that are nearer than this may stand the other way round. With e = 2^-24: exp2 and
// rcp are within 2 e, the argument's rounding moves e^-l by |l| 1.5 e relative and s (1 - s) |l| < 0.23, so a sigmoid
// is within 8 e; a softmax score, with a sum of 20 roundings, within 64 e of the row's largest score; adding the bias
// rounds by e |c|. The limit is four such errors.
__device__ __forceinline__ float gap_limit(bool sigmoid, float s_max, float c) {
    return (sigmoid ? 32.0f : 256.0f * s_max) * 0x1p-24f + fabsf(c) * 0x1p-21f;
}
// How far an fp32 group score may be from the definition's. It is the sum of two c, a and b, which may cancel: its
// error is that of the terms, two scores' and, with the sum's own rounding, at most 2 e (|a| + |b|), not one of the
// sum's size (biases of +-40 leave sums below 1 that are 4e-6 off). size: |a| + |b|, counted twice.
__device__ __forceinline__ float group_error(bool sigmoid, float s_max, float size) {
    return (sigmoid ? 16.0f : 128.0f * s_max) * 0x1p-24f + size * 0x1p-22f;
}

// LDS of the one wave of a workgroup. A row may have E picks.
template <int TOKENS>
struct RoutingLds {
    int E, G, K;
    __host__ __device__ int pitch() const { return (E + 3) / 4 * 4 + 4; }
    __host__ __device__ int picks_at() const { return 8 * TOKENS * K; }  // after the parts (double): 16 bits each
    __host__ __device__ int order_at() const { return picks_at() + 2 * TOKENS * E; }
    __host__ __device__ int scores_at() const { return (order_at() + 2 * E + 3) / 4 * 4; }
    __host__ __device__ int kept_at() const { return scores_at() + 4 * TOKENS * G; }
    __host__ __device__ int sizes_at() const { return kept_at() + 4 * TOKENS * G; }
    // c of the rows' experts, fp32; or, once the groups are scored, float64 values of one row and its groups
    __host__ __device__ int row_at() const { return (sizes_at() + 4 * TOKENS * G + 15) / 16 * 16; }
    __host__ __device__ int bytes(bool rows) const {
        const int scores = 4 * TOKENS * pitch(), exact = 8 * (E + G);
        return row_at() + (rows ? (scores > exact ? scores : exact) : 0);
    }
};

// Expert of lane l's register j: 16-byte (8-byte) pieces of 4 consecutive experts
template <int LANES, int C>
__device__ __forceinline__ int expert_of(int l, int j) {
    constexpr int V = C < 4 ? C : 4;
    return j / V * (LANES * V) + l * V + j % V;
}

// Lane l's logits of the row that starts at element `at`; -inf past E
template <typename L, int LANES, int C, bool VEC>
__device__ __forceinline__ void load_logits(const void* p, int64_t at, int E, int l, float (&v)[C]) {
    if constexpr (VEC && C >= 4) {
#pragma unroll
        for (int j = 0; j < C; j += 4) {
            const int e = expert_of<LANES, C>(l, j);
            if (e < E) {  // E % 4 == 0
                load4<L>(p, at + e, &v[j]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) v[j + i] = kLow;
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < C; ++j) {
            const int e = expert_of<LANES, C>(l, j);
            v[j] = e < E ? logit<L>(p, at + e) : kLow;
        }
    }
}

// c (what groups are scored by) of all experts of row t in float64, by the whole wave, to cs [E]; -inf where not
// available
template <typename L>
__device__ __forceinline__ void exact_scores(const GroupRouting& r, int64_t t, double* cs) {
    const int lane = lane_id(), E = r.E;
    double top = kNone, sum = 1.0;
    auto at = [&](int e) {
        const double x = static_cast<double>(logit<L>(r.logits, t * r.ld + e));
        return x > kNone ? x : kNone;  // NaN too
    };
    if (!r.sigmoid) {
#pragma unroll 1
        for (int e = lane; e < E; e += kWave) top = fmax(top, at(e));
#pragma unroll 1
        for (int d = kWave / 2; d > 0; d >>= 1) top = fmax(top, __shfl_xor(top, d, kWave));
        sum = 0.0;
    }
#pragma unroll 1
    for (int e = lane; e < E; e += kWave) {
        const double x = at(e);
        const double p = r.sigmoid ? exp(-x) : x == top ? 1.0 : exp(x - top);
        const double s = !(x > kNone) ? 0.0 : r.sigmoid ? 1.0 / (1.0 + p) : p;
        sum += s;
        cs[e] = x > kNone ? s : kNone;
    }
#pragma unroll 1
    for (int d = kWave / 2; d > 0; d >>= 1) sum += __shfl_xor(sum, d, kWave);
    for (int e = lane; e < E; e += kWave) {  // its own entries
        double c = cs[e];
        if (!r.sigmoid) c = c > kNone ? c / sum : kNone;
        if (r.bias) c += static_cast<double>(r.bias[e]);
        cs[e] = c > kNone ? c : kNone;
    }
    __syncthreads();
}

// Whether c comes before o in descending order, the lower index first among equals
__device__ __forceinline__ bool goes_before(double o, int oi, double c, int ci) { return o > c || (o == c && oi < ci); }

// LANES: lanes of a token. C: experts of a lane. VEC: rows allow loads of 4 experts.
template <typename L, int LANES, int C, bool VEC>
__global__ __launch_bounds__(kWave) void group_routing_kernel(GroupRouting r, int32_t* __restrict__ ids,
                                                              void* __restrict__ weights) {
    constexpr int kTokens = kWave / LANES;
    extern __shared__ __align__(16) char shared[];
    const int E = r.E, G = r.groups, K = r.K, size = E / G;
    const RoutingLds<kTokens> lay{E, G, K};
    double* parts = reinterpret_cast<double*>(shared);
    uint16_t* pick = reinterpret_cast<uint16_t*>(shared + lay.picks_at());  // [token][E]
    uint16_t* order = reinterpret_cast<uint16_t*>(shared + lay.order_at());
    float* gs = reinterpret_cast<float*>(shared + lay.scores_at());
    int* kept = reinterpret_cast<int*>(shared + lay.kept_at());
    float* sizes = reinterpret_cast<float*>(shared + lay.sizes_at());  // of the groups' terms, for group_error
    float* row = reinterpret_cast<float*>(shared + lay.row_at());
    double* cs = reinterpret_cast<double*>(row);
    double* cgs = cs + E;
    const int lane = lane_id(), tok = lane / LANES, l = lane % LANES;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * kTokens + tok;
    const bool valid = t < r.T;

    float v[C];  // logits, -inf where not available
    if (valid) {
        load_logits<L, LANES, C, VEC>(r.logits, t * r.ld, E, l, v);
    } else {
#pragma unroll
        for (int j = 0; j < C; ++j) v[j] = kLow;
    }
#pragma unroll
    for (int j = 0; j < C; ++j) v[j] = v[j] > kLow ? v[j] : kLow;  // NaN too
    const bool grouped = r.top_groups < G;
    const bool all_softmax = !r.sigmoid && !r.renormalize;  // weights over the whole row
    const bool scored = r.bias || (grouped && r.group_top == 2);
    float top = 0.0f, s_max = 1.0f;
    double whole = 1.0;  // sum of the row's e^(l - top)
    if (!r.sigmoid && (scored || all_softmax)) {
        int m = key_of(v[0]);
#pragma unroll
        for (int j = 1; j < C; ++j) m = max(m, key_of(v[j]));
        top = key_value(row_max_i<LANES>(m));
    }
    int key[C];
    float s[C];
    if (scored || all_softmax) {
        if (r.sigmoid) {
#pragma unroll
            for (int j = 0; j < C; ++j)  // 0 for -inf
                s[j] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v[j] * -1.4426950408889634f));
        } else {
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < C; ++j) {
                const float d = v[j] == top ? 0.0f : v[j] - top;
                s[j] = v[j] > kLow ? __builtin_amdgcn_exp2f(d * 1.4426950408889634f) : 0.0f;
                sum += s[j];
            }
            if (all_softmax) {  // in float64, so that a row's weights do not depend on how it is spread over lanes
                whole = 0.0;
#pragma unroll
                for (int j = 0; j < C; ++j) whole += static_cast<double>(s[j]);
                whole = row_sum<LANES>(whole);
            }
            sum = row_sum_f<LANES>(sum);
            s_max = sum > 0.0f ? __builtin_amdgcn_rcpf(sum) : 1.0f;
#pragma unroll
            for (int j = 0; j < C; ++j) s[j] *= s_max;
        }
    }
    if (r.bias) {
        float b[C];
        load_logits<F32, LANES, C, VEC>(r.bias, 0, E, l, b);
#pragma unroll
        for (int j = 0; j < C; ++j) {
            const float c = s[j] + b[j];
            key[j] = v[j] > kLow && c > kLow ? key_of(c) : kGone;
        }
    } else {
#pragma unroll
        for (int j = 0; j < C; ++j) key[j] = v[j] > kLow ? key_of(v[j]) : kGone;
    }
    if (grouped) {
        const bool by_score = r.group_top == 2 && !r.bias;
        auto entry = [&](int j) { return key[j] == kGone ? kLow : by_score ? s[j] : key_value(key[j]); };
        float* out = row + tok * lay.pitch();
#pragma unroll
        for (int j = 0; j < C; j += (C < 4 ? 1 : 4)) {  // a row's end may be written past E: the pitch has room
            const int e = expert_of<LANES, C>(l, j);
            if constexpr (C < 4) {
                if (e < E) out[e] = entry(j);
            } else if (e < E) {
                *reinterpret_cast<f32x4*>(out + e) = f32x4{entry(j), entry(j + 1), entry(j + 2), entry(j + 3)};
            }
        }
        __syncthreads();
        for (int i = lane; i < kTokens * G; i += kWave) {
            const int q = i / G, g = i - q * G;
            const float* c = row + q * lay.pitch() + g * size;
            float a = kLow, b = kLow;
            auto take = [&](float x) {
                b = fmaxf(b, fminf(a, x));
                a = fmaxf(a, x);
            };
            if (size % 4 == 0) {
#pragma unroll 4
                for (int n = 0; n < size; n += 4) {
                    const f32x4 x = *reinterpret_cast<const f32x4*>(c + n);
                    take(x[0]), take(x[1]), take(x[2]), take(x[3]);
                }
            } else {
#pragma unroll 4
                for (int n = 0; n < size; ++n) take(c[n]);
            }
            const bool two = r.group_top == 2 && b > kLow;
            gs[i] = two ? a + b : a;
            sizes[i] = a == -kLow ? 0.0f : fabsf(a) + (two ? fabsf(b) : 0.0f);  // an infinite bias decides by itself
        }
        __syncthreads();
        for (int i = lane; i < kTokens * G; i += kWave) {
            const int q = i / G, g = i - q * G;
            const float* o = gs + q * G;
            const float x = o[g];
            int before = 0;
#pragma unroll 8
            for (int n = 0; n < G; ++n) before += o[n] > x || (o[n] == x && n < g);
            kept[i] = before < r.top_groups;
        }
        __syncthreads();
        if (scored) {
            // the least that a group that stays may be, the most that one that does not may be; empty groups are exact
            int least = 2147483647, most = kGone;
#pragma unroll 1
            for (int g = l; g < G; g += LANES) {
                const float x = gs[tok * G + g], err = group_error(r.sigmoid, s_max, sizes[tok * G + g]);
                if (!(x > kLow)) continue;
                const float low = x - err;
                if (!kept[tok * G + g]) most = max(most, key_of(x + err));
                else least = min(least, key_of(low > kLow ? low : kLow));  // NaN, where x and err are infinite
            }
            least = row_min_i<LANES>(least);
            most = row_max_i<LANES>(most);
            uint64_t open = __ballot(valid && most != kGone && least <= most);
#pragma unroll 1
            for (int q = 0; open && q < kTokens; ++q) {
                if (!((open >> (q * LANES)) & 1)) continue;
                exact_scores<L>(r, static_cast<int64_t>(blockIdx.x) * kTokens + q, cs);
#pragma unroll 1
                for (int g = lane; g < G; g += kWave) {
                    double a = kNone, b = kNone;
                    for (int e = g * size; e < (g + 1) * size; ++e) {
                        b = fmax(b, fmin(a, cs[e]));
                        a = fmax(a, cs[e]);
                    }
                    cgs[g] = r.group_top == 2 && b > kNone ? a + b : a;
                }
                __syncthreads();
#pragma unroll 1
                for (int g = lane; g < G; g += kWave) {
                    int before = 0;
                    for (int o = 0; o < G; ++o) before += goes_before(cgs[o], o, cgs[g], g);
                    kept[q * G + g] = before < r.top_groups;
                }
                __syncthreads();
            }
        }
        const int* mine = kept + tok * G;
        if (C >= 4 && size % 4 == 0) {  // a piece's experts are of one group
#pragma unroll
            for (int j = 0; j < C; j += 4) {
                const int e = expert_of<LANES, C>(l, j);
                if (e >= E || mine[(e * r.size_inverse) >> 16]) continue;
#pragma unroll
                for (int i = j; i < min(j + 4, C); ++i) key[i] = kGone;
            }
        } else {
#pragma unroll
            for (int j = 0; j < C; ++j) {
                const int e = expert_of<LANES, C>(l, j);
                if (e < E && !mine[(e * r.size_inverse) >> 16]) key[j] = kGone;
            }
        }
    }
    int picks = K;         // of this row: K, and those that are not told from the K-th
    bool reorder = false;  // two of them are nearer than their keys tell apart
    if (r.bias || !std::is_same_v<L, F32>) {
        // Keys with 255 - e in their low 8 bits: the maximum is the pick, and the lowest index wins. Half logits leave
        // those bits free; c loses them, up to 2^-15 of it, which counts as an error like fp32's own.
#pragma unroll
        for (int j = 0; j < C; ++j)
            key[j] = key[j] == kGone ? kGone : (key[j] & ~(kMaxE - 1)) | (kMaxE - 1 - expert_of<LANES, C>(l, j));
        int last = kGone;
#pragma unroll 1
        for (int k = 0;; ++k) {
            int m = key[0];
#pragma unroll
            for (int j = 1; j < C; ++j) m = max(m, key[j]);
            m = row_max_i<LANES>(m);
            if (r.bias) {
                const float x = key_value(last & ~(kMaxE - 1)), y = key_value(m & ~(kMaxE - 1));
                const bool clear = x - y > gap_limit(r.sigmoid, s_max, x) + fabsf(y) * 0x1p-15f;
                if (!clear && last != kGone && m != kGone && k <= picks) {
                    reorder = true;
                    picks = max(picks, k + 1);
                }
                last = m;
            }
            if (k >= K && (k == K + kMore || !__any(k < picks))) break;
            if (l == 0 && k < picks)
                pick[tok * E + k] = static_cast<uint16_t>(m == kGone ? kNoPick : kMaxE - 1 - (m & (kMaxE - 1)));
#pragma unroll
            for (int j = 0; j < C; ++j) key[j] = key[j] == m ? kGone : key[j];
        }
    } else {
        constexpr int kStep = C < 4 ? C : 4;
#pragma unroll 1
        for (int k = 0; k < K; ++k) {
            int m = key[0];
#pragma unroll
            for (int j = 1; j < C; ++j) m = max(m, key[j]);
            m = row_max_i<LANES>(m);
            int jw = -1;
#pragma unroll
            for (int j = C - 1; j >= 0; --j) jw = key[j] == m ? j : jw;
            const int e = row_min_i<LANES>(jw < 0 ? kMaxE : expert_of<LANES, C>(l, jw));
            if (l == 0) pick[tok * E + k] = static_cast<uint16_t>(m == kGone ? kNoPick : e);
            const int mine = e / kStep % LANES == l ? e / (LANES * kStep) * kStep + e % kStep : -1;  // its register
#pragma unroll
            for (int j = 0; j < C; ++j) key[j] = mine == j ? kGone : key[j];
        }
    }
    __syncthreads();
    const uint64_t redo = __ballot(reorder && valid), select = __ballot(picks > K + kMore && valid);
#pragma unroll 1
    for (int q = 0; redo && q < kTokens; ++q) {
        if (!((redo >> (q * LANES)) & 1)) continue;
        const int64_t tq = static_cast<int64_t>(blockIdx.x) * kTokens + q;
        const int n = __shfl(picks, q * LANES, kWave);
        uint16_t* of = pick + q * E;
        const bool whole_row = (select >> (q * LANES)) & 1;
        if (r.sigmoid && !whole_row) {  // the picks' alone
            for (int k = lane; k < n; k += kWave) {
                const int e = of[k];
                if (e == kNoPick) continue;
                const double x = static_cast<double>(logit<L>(r.logits, tq * r.ld + e));
                cs[e] = 1.0 / (1.0 + exp(-x)) + static_cast<double>(r.bias[e]);
            }
            __syncthreads();
        } else {
            exact_scores<L>(r, tq, cs);
        }
        if (whole_row) {
            double c[kMaxE / kWave];  // of expert i * 64 + lane
#pragma unroll
            for (int i = 0; i < kMaxE / kWave; ++i) {
                const int e = i * kWave + lane;
                c[i] = e < E && (!grouped || kept[q * G + ((e * r.size_inverse) >> 16)]) ? cs[e] : kNone;
            }
#pragma unroll 1
            for (int k = 0; k < K; ++k) {
                double m = c[0];
#pragma unroll
                for (int i = 1; i < kMaxE / kWave; ++i) m = fmax(m, c[i]);
                m = wave_max_d(m);
                int e = kNoPick;
#pragma unroll
                for (int i = kMaxE / kWave - 1; i >= 0; --i) {  // the lowest index last
                    const uint64_t at = __ballot(c[i] == m);
                    if (m > kNone && at) e = i * kWave + __builtin_ctzll(at);
                }
#pragma unroll
                for (int i = 0; i < kMaxE / kWave; ++i) c[i] = e == i * kWave + lane ? kNone : c[i];
                if (lane == 0) of[k] = static_cast<uint16_t>(e);
            }
            __syncthreads();
            continue;
        }
#pragma unroll 1
        for (int k = lane; k < n; k += kWave) {
            const int e = of[k];
            int before = k;  // empty picks, at the end, stay
            if (e != kNoPick) {
                before = 0;
                for (int o = 0; o < n; ++o) before += of[o] != kNoPick && goes_before(cs[of[o]], of[o], cs[e], e);
            }
            order[before] = static_cast<uint16_t>(e);
        }
        __syncthreads();
        for (int k = lane; k < K; k += kWave) of[k] = order[k];
        __syncthreads();
    }
    if (!valid) return;
    // Weights in float64: K values of a row. Renormalised, the scores are taken relative to the largest of the picks:
    // their ratios hold where the scores themselves would underflow.
    const uint16_t* my = pick + tok * E;
    double* part = parts + tok * K;
    int ref_key = kGone;
    const float first = l < K && my[l] != kNoPick ? logit<L>(r.logits, t * r.ld + my[l]) : 0.0f;
    auto chosen = [&](int k) { return k < LANES ? first : logit<L>(r.logits, t * r.ld + my[k]); };
    if (r.renormalize) {
        for (int k = l; k < K; k += LANES) {
            if (my[k] == kNoPick) continue;
            const float x = chosen(k);
            ref_key = max(ref_key, key_of(r.sigmoid ? fminf(x, 0.0f) : x));
        }
        ref_key = row_max_i<LANES>(ref_key);
    }
    const double ref = r.renormalize ? static_cast<double>(key_value(ref_key))
                       : r.sigmoid   ? 0.0
                                     : static_cast<double>(top);
    double total = 0.0;
    for (int k = l; k < K; k += LANES) {
        double p = 0.0;
        if (my[k] != kNoPick) {
            const double x = static_cast<double>(chosen(k));
            if (r.sigmoid) p = exp(fmin(x, 0.0) - ref) / (1.0 + exp(-fabs(x)));
            else p = x == ref ? 1.0 : exp(x - ref);
        }
        part[k] = p;
        total += p;
    }
    double factor = static_cast<double>(r.scale);
    if (r.renormalize) {
        total = row_sum<LANES>(total);
        factor = total > 0.0 ? factor / total : 0.0;
    } else if (!r.sigmoid) {
        factor = whole > 0.0 ? factor / whole : 0.0;
    }
    for (int k = l; k < K; k += LANES) {  // each lane its own parts
        ids[t * K + k] = my[k] == kNoPick ? -1 : my[k];
        const float w = static_cast<float>(part[k] * factor);
        if (r.weights_type == MOE_DT_FLOAT32) put<F32>(weights, t * K + k, w);
        else put<F16>(weights, t * K + k, w);
    }
}

template <typename L>
__device__ __forceinline__ void store4_logits(void* p, int64_t i, const float* v) {
    if constexpr (std::is_same_v<L, F32>) {
        *reinterpret_cast<f32x4*>(static_cast<float*>(p) + i) = f32x4{v[0], v[1], v[2], v[3]};
    } else {
        uint16_t b[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) put<L>(b, j, v[j]);
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) =
            make_uint2(b[0] | (static_cast<uint32_t>(b[1]) << 16), b[2] | (static_cast<uint32_t>(b[3]) << 16));
    }
}

// Gradient of the weights of `ids` to the logits. p = s / sum of the K chosen s, g = grad_w, all times scale:
//   renormalised  softmax: dl_k = p_k (g_k - sum g p)          sigmoid: the same times (1 - s_k)
//   not           sigmoid: dl_k = g_k s_k (1 - s_k)            softmax: dl_e = s_e (g_e [e chosen] - sum g s)
// Where one expert has nearly all of a row, g_k nearly is that sum, and the difference is made of the other picks'
// terms: scores of the picks, their sums, the mean and the difference are float64 (of the whole row fp32). The scale
// comes last and the picks' scores have 29 bits, so that g s is exact: one renormalised weight is constant, and its
// gradient is 0, since g s / s is g.
// Bound by its bytes (T E written, and read in the last form; in the others only the picks' logits are read). 16 lanes
// have a token, a wave four. A lane has every 16th pick; their terms are added into a row of LDS one after another, so
// an id that a caller's list holds twice adds up in a fixed order, and the row leaves in whole vectors.
template <typename L, int C, bool VEC>
__global__ __launch_bounds__(kWave) void group_routing_grad_kernel(GroupRouting r, const void* __restrict__ grad_w,
                                                                   const int32_t* __restrict__ ids,
                                                                   void* __restrict__ grad_logits) {
    extern __shared__ __align__(16) char shared[];
    const int E = r.E, K = r.K, pitch = (E + 3) / 4 * 4 + 4;
    const int lane = lane_id(), tok = lane / kRow, l = lane % kRow;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * kRowTokens + tok;
    const bool valid = t < r.T;
    float* row = reinterpret_cast<float*>(shared) + tok * pitch;
    const bool softmax_all = !r.sigmoid && !r.renormalize;

    struct Pick {
        int id;  // -1: outside [0, E), or its expert is not available
        float x, g;
    };
    auto load_pick = [&](int k) {
        Pick p{-1, kLow, 0.0f};
        if (!valid || k >= K) return p;
        const int e = ids[t * K + k];
        if (e < 0 || e >= E) return p;
        p.x = logit<L>(r.logits, t * r.ld + e);
        if (!(p.x > kLow)) return p;
        p.id = e;
        p.g = r.weights_type == MOE_DT_FLOAT32   ? logit<F32>(grad_w, t * K + k)
              : r.weights_type == MOE_DT_FLOAT16 ? logit<F16>(grad_w, t * K + k)
                                                 : logit<B16>(grad_w, t * K + k);
        return p;
    };
    const Pick first = load_pick(l);
    auto pick_at = [&](int k) { return k < kRow ? first : load_pick(k); };

    // Scores up to a factor e^-top: of the row's softmax where all of it counts, else, renormalised, relative to the
    // largest of the picks, so that picks far below the row's best keep their ratios.
    float s[C], top = 0.0f;
    double inv = 1.0;  // one over the row's sum
    if (softmax_all) {
        float v[C];
        if (valid) {
            load_logits<L, kRow, C, VEC>(r.logits, t * r.ld, E, l, v);
        } else {
#pragma unroll
            for (int j = 0; j < C; ++j) v[j] = kLow;
        }
        int m = kGone;
#pragma unroll
        for (int j = 0; j < C; ++j) {
            v[j] = v[j] > kLow ? v[j] : kLow;
            m = max(m, key_of(v[j]));
        }
        top = key_value(row_max_i<kRow>(m));
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < C; ++j) {
            const float d = v[j] == top ? 0.0f : v[j] - top;
            s[j] = v[j] > kLow ? __builtin_amdgcn_exp2f(d * 1.4426950408889634f) : 0.0f;
            sum += static_cast<double>(s[j]);
        }
        sum = row_sum_d(sum);
        inv = sum > 0.0 ? 1.0 / sum : 0.0;
    } else if (r.renormalize) {
        int m = kGone;
        for (int k = l; k < K; k += kRow) {
            const Pick p = pick_at(k);
            if (p.id >= 0) m = max(m, key_of(r.sigmoid ? fminf(p.x, 0.0f) : p.x));
        }
        m = row_max_i<kRow>(m);
        top = m == kGone ? 0.0f : key_value(m);
    }
    // A pick's score, and for the sigmoid one less it, in LDS until the sums are known: entry k is lane k % 16's alone
    double2* scores = reinterpret_cast<double2*>(shared + kRowTokens * pitch * 4) + tok * K;
    double total = 0.0, dot = 0.0;  // sums of s and g s over the picks
#pragma unroll 1
    for (int k = l; k < K; k += kRow) {
        const Pick p = pick_at(k);
        if (p.id < 0) continue;
        const double x = static_cast<double>(p.x), at_top = static_cast<double>(top);
        const double lead = r.sigmoid ? fmin(x, 0.0) : x;
        double sk = lead == at_top ? 1.0 : exp(lead - at_top), rest = 0.0;
        if (r.sigmoid) {
            const double q = exp(-fabs(x));
            sk /= 1.0 + q;
            rest = (x >= 0.0 ? q : 1.0) / (1.0 + q);
        }
        sk = __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, sk) & ~uint64_t{0xffffff});  // 29 bits
        scores[k] = make_double2(sk, rest);
        total += sk;
        dot += static_cast<double>(p.g) * sk;
    }
    total = row_sum_d(total);
    dot = row_sum_d(dot);
    const bool any = total > 0.0;
    const double norm = !r.renormalize ? 1.0 : any ? 1.0 / total : 0.0;
    const double mean = softmax_all ? dot * inv : r.renormalize && any ? dot / total : 0.0;
    const double scale = static_cast<double>(r.scale);

#pragma unroll
    for (int j = 0; j < C; ++j) {
        const int e = expert_of<kRow, C>(l, j);
        if (e < E) row[e] = 0.0f;
    }
    __syncthreads();
    for (int k0 = 0; k0 < K; k0 += kRow) {
        const Pick p = pick_at(k0 + l);
        float d = 0.0f;
        if (softmax_all) {
            d = p.g;
        } else if (p.id >= 0) {
            const double2 sk = scores[k0 + l];
            const double dw = scale * (static_cast<double>(p.g) - mean) * (sk.x * norm);
            d = static_cast<float>(r.sigmoid ? dw * sk.y : dw);
        }
        for (int i = 0; i < kRow && k0 + i < K; ++i) {
            if (l == i && p.id >= 0) row[p.id] += d;
            __syncthreads();  // one wave: orders the additions
        }
    }
    if (!valid) return;
    const double all = scale * inv;
    auto from_all = [&](float g, float sj) {
        return static_cast<float>((static_cast<double>(g) - mean) * (all * static_cast<double>(sj)));
    };
#pragma unroll
    for (int j = 0; j < C; j += (VEC && C >= 4 ? 4 : 1)) {
        const int e = expert_of<kRow, C>(l, j);
        if (e >= E) continue;
        if constexpr (VEC && C >= 4) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(row + e);
            float v[4] = {a[0], a[1], a[2], a[3]};
            if (softmax_all) {
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = from_all(v[i], s[j + i]);
            }
            store4_logits<L>(grad_logits, t * E + e, v);
        } else {
            put<L>(grad_logits, t * E + e, softmax_all ? from_all(row[e], s[j]) : row[e]);
        }
    }
}

// Up to two rows a SIMD a token of more than 64 experts has a wave, whose chain is shorter: E = 256 with bias and
// groups, T = 1 5.8 us (a DPP row 7.2), T = 2048 8.8 (10.5), T = 4096 10.8 (11.6), there without a bias 9.4 (7.9). At
// 64 experts both take 4.9 us at T = 1 and the DPP row less from there on.
constexpr int64_t kWaveRows = 2048;

// Rows of 4-expert pieces that one load can read
bool vector_logits(const GroupRouting& r) {
    const uintptr_t mask = r.logits_type == MOE_DT_FLOAT32 ? 15 : 7;
    return r.E % 4 == 0 && r.ld % 4 == 0 && (reinterpret_cast<uintptr_t>(r.logits) & mask) == 0 &&
           (reinterpret_cast<uintptr_t>(r.bias) & 15) == 0;
}

template <typename L, int LANES, int C, bool VEC>
hipError_t run_routing_vec(const GroupRouting& r, int32_t* ids, void* weights, hipStream_t stream) {
    constexpr int kTokens = kWave / LANES;
    TraceScope trace("moe_group_routing", stream);
    group_routing_kernel<L, LANES, C, VEC>
        <<<static_cast<unsigned>((r.T + kTokens - 1) / kTokens), kWave,
           RoutingLds<kTokens>{r.E, r.groups, r.K}.bytes(r.bias || r.top_groups < r.groups), stream>>>(r, ids, weights);
    return hipGetLastError();
}
template <typename L, int LANES, int C>
hipError_t run_routing_lanes(const GroupRouting& r, int32_t* ids, void* weights, hipStream_t stream) {
    return vector_logits(r) ? run_routing_vec<L, LANES, C, true>(r, ids, weights, stream)
                            : run_routing_vec<L, LANES, C, false>(r, ids, weights, stream);
}
template <typename L, int C>
hipError_t run_routing(const GroupRouting& r, int32_t* ids, void* weights, hipStream_t stream) {
    if (C > 4 && r.T <= kWaveRows) return run_routing_lanes<L, kWave, 4>(r, ids, weights, stream);
    return run_routing_lanes<L, kRow, C>(r, ids, weights, stream);
}
template <typename L, int C, bool VEC>
hipError_t run_grad_vec(const GroupRouting& r, const void* gw, const int32_t* ids, void* gl, hipStream_t stream) {
    TraceScope trace("moe_group_routing_grad", stream);
    const int lds = kRowTokens * (((r.E + 3) / 4 * 4 + 4) * 4 + r.K * 16);
    group_routing_grad_kernel<L, C, VEC><<<static_cast<unsigned>((r.T + kRowTokens - 1) / kRowTokens), kWave, lds,
                                           stream>>>(r, gw, ids, gl);
    return hipGetLastError();
}
template <typename L, int C>
hipError_t run_grad(const GroupRouting& r, const void* gw, const int32_t* ids, void* gl, hipStream_t stream) {
    const bool vec = vector_logits(r) && (reinterpret_cast<uintptr_t>(gl) & 15) == 0;
    return vec ? run_grad_vec<L, C, true>(r, gw, ids, gl, stream) : run_grad_vec<L, C, false>(r, gw, ids, gl, stream);
}

template <typename F>
hipError_t by_type(const GroupRouting& r, F&& f) {
    const int c = (r.E + kRow - 1) / kRow;
    auto with = [&](auto type) {
        if (c <= 1) return f(type, std::integral_constant<int, 1>());
        if (c <= 4) return f(type, std::integral_constant<int, 4>());
        if (c <= 8) return f(type, std::integral_constant<int, 8>());
        return f(type, std::integral_constant<int, 16>());
    };
    if (r.logits_type == MOE_DT_FLOAT32) return with(F32());
    return r.logits_type == MOE_DT_FLOAT16 ? with(F16()) : with(B16());
}

}  // namespace

hipError_t launch_group_routing(const GroupRouting& r, int32_t* ids, void* weights, hipStream_t stream) {
    return by_type(r, [&](auto type, auto c) {
        return run_routing<decltype(type), decltype(c)::value>(r, ids, weights, stream);
    });
}
hipError_t launch_group_routing_grad(const GroupRouting& r, const void* grad_weights, const int32_t* ids,
                                     void* grad_logits, hipStream_t stream) {
    return by_type(r, [&](auto type, auto c) {
        return run_grad<decltype(type), decltype(c)::value>(r, grad_weights, ids, grad_logits, stream);
    });
}

}  // namespace moe
