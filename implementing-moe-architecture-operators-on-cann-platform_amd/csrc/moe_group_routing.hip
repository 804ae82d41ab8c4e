// moe_group_routing.hip -- MoeRoutingGroupTopK and its gradient for gfx950: from logits [T, E] to experts and weights.
//
// The reference routes by softmax and top-K alone (op_kernel/moe_routing.cpp:238-369). Here
//   s = sigmoid(l) or softmax(l),  c = s + bias
//   groups of E / G consecutive experts, each scored by its best c or the sum of its two best; the best topGroups stay
//   the K best c among them in descending order, ties to the lowest index; w = scale * s, over the K's sum if asked
// An expert whose logit or c is NaN or -inf is not available; picks with no expert left are id -1, weight 0.
// c is compared in float64: fp32 scores that agree to their last bit would be picked in an order that depends on how
// the exponential was rounded.
#include "moe_device.h"
#include "moe_launch.h"
#include "moe_ops.h"

#include <type_traits>

namespace moe {

namespace {

constexpr int kThreads = 256;
constexpr int kLanes = 16;                     // lanes of one token
constexpr int kTokens = kThreads / kLanes;     // tokens of a workgroup
constexpr int kMaxE = 256;
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

template <typename V>
__device__ __forceinline__ V row_max(V v) {
#pragma unroll
    for (int d = kLanes / 2; d > 0; d >>= 1) {
        const V o = __shfl_xor(v, d, kLanes);
        v = o > v ? o : v;
    }
    return v;
}
template <typename V>
__device__ __forceinline__ V row_sum(V v) {
#pragma unroll
    for (int d = kLanes / 2; d > 0; d >>= 1) v += __shfl_xor(v, d, kLanes);
    return v;
}

// LDS: c [kTokens][E], group scores [kTokens][G] (double), picked scores [kTokens][K] (double), picks [kTokens][K]
// (int), kept groups [kTokens][G] (int)
int routing_lds(int E, int G, int K) { return kTokens * (E * 8 + G * 8 + K * 8 + K * 4 + G * 4); }

// C: experts of a lane (lane, lane + 16, ...), at most
template <typename L, int C>
__global__ __launch_bounds__(kThreads) void group_routing_kernel(GroupRouting r, int32_t* __restrict__ ids,
                                                                 void* __restrict__ weights) {
    extern __shared__ __align__(16) char shared[];
    const int E = r.E, G = r.groups, K = r.K, size = E / G;
    double* cs = reinterpret_cast<double*>(shared);
    double* gs = cs + kTokens * E;
    double* ps = gs + kTokens * G;
    int* pick = reinterpret_cast<int*>(ps + kTokens * K);
    int* kept = pick + kTokens * K;
    const int tid = static_cast<int>(threadIdx.x), tok = tid / kLanes, l = tid % kLanes;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * kTokens + tok;
    const bool valid = t < r.T;

    double s[C], c[C], lg[C];  // scores, what is compared, logits
    bool open[C];
    double top = kNone;
#pragma unroll
    for (int j = 0; j < C; ++j) {
        const int e = l + j * kLanes;
        double v = kNone;
        if (valid && e < E) v = static_cast<double>(logit<L>(r.logits, t * r.ld + e));
        open[j] = v > kNone;  // false for NaN too
        lg[j] = s[j] = v;
        if (open[j] && v > top) top = v;
    }
    if (r.sigmoid) {
#pragma unroll
        for (int j = 0; j < C; ++j) s[j] = open[j] ? 1.0 / (1.0 + exp(-s[j])) : 0.0;
    } else {
        top = row_max(top);
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < C; ++j) {
            s[j] = open[j] ? (s[j] == top ? 1.0 : exp(s[j] - top)) : 0.0;
            sum += s[j];
        }
        sum = row_sum(sum);
#pragma unroll
        for (int j = 0; j < C; ++j) s[j] = open[j] ? s[j] / sum : 0.0;
    }
#pragma unroll
    for (int j = 0; j < C; ++j) {
        const int e = l + j * kLanes;
        c[j] = kNone;
        if (open[j]) {
            c[j] = r.bias ? s[j] + static_cast<double>(r.bias[e]) : s[j];
            if (!(c[j] > kNone)) c[j] = kNone;
        }
    }
    if (r.top_groups < G) {
#pragma unroll
        for (int j = 0; j < C; ++j) {
            const int e = l + j * kLanes;
            if (e < E) cs[tok * E + e] = c[j];
        }
        __syncthreads();
        for (int i = tid; i < kTokens * G; i += kThreads) {
            const double* row = cs + (i / G) * E + (i % G) * size;
            double a = kNone, b = kNone;
            for (int e = 0; e < size; ++e) {
                const double v = row[e];
                if (v > a) {
                    b = a;
                    a = v;
                } else if (v > b) {
                    b = v;
                }
            }
            gs[i] = r.group_top == 2 && b > kNone ? a + b : a;
        }
        __syncthreads();
        for (int i = tid; i < kTokens * G; i += kThreads) {
            const double* row = gs + i / G * G;
            const int me = i % G;
            const double v = row[me];
            int before = 0;
            for (int o = 0; o < G; ++o) before += row[o] > v || (row[o] == v && o < me);
            kept[i] = before < r.top_groups;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < C; ++j) {
            const int e = l + j * kLanes;
            if (e < E && !kept[tok * G + e / size]) c[j] = kNone;
        }
    }
    for (int k = 0; k < K; ++k) {
        double best = kNone;
        int at = kMaxE;
#pragma unroll
        for (int j = 0; j < C; ++j)
            if (c[j] > best) {  // ascending e: the lowest index of equals stays
                best = c[j];
                at = l + j * kLanes;
            }
#pragma unroll
        for (int d = kLanes / 2; d > 0; d >>= 1) {
            const double ob = __shfl_xor(best, d, kLanes);
            const int oa = __shfl_xor(at, d, kLanes);
            if (ob > best || (ob == best && oa < at)) {
                best = ob;
                at = oa;
            }
        }
        if (at == kMaxE) {
            if (l == 0) {
                pick[tok * K + k] = -1;
                ps[tok * K + k] = r.renormalize ? kNone : 0.0;
            }
        } else {
#pragma unroll
            for (int j = 0; j < C; ++j)
                if (l + j * kLanes == at) {
                    pick[tok * K + k] = at;
                    ps[tok * K + k] = r.renormalize ? lg[j] : s[j];
                    c[j] = kNone;
                }
        }
    }
    __syncthreads();
    if (!valid) return;
    // Renormalised, the scores are taken relative to the largest of the picks: their ratios hold where the scores
    // themselves would underflow.
    const double* p = ps + tok * K;
    double ref = kNone, sum = 0.0;
    auto part = [&](double v) {
        if (!(v > kNone)) return 0.0;
        if (r.sigmoid) return exp(fmin(v, 0.0) - ref) / (1.0 + exp(-fabs(v)));
        return v == ref ? 1.0 : exp(v - ref);
    };
    if (r.renormalize) {
        for (int k = 0; k < K; ++k) ref = fmax(ref, r.sigmoid ? fmin(p[k], 0.0) : p[k]);
        for (int k = 0; k < K; ++k) sum += part(p[k]);
    }
    for (int k = l; k < K; k += kLanes) {
        ids[t * K + k] = pick[tok * K + k];
        const double q = !r.renormalize ? p[k] : sum > 0.0 ? part(p[k]) / sum : 0.0;
        const float w = static_cast<float>(q * static_cast<double>(r.scale));
        if (r.weights_type == MOE_DT_FLOAT32) put<F32>(weights, t * K + k, w);
        else put<F16>(weights, t * K + k, w);
    }
}

// Gradient of the weights of `ids` to the logits. p = s / sum of the K chosen s, g = scale * grad_w:
//   renormalised  softmax: dl_k = p_k (g_k - sum g p)          sigmoid: the same times (1 - s_k)
//   not           sigmoid: dl_k = g_k s_k (1 - s_k)            softmax: dl_e = s_e (g_e [e chosen] - sum g s)
// 16 lanes have a token. Every expert's lane goes over the K picks itself, so an id that a caller's list holds twice
// adds up in a fixed order and no lane writes another's element.
template <typename L, int C>
__global__ __launch_bounds__(kThreads) void group_routing_grad_kernel(GroupRouting r, const void* __restrict__ grad_w,
                                                                      const int32_t* __restrict__ ids,
                                                                      void* __restrict__ grad_logits) {
    const int E = r.E, K = r.K;
    const int tid = static_cast<int>(threadIdx.x), tok = tid / kLanes, l = tid % kLanes;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * kTokens + tok;
    if (t >= r.T) return;
    const int32_t* id = ids + t * K;
    auto g_of = [&](int k) {
        const float g = r.weights_type == MOE_DT_FLOAT32 ? logit<F32>(grad_w, t * K + k)
                                                         : r.weights_type == MOE_DT_FLOAT16
                                                               ? logit<F16>(grad_w, t * K + k)
                                                               : logit<B16>(grad_w, t * K + k);
        return g * r.scale;
    };
    constexpr float kLow = -__builtin_huge_valf();
    const bool softmax_all = !r.sigmoid && !r.renormalize;
    float lg[C], top = r.sigmoid && !r.renormalize ? 0.0f : kLow, sum = 0.0f;
#pragma unroll
    for (int j = 0; j < C; ++j) {
        const int e = l + j * kLanes;
        lg[j] = e < E ? logit<L>(r.logits, t * r.ld + e) : kLow;
    }
    // Scores up to a factor e^-top: of the row's softmax where all of it counts, else, renormalised, relative to the
    // largest of the picks, so that picks far below the row's best keep their ratios.
    if (softmax_all) {
#pragma unroll
        for (int j = 0; j < C; ++j)
            if (lg[j] > top) top = lg[j];
        top = row_max(top);
    } else if (r.renormalize) {
        for (int k = 0; k < K; ++k) {
            const int e = id[k];
            if (e < 0 || e >= E) continue;
            const float v = logit<L>(r.logits, t * r.ld + e), x = r.sigmoid ? fminf(v, 0.0f) : v;
            if (v > kLow && x > top) top = x;
        }
    }
    auto score = [&](float v) {
        if (!(v > kLow)) return 0.0f;
        if (r.sigmoid) return expf(fminf(v, 0.0f) - top) / (1.0f + expf(-fabsf(v)));
        return v == top ? 1.0f : expf(v - top);
    };
    if (softmax_all) {
#pragma unroll
        for (int j = 0; j < C; ++j) sum += score(lg[j]);
        sum = row_sum(sum);
    }
    const float inv = softmax_all ? (sum > 0.0f ? 1.0f / sum : 0.0f) : 1.0f;
    float total = 0.0f, dot = 0.0f;  // sum s, sum g s over the picks
    for (int k = 0; k < K; ++k) {
        const int e = id[k];
        if (e < 0 || e >= E) continue;
        const float s = score(logit<L>(r.logits, t * r.ld + e)) * inv;
        if (s > 0.0f) {
            total += s;
            dot += g_of(k) * s;
        }
    }
    const float mean = r.renormalize ? (total > 0.0f ? dot / total : 0.0f) : dot;
    const float norm = r.renormalize ? (total > 0.0f ? 1.0f / total : 0.0f) : 1.0f;
#pragma unroll
    for (int j = 0; j < C; ++j) {
        const int e = l + j * kLanes;
        if (e >= E) continue;
        float d = 0.0f;
        bool hit = false;
        for (int k = 0; k < K; ++k) {
            if (id[k] != e) continue;
            const float g = g_of(k);
            d += r.renormalize ? g - mean : g;
            hit = true;
        }
        if (softmax_all) d -= mean;
        if (softmax_all || hit) {  // without a pick in the row there is nothing the scores are relative to
            if (r.sigmoid) d *= expf(fminf(-lg[j], 0.0f)) / (1.0f + expf(-fabsf(lg[j])));  // 1 - s
            const float s = score(lg[j]) * inv;
            d = s > 0.0f ? d * s * norm : 0.0f;
        }
        put<L>(grad_logits, t * E + e, d);
    }
}

template <typename L, int C>
hipError_t run_routing(const GroupRouting& r, int32_t* ids, void* weights, hipStream_t stream) {
    const int lds = routing_lds(r.E, r.groups, r.K);
    auto fn = &group_routing_kernel<L, C>;
    const hipError_t err = ensure_lds_limit(reinterpret_cast<const void*>(fn), routing_lds(kMaxE, kMaxE, kMaxE));
    if (err != hipSuccess) return err;
    TraceScope trace("moe_group_routing", stream);
    fn<<<static_cast<unsigned>((r.T + kTokens - 1) / kTokens), kThreads, lds, stream>>>(r, ids, weights);
    return hipGetLastError();
}
template <typename L, int C>
hipError_t run_grad(const GroupRouting& r, const void* gw, const int32_t* ids, void* gl, hipStream_t stream) {
    TraceScope trace("moe_group_routing_grad", stream);
    group_routing_grad_kernel<L, C>
        <<<static_cast<unsigned>((r.T + kTokens - 1) / kTokens), kThreads, 0, stream>>>(r, gw, ids, gl);
    return hipGetLastError();
}

template <typename F>
hipError_t by_type(const GroupRouting& r, F&& f) {
    const int c = (r.E + kLanes - 1) / kLanes;
    auto with = [&](auto type) {
        if (c <= 1) return f(type, std::integral_constant<int, 1>());
        if (c <= 4) return f(type, std::integral_constant<int, 4>());
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
