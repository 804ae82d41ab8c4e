// moe_combine_grad.hip -- MoeCombineGrad for gfx950: the gradients of y[t, :] = sum_k weights[t, k] *
// expert_out[t, k, :].
//
//   grad_expert_out[t, k, :] = weights[t, k] * grad_y[t, :]
//   grad_weights[t, k]       = sum_h grad_y[t, h] * expert_out[t, k, h]
//
// The forward is the reference's op_kernel/moe_combine.cpp:80-111; it has no gradient there.
// Pure streaming: T (2 K + 1) H 2 bytes. One pass: a thread holds 8 hidden elements of grad_y and, for up to 8 experts
// at a time, loads their rows, adds to their dot products and writes their gradient rows. A wave has a token to itself,
// or four waves share it; the dot products are added over the lanes and then over the waves in a fixed order.
// T = 16384, H = 2048, K = 6: 872 MB in 144 us, 6.07 TB/s (a copy of 1 GB: 5.0). T = 128, K = 2: 4 us, of a call of 7.
#include "moe_device.h"
#include "moe_launch.h"

namespace moe {

namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 8;  // experts in flight per thread
// expert_out and its gradient together beyond the 256 MB Infinity Cache go past it (non-temporal): T = 16384, K = 6 144
// us, through the cache 171 us
constexpr int64_t kStreamBytes = int64_t(128) << 20;
constexpr int64_t kMaxBlocks = int64_t(1) << 22;  // of a launch: 2^30 threads, HIP's limit is 2^32

template <int WAVES, bool NT>  // waves of one token: 1 or 4
__global__ __launch_bounds__(kThreads) void combine_grad_kernel(const uint16_t* __restrict__ grad_y,
                                                                const uint16_t* __restrict__ expert_out,
                                                                const uint16_t* __restrict__ weights,
                                                                uint16_t* __restrict__ grad_eo,
                                                                uint16_t* __restrict__ grad_w, int64_t T, int H,
                                                                int K) {
    __shared__ float part[4][kBatch];
    const int wave = static_cast<int>(threadIdx.x) / kWave, lane = lane_id();
    constexpr int kTokens = 4 / WAVES;  // of a workgroup at a time; more than kMaxBlocks workgroups' take turns
    const int first = (WAVES == 1 ? lane : static_cast<int>(threadIdx.x)) * 8;
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * kTokens + (WAVES == 1 ? wave : 0); t < T;
         t += static_cast<int64_t>(gridDim.x) * kTokens) {
        const uint16_t* dy = grad_y + t * H;
        for (int k0 = 0; k0 < K; k0 += kBatch) {
            float dot[kBatch] = {}, w[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) w[u] = k0 + u < K ? f16_bits_to_f32(weights[t * K + k0 + u]) : 0.0f;
            for (int c = first; c < H; c += WAVES * kWave * 8) {
                const f16x8 d = load_f16x8(dy + c);
                f16x8 o[kBatch];
#pragma unroll
                for (int u = 0; u < kBatch; ++u)
                    if (k0 + u < K) {
                        const uint16_t* at = expert_out + (t * K + k0 + u) * H + c;
                        o[u] = NT ? load_f16x8_stream(at) : load_f16x8(at);
                    }
#pragma unroll
                for (int u = 0; u < kBatch; ++u) {
                    if (k0 + u < K) {
                        f16x8 v;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float g = static_cast<float>(d[j]);
                            dot[u] += g * static_cast<float>(o[u][j]);
                            v[j] = static_cast<f16>(w[u] * g);
                        }
                        uint16_t* at = grad_eo + (t * K + k0 + u) * H + c;
                        if (NT) __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), reinterpret_cast<u32x4*>(at));
                        else *reinterpret_cast<f16x8*>(at) = v;
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < kBatch; ++u)
#pragma unroll
                for (int d = kWave / 2; d > 0; d >>= 1) dot[u] += __shfl_xor(dot[u], d, kWave);
            if (WAVES == 1) {
                float v = dot[0];
#pragma unroll
                for (int u = 1; u < kBatch; ++u) v = lane == u ? dot[u] : v;
                if (lane < kBatch && k0 + lane < K) grad_w[t * K + k0 + lane] = f32_to_f16_bits(v);
            } else {
                if (lane == 0) {
#pragma unroll
                    for (int u = 0; u < kBatch; ++u) part[wave][u] = dot[u];
                }
                __syncthreads();
                const int u = static_cast<int>(threadIdx.x);
                if (u < kBatch && k0 + u < K)
                    grad_w[t * K + k0 + u] = f32_to_f16_bits(part[0][u] + part[1][u] + part[2][u] + part[3][u]);
                __syncthreads();
            }
        }
    }
}

}  // namespace

hipError_t launch_combine_grad(const uint16_t* grad_y, const uint16_t* expert_out, const uint16_t* weights,
                               uint16_t* grad_eo, uint16_t* grad_w, int64_t T, int H, int K, hipStream_t stream) {
    TraceScope trace("moe_combine_grad", stream);
    const bool nt = T * K * H * 2 > kStreamBytes;
    // a wave a token once that gives every SIMD two waves
    const bool one = T >= 2048;
    const int64_t blocks = one ? (T + 3) / 4 : T;
    const unsigned grid = static_cast<unsigned>(blocks < kMaxBlocks ? blocks : kMaxBlocks);
    if (one && nt)
        combine_grad_kernel<1, true>
            <<<grid, kThreads, 0, stream>>>(grad_y, expert_out, weights, grad_eo, grad_w, T, H, K);
    else if (one)
        combine_grad_kernel<1, false>
            <<<grid, kThreads, 0, stream>>>(grad_y, expert_out, weights, grad_eo, grad_w, T, H, K);
    else if (nt)
        combine_grad_kernel<4, true>
            <<<grid, kThreads, 0, stream>>>(grad_y, expert_out, weights, grad_eo, grad_w, T, H, K);
    else
        combine_grad_kernel<4, false>
            <<<grid, kThreads, 0, stream>>>(grad_y, expert_out, weights, grad_eo, grad_w, T, H, K);
    return hipGetLastError();
}

}  // namespace moe
