// moe_norm.hip -- MoeAddRmsNorm, MoeAddRmsNormQuant, MoeAddRmsNormGrad and MoeQuantize for gfx950.
//
// v = x + residual in fp32, y = v r gamma with r = 1 / sqrt(mean v^2 + eps). The 8-bit form of a row is q = rint(p 127
// / max |p|): with p = v gamma the factor r, which a row has in common, cancels, so q needs no sum and is the same
// whatever the order of the sums; r enters the scale alone, max |p| r / 127. The gradient with u = v r: grad_v = r
// (grad_y gamma - u mean(grad_y gamma u)) + grad_sum, grad_gamma = the column sums of grad_y u.
//
// Memory bounds them: a row is read once into the registers of 1 to 16 waves (8 values a lane and step), reduced, and
// written from there; rows above 32768 values are read twice. Squares are added in fp64, which neither overflows nor
// loses a small row, and takes no time that memory does not hide. Reductions go over the lanes by DPP and then over the
// waves through LDS, in a fixed order.
//   T = 16381, H = 2048 bf16, x + residual -> sum, y, q  58.6 us, 5.15 TB/s (a copy of 1 GB: 5.13)
//   98304 rows of 1408 bf16 -> q                         72.3 us, 5.75 TB/s
//   gradient of T = 8192, H = 2048 fp16 with grad_sum    29.7 us, 4.5 TB/s, and 4.4 for the workgroups' column sums
//   T = 1, H = 7168                                      4.3 us, a row's latency: of a call of 8.6
#include "moe_ops.h"
#include "moe_rows.h"

namespace moe {

namespace {

constexpr int64_t kMaxBlocks = int64_t(1) << 20;  // of a launch

// Sum and largest (TWO: two sums) over the WAVES waves of a row, the same on every lane; `ex`: LDS for the waves' parts
template <int WAVES>
struct RowExchange {
    double a[WAVES], b[WAVES];
    uint32_t top[WAVES];
};
template <int WAVES, bool TWO>
__device__ __forceinline__ void reduce_row(RowExchange<WAVES>& ex, double& a, double& b, uint32_t& top) {
    a = wave_sum(a);
    if (TWO) b = wave_sum(b);
    else top = wave_max(top);
    if (WAVES == 1) return;
    const int wave = static_cast<int>(threadIdx.x) / kWave % WAVES;
    if (lane_id() == 0) {
        ex.a[wave] = a;
        if (TWO) ex.b[wave] = b;
        else ex.top[wave] = top;
    }
    __syncthreads();
    a = ex.a[0];
    b = ex.b[0];
    top = ex.top[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) {
        a += ex.a[w];
        if (TWO) b += ex.b[w];
        else top = max(top, ex.top[w]);
    }
    __syncthreads();  // read before the next row's parts
}

// r of a row as f r', f a power of two that keeps r' and f v in fp32's range for any finite v
struct RowFactor {
    float f, r;
};
__device__ __forceinline__ RowFactor row_factor(double squares, int H, float eps) {
    const double m = squares / H + static_cast<double>(eps);
    RowFactor s;
    s.f = m > 0x1p100 ? 0x1p-80f : m < 0x1p-100 ? 0x1p100f : 1.0f;
    s.r = 1.0f / sqrtf(static_cast<float>(m * s.f * s.f));
    return s;
}

__device__ __forceinline__ uint32_t magnitude(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

// NORM: the norm (its result, its 8-bit form or both), gamma of type G; else the 8-bit form of x itself. CHUNKS steps
// of V values a lane hold a row; 0: any length, read twice.
template <typename T, typename G, int WAVES, int CHUNKS, int V, bool NORM>
__global__ __launch_bounds__(WAVES == 1 ? 256 : WAVES * kWave) void norm_kernel(NormArgs n) {
    using Bits = typename T::Bits;
    constexpr int kRows = WAVES == 1 ? 4 : 1;  // rows of a workgroup at a time
    constexpr int kStep = WAVES * kWave * V;
    constexpr int kSteps = CHUNKS > 0 ? CHUNKS : 1;
    __shared__ RowExchange<WAVES> ex;
    const int wave = static_cast<int>(threadIdx.x) / kWave;
    const int lead = WAVES == 1 ? lane_id() : static_cast<int>(threadIdx.x);
    const bool ragged = n.H % V != 0;
    const typename G::Bits* gamma = static_cast<const typename G::Bits*>(n.gamma);
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + (WAVES == 1 ? wave : 0); row < n.rows;
         row += static_cast<int64_t>(gridDim.x) * kRows) {
        const Bits* x = static_cast<const Bits*>(n.x) + row * n.ldx;
        const Bits* res = NORM && n.residual ? static_cast<const Bits*>(n.residual) + row * n.ldr : nullptr;
        float v[kSteps][V];
        Step<V> at[kSteps];
        double squares = 0.0, unused = 0.0;
        uint32_t top = 0;
        auto load = [&](int col) __attribute__((always_inline)) {  // kSteps steps from col on
            RawRow<T, V> a[kSteps], b[kSteps];
#pragma unroll
            for (int c = 0; c < kSteps; ++c) {
                at[c] = step_at<V>(col + c * kStep, n.H);
                a[c].load(x + at[c].at);
            }
            if (NORM && res) {
#pragma unroll
                for (int c = 0; c < kSteps; ++c) b[c].load(res + at[c].at);
            }
#pragma unroll
            for (int c = 0; c < kSteps; ++c)
#pragma unroll
                for (int j = 0; j < V; ++j) v[c][j] = NORM && res ? a[c].get(j) + b[c].get(j) : a[c].get(j);
        };
        auto take = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int c = 0; c < kSteps; ++c) {
                if (NORM) {
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const double d = (ragged ? j >= at[c].skip : at[c].live) ? v[c][j] : 0.0f;
                        squares += d * d;
                    }
                }
                if (!NORM || n.q) {
                    float g[V];
                    if (NORM) load_row<G, V>(gamma + at[c].at, g);
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const uint32_t m = magnitude(NORM ? v[c][j] * g[j] : v[c][j]);
                        top = max(top, at[c].live ? m : 0u);
                    }
                }
            }
        };
        RowFactor s{1.0f, 1.0f};
        RowQuant quant{};
        auto finish = [&]() __attribute__((always_inline)) {
            reduce_row<WAVES, false>(ex, squares, unused, top);
            if (NORM) s = row_factor(squares, n.H, n.eps);
            if (!n.q) return;
            quant = row_quant(top);
            if (lead != 0) return;
            const float t = __builtin_bit_cast(float, top), scale = (NORM ? t * s.f * s.r : t) / 127.0f;
            n.scale[row] = quant.finite ? scale : __builtin_nanf("");
        };
        auto put = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int c = 0; c < kSteps; ++c) {
                if (!at[c].live) continue;
                const int64_t to = row * n.H + at[c].at;
                if (!NORM) {
                    store_quant<V>(n.q + to, v[c], quant);
                    continue;
                }
                float g[V], y[V];
                load_row<G, V>(gamma + at[c].at, g);
                if (n.sum) store_row<T, V>(static_cast<Bits*>(n.sum) + to, v[c]);
                if (n.y) {
#pragma unroll
                    for (int j = 0; j < V; ++j) y[j] = v[c][j] * s.f * s.r * g[j];
                    store_row<T, V>(static_cast<Bits*>(n.y) + to, y);
                }
                if (n.q) {
#pragma unroll
                    for (int j = 0; j < V; ++j) y[j] = v[c][j] * g[j];
                    store_quant<V>(n.q + to, y, quant);
                }
            }
        };
        if (CHUNKS > 0) {
            load(lead * V);
            take();
            finish();
            put();
        } else {
            for (int col = lead * V; col < n.H; col += kStep) {
                load(col);
                take();
            }
            finish();
            for (int col = lead * V; col < n.H; col += kStep) {
                load(col);
                put();
            }
        }
    }
}

// The gradient. A workgroup walks rows, at least 8 waves' worth at a time, and keeps its share of grad_gamma's column
// sums in registers; they leave as one row of `part` for each workgroup. us of both launches with 4, 8 and 16 waves a
// workgroup: T = 8192, H = 2048 30.8, 30.4, 33.7; T = 16384, H = 512 19.4, 17.6, 19.3; T = 4096, H = 4096 30.7, 29.8,
// 32.7 (fewer rows of `part`, but more waves wait for each other)
constexpr int kGradWaves = 8;
constexpr int grad_waves(int H) {  // of a row, two steps each
    return H <= 1024 ? 1 : H <= 2048 ? 2 : H <= 4096 ? 4 : H <= 8192 ? 8 : 16;
}
constexpr int grad_threads(int waves) { return (waves < kGradWaves ? kGradWaves : waves) * kWave; }
template <typename T, typename G, int WAVES, int STEPS, int V>
__global__ __launch_bounds__(grad_threads(WAVES)) void norm_grad_kernel(NormArgs n) {
    using Bits = typename T::Bits;
    constexpr int kRows = grad_threads(WAVES) / (WAVES * kWave);
    constexpr int kStep = WAVES * kWave * V;
    __shared__ RowExchange<WAVES> ex[kRows];
    __shared__ float sums[kRows > 1 ? kRows - 1 : 1][kRows > 1 ? STEPS * kStep : 1];
    const int team = static_cast<int>(threadIdx.x) / (WAVES * kWave);
    const int lead = static_cast<int>(threadIdx.x) % (WAVES * kWave);
    const typename G::Bits* gamma = static_cast<const typename G::Bits*>(n.gamma);
    Step<V> at[STEPS];
#pragma unroll
    for (int c = 0; c < STEPS; ++c) at[c] = step_at<V>(lead * V + c * kStep, n.H);
    float gg[STEPS][V] = {};
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * kRows; base < n.rows;
         base += static_cast<int64_t>(gridDim.x) * kRows) {
        const bool live = base + team < n.rows;  // past the last row: that row again, for nothing
        const int64_t row = live ? base + team : n.rows - 1;
        const Bits* x = static_cast<const Bits*>(n.x) + row * n.ldx;
        const Bits* gy = static_cast<const Bits*>(n.grad_y) + row * n.ldy;
        RawRow<T, V> v[STEPS], d[STEPS], add[STEPS];
        double squares = 0.0, dot = 0.0;
        uint32_t unused = 0;
#pragma unroll
        for (int c = 0; c < STEPS; ++c) {
            v[c].load(x + at[c].at);
            d[c].load(gy + at[c].at);
        }
        if (n.grad_sum) {
#pragma unroll
            for (int c = 0; c < STEPS; ++c)
                add[c].load(static_cast<const Bits*>(n.grad_sum) + row * n.lds + at[c].at);
        }
#pragma unroll
        for (int c = 0; c < STEPS; ++c) {
            float g[V];
            load_row<G, V>(gamma + at[c].at, g);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const bool counts = j >= at[c].skip;  // past the row none does
                const double a = counts ? v[c].get(j) : 0.0f;
                squares += a * a;
                dot += static_cast<double>(counts ? d[c].get(j) * g[j] : 0.0f) * a;
            }
        }
        reduce_row<WAVES, true>(ex[team], squares, dot, unused);
        if (!live) continue;
        const RowFactor s = row_factor(squares, n.H, n.eps);
        const float r = s.f * s.r;
        const float mean = static_cast<float>(dot * s.f * s.r / n.H);  // of grad_y gamma u
#pragma unroll
        for (int c = 0; c < STEPS; ++c) {
            float g[V], gx[V];
            load_row<G, V>(gamma + at[c].at, g);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float u = v[c].get(j) * s.f * s.r, gv = d[c].get(j);
                gg[c][j] += gv * u;
                gx[j] = r * (gv * g[j] - u * mean);
                if (n.grad_sum) gx[j] += add[c].get(j);
            }
            if (n.y && at[c].live) store_row<T, V>(static_cast<Bits*>(n.y) + row * n.H + at[c].at, gx);
        }
    }
    if (!n.part) return;
    if (kRows > 1) {  // the teams' sums, added in order
        if (team > 0) {
#pragma unroll
            for (int c = 0; c < STEPS; ++c)
                if (at[c].live) store_row<F32, V>(&sums[team - 1][at[c].at], gg[c]);
        }
        __syncthreads();
        if (team > 0) return;
#pragma unroll
        for (int t = 0; t + 1 < kRows; ++t)
#pragma unroll
            for (int c = 0; c < STEPS; ++c) {
                float other[V];
                load_row<F32, V>(&sums[t][at[c].at], other);
#pragma unroll
                for (int j = 0; j < V; ++j) gg[c][j] += other[j];
            }
    }
    float* out = n.part + static_cast<int64_t>(blockIdx.x) * n.H;
#pragma unroll
    for (int c = 0; c < STEPS; ++c)
        if (at[c].live) store_row<F32, V>(out + at[c].at, gg[c]);
}

// grad_gamma: the workgroups' rows, 32 columns a workgroup (whole lines; 16 columns took 1 to 2 us more); 32 groups add
// every 32nd row, 8 of them 4 groups' sums, and one those
constexpr int kSumThreads = 1024, kSumCols = 32;
template <typename G>
__global__ __launch_bounds__(kSumThreads) void gamma_sum_kernel(const float* __restrict__ part,
                                                                typename G::Bits* __restrict__ out, int H, int rows) {
    constexpr int kCols = kSumCols, kGroups = kSumThreads / kCols, kFirst = 8;
    __shared__ float sums[kGroups][kCols], eighths[kFirst][kCols];
    const int i = static_cast<int>(threadIdx.x) % kCols, q = static_cast<int>(threadIdx.x) / kCols;
    const int col = static_cast<int>(blockIdx.x) * kCols + i;
    float s = 0.0f;
    if (col < H) {
#pragma unroll 16
        for (int b = q; b < rows; b += kGroups) s += part[static_cast<int64_t>(b) * H + col];
    }
    sums[q][i] = s;
    __syncthreads();
    if (q < kFirst) {
        s = 0.0f;
#pragma unroll
        for (int g = 0; g < kGroups / kFirst; ++g) s += sums[q + g * kFirst][i];
        eighths[q][i] = s;
    }
    __syncthreads();
    if (q != 0 || col >= H) return;
    s = 0.0f;
#pragma unroll
    for (int g = 0; g < kFirst; ++g) s += eighths[g][i];
    out[col] = G::store(s);
}

// Waves of a row, and the steps that hold it (0: none do). Where there are rows enough for every SIMD a row has two
// steps in flight for as few waves as that takes; few rows are spread over as many waves as have one step each.
//   x + residual with y and its 8-bit form, bf16, us with 1, 2, 4 waves: T = 16384, H = 512 18 / 22 / 34; H = 1024 32 /
//   31 / 42; H = 2048 74 (four steps) / 58 / 59; T = 98304, H = 1408 328 / 244 / 260
struct Shape {
    int waves, steps;
};
Shape norm_shape(int64_t rows, int H) {
    const int reach = rows >= 2048 ? 1024 : 512;  // values that a wave holds
    for (int waves = 1; waves <= 16; waves *= 2)
        if (H <= waves * reach) return Shape{waves, (H + waves * 512 - 1) / (waves * 512)};
    return Shape{16, H <= 16384 ? 2 : H <= 32768 ? 4 : 0};
}
unsigned norm_grid(int64_t rows, int waves) {
    const int64_t blocks = waves == 1 ? (rows + 3) / 4 : rows;
    return static_cast<unsigned>(blocks < kMaxBlocks ? blocks : kMaxBlocks);
}

template <typename T, typename G, int WAVES, int CHUNKS, bool NORM, int V = 8>
hipError_t run_norm(const NormArgs& n, hipStream_t stream) {
    norm_kernel<T, G, WAVES, CHUNKS, V, NORM>
        <<<norm_grid(n.rows, WAVES), WAVES == 1 ? 256 : WAVES * kWave, 0, stream>>>(n);
    return hipGetLastError();
}
template <typename T, typename G, bool NORM>
hipError_t run_norm_any(const NormArgs& n, hipStream_t stream) {
    if (n.H < 8) return run_norm<T, G, 1, 1, NORM, 1>(n, stream);
    const Shape s = norm_shape(n.rows, n.H);
    switch (s.waves * 8 + s.steps) {
        case 1 * 8 + 1: return run_norm<T, G, 1, 1, NORM>(n, stream);
        case 1 * 8 + 2: return run_norm<T, G, 1, 2, NORM>(n, stream);
        case 2 * 8 + 1: return run_norm<T, G, 2, 1, NORM>(n, stream);
        case 2 * 8 + 2: return run_norm<T, G, 2, 2, NORM>(n, stream);
        case 4 * 8 + 1: return run_norm<T, G, 4, 1, NORM>(n, stream);
        case 4 * 8 + 2: return run_norm<T, G, 4, 2, NORM>(n, stream);
        case 8 * 8 + 1: return run_norm<T, G, 8, 1, NORM>(n, stream);
        case 8 * 8 + 2: return run_norm<T, G, 8, 2, NORM>(n, stream);
        case 16 * 8 + 1: return run_norm<T, G, 16, 1, NORM>(n, stream);
        case 16 * 8 + 2: return run_norm<T, G, 16, 2, NORM>(n, stream);
        case 16 * 8 + 4: return run_norm<T, G, 16, 4, NORM>(n, stream);
        default: return run_norm<T, G, 16, 0, NORM>(n, stream);
    }
}

template <typename T, typename G, int WAVES, int STEPS, int V = 8>
hipError_t run_norm_grad(const NormArgs& n, int blocks, hipStream_t stream) {
    norm_grad_kernel<T, G, WAVES, STEPS, V><<<blocks, grad_threads(WAVES), 0, stream>>>(n);
    return hipGetLastError();
}
template <typename T, typename G>
hipError_t run_norm_grad_any(const NormArgs& n, int blocks, hipStream_t stream) {
    if (n.H < 8) return run_norm_grad<T, G, 1, 1, 1>(n, blocks, stream);
    if (n.H <= 512) return run_norm_grad<T, G, 1, 1>(n, blocks, stream);
    switch (grad_waves(n.H)) {
        case 1: return run_norm_grad<T, G, 1, 2>(n, blocks, stream);
        case 2: return run_norm_grad<T, G, 2, 2>(n, blocks, stream);
        case 4: return run_norm_grad<T, G, 4, 2>(n, blocks, stream);
        case 8: return run_norm_grad<T, G, 8, 2>(n, blocks, stream);
        default: return run_norm_grad<T, G, 16, 2>(n, blocks, stream);
    }
}

// f(row type, gamma type) for the types of a call
template <typename F>
hipError_t by_type(int type, bool gamma_f32, F&& f) {
    if (type == MOE_DT_FLOAT32) return f(F32(), F32());
    if (type == MOE_DT_FLOAT16) return gamma_f32 ? f(Half(), F32()) : f(Half(), Half());
    return gamma_f32 ? f(Bf16(), F32()) : f(Bf16(), Bf16());
}

}  // namespace

hipError_t launch_norm(const NormArgs& n, int type, bool norm, hipStream_t stream) {
    TraceScope trace(norm ? "moe_norm" : "moe_quantize", stream);
    if (!norm)
        return by_type(type, false, [&](auto t, auto) { return run_norm_any<decltype(t), F32, false>(n, stream); });
    return by_type(type, n.gamma_f32, [&](auto t, auto g) {
        return run_norm_any<decltype(t), decltype(g), true>(n, stream);
    });
}

// Workgroups of the gradient, 16 waves on every CU at most. T = 8192, H = 2048, us of both launches with workgroups of 4
// waves: 2 waves a row and 1024 workgroups 31.5, 512 34.0; 1 wave (four steps) 33.1 with 512; 4 waves (one step) 33.5
// with 1024
int norm_grad_blocks(int64_t rows, int H) {
    const int waves = grad_waves(H);
    const int64_t each = waves < kGradWaves ? kGradWaves / waves : 1, most = waves <= kGradWaves ? 512 : 256;
    const int64_t blocks = (rows + each - 1) / each;
    return static_cast<int>(blocks < 1 ? 1 : blocks < most ? blocks : most);
}

hipError_t launch_norm_grad(const NormArgs& n, int type, void* grad_gamma, hipStream_t stream) {
    const int blocks = norm_grad_blocks(n.rows, n.H);
    hipError_t err;
    {
        TraceScope trace("moe_norm_grad", stream);
        err = by_type(type, n.gamma_f32, [&](auto t, auto g) {
            return run_norm_grad_any<decltype(t), decltype(g)>(n, blocks, stream);
        });
    }
    if (err != hipSuccess || !grad_gamma) return err;
    TraceScope trace("moe_norm_gamma", stream);
    const int grid = (n.H + kSumCols - 1) / kSumCols;
    return by_type(type, n.gamma_f32, [&](auto, auto g) {
        using G = decltype(g);
        gamma_sum_kernel<G><<<grid, kSumThreads, 0, stream>>>(n.part, static_cast<typename G::Bits*>(grad_gamma), n.H,
                                                              blocks);
        return hipGetLastError();
    });
}

}  // namespace moe
