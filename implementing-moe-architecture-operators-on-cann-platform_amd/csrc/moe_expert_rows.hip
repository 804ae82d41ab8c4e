// moe_expert_rows.hip -- MoePermute, MoeUnpermute and MoeUnpermuteGrad for gfx950: tokens sorted by expert, and back.
//
// The T K picks (token t, k) are sorted by expert, those of one expert in the order of their slots t K + k, and token t's
// row is copied to the places of its picks. Picks of no expert stand behind the others, in slot order too, with zero
// rows; position[t, k] is a pick's place p, or -1 - p of a pick of no expert, so every row has exactly one pick.
//   back       y[t] = sum_k weights[t, k] rows[position[t, k]], fp32 sums in ascending k
//   gradients  of rows: weights[t, k] grad_y[t] at position[t, k] (zeros for a pick of no expert); of weights[t, k]:
//              <grad_y[t], rows[position[t, k]]>; the gradient of MoePermute is the way back without weights
// Memory bounds all three: a token's row is read once and its K copies are written, or the other way round. No atomics:
// a pick's place is offsets[expert] + the expert's picks in earlier chunks + its rank in its chunk.
#include "moe_ops.h"
#include "moe_rows.h"

namespace moe {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / kWave;
constexpr int kBuckets = 257;  // 256 experts and the picks of none
constexpr int kPasses = 4;     // slots of a lane in one ranking
constexpr int kChunkSlots = kThreads * kPasses;
constexpr int64_t kStreamBytes = int64_t(128) << 20;  // results beyond this go past the caches
constexpr int64_t kMaxBlocks = int64_t(1) << 20;      // of a launch

// Ranks the slots [s0, s0 + count) by bucket, count <= kChunkSlots: wave w has R consecutive ones from w R on, 64 at a
// time. Lanes of the same bucket find each other with ballots over the bucket's bits, so a slot's place among the wave's
// earlier ones is a popcount, and a count for each (wave, bucket) in LDS carries it on. counts[w][b]: the wave's slots,
// then (scanned) those of the waves before; total[b]: the chunk's.
struct Ranking {
    int bucket[kPasses], rank[kPasses];
    int R, first;
};
__device__ __forceinline__ void rank_chunk(const int32_t* ids, int64_t s0, int count, int E, int* counts, int* total,
                                           Ranking& k) {
    const int tid = static_cast<int>(threadIdx.x), lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    k.R = (count + kThreads - 1) / kThreads * kWave;
    k.first = wave * k.R;
    const int end = min(count, k.first + k.R);
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
        const int s = k.first + i * kWave + lane;
        const int e = s < end && i * kWave < k.R ? ids[s0 + s] : -1;
        k.bucket[i] = s < end && i * kWave < k.R ? (e >= 0 && e < E ? e : E) : -1;
    }
    const int B = E + 1;
    for (int i = tid; i < kWaves * B; i += kThreads) counts[i] = 0;
    __syncthreads();
    const int bits = 32 - __builtin_clz(E);  // of the largest bucket, E
    const uint64_t below = (uint64_t{1} << lane) - 1;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
        k.rank[i] = 0;
        if (i * kWave >= k.R || k.first + i * kWave >= end) continue;  // uniform
        const bool valid = k.bucket[i] >= 0;
        uint64_t same = __ballot(valid);
        for (int b = 0; b < bits; ++b) {
            const bool bit = (k.bucket[i] >> b) & 1;
            const uint64_t m = __ballot(bit);
            same &= bit ? m : ~m;
        }
        const int before = __popcll(same & below);
        if (valid) {
            k.rank[i] = counts[wave * B + k.bucket[i]] + before;
            // the bucket's first lane advances the count; every lane's read above is issued first
            if (before == 0) counts[wave * B + k.bucket[i]] += __popcll(same);
        }
    }
    __syncthreads();
    for (int b = tid; b < B; b += kThreads) {
        int sum = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const int c = counts[w * B + b];
            counts[w * B + b] = sum;
            sum += c;
        }
        total[b] = sum;
    }
    __syncthreads();
}

// Exclusive sums over the buckets, by the first 5 waves; `part`: LDS of 8 ints. Every thread calls it; it ends with a
// barrier.
__device__ __forceinline__ void scan_buckets(const int* total, int B, int* start, int* part) {
    const int tid = static_cast<int>(threadIdx.x), lane = lane_id(), wave = tid / kWave;
    const int v = tid < B ? total[tid] : 0;
    int incl = v;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const int o = __shfl_up(incl, d, kWave);
        if (lane >= d) incl += o;
    }
    if (wave < 8 && lane == kWave - 1) part[wave] = incl;
    __syncthreads();
    if (tid < B) {
        int carry = 0;
        for (int w = 0; w < wave; ++w) carry += part[w];
        start[tid] = carry + incl - v;
    }
    __syncthreads();
}

// Slots of a chunk, whole tokens, and chunks
struct Chunks {
    int64_t tokens, count;
};
__host__ __device__ __forceinline__ Chunks chunks_of(int64_t T, int K) {
    const int64_t tokens = kChunkSlots / K;  // K <= E <= 256
    return Chunks{tokens, (T + tokens - 1) / tokens};
}

// One chunk a workgroup: ranks[s] within the chunk, and the chunk's counts
__global__ __launch_bounds__(kThreads) void sort_count_kernel(SortArgs a) {
    __shared__ int counts[kWaves * kBuckets], total[kBuckets];
    const Chunks c = chunks_of(a.T, a.K);
    const int64_t s0 = static_cast<int64_t>(blockIdx.x) * c.tokens * a.K;
    const int count = static_cast<int>(min(c.tokens * a.K, a.T * a.K - s0));
    Ranking k;
    rank_chunk(a.ids, s0, count, a.E, counts, total, k);
    const int B = a.E + 1, lane = lane_id(), wave = static_cast<int>(threadIdx.x) / kWave;
    int32_t* ranks = a.scratch + c.count * B;
#pragma unroll
    for (int i = 0; i < kPasses; ++i)
        if (k.bucket[i] >= 0)
            ranks[s0 + k.first + i * kWave + lane] = counts[wave * B + k.bucket[i]] + k.rank[i];
    for (int b = static_cast<int>(threadIdx.x); b < B; b += kThreads)
        a.scratch[static_cast<int64_t>(blockIdx.x) * B + b] = total[b];
}

// Bytes of a row copied to up to 16 places by one wave: 16 a lane and step, 4 steps' loads first. The last step of a row
// that is no multiple of 16 long begins 16 before its end; shorter rows go byte by byte.
template <bool NT>
__device__ __forceinline__ void copy_row(const char* src, char* rows, int64_t row_bytes, const int (&place)[16], int n) {
    constexpr int kBatch = 4;
    const int lane = lane_id();
    if (row_bytes < 16) {
        const char v = lane < row_bytes ? src[lane] : 0;
#pragma unroll
        for (int k = 0; k < 16; ++k)
            if (k < n && lane < row_bytes)
                rows[(place[k] >= 0 ? place[k] : ~place[k]) * row_bytes + lane] = place[k] >= 0 ? v : 0;
        return;
    }
    for (int64_t b0 = 0; b0 < row_bytes; b0 += kBatch * kWave * 16) {
        u32x4 v[kBatch];
        int64_t at[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            at[u] = b0 + (u * kWave + lane) * 16;
            v[u] = *reinterpret_cast<const u32x4_any*>(src + min(at[u], row_bytes - 16));
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            if (k >= n) continue;
            char* dst = rows + (place[k] >= 0 ? place[k] : ~place[k]) * row_bytes;
#pragma unroll
            for (int u = 0; u < kBatch; ++u)
                if (at[u] < row_bytes)
                    store16<NT>(dst + min(at[u], row_bytes - 16), place[k] >= 0 ? v[u] : u32x4{0, 0, 0, 0});
        }
    }
}

// The places of a chunk's picks and the copies of its tokens. SINGLE: every workgroup ranks all slots (one chunk) for
// itself, one launch; else the ranks and counts come from sort_count_kernel. Workgroup b of `per` for a chunk copies the
// chunk's tokens [b tokens / per, (b + 1) tokens / per).
template <bool SINGLE, bool NT>
__global__ __launch_bounds__(kThreads) void sort_copy_kernel(SortArgs a, int per) {
    __shared__ int counts[kWaves * kBuckets], total[kBuckets], start[kBuckets], part[8];
    __shared__ int place[SINGLE ? kChunkSlots : 1];
    const int tid = static_cast<int>(threadIdx.x), lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int B = a.E + 1;
    const Chunks c = chunks_of(a.T, a.K);
    const int64_t chunk = static_cast<int64_t>(blockIdx.x) / per;
    const int piece = static_cast<int>(blockIdx.x) % per;
    const int64_t t0 = chunk * c.tokens, tokens = min(c.tokens, a.T - t0);
    const int64_t first = t0 + tokens * piece / per, last = t0 + tokens * (piece + 1) / per;
    const int32_t* ranks = a.scratch + c.count * B;
    if (SINGLE) {
        Ranking k;
        rank_chunk(a.ids, 0, static_cast<int>(a.T * a.K), a.E, counts, total, k);
        scan_buckets(total, B, start, part);
#pragma unroll
        for (int i = 0; i < kPasses; ++i)
            if (k.bucket[i] >= 0) {
                const int p = start[k.bucket[i]] + counts[wave * B + k.bucket[i]] + k.rank[i];
                place[k.first + i * kWave + lane] = k.bucket[i] < a.E ? p : ~p;
            }
        __syncthreads();
    } else {
        // column sums of the counts over all chunks (total) and over those before this one (kept in counts)
        for (int b = tid; b < B; b += kThreads) {
            int sum = 0, before = 0;
#pragma unroll 8
            for (int64_t i = 0; i < c.count; ++i) {
                const int v = a.scratch[i * B + b];
                before += i < chunk ? v : 0;
                sum += v;
            }
            total[b] = sum;
            counts[b] = before;
        }
        __syncthreads();
        scan_buckets(total, B, start, part);
    }
    if (blockIdx.x == 0)
        for (int b = tid; b < B; b += kThreads) a.offsets[b] = start[b];
    const int64_t row_bytes = static_cast<int64_t>(a.H) * a.bytes;
    for (int64_t t = first + wave; t < last; t += kWaves) {
        const char* src = static_cast<const char*>(a.x) + t * a.ldx * a.bytes;
        const float scale = a.scale ? a.scale[t] : 0.0f;
        for (int k0 = 0; k0 < a.K; k0 += 16) {
            const int n = min(16, a.K - k0);
            int p[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                if (k >= n) continue;
                const int64_t s = t * a.K + k0 + k;
                if (SINGLE) {
                    p[k] = place[s];
                } else {
                    const int e = a.ids[s], b = e >= 0 && e < a.E ? e : a.E;
                    const int at = start[b] + counts[b] + ranks[s];
                    p[k] = b < a.E ? at : ~at;
                }
            }
            if (lane == 0) {
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    if (k >= n) continue;
                    a.position[t * a.K + k0 + k] = p[k];
                    if (a.scale) a.row_scale[p[k] >= 0 ? p[k] : ~p[k]] = p[k] >= 0 ? scale : 0.0f;
                }
            }
            copy_row<NT>(src, static_cast<char*>(a.rows), row_bytes, p, n);
        }
    }
}

__device__ __forceinline__ float load_weight(const void* w, int64_t at, int type) {
    if (type == MOE_DT_FLOAT32) return static_cast<const float*>(w)[at];
    const uint16_t b = static_cast<const uint16_t*>(w)[at];
    return type == MOE_DT_FLOAT16 ? Half::load(b) : Bf16::load(b);
}
__device__ __forceinline__ void store_weight(void* w, int64_t at, int type, float v) {
    if (type == MOE_DT_FLOAT32) static_cast<float*>(w)[at] = v;
    else static_cast<uint16_t*>(w)[at] = type == MOE_DT_FLOAT16 ? Half::store(v) : Bf16::store(v);
}

constexpr int kUnsortThreads = 256;

// A thread has V values of a token; up to 8 rows are loaded before they are added, in ascending k
template <typename T, int V>
__global__ __launch_bounds__(kUnsortThreads) void unsort_kernel(UnsortArgs a) {
    using Bits = typename T::Bits;
    constexpr int kBatch = 8;
    const int steps = (a.H + V - 1) / V;
    const int64_t work = a.T * steps;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kUnsortThreads + threadIdx.x; i < work;
         i += static_cast<int64_t>(gridDim.x) * kUnsortThreads) {
        const int64_t t = i / steps;
        const int col = step_at<V>(static_cast<int>(i - t * steps) * V, a.H).at;
        float y[V] = {};
        for (int k0 = 0; k0 < a.K; k0 += kBatch) {
            RawRow<T, V> v[kBatch];
            float w[kBatch];
            bool live[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int p = k0 + u < a.K ? a.position[t * a.K + k0 + u] : -1;
                live[u] = p >= 0 && p < a.R;
                if (!live[u]) continue;
                v[u].load(static_cast<const Bits*>(a.rows) + static_cast<int64_t>(p) * a.H + col);
                w[u] = a.weights ? load_weight(a.weights, t * a.K + k0 + u, a.weights_type) : 1.0f;
            }
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                if (!live[u]) continue;
#pragma unroll
                for (int j = 0; j < V; ++j) y[j] += w[u] * v[u].get(j);
            }
        }
        store_row<T, V>(static_cast<Bits*>(a.y) + t * a.H + col, y);
    }
}

// One or four waves a token; the dot products are added over the lanes and then over the waves in a fixed order
template <typename T, int WAVES, int V, bool NT>
__global__ __launch_bounds__(kUnsortThreads) void unsort_grad_kernel(UnsortArgs a) {
    using Bits = typename T::Bits;
    constexpr int kBatch = 8, kTokens = 4 / WAVES;
    __shared__ float part[4][kBatch];
    const int tid = static_cast<int>(threadIdx.x), wave = tid / kWave, lane = lane_id();
    const int first = (WAVES == 1 ? lane : tid) * V;
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * kTokens + (WAVES == 1 ? wave : 0); t < a.T;
         t += static_cast<int64_t>(gridDim.x) * kTokens) {
        const Bits* gy = static_cast<const Bits*>(a.grad_y) + t * a.ldy;
        for (int k0 = 0; k0 < a.K; k0 += kBatch) {
            float dot[kBatch] = {}, w[kBatch];
            int row[kBatch];  // -1: none, nothing is read or written
            bool live[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int64_t at = t * a.K + k0 + u;
                const int p = k0 + u < a.K ? a.position[at] : 0;
                row[u] = p >= 0 ? p : ~p;
                if (k0 + u >= a.K || row[u] >= a.R) row[u] = -1;
                live[u] = p >= 0 && row[u] >= 0;
                w[u] = !live[u] ? 0.0f : a.weights ? load_weight(a.weights, at, a.weights_type) : 1.0f;
            }
            for (int c = first; c < a.H; c += WAVES * kWave * V) {
                const Step<V> s = step_at<V>(c, a.H);
                RawRow<T, V> d, v[kBatch];
                d.load(gy + s.at);
                if (a.weights) {
#pragma unroll
                    for (int u = 0; u < kBatch; ++u)
                        if (live[u])
                            v[u].load(static_cast<const Bits*>(a.rows) + static_cast<int64_t>(row[u]) * a.H + s.at);
                }
#pragma unroll
                for (int u = 0; u < kBatch; ++u) {
                    if (row[u] < 0) continue;
                    float g[V];
#pragma unroll
                    for (int j = 0; j < V; ++j) g[j] = live[u] ? w[u] * d.get(j) : 0.0f;
                    if (a.weights && live[u]) {
#pragma unroll
                        for (int j = 0; j < V; ++j) dot[u] += j >= s.skip ? d.get(j) * v[u].get(j) : 0.0f;
                    }
                    store_row<T, V, NT>(static_cast<Bits*>(a.y) + static_cast<int64_t>(row[u]) * a.H + s.at, g);
                }
            }
            if (!a.weights) continue;
#pragma unroll
            for (int u = 0; u < kBatch; ++u)
#pragma unroll
                for (int s = kWave / 2; s > 0; s >>= 1) dot[u] += __shfl_xor(dot[u], s, kWave);
            if (WAVES == 1) {
                float v = dot[0];
#pragma unroll
                for (int u = 1; u < kBatch; ++u) v = lane == u ? dot[u] : v;
                if (lane < kBatch && k0 + lane < a.K) store_weight(a.grad_weights, t * a.K + k0 + lane, a.weights_type, v);
            } else {
                if (lane == 0) {
#pragma unroll
                    for (int u = 0; u < kBatch; ++u) part[wave][u] = dot[u];
                }
                __syncthreads();
                if (tid < kBatch && k0 + tid < a.K)
                    store_weight(a.grad_weights, t * a.K + k0 + tid, a.weights_type,
                                 part[0][tid] + part[1][tid] + part[2][tid] + part[3][tid]);
                __syncthreads();
            }
        }
    }
}

template <typename T>
void run_unsort(const UnsortArgs& u, unsigned grid, hipStream_t stream) {
    if (u.H < 8) unsort_kernel<T, 1><<<grid, kUnsortThreads, 0, stream>>>(u);
    else unsort_kernel<T, 8><<<grid, kUnsortThreads, 0, stream>>>(u);
}

template <typename T>
void run_unsort_grad(const UnsortArgs& u, unsigned grid, bool one, bool nt, hipStream_t stream) {
    if (u.H < 8) unsort_grad_kernel<T, 1, 1, false><<<grid, kUnsortThreads, 0, stream>>>(u);
    else if (one && nt) unsort_grad_kernel<T, 1, 8, true><<<grid, kUnsortThreads, 0, stream>>>(u);
    else if (one) unsort_grad_kernel<T, 1, 8, false><<<grid, kUnsortThreads, 0, stream>>>(u);
    else if (nt) unsort_grad_kernel<T, 4, 8, true><<<grid, kUnsortThreads, 0, stream>>>(u);
    else unsort_grad_kernel<T, 4, 8, false><<<grid, kUnsortThreads, 0, stream>>>(u);
}

}  // namespace

// chunks' counts [chunks][E + 1], ranks [T K]
size_t sort_scratch_bytes(int64_t T, int E, int K) {
    if (T * K <= kChunkSlots) return 0;
    return static_cast<size_t>(chunks_of(T, K).count * (E + 1) + T * K) * sizeof(int32_t);
}

hipError_t launch_sort(const SortArgs& s, hipStream_t stream) {
    const bool nt = s.T * s.K * s.H * s.bytes > kStreamBytes;
    if (s.T * s.K <= kChunkSlots) {
        TraceScope trace("moe_sort_rows", stream);
        const int64_t most = (s.T + kWaves - 1) / kWaves;  // workgroups that have tokens
        const int per = static_cast<int>(most < 1 ? 1 : most < 256 ? most : 256);
        if (nt) sort_copy_kernel<true, true><<<per, kThreads, 0, stream>>>(s, per);
        else sort_copy_kernel<true, false><<<per, kThreads, 0, stream>>>(s, per);
        return hipGetLastError();
    }
    const Chunks c = chunks_of(s.T, s.K);
    {
        TraceScope trace("moe_sort_count", stream);
        sort_count_kernel<<<static_cast<unsigned>(c.count), kThreads, 0, stream>>>(s);
    }
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    TraceScope trace("moe_sort_rows", stream);
    const int per = static_cast<int>(c.count < 512 ? (512 + c.count - 1) / c.count : 1);
    const unsigned grid = static_cast<unsigned>(c.count * per);
    if (nt) sort_copy_kernel<false, true><<<grid, kThreads, 0, stream>>>(s, per);
    else sort_copy_kernel<false, false><<<grid, kThreads, 0, stream>>>(s, per);
    return hipGetLastError();
}

hipError_t launch_unsort(const UnsortArgs& u, hipStream_t stream) {
    TraceScope trace("moe_unsort_rows", stream);
    const int64_t steps = u.H < 8 ? u.H : (u.H + 7) / 8, blocks = (u.T * steps + kUnsortThreads - 1) / kUnsortThreads;
    const unsigned grid = static_cast<unsigned>(blocks < kMaxBlocks ? blocks : kMaxBlocks);
    if (u.type == MOE_DT_FLOAT32) run_unsort<F32>(u, grid, stream);
    else if (u.type == MOE_DT_FLOAT16) run_unsort<Half>(u, grid, stream);
    else run_unsort<Bf16>(u, grid, stream);
    return hipGetLastError();
}

hipError_t launch_unsort_grad(const UnsortArgs& u, hipStream_t stream) {
    TraceScope trace("moe_unsort_grad", stream);
    const bool one = u.T >= 2048 || u.H < 8;  // a wave a token once that gives every SIMD two waves
    const bool nt = u.R * u.H * (u.type == MOE_DT_FLOAT32 ? 4 : 2) > kStreamBytes;
    const int64_t blocks = one ? (u.T + 3) / 4 : u.T;
    const unsigned grid = static_cast<unsigned>(blocks < kMaxBlocks ? blocks : kMaxBlocks);
    if (u.type == MOE_DT_FLOAT32) run_unsort_grad<F32>(u, grid, one, nt, stream);
    else if (u.type == MOE_DT_FLOAT16) run_unsort_grad<Half>(u, grid, one, nt, stream);
    else run_unsort_grad<Bf16>(u, grid, one, nt, stream);
    return hipGetLastError();
}

}  // namespace moe
