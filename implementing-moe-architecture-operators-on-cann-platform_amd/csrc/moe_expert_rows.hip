// moe_expert_rows.hip -- MoePermute, MoeUnpermute and MoeUnpermuteGrad for gfx950: tokens sorted by expert, and back.
//
// The T K picks (token t, k) are sorted by expert, those of one expert in the order of their slots t K + k, and token
// t's row is copied to the places of its picks. Picks of no expert stand behind the others, in slot order too, with
// zero rows; position[t, k] is a pick's place p, or -1 - p of a pick of no expert, so every row has exactly one pick.
//   back       y[t] = sum_k weights[t, k] rows[position[t, k]], fp32 sums in ascending k
//   gradients  of rows: weights[t, k] grad_y[t] at position[t, k] (zeros for a pick of no expert); of weights[t, k]:
//              <grad_y[t], rows[position[t, k]]>; the gradient of MoePermute is the way back without weights
//   any positions: a row's gradient is the sum over the picks that name it, in ascending order, so every row's picks
//              are found first (lists by atomic exchange, whose order decides nothing)
// Memory bounds all three: a token's row is read once and its K copies are written, or the other way round; a wave
// works on one token, so its picks' places and weights are read once and stand in scalar registers. Sorting has no
// atomics: a pick's place is offsets[expert] + the expert's picks in earlier chunks + its rank in its chunk.
//   T = 16384, H = 2048, K = 6, E = 64, fp16/bf16: sorting 5.0 + 85 us, 5.2 TB/s over both; back 78 us, 6.0 TB/s (with
//   the places read by every thread 108); gradient 205 us, 4.3 TB/s; of any positions 192
//   T = 1021, H = 1057, K = 8, E = 256: sorting 16 us (one launch), back 8, gradient 12.5 (rows on odd addresses: 12 at
//   1056), of any positions 20
#include "moe_ops.h"
#include "moe_rows.h"

namespace moe {

namespace {

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / kWave;
constexpr int kCopyThreads = 256;
constexpr int kBuckets = 257;            // 256 experts and the picks of none
constexpr int kSingleSlots = 8 * kSortThreads;
constexpr int64_t kStreamBytes = int64_t(128) << 20;  // beyond this rows go past the caches
constexpr int64_t kMaxBlocks = int64_t(1) << 20;      // of a launch

// Ranks `count` slots, at most 64 PASSES a wave, by bucket: wave w has R consecutive ones from w R on, 64 at a time.
// Lanes of the same bucket find each other with ballots over the bucket's bits, so a slot's place among the wave's
// earlier ones is a popcount, and a count for each (wave, bucket) in LDS carries it on. counts[w][b]: in the end the
// slots of b in the waves before w; total[b]: all of them.
template <int PASSES>
struct Ranking {
    int bucket[PASSES], rank[PASSES];  // bucket -1: no slot
    int first, R;
};
template <int PASSES>
__device__ __forceinline__ void rank_slots_of(const int32_t* ids, int count, int E, int* counts, int* total,
                                              Ranking<PASSES>& k) {
    const int tid = static_cast<int>(threadIdx.x), lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    k.R = (count + kSortThreads - 1) / kSortThreads * kWave;
    k.first = wave * k.R;
    const int end = min(count, k.first + k.R);
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int s = k.first + i * kWave + lane;
        const int e = s < end ? ids[s] : -1;
        k.bucket[i] = s >= end ? -1 : e >= 0 && e < E ? e : E;
    }
    const int B = E + 1;
    for (int i = tid; i < kSortWaves * B; i += kSortThreads) counts[i] = 0;
    __syncthreads();
    const int bits = 32 - __builtin_clz(E);  // of the largest bucket, E
    const uint64_t below = (uint64_t{1} << lane) - 1;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        k.rank[i] = 0;
        if (k.first + i * kWave >= end) continue;  // uniform
        const bool valid = k.bucket[i] >= 0;
        uint64_t same = __ballot(valid);
        for (int b = 0; b < bits; ++b) {
            const bool bit = (k.bucket[i] >> b) & 1;
            const uint64_t m = __ballot(bit);
            same &= bit ? m : ~m;
        }
        const int before = __popcll(same & below);
        int* const count_of = counts + wave * B + (valid ? k.bucket[i] : 0);
        const int had = *count_of;
        k.rank[i] = had + before;
        // the bucket's first lane advances the count, when every lane has read it and before any reads it again
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (valid && before == 0) *count_of = had + __popcll(same);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    __syncthreads();
    for (int b = tid; b < B; b += kSortThreads) {
        int sum = 0;
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) {
            const int c = counts[w * B + b];
            counts[w * B + b] = sum;
            sum += c;
        }
        total[b] = sum;
    }
    __syncthreads();
}

// start[b]: the experts' exclusive sums, and of the picks of none all experts'. By the first 256 threads; every thread
// calls it, and it ends with a barrier.
__device__ __forceinline__ void scan_buckets(const int* total, int E, int* start) {
    __shared__ int part[4];
    const int tid = static_cast<int>(threadIdx.x), lane = lane_id(), wave = tid / kWave;
    const int v = tid < E ? total[tid] : 0;
    int incl = v;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const int o = __shfl_up(incl, d, kWave);
        if (lane >= d) incl += o;
    }
    if (wave < 4 && lane == kWave - 1) part[wave] = incl;
    __syncthreads();
    if (tid < E) {
        for (int w = 0; w < wave; ++w) incl += part[w];
        start[tid] = incl - v;
        if (tid == E - 1) start[E] = incl;
    }
    __syncthreads();
}

// Whole tokens of a chunk, whose picks one workgroup ranks, and chunks: 1024 picks each, 4096 from 2^18 of them on
struct Chunks {
    int tokens, slots;
    int64_t count;
};
__host__ __device__ __forceinline__ Chunks chunks_of(int64_t T, int K) {
    const int slots = T * K < int64_t(1) << 18 ? kSortThreads : 4 * kSortThreads;
    const int tokens = slots / K;  // K <= 256
    return Chunks{tokens, slots, (T + tokens - 1) / tokens};
}

// One chunk a workgroup: each slot's rank within the chunk, and the chunk's counts
template <int PASSES>
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(SortArgs a) {
    __shared__ int counts[kSortWaves * kBuckets], total[kBuckets];
    const Chunks c = chunks_of(a.T, a.K);
    const int64_t s0 = static_cast<int64_t>(blockIdx.x) * c.tokens * a.K;
    const int count = static_cast<int>(min(static_cast<int64_t>(c.tokens) * a.K, a.T * a.K - s0));
    Ranking<PASSES> k;
    rank_slots_of<PASSES>(a.ids + s0, count, a.E, counts, total, k);
    const int B = a.E + 1, lane = lane_id(), wave = static_cast<int>(threadIdx.x) / kWave;
    int32_t* ranks = a.scratch + c.count * B;
#pragma unroll
    for (int i = 0; i < PASSES; ++i)
        if (k.bucket[i] >= 0)
            ranks[s0 + k.first + i * kWave + lane] = counts[wave * B + k.bucket[i]] + k.rank[i];
    for (int b = static_cast<int>(threadIdx.x); b < B; b += kSortThreads)
        a.scratch[static_cast<int64_t>(blockIdx.x) * B + b] = total[b];
}

// Bytes of a row copied to up to 16 places by one wave: 16 a lane and step, 4 steps' loads first. The last step of a
// row that is no multiple of 16 long begins 16 before its end; shorter rows go byte by byte.
template <bool NT>
__device__ __forceinline__ void copy_row(const char* src, char* rows, int64_t row_bytes, const int (&place)[16],
                                         int n) {
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

// A token's picks, 16 at a time: their places written down and its row copied there by the wave. place(k): of pick k.
template <bool NT, typename F>
__device__ __forceinline__ void copy_token(const SortArgs& a, int64_t t, F&& place) {
    const int64_t row_bytes = static_cast<int64_t>(a.H) * a.bytes;
    const char* src = static_cast<const char*>(a.x) + t * a.ldx * a.bytes;
    for (int k0 = 0; k0 < a.K; k0 += 16) {
        const int n = min(16, a.K - k0), lane = lane_id();
        const int mine = lane < n ? place(k0 + lane) : 0;
        if (lane < n) {
            a.position[t * a.K + k0 + lane] = mine;
            if (a.scale) a.row_scale[mine >= 0 ? mine : ~mine] = mine >= 0 ? a.scale[t] : 0.0f;
        }
        int p[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) p[k] = __builtin_amdgcn_readlane(mine, k);
        copy_row<NT>(src, static_cast<char*>(a.rows), row_bytes, p, n);
    }
}

// Few picks, one launch: every workgroup ranks all of them for itself and copies its share of the tokens
template <int PASSES>
__global__ __launch_bounds__(kSortThreads) void sort_single_kernel(SortArgs a) {
    __shared__ int counts[kSortWaves * kBuckets], total[kBuckets], start[kBuckets];
    __shared__ int places[PASSES * kSortThreads];
    const int tid = static_cast<int>(threadIdx.x), lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int B = a.E + 1, S = static_cast<int>(a.T) * a.K;
    Ranking<PASSES> k;
    rank_slots_of<PASSES>(a.ids, S, a.E, counts, total, k);
    scan_buckets(total, a.E, start);
#pragma unroll
    for (int i = 0; i < PASSES; ++i)
        if (k.bucket[i] >= 0) {
            const int p = start[k.bucket[i]] + counts[wave * B + k.bucket[i]] + k.rank[i];
            places[k.first + i * kWave + lane] = k.bucket[i] < a.E ? p : ~p;
        }
    __syncthreads();
    if (blockIdx.x == 0)
        for (int b = tid; b < B; b += kSortThreads) a.offsets[b] = start[b];
    for (int64_t t = static_cast<int64_t>(wave) * gridDim.x + blockIdx.x; t < a.T;
         t += static_cast<int64_t>(kSortWaves) * gridDim.x)
        copy_token<false>(a, t, [&](int k) { return places[t * a.K + k]; });
}

// The copies from sort_count_kernel's ranks and counts. Workgroup b of `per` for a chunk adds the counts of all chunks
// and of those before its own, and copies the chunk's tokens [b tokens / per, (b + 1) tokens / per).
template <bool NT>
__global__ __launch_bounds__(kCopyThreads) void sort_copy_kernel(SortArgs a, int per) {
    constexpr int kWaves = kCopyThreads / kWave;
    __shared__ int total[kBuckets], before[kBuckets], start[kBuckets];
    __shared__ int part[2][kCopyThreads];
    const int tid = static_cast<int>(threadIdx.x), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int B = a.E + 1;
    const Chunks c = chunks_of(a.T, a.K);
    const int64_t chunk = static_cast<int64_t>(blockIdx.x) / per;
    const int piece = static_cast<int>(blockIdx.x) % per;
    const int64_t t0 = chunk * c.tokens, tokens = min(static_cast<int64_t>(c.tokens), a.T - t0);
    const int64_t first = t0 + tokens * piece / per, last = t0 + tokens * (piece + 1) / per;
    const int32_t* ranks = a.scratch + c.count * B;
    // `lanes` threads for each of as many buckets as that leaves, every lanes-th chunk each; their sums meet in LDS
    const int width = min(B, kCopyThreads), lanes = kCopyThreads / width, own = tid % width, j = tid / width;
    for (int b0 = 0; b0 < B; b0 += width) {
        const int b = b0 + own;
        int sum = 0, pre = 0;
        if (b < B && j < lanes) {
#pragma unroll 8
            for (int64_t i = j; i < c.count; i += lanes) {
                const int v = a.scratch[i * B + b];
                pre += i < chunk ? v : 0;
                sum += v;
            }
        }
        part[0][tid] = sum;
        part[1][tid] = pre;
        __syncthreads();
        if (j == 0 && b < B) {
            for (int l = 1; l < lanes; ++l) {
                sum += part[0][tid + l * width];
                pre += part[1][tid + l * width];
            }
            total[b] = sum;
            before[b] = pre;
        }
        __syncthreads();
    }
    scan_buckets(total, a.E, start);
    if (blockIdx.x == 0)
        for (int b = tid; b < B; b += kCopyThreads) a.offsets[b] = start[b];
    for (int64_t t = first + wave; t < last; t += kWaves)
        copy_token<NT>(a, t, [&](int k) {
            const int64_t s = t * a.K + k;
            const int e = a.ids[s], b = e >= 0 && e < a.E ? e : a.E;
            const int p = start[b] + before[b] + ranks[s];
            return b < a.E ? p : ~p;
        });
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

// A wave has STEPS steps of V values a lane of a token; up to 8 rows are loaded before they are added, in ascending k.
// The picks' places and weights are read once, a pick a lane.
template <typename T, int V, int STEPS, bool NT>
__global__ __launch_bounds__(kUnsortThreads) void unsort_kernel(UnsortArgs a) {
    using Bits = typename T::Bits;
    constexpr int kBatch = 8, kSpan = STEPS * kWave * V, kWaves = kUnsortThreads / kWave;
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const int spans = (a.H + kSpan - 1) / kSpan;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kWaves + wave; i < a.T * spans;
         i += static_cast<int64_t>(gridDim.x) * kWaves) {
        const int64_t t = i / spans;
        Step<V> at[STEPS];
#pragma unroll
        for (int c = 0; c < STEPS; ++c)
            at[c] = step_at<V>(static_cast<int>(i - t * spans) * kSpan + (c * kWave + lane) * V, a.H);
        float y[STEPS][V] = {};
        for (int k0 = 0; k0 < a.K; k0 += kBatch) {
            int p = -1;
            float w = 0.0f;
            if (lane < kBatch && k0 + lane < a.K) {
                p = a.position[t * a.K + k0 + lane];
                if (p >= a.R) p = -1;
                if (p >= 0) w = a.weights ? load_weight(a.weights, t * a.K + k0 + lane, a.weights_type) : 1.0f;
            }
            RawRow<T, V> v[kBatch][STEPS];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int row = __builtin_amdgcn_readlane(p, u);
                if (row < 0) continue;
                const Bits* src = static_cast<const Bits*>(a.rows) + static_cast<int64_t>(row) * a.H;
#pragma unroll
                for (int c = 0; c < STEPS; ++c) v[u][c].template load<NT>(src + at[c].at);
            }
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                if (__builtin_amdgcn_readlane(p, u) < 0) continue;
                const float weight = of_lane(w, u);
#pragma unroll
                for (int c = 0; c < STEPS; ++c)
#pragma unroll
                    for (int j = 0; j < V; ++j) y[c][j] += weight * v[u][c].get(j);
            }
        }
#pragma unroll
        for (int c = 0; c < STEPS; ++c)
            if (at[c].live) store_row<T, V>(static_cast<Bits*>(a.y) + t * a.H + at[c].at, y[c]);
    }
}

// Lists of the picks that name a row: heads[row], then links[pick]; -1 ends one
__global__ __launch_bounds__(kUnsortThreads) void unsort_heads_kernel(UnsortArgs a) {
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kUnsortThreads + threadIdx.x; i < a.R;
         i += static_cast<int64_t>(gridDim.x) * kUnsortThreads)
        a.heads[i] = -1;
}
__global__ __launch_bounds__(kUnsortThreads) void unsort_links_kernel(UnsortArgs a) {
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kUnsortThreads + threadIdx.x; i < a.T * a.K;
         i += static_cast<int64_t>(gridDim.x) * kUnsortThreads) {
        const int p = a.position[i];
        if (p >= 0 && p < a.R) a.links[i] = atomicExch(a.heads + p, static_cast<int>(i));
    }
}

// The gradient's rows that not exactly one pick names: zeros, or the picks' sum in ascending order. A wave looks at 8
// rows. It takes up to 64 picks from a row's list and ranks them; for a row of more, which at most every 64th can be,
// it reads all positions again. T = 16384, K = 6, H = 2048, all four launches: pairs of picks 208 us, 64 to a row 1.0
// ms, 65 to a row 9.8, all on one 80.
template <typename T, int V>
__global__ __launch_bounds__(kUnsortThreads) void unsort_rest_kernel(UnsortArgs a) {
    using Bits = typename T::Bits;
    constexpr int kRows = 8, kBatch = 8, kWaves = kUnsortThreads / kWave;
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const int64_t picks = a.T * a.K;
    for (int64_t base = (static_cast<int64_t>(blockIdx.x) * kWaves + wave) * kRows; base < a.R;
         base += static_cast<int64_t>(gridDim.x) * kWaves * kRows) {
        int head = -1;
        bool open = false;
        if (lane < kRows && base + lane < a.R) {
            head = a.heads[base + lane];
            open = head < 0 || a.links[head] >= 0;
        }
        for (uint64_t left = __ballot(open); left != 0; left &= left - 1) {
            const int64_t row = base + __builtin_ctzll(left);
            int pick = __builtin_amdgcn_readlane(head, __builtin_ctzll(left)), mine = 0, n = 0;
            for (; pick >= 0 && n < kWave; ++n) {
                mine = lane == n ? pick : mine;
                pick = __builtin_amdgcn_readfirstlane(a.links[pick]);
            }
            const bool more = pick >= 0;
            int rank = 0;  // of this lane's pick; lanes without one take the places behind
            for (int i = 0; i < n; ++i) rank += __builtin_amdgcn_readlane(mine, i) < mine;
            mine = __builtin_amdgcn_ds_permute((lane < n ? rank : lane) * 4, mine);
            for (int c = 0; c < a.H; c += kWave * V) {
                const Step<V> s = step_repeating<V>(c + lane * V, a.H);
                float y[V] = {};
                // adds the picks of `bits` from the lowest on, 8 loads at a time
                auto add = [&](uint64_t bits, auto&& pick_of) __attribute__((always_inline)) {
                    while (bits != 0) {
                        int64_t at[kBatch];
                        float w[kBatch];
                        RawRow<T, V> d[kBatch];
#pragma unroll
                        for (int u = 0; u < kBatch; ++u) {
                            at[u] = bits != 0 ? pick_of(__builtin_ctzll(bits)) : -1;
                            bits &= bits - 1;
                            if (at[u] < 0) continue;
                            d[u].load(static_cast<const Bits*>(a.grad_y) + at[u] / a.K * a.ldy + s.at);
                            w[u] = a.weights ? load_weight(a.weights, at[u], a.weights_type) : 1.0f;
                        }
#pragma unroll
                        for (int u = 0; u < kBatch; ++u) {
                            if (at[u] < 0) continue;
#pragma unroll
                            for (int j = 0; j < V; ++j) y[j] += w[u] * d[u].get(j);
                        }
                    }
                };
                if (more) {
                    for (int64_t from = 0; from < picks; from += kWave) {
                        const int p = from + lane < picks ? a.position[from + lane] : -1;
                        add(__ballot(p == row), [&](int bit) { return from + bit; });
                    }
                } else if (n > 0) {
                    add(~uint64_t{0} >> (kWave - n),
                        [&](int bit) { return static_cast<int64_t>(__builtin_amdgcn_readlane(mine, bit)); });
                }
                store_row<T, V>(static_cast<Bits*>(a.y) + row * a.H + s.at, y);
            }
        }
    }
}

// 1, 2 or 4 waves a token, 8 of its rows at a time; the picks' places and weights are read once, a pick a lane. The dot
// products are added over the lanes and then over the waves in a fixed order. ANY: positions that are not MoePermute's;
// the rows that not exactly one pick names are unsort_rest_kernel's.
template <typename T, int WAVES, int V, bool NT, bool ANY>
__global__ __launch_bounds__(kUnsortThreads) void unsort_grad_kernel(UnsortArgs a) {
    using Bits = typename T::Bits;
    constexpr int kBatch = 8, kTokens = kUnsortThreads / (WAVES * kWave);
    __shared__ float part[kUnsortThreads / kWave][kBatch];
    const int tid = static_cast<int>(threadIdx.x), lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave), team = wave / WAVES;
    const int first = wave % WAVES * kWave * V;
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * kTokens; base < a.T;
         base += static_cast<int64_t>(gridDim.x) * kTokens) {
        const bool token = base + team < a.T;
        const int64_t t = token ? base + team : a.T - 1;
        const Bits* gy = static_cast<const Bits*>(a.grad_y) + t * a.ldy;
        for (int k0 = 0; k0 < a.K; k0 += kBatch) {
            // of pick k0 + lane: its row (past the rows: none, nothing is read or written), whether an expert has it
            int row = -1;
            bool live = false, sole = true;
            float w = 0.0f;
            if (token && lane < kBatch && k0 + lane < a.K) {
                const int64_t at = t * a.K + k0 + lane;
                const int p = a.position[at];
                row = p >= 0 ? p : ~p;
                if (row >= a.R) row = -1;
                live = p >= 0 && row >= 0;
                if (ANY) sole = live && a.heads[row] == at && a.links[at] < 0;
                if (live) w = a.weights ? load_weight(a.weights, at, a.weights_type) : 1.0f;
            }
            const uint64_t lives = __ballot(live), soles = __ballot(sole);
            float dot[kBatch] = {};
            // a wave's lanes go through this together, since readlane is for active ones
            for (int c = first; c < a.H; c += WAVES * kWave * V) {
                const Step<V> s = step_repeating<V>(c + lane * V, a.H);
                RawRow<T, V> d, v[kBatch];
                d.load(gy + s.at);
                if (a.weights) {
#pragma unroll
                    for (int u = 0; u < kBatch; ++u)
                        if (lives >> u & 1) {
                            const int64_t from = __builtin_amdgcn_readlane(row, u);
                            v[u].template load<NT>(static_cast<const Bits*>(a.rows) + from * a.H + s.at);
                        }
                }
#pragma unroll
                for (int u = 0; u < kBatch; ++u) {
                    const int to = __builtin_amdgcn_readlane(row, u);
                    const bool on = lives >> u & 1;
                    if (ANY ? !on : to < 0) continue;
                    const float weight = of_lane(w, u);
                    float g[V];
#pragma unroll
                    for (int j = 0; j < V; ++j) g[j] = on ? weight * d.get(j) : 0.0f;
                    if (a.weights && on) {
#pragma unroll
                        for (int j = 0; j < V; ++j) dot[u] += j >= s.skip ? d.get(j) * v[u].get(j) : 0.0f;
                    }
                    if (!ANY || soles >> u & 1)
                        store_row<T, V, NT>(static_cast<Bits*>(a.y) + static_cast<int64_t>(to) * a.H + s.at, g);
                }
            }
            if (!a.weights) continue;
#pragma unroll
            for (int u = 0; u < kBatch; ++u) dot[u] = wave_sum(dot[u]);
            float v = dot[0];
#pragma unroll
            for (int u = 1; u < kBatch; ++u) v = lane == u ? dot[u] : v;
            if (WAVES > 1) {
                if (lane < kBatch) part[wave][lane] = v;
                __syncthreads();
                if (lane < kBatch) {
                    v = part[team * WAVES][lane];
#pragma unroll
                    for (int x = 1; x < WAVES; ++x) v += part[team * WAVES + x][lane];
                }
                __syncthreads();
            }
            if (token && wave % WAVES == 0 && lane < kBatch && k0 + lane < a.K)
                store_weight(a.grad_weights, t * a.K + k0 + lane, a.weights_type, v);
        }
    }
}

template <typename T, int V, int STEPS, bool NT>
void run_unsort(const UnsortArgs& u, hipStream_t stream) {
    constexpr int kWaves = kUnsortThreads / kWave;
    const int64_t spans = (u.H + STEPS * kWave * V - 1) / (STEPS * kWave * V);
    const int64_t blocks = (u.T * spans + kWaves - 1) / kWaves;
    unsort_kernel<T, V, STEPS, NT>
        <<<static_cast<unsigned>(blocks < kMaxBlocks ? blocks : kMaxBlocks), kUnsortThreads, 0, stream>>>(u);
}
template <typename T>
void run_unsort_any(const UnsortArgs& u, hipStream_t stream) {
    const bool nt = u.R * u.H * static_cast<int64_t>(sizeof(typename T::Bits)) > kStreamBytes;
    const bool two = u.T >= 2048 && u.H > 512;
    if (u.H < 8) run_unsort<T, 1, 1, false>(u, stream);
    else if (two) nt ? run_unsort<T, 8, 2, true>(u, stream) : run_unsort<T, 8, 2, false>(u, stream);
    else nt ? run_unsort<T, 8, 1, true>(u, stream) : run_unsort<T, 8, 1, false>(u, stream);
}

template <typename T, int WAVES, int V>
void run_unsort_grad(const UnsortArgs& u, hipStream_t stream) {
    constexpr int kTokens = kUnsortThreads / (WAVES * kWave);
    const int64_t blocks = (u.T + kTokens - 1) / kTokens;
    const unsigned grid = static_cast<unsigned>(blocks < kMaxBlocks ? blocks : kMaxBlocks);
    const bool nt = u.R * u.H * static_cast<int64_t>(sizeof(typename T::Bits)) > kStreamBytes;
    if (u.heads) {
        if (nt) unsort_grad_kernel<T, WAVES, V, true, true><<<grid, kUnsortThreads, 0, stream>>>(u);
        else unsort_grad_kernel<T, WAVES, V, false, true><<<grid, kUnsortThreads, 0, stream>>>(u);
    } else {
        if (nt) unsort_grad_kernel<T, WAVES, V, true, false><<<grid, kUnsortThreads, 0, stream>>>(u);
        else unsort_grad_kernel<T, WAVES, V, false, false><<<grid, kUnsortThreads, 0, stream>>>(u);
    }
}
unsigned threads_grid(int64_t items, int each) {
    const int64_t blocks = (items + each - 1) / each;
    return static_cast<unsigned>(blocks < kMaxBlocks ? blocks : kMaxBlocks);
}
// A wave a token once that gives every SIMD two of them, or where it has a token's row in one step
template <typename T>
void run_unsort_grad_any(const UnsortArgs& u, hipStream_t stream) {
    if (u.H < 8) run_unsort_grad<T, 1, 1>(u, stream);
    else if (u.T >= 2048 || u.H <= 512) run_unsort_grad<T, 1, 8>(u, stream);
    else if (u.H <= 1024) run_unsort_grad<T, 2, 8>(u, stream);
    else run_unsort_grad<T, 4, 8>(u, stream);
    if (!u.heads) return;
    const unsigned grid = threads_grid(u.R, kUnsortThreads / kWave * 8);
    if (u.H < 8) unsort_rest_kernel<T, 1><<<grid, kUnsortThreads, 0, stream>>>(u);
    else unsort_rest_kernel<T, 8><<<grid, kUnsortThreads, 0, stream>>>(u);
}

}  // namespace

// chunks' counts [chunks][E + 1], ranks [T K]
size_t sort_scratch_bytes(int64_t T, int E, int K) {
    if (T * K <= kSingleSlots) return 0;
    return static_cast<size_t>(chunks_of(T, K).count * (E + 1) + T * K) * sizeof(int32_t);
}

hipError_t launch_sort(const SortArgs& s, hipStream_t stream) {
    const int64_t S = s.T * s.K;
    if (S <= kSingleSlots) {
        TraceScope trace("moe_sort_rows", stream);
        const int grid = static_cast<int>(s.T < 1 ? 1 : s.T < 256 ? s.T : 256);
        if (S <= kSortThreads) sort_single_kernel<1><<<grid, kSortThreads, 0, stream>>>(s);
        else sort_single_kernel<kSingleSlots / kSortThreads><<<grid, kSortThreads, 0, stream>>>(s);
        return hipGetLastError();
    }
    const Chunks c = chunks_of(s.T, s.K);
    {
        TraceScope trace("moe_sort_count", stream);
        if (c.slots == kSortThreads)
            sort_count_kernel<1><<<static_cast<unsigned>(c.count), kSortThreads, 0, stream>>>(s);
        else
            sort_count_kernel<4><<<static_cast<unsigned>(c.count), kSortThreads, 0, stream>>>(s);
    }
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    TraceScope trace("moe_sort_rows", stream);
    // a token a wave, but no more than 2048 workgroups where a chunk has one
    constexpr int kWaves = kCopyThreads / kWave;
    const int64_t most = c.count < 2048 ? 2048 / c.count : 1, want = (c.tokens + kWaves - 1) / kWaves;
    const int per = static_cast<int>(want < most ? want : most);
    const unsigned grid = static_cast<unsigned>(c.count * per);
    if (S * s.H * s.bytes > kStreamBytes) sort_copy_kernel<true><<<grid, kCopyThreads, 0, stream>>>(s, per);
    else sort_copy_kernel<false><<<grid, kCopyThreads, 0, stream>>>(s, per);
    return hipGetLastError();
}

hipError_t launch_unsort(const UnsortArgs& u, hipStream_t stream) {
    TraceScope trace("moe_unsort_rows", stream);
    if (u.type == MOE_DT_FLOAT32) run_unsort_any<F32>(u, stream);
    else if (u.type == MOE_DT_FLOAT16) run_unsort_any<Half>(u, stream);
    else run_unsort_any<Bf16>(u, stream);
    return hipGetLastError();
}

hipError_t launch_unsort_grad(const UnsortArgs& u, hipStream_t stream) {
    TraceScope trace("moe_unsort_grad", stream);
    if (u.heads) {
        unsort_heads_kernel<<<threads_grid(u.R, kUnsortThreads), kUnsortThreads, 0, stream>>>(u);
        unsort_links_kernel<<<threads_grid(u.T * u.K, kUnsortThreads), kUnsortThreads, 0, stream>>>(u);
    }
    if (u.type == MOE_DT_FLOAT32) run_unsort_grad_any<F32>(u, stream);
    else if (u.type == MOE_DT_FLOAT16) run_unsort_grad_any<Half>(u, stream);
    else run_unsort_grad_any<Bf16>(u, stream);
    return hipGetLastError();
}

}  // namespace moe
