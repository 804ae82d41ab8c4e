// moe_linear_tiled.hip -- the dense product on 256 x 256 tiles, for the sizes that the matrix cores bound.
//
// C[m][n] = sum_k P[m][k] Q[n][k] as in moe_linear.hip, operands that 16-byte copies can read. The main loop is that of
// the expert GEMMs (moe_ffn_tiled.hip, where its choices are measured): 8 waves (2 x 4) of 128 x 64, two LDS slots of
// four 16 KB half tiles (P rows 0-127 and 128-255, two halves of Q rows), a stage of 64 k as two pairs of ticks (LDS
// reads and copies, then 32 MFMAs), waves 4-7 one tick behind waves 0-3, persistent workgroups whose ring runs on
// across tiles. New here: either operand may be stored by k (a half tile is then 64 k x 128 rows and its fragments come
// out of ds_read_b64_tr_b16), k of any length (copies past the end read zeros), tiles in bands of 8 m-tiles (the 32
// workgroups of an XCD then read 8 + 4 panels a stage, not 32 + 1), and the epilogue of moe_gemm.h.
//
// Matrix cores and the clock they leave bound it. T = 16381, H = 2048, N = 2816 SwiGLU bf16: 282-293 us with the
// epilogue, 1290-1340 TFLOP/s (8192^3 by the library: 1413); grad_x of a T = 8192 step 148 us, 1277 TFLOP/s.
// grad_weight there has 176 tiles for 256 CUs and takes 200 us: tiles of 256 x 192 (242 of them) took 170 us where
// these took 177, and 168 to 199 us where these took 137 to 142 on full rounds, so a product is not bound by the CUs it
// leaves idle.
#include "moe_gemm.h"

namespace moe {

namespace {

constexpr int kBM = 256, kBN = 256, kBK = 64;
constexpr int kThreads = 512;
constexpr int kHalfTile = 128 * kBK;          // halfs of a half tile
constexpr int kStageHalfs = 4 * kHalfTile;
constexpr int kEpiBytes = 4096;               // per wave: 16 rows x 64 columns of fp32
constexpr int kLdsBytes = 2 * kStageHalfs * 2 + kThreads / kWave * kEpiBytes;
constexpr int kXcds = 8;
constexpr int kBand = 8;                      // m-tiles of a band
constexpr uint32_t kPastEnd = 0x80000000u;    // a buffer offset past every buffer: the load returns zeros

__device__ __forceinline__ void ring_barrier() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    __builtin_amdgcn_sched_barrier(0);
}

// The lane index read afresh: what is derived from it at a tile change is then not kept in registers through the main
// loop, where accumulators and fragments leave no room.
__device__ __forceinline__ int lane_fresh() {
    int v;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(v));
    return v;
}

struct Tile {
    int m0, n0;
};

// Where a tile's copies come from. Per half tile wave w issues instructions 2 w and 2 w + 1, each 64 granules of 16
// bytes: by rows 8 rows of 8 granules, granule g of row r standing at g ^ ((r >> 1) & 7); by k 4 k of 16 granules (8
// rows each), granule g of k standing at g ^ (2 f(k)), f(k) = (k & 3) | (k >> 3 & 1) << 2. Offsets are relative to the
// tile's first row (by rows) or the stage's first k (by k).
struct CopyPlan {
    uint32_t po[2][2], qo[2][2];  // [half][instruction]
    const uint16_t* pb;
    const uint16_t* qb[2];
};

template <typename T, bool PK, bool QK, bool SWIGLU>
__global__ __launch_bounds__(kThreads) void gemm_tiled_kernel(GemmArgs g, int mtiles, int ntiles) {
    extern __shared__ __align__(16) uint16_t lds[];
    const int tid = static_cast<int>(threadIdx.x), lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int row16 = lane & 15, kg = lane >> 4;
    const int wm = wave >> 2, wn = wave & 3;
    const int nst = max(2, (g.k + kBK - 1) / kBK);  // the ring runs two stages ahead; a second one past k is zeros

    // XCD x has the tiles [x per_xcd, (x + 1) per_xcd), dealt round-robin to its workgroups
    const int total = mtiles * ntiles;
    const int nloc = static_cast<int>(gridDim.x) / kXcds;
    const int x = static_cast<int>(blockIdx.x) % kXcds, li = static_cast<int>(blockIdx.x) / kXcds;
    const int per_xcd = (total + kXcds - 1) / kXcds;
    auto tile_at = [&](int i, Tile& t) __attribute__((always_inline)) -> bool {
        const int loc = li + i * nloc, at = x * per_xcd + loc;
        if (loc >= per_xcd || at >= total) return false;
        const int band = at / (kBand * ntiles), r = at - band * kBand * ntiles;
        const int rows = min(kBand, mtiles - band * kBand);
        const int nt = r / rows;
        t.m0 = __builtin_amdgcn_readfirstlane((band * kBand + r - nt * rows) * kBM);
        t.n0 = __builtin_amdgcn_readfirstlane(nt * (SWIGLU ? kBN / 2 : kBN));
        return true;
    };
    Tile cur;
    if (!tile_at(0, cur)) return;

    // k of the stage that this lane's granule of instruction j holds (by rows: its first of 8)
    auto granule_k = [&](bool by_k, int j, int ln) __attribute__((always_inline)) {
        const int i = wave * 2 + j;
        return by_k ? i * 4 + ln / 16 : ((ln % 8) ^ (((i * 8 + ln / 8) >> 1) & 7)) * 8;
    };
    // operand row (of the half tile) that it starts at
    auto granule_row = [&](bool by_k, int j, int ln) __attribute__((always_inline)) {
        const int i = wave * 2 + j;
        if (!by_k) return i * 8 + ln / 8;
        const int k = i * 4 + ln / 16, f = (k & 3) | (((k >> 3) & 1) << 2);
        return ((ln % 16) ^ (f << 1)) * 8;
    };
    auto make_plan = [&](const Tile& t, CopyPlan& c) __attribute__((always_inline)) {
        const int ln = lane_fresh();
        const uint32_t pp = static_cast<uint32_t>(g.ldp) * 2, qp = static_cast<uint32_t>(g.ldq) * 2;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int pk = granule_k(PK, j, ln), pr = granule_row(PK, j, ln);
            const int qk = granule_k(QK, j, ln), qr = granule_row(QK, j, ln);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = h * 128 + pr;
                const uint32_t po = PK ? pk * pp + (t.m0 + row) * 2u : row * pp + pk * 2u;
                c.po[h][j] = t.m0 + row < g.m ? po : kPastEnd;
                // SwiGLU: half 0 the gate rows, half 1 the up rows of the same columns. Else wave column wn has columns
                // wn * 64 + h * 32 + [0, 32) of half h.
                const int col = SWIGLU ? qr : (qr >> 5) * 64 + h * 32 + (qr & 31);
                const uint32_t up = SWIGLU && QK && h ? static_cast<uint32_t>(g.up) : 0u;
                const uint32_t qo = QK ? qk * qp + (t.n0 + col + up) * 2u : col * qp + qk * 2u;
                c.qo[h][j] = t.n0 + col < g.n ? qo : kPastEnd;
            }
        }
        c.pb = g.p + (PK ? 0 : static_cast<int64_t>(t.m0) * g.ldp);
        c.qb[0] = g.q + (QK ? 0 : static_cast<int64_t>(t.n0) * g.ldq);
        c.qb[1] = c.qb[0] + (SWIGLU && !QK ? static_cast<int64_t>(g.up) * g.ldq : 0);
    };
    // One half tile of stage kc into ring slot q % 2. By rows the k offset is the instruction's scalar one, by k it
    // moves the base, so an operand may be larger than 4 GiB. Granules from k on read zeros.
    const int pgk[2] = {granule_k(PK, 0, lane), granule_k(PK, 1, lane)};
    const int qgk[2] = {granule_k(QK, 0, lane), granule_k(QK, 1, lane)};
    auto copy = [&](bool by_k, const uint16_t* base, int64_t ld, const uint32_t (&off)[2], const int (&gk)[2],
                    uint16_t* s, int kc) __attribute__((always_inline)) {
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint16_t*>(by_k ? base + static_cast<int64_t>(kc) * kBK * ld : base), 0, 0x7fffffff, 0x00020000);
        const int left = g.k - kc * kBK;
#pragma unroll
        for (int j = 0; j < 2; ++j)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                r, (__attribute__((address_space(3))) void*)(s + (wave * 2 + j) * 512), 16,
                static_cast<int>(gk[j] < left ? off[j] : kPastEnd), by_k ? 0 : kc * kBK * 2, 0, 1);
    };
    auto copyP = [&](int q, int h, int kc, const CopyPlan& c) __attribute__((always_inline)) {
        copy(PK, c.pb, g.ldp, c.po[h], pgk, lds + (q & 1) * kStageHalfs + h * kHalfTile, kc);
    };
    auto copyQ = [&](int q, int h, int kc, const CopyPlan& c) __attribute__((always_inline)) {
        copy(QK, c.qb[h], g.ldq, c.qo[h], qgk, lds + (q & 1) * kStageHalfs + (2 + h) * kHalfTile, kc);
    };

    // Fragments of one P half (4 blocks, both 32-k steps) and of both Q halves (2 blocks each)
    using Acc = f32x4[2][4][2];
    s16x8 fp[2][4], fq0[2][2], fq1[2][2];
    const int sw = (row16 >> 1) & 7;
    auto rdP = [&](int q, int h) __attribute__((always_inline)) {
        const uint16_t* s = lds + (q & 1) * kStageHalfs + h * kHalfTile;
        if constexpr (PK) {
            const uint32_t addr[4] = {
                transposed_address(s, wm * 64, lane), transposed_address(s, wm * 64 + 16, lane),
                transposed_address(s, wm * 64 + 32, lane), transposed_address(s, wm * 64 + 48, lane)};
            read_transposed(addr, fp);
        } else {
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    fp[kk][i] = *reinterpret_cast<const s16x8*>(s + (wm * 64 + i * 16 + row16) * kBK +
                                                                (((kk * 4 + kg) ^ sw) * 8));
        }
    };
    auto rdQ = [&](int q, int h, s16x8 (&f)[2][2]) __attribute__((always_inline)) {
        const uint16_t* s = lds + (q & 1) * kStageHalfs + (2 + h) * kHalfTile;
        if constexpr (QK) {
            const uint32_t addr[2] = {transposed_address(s, wn * 32, lane), transposed_address(s, wn * 32 + 16, lane)};
            read_transposed(addr, f);
        } else {
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    f[kk][j] = *reinterpret_cast<const s16x8*>(s + (wn * 32 + j * 16 + row16) * kBK +
                                                               (((kk * 4 + kg) ^ sw) * 8));
        }
    };
    // Ends a memory tick: the fragments are in registers and all but this wave's youngest 8 copies have landed
    auto tick_m = [&]() __attribute__((always_inline)) {
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(8) & 0xf0ffu);
        ring_barrier();
    };
    auto tick_c = [&](Acc& c, bool zero) __attribute__((always_inline)) {
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    c[j >> 1][i][j & 1] = T::mfma(j < 2 ? fq0[kk][j & 1] : fq1[kk][j & 1], fp[kk][i],
                                                  zero && kk == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : c[j >> 1][i][j & 1]);
        ring_barrier();
    };
    // half1 refills the second P half of stage q + 1 (stage kc of c), half2 the other three half tiles of stage q + 2
    auto half1 = [&](Acc (&acc)[2], int q, bool first, int kc, const CopyPlan& c) __attribute__((always_inline)) {
        if (PK || QK) copyP(q + 1, 1, kc, c);  // transposed reads wait for their data: the copies go first
        rdP(q, 0);
        rdQ(q, 0, fq0);
        rdQ(q, 1, fq1);
        if (!PK && !QK) copyP(q + 1, 1, kc, c);
        tick_m();
        tick_c(acc[0], first);
    };
    auto half2 = [&](Acc (&acc)[2], int q, bool first, int kc, const CopyPlan& c) __attribute__((always_inline)) {
        if (!PK) rdP(q, 1);
        copyP(q, 0, kc, c);
        copyQ(q, 0, kc, c);
        copyQ(q, 1, kc, c);
        if (PK) rdP(q, 1);
        tick_m();
        tick_c(acc[1], first);
    };

    // acc[a][b][i][j]: rows a * 128 + wm * 64 + i * 16 + row16, columns of Q half b, 4 consecutive ones from 4 kg on.
    // The 8 blocks of 16 rows share one copy of the epilogue's code: unrolled, its activations are too long for the
    // accumulators to stay in registers.
    auto epilogue = [&](const Acc (&acc)[2], const Tile& t) __attribute__((always_inline)) {
        const int ln = lane_fresh(), row16 = ln & 15, kg = ln >> 4;
        const bool vec = vector_rows(g), lines = whole_lines(g, vec);
        float* stg = reinterpret_cast<float*>(lds + 2 * kStageHalfs) + wave * (kEpiBytes / 4);
        auto put = [&](int i) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < 4; ++j) put_block<4>(stg, row16, kg, j, acc[i >> 2][j >> 1][i & 3][j & 1]);
        };
#pragma unroll 1
        for (int i = 0; i < 8; ++i) {
            switch (i) {
                case 0: put(0); break;
                case 1: put(1); break;
                case 2: put(2); break;
                case 3: put(3); break;
                case 4: put(4); break;
                case 5: put(5); break;
                case 6: put(6); break;
                default: put(7); break;
            }
            store_block<T, SWIGLU, 4>(g, stg, ln, t.m0 + (i >> 2) * 128 + wm * 64 + (i & 3) * 16,
                                      t.n0 + wn * (SWIGLU ? 32 : 64), vec, lines);
        }
    };

    CopyPlan plan;
    make_plan(cur, plan);
#pragma unroll
    for (int st = 0; st < 2; ++st) {
        copyP(st, 0, st, plan);
        copyQ(st, 0, st, plan);
        copyQ(st, 1, st, plan);
        __builtin_amdgcn_sched_barrier(0);
        if (st == 0) copyP(st, 1, st, plan);
        __builtin_amdgcn_sched_barrier(0);  // stage 0 first: the counted wait below covers its first three half tiles
    }
    tick_m();
    int q0 = 0;  // ring index of the tile's first stage
    for (int i = 0;; ++i) {
        Tile nxt = cur;
        const bool has_next = tile_at(i + 1, nxt);
        // the last two stages copy the next tile's first two; after the last tile, stages past k: zeros, no traffic
        const int kc0 = has_next ? 0 : nst, kc1 = has_next ? 1 : nst;
        if (wm) ring_barrier();  // waves 4-7 run one tick behind waves 0-3
        Acc acc[2];
        auto full = [&](int s, bool first) __attribute__((always_inline)) {
            half1(acc, q0 + s, first, s + 1, plan);
            half2(acc, q0 + s, first, s + 2, plan);
        };
        if (nst > 2) {
            full(0, true);
            for (int s = 1; s + 2 < nst; ++s) full(s, false);
            half1(acc, q0 + nst - 2, false, nst - 1, plan);
        } else {
            half1(acc, q0, true, 1, plan);
        }
        if (has_next) make_plan(nxt, plan);
        half2(acc, q0 + nst - 2, nst == 2, kc0, plan);
        half1(acc, q0 + nst - 1, false, kc0, plan);
        half2(acc, q0 + nst - 1, false, kc1, plan);
        if (!wm) ring_barrier();
        epilogue(acc, cur);
        if (!has_next) break;
        cur = nxt;
        q0 += nst;
    }
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // the surplus copies have landed before the workgroup ends
}

template <typename T, bool PK, bool QK, bool SWIGLU>
hipError_t run_tiled(const GemmArgs& g, hipStream_t stream) {
    auto fn = &gemm_tiled_kernel<T, PK, QK, SWIGLU>;
    const void* p = reinterpret_cast<const void*>(fn);
    const int bn = SWIGLU ? kBN / 2 : kBN;
    const int mtiles = (g.m + kBM - 1) / kBM, ntiles = (g.n + bn - 1) / bn;
    int grid = resident_workgroups(p, kThreads, kLdsBytes) / kXcds * kXcds;
    const int most = (mtiles * ntiles + kXcds - 1) / kXcds * kXcds;
    if (grid < kXcds) grid = kXcds;
    if (grid > most) grid = most;
    TraceScope trace("moe_linear_gemm_tiled", stream);
    fn<<<grid, kThreads, kLdsBytes, stream>>>(g, mtiles, ntiles);
    return hipGetLastError();
}

template <typename T>
hipError_t run_tiled_any(const GemmArgs& g, bool p_by_k, bool q_by_k, hipStream_t stream) {
    if (p_by_k) return run_tiled<T, true, true, false>(g, stream);
    if (g.act == kActSwiglu)
        return q_by_k ? run_tiled<T, false, true, true>(g, stream) : run_tiled<T, false, false, true>(g, stream);
    return q_by_k ? run_tiled<T, false, true, false>(g, stream) : run_tiled<T, false, false, false>(g, stream);
}

template <typename T>
hipError_t prepare() {
    for (const void* fn : {reinterpret_cast<const void*>(&gemm_tiled_kernel<T, true, true, false>),
                           reinterpret_cast<const void*>(&gemm_tiled_kernel<T, false, true, true>),
                           reinterpret_cast<const void*>(&gemm_tiled_kernel<T, false, false, true>),
                           reinterpret_cast<const void*>(&gemm_tiled_kernel<T, false, true, false>),
                           reinterpret_cast<const void*>(&gemm_tiled_kernel<T, false, false, false>)}) {
        const hipError_t err = ensure_lds_limit(fn, kLdsBytes);
        if (err != hipSuccess) return err;
    }
    return hipSuccess;
}

}  // namespace

hipError_t prepare_gemm_tiled() {
    const hipError_t err = prepare<Half>();
    return err == hipSuccess ? prepare<Bf16>() : err;
}

hipError_t launch_gemm_tiled(const GemmArgs& g, bool p_by_k, bool q_by_k, bool bf16, hipStream_t stream) {
    return bf16 ? run_tiled_any<Bf16>(g, p_by_k, q_by_k, stream) : run_tiled_any<Half>(g, p_by_k, q_by_k, stream);
}

}  // namespace moe
