// moe_linear.hip -- MoeLinear and MoeLinearGrad for gfx950: y = act(x W^T + b) + r and its gradients.
//
// No counterpart in the reference, whose products are the expert FFN's (op_kernel/moe_expert_ffn.cpp:265-394).
// Every product here is C[m][n] = sum_k P[m][k] Q[n][k] with fp16 or bf16 operands and fp32 sums (MFMA):
//   forward    P = x  (by rows), Q = W (by rows, or by k when W is a transposed view)
//   grad_x     P = dz (by rows), Q = W read the other way round
//   grad_W     P = dz (by k: its T rows are the reduction), Q = x (by k)
// The tiles here, 32 to 256 rows by 128, are for products that do not fill the GPU with 256 x 256 ones; where even
// these leave CUs idle the product is split over k and a second launch adds the pieces in order. What bounds them is
// the copies into LDS: 24 KB a stage and two workgroups a CU, 0.65 us for both (64 rows), is 19 TB/s over the GPU, and
// 128 and 256 rows come to 18 and 13 TB/s. So the taller tile wins until the pieces' sums cost more than its reads
// save.
//   T = 4097, H = 7168, N = 256 (130 tiles of 64 rows in 3 pieces): 25.6 + 4.2 us, of which x from HBM alone is 11
//   both gradients' products at T = 1000, H = 1056, N = 733, one launch of 256 workgroups: 10.9 + 3.2 us
#include "moe_gemm.h"

namespace moe {

namespace {

constexpr int kBN = 128;      // Q rows of a tile (SwiGLU: 64 gate and the matching 64 up rows)
constexpr int kBK = 64;       // k of a stage
constexpr int kXcds = 8;
constexpr uint32_t kPastEnd = 0x80000000u;  // a buffer offset past every buffer: the load returns zeros

// Waves of a workgroup: each has 64 x 64 of a tile (narrower below 128 rows)
constexpr int mid_waves(int bm) { return bm == 256 ? 8 : 4; }
constexpr int mid_threads(int bm) { return mid_waves(bm) * kWave; }
// Stages in the LDS ring: one 144 KB workgroup a CU at 256 rows, two of 64 KB at 128, two of 72 or 80 KB below
constexpr int ring_stages(int bm) { return bm == 128 ? 2 : bm == 32 ? 4 : 3; }
constexpr int mid_lds_bytes(int bm) { return ring_stages(bm) * (bm + kBN) * kBK * 2; }

__device__ __forceinline__ void ring_barrier() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    __builtin_amdgcn_sched_barrier(0);
}

// Where the 16 bytes that lane `lane` of copy instruction `i` writes to LDS come from. Direct-to-LDS copies write 64
// consecutive 16-byte granules, so the layout's swizzle is in which granule each lane fetches.
//   by rows: an LDS row is one operand row, 64 k = 8 granules; granule g of row r stands at g ^ ((r >> 1) & 7), so the
//            16 rows one ds_read_b128 touches spread over all banks.
//   by k:    an LDS row is one k, ROWS operand rows = ROWS / 8 granules; its 32-byte pairs stand at pair ^ f(k), f over
//            (k & 3, k >> 3 & 1), so the 8 k that half a wave's ds_read_b64_tr_b16 touches spread over all banks.
struct Granule {
    int row;  // by rows: operand row of the tile; by k: k of the stage
    int el;   // by rows: first k of the stage; by k: first operand row of the tile
};
// 256 rows by k are two such tiles of 128 one after the other.
template <bool BY_K, int ROWS>
__device__ __forceinline__ Granule granule_of(int i, int lane) {
    static_assert(!BY_K || ROWS % 128 == 0, "the swizzle by k permutes 8 pairs of granules");
    if (!BY_K) {
        const int r = i * 8 + lane / 8;
        return Granule{r, ((lane % 8) ^ ((r >> 1) & 7)) * 8};
    }
    const int k = i % 16 * 4 + lane / 16, f = (k & 3) | (((k >> 3) & 1) << 2);
    return Granule{k, i / 16 * 128 + ((lane % 16) ^ (f << 1)) * 8};
}

// Fragments of N blocks of 16 operand rows from r0 on, both 32-k steps: lane (row16, kg) gets 8 k of one row.
template <bool BY_K, int N>
__device__ __forceinline__ void read_fragments(const uint16_t* tile, int r0, int lane, s16x8 (&f)[2][N]) {
    if constexpr (BY_K) {
        uint32_t addr[N];
#pragma unroll
        for (int n = 0; n < N; ++n) addr[n] = transposed_address(tile + r0 / 128 * 128 * kBK, r0 % 128 + n * 16, lane);
        read_transposed(addr, f);
    } else {
        const int row16 = lane & 15, kg = lane >> 4, sw = (row16 >> 1) & 7;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
            for (int n = 0; n < N; ++n)
                f[kk][n] = *reinterpret_cast<const s16x8*>(tile + (r0 + n * 16 + row16) * kBK +
                                                           (((kk * 4 + kg) ^ sw) * 8));
    }
}

// 8 consecutive elements (of a row's k, or by k of rows) from an operand of any alignment, zeros past its end
__device__ __forceinline__ s16x8 load_granule(const uint16_t* p, int64_t ld, bool by_k, int row, int k, int rows,
                                              int k1) {
    const int valid = row >= rows || k >= k1 ? 0 : by_k ? rows - row : k1 - k;
    return load8(p + (by_k ? static_cast<int64_t>(k) * ld + row : static_cast<int64_t>(row) * ld + k), valid,
                 by_k ? row : k);
}

// C[m][n] tile of BM x 128, one ring of direct-to-LDS stages, one barrier a stage.
// DIRECT: both operands allow 16-byte copies (bases and row pitches 16-byte aligned, by rows k % 8 == 0). Otherwise the
// granules come through registers (loads of any alignment) and are written to the same layout.
// block of grid: this product's share of the launch, grid a multiple of the XCDs.
template <typename T, bool PK, bool QK, int BM, bool SWIGLU, bool DIRECT>
__device__ __forceinline__ void gemm_mid(const GemmArgs& g, int mtiles, int ntiles, int block, int grid,
                                         uint16_t* lds) {
    constexpr int NS = ring_stages(BM);
    constexpr int WAVES = mid_waves(BM);
    constexpr int WM = BM >= 128 ? BM / 64 : 1, WN = WAVES / WM;  // waves along m and n
    constexpr int FM = BM / WM / 16, FN = kBN / WN / 16;  // 16 x 16 blocks of a wave
    constexpr int PC = BM / 8 / WAVES, QC = kBN / 8 / WAVES;  // copy instructions per wave and stage
    constexpr int kSlot = (BM + kBN) * kBK;
    const int tid = static_cast<int>(threadIdx.x), lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int wm = wave / WN, wn = wave % WN;
    const int row16 = lane & 15, kg = lane >> 4;

    // Workgroups go round-robin over the XCDs; each XCD takes a contiguous run of the items. The tiles that read the
    // same piece of the larger operand are neighbours in it, so that piece reaches that XCD's L2 once.
    const int item = block % kXcds * (grid / kXcds) + block / kXcds;
    if (item >= mtiles * ntiles * g.splits) return;
    const bool n_first = mtiles > ntiles;
    const int inner = n_first ? ntiles : mtiles, outer = item / inner;
    const int outers = n_first ? mtiles : ntiles;
    const int i0 = item - outer * inner, sp = outer / outers, o0 = outer - sp * outers;
    const int mt = n_first ? o0 : i0, nt = n_first ? i0 : o0;
    const int k0 = sp * g.split_k, k1 = min(g.k, k0 + g.split_k);
    const int nst = max(1, (k1 - k0 + kBK - 1) / kBK);
    const int m0 = mt * BM, n0 = nt * (SWIGLU ? kBN / 2 : kBN);

    // Q row of tile row r. SwiGLU: a wave's rows are half gate, half up, of the same output columns.
    auto q_col = [&](int r) {
        if (!SWIGLU) return n0 + r;
        constexpr int kHalf = kBN / WN / 2;
        return n0 + r / (2 * kHalf) * kHalf + r % kHalf;
    };
    auto q_up = [&](int r) { return SWIGLU && (r / (kBN / WN / 2)) % 2 == 1; };

    int prow[PC], pel[PC], qrow[QC], qel[QC];
#pragma unroll
    for (int c = 0; c < PC; ++c) {
        const Granule a = granule_of<PK, BM>(wave * PC + c, lane);
        prow[c] = a.row;
        pel[c] = a.el;
    }
#pragma unroll
    for (int c = 0; c < QC; ++c) {
        const Granule a = granule_of<QK, kBN>(wave * QC + c, lane);
        qrow[c] = a.row;
        qel[c] = a.el;
    }
    // Byte offsets of this lane's granules, relative to (by rows) the tile's first row, (by k) the stage's first k;
    // past every buffer where the operand has no such row. 64-bit arithmetic is in the bases alone, so an operand may
    // be larger than 4 GiB. By rows the k offset of a stage is the instruction's scalar one.
    uint32_t poff[PC], qoff[QC];
    if (DIRECT) {
        const uint32_t ppitch = static_cast<uint32_t>(g.ldp) * 2, qpitch = static_cast<uint32_t>(g.ldq) * 2;
#pragma unroll
        for (int c = 0; c < PC; ++c) {
            const int row = m0 + (PK ? pel[c] : prow[c]);
            poff[c] = row < g.m ? prow[c] * ppitch + (PK ? row : pel[c]) * 2u : kPastEnd;
        }
#pragma unroll
        for (int c = 0; c < QC; ++c) {
            const int tr = QK ? qel[c] : qrow[c], col = q_col(tr);
            const uint32_t off = QK ? qrow[c] * qpitch + (col + (q_up(tr) ? g.up : 0)) * 2u
                                    : (col - n0) * qpitch + qel[c] * 2u;
            qoff[c] = col < g.n ? off : kPastEnd;
        }
    }
    const uint16_t* pbase = g.p + (PK ? 0 : static_cast<int64_t>(m0) * g.ldp);
    const uint16_t* qbase = g.q + (QK ? 0 : static_cast<int64_t>(n0) * g.ldq);
    auto copy_stage = [&](int s) __attribute__((always_inline)) {
        uint16_t* slot = lds + (s % NS) * kSlot;
        const int kc = k0 + s * kBK;
        if (DIRECT) {
            const int left = k1 - kc;  // granules from here on are zeros
            const __amdgpu_buffer_rsrc_t pr = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<uint16_t*>(PK ? pbase + static_cast<int64_t>(kc) * g.ldp : pbase), 0, 0x7fffffff,
                0x00020000);
#pragma unroll
            for (int c = 0; c < PC; ++c)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    pr, (__attribute__((address_space(3))) void*)(slot + (wave * PC + c) * 512), 16,
                    static_cast<int>((PK ? prow[c] : pel[c]) < left ? poff[c] : kPastEnd), PK ? 0 : kc * 2, 0, 0);
#pragma unroll
            for (int c = 0; c < QC; ++c) {
                // by rows a copy instruction covers 8 rows, all gate or all up: the base tells them apart, so that the
                // offsets stay within the tile
                const int64_t up = !QK && q_up((wave * QC + c) * 8) ? static_cast<int64_t>(g.up) * g.ldq : 0;
                const __amdgpu_buffer_rsrc_t qr = __builtin_amdgcn_make_buffer_rsrc(
                    const_cast<uint16_t*>(QK ? qbase + static_cast<int64_t>(kc) * g.ldq : qbase + up), 0, 0x7fffffff,
                    0x00020000);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    qr, (__attribute__((address_space(3))) void*)(slot + BM * kBK + (wave * QC + c) * 512), 16,
                    static_cast<int>((QK ? qrow[c] : qel[c]) < left ? qoff[c] : kPastEnd), QK ? 0 : kc * 2, 0, 0);
            }
        } else {
#pragma unroll
            for (int c = 0; c < PC; ++c) {
                const int row = m0 + (PK ? pel[c] : prow[c]), k = kc + (PK ? prow[c] : pel[c]);
                const s16x8 v = load_granule(g.p, g.ldp, PK, row, k, g.m, k1);
                *reinterpret_cast<s16x8*>(slot + (wave * PC + c) * 512 + lane * 8) = v;
            }
#pragma unroll
            for (int c = 0; c < QC; ++c) {
                const int tr = QK ? qel[c] : qrow[c], up = q_up(tr) ? g.up : 0;
                const s16x8 v =
                    load_granule(g.q, g.ldq, QK, q_col(tr) + up, kc + (QK ? qrow[c] : qel[c]), g.n + up, k1);
                *reinterpret_cast<s16x8*>(slot + BM * kBK + (wave * QC + c) * 512 + lane * 8) = v;
            }
        }
    };

    f32x4 acc[FN][FM];
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int i = 0; i < FM; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};

#pragma unroll
    for (int s = 0; s < NS - 1; ++s) copy_stage(s);  // stages past the last are all past k1: zeros, no traffic
    for (int s = 0; s < nst; ++s) {
        // this wave's reads of stage s - 1 are in registers and its copies of stage s have landed; after the barrier
        // so have everyone's, and the slot of stage s - 1 may be filled again
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(vmcnt_imm((NS - 2) * (PC + QC)) & 0xf0ffu);
        ring_barrier();
        copy_stage(s + NS - 1);
        const uint16_t* tp = lds + (s % NS) * kSlot;
        const uint16_t* tq = tp + BM * kBK;
        s16x8 fp[2][FM], fq[2][FN];
        read_fragments<PK, FM>(tp, wm * (BM / WM), lane, fp);
        read_fragments<QK, FN>(tq, wn * (kBN / WN), lane, fq);
        __builtin_amdgcn_sched_barrier(0);  // all reads are on their way before the first product
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int i = 0; i < FM; ++i) acc[j][i] = T::mfma(fq[kk][j], fp[kk][i], acc[j][i]);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0) & 0xf0ffu);  // the surplus copies have landed

    // acc[j][i]: D[Q row 4 kg + r of block j][P row row16 of block i], 4 consecutive columns of one row
    constexpr int FO = SWIGLU ? FN / 2 : FN;
    const int r0 = m0 + wm * (BM / WM), c0 = n0 + wn * (FO * 16);
    if (g.splits > 1) {
        const int64_t pld = part_ld(g.n, SWIGLU), pcols = part_cols(g.n);
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const int row = r0 + i * 16 + row16;
            if (row >= g.m) continue;
#pragma unroll
            for (int j = 0; j < FO; ++j) {
                const int col = c0 + j * 16 + kg * 4;
                if (col >= g.n) continue;
                float* dst = g.partial + (static_cast<int64_t>(sp) * g.m + row) * pld + col;
                *reinterpret_cast<f32x4*>(dst) = acc[j][i];
                if (SWIGLU) *reinterpret_cast<f32x4*>(dst + pcols) = acc[j + FO][i];
            }
        }
        return;
    }
    ring_barrier();  // everyone's reads and copies are over: the ring's room is the epilogue's
    const bool vec = vector_rows(g), lines = whole_lines(g, vec);
    float* stg = reinterpret_cast<float*>(lds) + wave * (FN * 256);
    auto put = [&](int i) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < FN; ++j) put_block<FN>(stg, row16, kg, j, acc[j][i]);
    };
#pragma unroll 1
    for (int i = 0; i < FM; ++i) {  // one copy of the epilogue's code
        switch (i) {
            case 0: put(0); break;
            case 1: put(1); break;
            case 2: put(FM > 2 ? 2 : 0); break;
            default: put(FM > 3 ? 3 : 0); break;
        }
        store_block<T, SWIGLU, FN>(g, stg, lane, r0 + i * 16, c0, vec, lines);
    }
}

template <typename T, bool PK, bool QK, int BM, bool SWIGLU, bool DIRECT>
__global__ __launch_bounds__(mid_threads(BM)) __attribute__((amdgpu_waves_per_eu(2, 2))) void gemm_mid_kernel(
    GemmArgs g, int mtiles, int ntiles) {
    extern __shared__ __align__(16) uint16_t lds[];
    gemm_mid<T, PK, QK, BM, SWIGLU, DIRECT>(g, mtiles, ntiles, static_cast<int>(blockIdx.x),
                                            static_cast<int>(gridDim.x), lds);
}

// Both gradient products in one launch: neither needs the other, and small ones leave the GPU half empty. The first
// x_blocks workgroups have grad_x.
template <typename T, bool QK, int BM>
__global__ __launch_bounds__(mid_threads(BM)) __attribute__((amdgpu_waves_per_eu(2, 2))) void gemm_pair_kernel(
    GemmArgs x, GemmArgs w, int x_blocks) {
    extern __shared__ __align__(16) uint16_t lds[];
    const int block = static_cast<int>(blockIdx.x);
    if (block < x_blocks)
        gemm_mid<T, false, QK, BM, false, true>(x, (x.m + BM - 1) / BM, (x.n + kBN - 1) / kBN, block, x_blocks, lds);
    else
        gemm_mid<T, true, true, 128, false, true>(w, (w.m + 127) / 128, (w.n + kBN - 1) / kBN, block - x_blocks,
                                                  static_cast<int>(gridDim.x) - x_blocks, lds);
}

int mid_grid(const GemmArgs& g, int bm, int bn) {
    const int64_t items = static_cast<int64_t>((g.m + bm - 1) / bm) * ((g.n + bn - 1) / bn) * g.splits;
    return static_cast<int>((items + kXcds - 1) / kXcds * kXcds);
}

template <typename T, bool PK, bool QK, int BM, bool SWIGLU, bool DIRECT>
hipError_t run_mid(const GemmArgs& g, hipStream_t stream) {
    constexpr int kCols = SWIGLU ? kBN / 2 : kBN;
    TraceScope trace("moe_linear_gemm", stream);
    gemm_mid_kernel<T, PK, QK, BM, SWIGLU, DIRECT>
        <<<mid_grid(g, BM, kCols), mid_threads(BM), mid_lds_bytes(BM), stream>>>(g, (g.m + BM - 1) / BM,
                                                                                (g.n + kCols - 1) / kCols);
    return hipGetLastError();
}

template <typename T, bool QK, int BM>
hipError_t run_pair(const GemmArgs& x, const GemmArgs& w, hipStream_t stream) {
    constexpr int kLds = mid_lds_bytes(BM) > mid_lds_bytes(128) ? mid_lds_bytes(BM) : mid_lds_bytes(128);
    const int x_blocks = mid_grid(x, BM, kBN);
    TraceScope trace("moe_linear_gemm", stream);
    gemm_pair_kernel<T, QK, BM><<<x_blocks + mid_grid(w, 128, kBN), mid_threads(BM), kLds, stream>>>(x, w, x_blocks);
    return hipGetLastError();
}
template <typename T>
hipError_t run_pair_any(const GemmArgs& x, const GemmArgs& w, bool q_by_k, int bm, hipStream_t stream) {
    if (bm == 32) return q_by_k ? run_pair<T, true, 32>(x, w, stream) : run_pair<T, false, 32>(x, w, stream);
    if (bm == 64) return q_by_k ? run_pair<T, true, 64>(x, w, stream) : run_pair<T, false, 64>(x, w, stream);
    return q_by_k ? run_pair<T, true, 128>(x, w, stream) : run_pair<T, false, 128>(x, w, stream);
}

template <typename T, bool PK, bool QK, int BM, bool SWIGLU>
hipError_t run_mid_direct(const GemmArgs& g, bool direct, hipStream_t stream) {
    return direct ? run_mid<T, PK, QK, BM, SWIGLU, true>(g, stream) : run_mid<T, PK, QK, BM, SWIGLU, false>(g, stream);
}

template <typename T>
hipError_t run_mid_any(const GemmArgs& g, bool p_by_k, bool q_by_k, bool direct, int bm, hipStream_t stream) {
    const bool swiglu = g.act == kActSwiglu;
    if (p_by_k) return bm == 256 ? run_mid<T, true, true, 256, false, true>(g, stream)
                                 : run_mid_direct<T, true, true, 128, false>(g, direct, stream);
    if (bm == 256) {  // direct operands only
        if (q_by_k) return swiglu ? run_mid<T, false, true, 256, true, true>(g, stream)
                                  : run_mid<T, false, true, 256, false, true>(g, stream);
        return swiglu ? run_mid<T, false, false, 256, true, true>(g, stream)
                      : run_mid<T, false, false, 256, false, true>(g, stream);
    }
    if (bm == 128) {
        if (q_by_k) return swiglu ? run_mid_direct<T, false, true, 128, true>(g, direct, stream)
                                  : run_mid_direct<T, false, true, 128, false>(g, direct, stream);
        return swiglu ? run_mid_direct<T, false, false, 128, true>(g, direct, stream)
                      : run_mid_direct<T, false, false, 128, false>(g, direct, stream);
    }
    if (bm == 64) {
        if (q_by_k) return swiglu ? run_mid_direct<T, false, true, 64, true>(g, direct, stream)
                                  : run_mid_direct<T, false, true, 64, false>(g, direct, stream);
        return swiglu ? run_mid_direct<T, false, false, 64, true>(g, direct, stream)
                      : run_mid_direct<T, false, false, 64, false>(g, direct, stream);
    }
    if (q_by_k) return swiglu ? run_mid_direct<T, false, true, 32, true>(g, direct, stream)
                              : run_mid_direct<T, false, true, 32, false>(g, direct, stream);
    return swiglu ? run_mid_direct<T, false, false, 32, true>(g, direct, stream)
                  : run_mid_direct<T, false, false, 32, false>(g, direct, stream);
}

// Adds the splits' sums in order and applies the epilogue; a thread has 4 columns of a row.
constexpr int kReduceThreads = 256;
int64_t reduce_blocks(const GemmArgs& g) { return (part_cols(g.n) / 4 * g.m + kReduceThreads - 1) / kReduceThreads; }
template <typename T, bool SWIGLU>
__device__ __forceinline__ void gemm_reduce(const GemmArgs& g, int block) {
    const int64_t pcols = part_cols(g.n), pld = part_ld(g.n, SWIGLU), per_row = pcols / 4;
    const int64_t idx = static_cast<int64_t>(block) * kReduceThreads + threadIdx.x;
    if (idx >= per_row * g.m) return;
    const int64_t row = idx / per_row;
    const int col = static_cast<int>(idx % per_row) * 4;
    const float* src = g.partial + row * pld + col;
    const int64_t step = static_cast<int64_t>(g.m) * pld;
    f32x4 z = *reinterpret_cast<const f32x4*>(src), u = {0.f, 0.f, 0.f, 0.f};
    if (SWIGLU) u = *reinterpret_cast<const f32x4*>(src + pcols);
#pragma unroll 4
    for (int s = 1; s < g.splits; ++s) {
        z += *reinterpret_cast<const f32x4*>(src + s * step);
        if (SWIGLU) u += *reinterpret_cast<const f32x4*>(src + s * step + pcols);
    }
    store4<T, SWIGLU>(g, row, col, z, u, vector_rows(g));
}
template <typename T, bool SWIGLU>
__global__ __launch_bounds__(kReduceThreads) void gemm_reduce_kernel(GemmArgs g) {
    gemm_reduce<T, SWIGLU>(g, static_cast<int>(blockIdx.x));
}

// What is left of a training step's gradients in one launch: the split products' sums and the bias's column sums
template <typename T>
__global__ __launch_bounds__(kReduceThreads) void grad_tail_kernel(GradTail t) {
    int block = static_cast<int>(blockIdx.x);
    if (block < t.x_blocks) return gemm_reduce<T, false>(t.x, block);
    block -= t.x_blocks;
    if (block < t.w_blocks) return gemm_reduce<T, false>(t.w, block);
    column_sums<T>(t.sums, t.bias_grad, t.Z, t.sum_rows, block - t.w_blocks);
}

template <typename T>
hipError_t prepare_256() {
    for (const void* fn : {reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, false, 256, false, true>),
                           reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, false, 256, true, true>),
                           reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, true, 256, false, true>),
                           reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, true, 256, true, true>),
                           reinterpret_cast<const void*>(&gemm_mid_kernel<T, true, true, 256, false, true>)}) {
        const hipError_t err = ensure_lds_limit(fn, mid_lds_bytes(256));
        if (err != hipSuccess) return err;
    }
    return hipSuccess;
}

template <typename T, int BM>
hipError_t prepare_bm() {
    const int lds = mid_lds_bytes(BM);
    for (const void* fn : {reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, false, BM, false, true>),
                           reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, false, BM, true, true>),
                           reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, true, BM, false, true>),
                           reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, true, BM, true, true>),
                           reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, false, BM, false, false>),
                           reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, false, BM, true, false>),
                           reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, true, BM, false, false>),
                           reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, true, BM, true, false>),
                           reinterpret_cast<const void*>(&gemm_pair_kernel<T, false, BM>),
                           reinterpret_cast<const void*>(&gemm_pair_kernel<T, true, BM>)}) {
        const hipError_t err = ensure_lds_limit(fn, lds);
        if (err != hipSuccess) return err;
    }
    return hipSuccess;
}

}  // namespace

hipError_t launch_gemm_mid(const GemmArgs& g, bool p_by_k, bool q_by_k, bool bf16, bool direct, int bm,
                           hipStream_t stream) {
    return bf16 ? run_mid_any<Bf16>(g, p_by_k, q_by_k, direct, bm, stream)
                : run_mid_any<Half>(g, p_by_k, q_by_k, direct, bm, stream);
}

hipError_t launch_gemm_reduce(const GemmArgs& g, bool bf16, hipStream_t stream) {
    const bool swiglu = g.act == kActSwiglu;
    const int64_t work = part_cols(g.n) / 4 * g.m;
    const int grid = static_cast<int>((work + kReduceThreads - 1) / kReduceThreads);
    TraceScope trace("moe_linear_reduce", stream);
    if (bf16) {
        if (swiglu) gemm_reduce_kernel<Bf16, true><<<grid, kReduceThreads, 0, stream>>>(g);
        else gemm_reduce_kernel<Bf16, false><<<grid, kReduceThreads, 0, stream>>>(g);
    } else {
        if (swiglu) gemm_reduce_kernel<Half, true><<<grid, kReduceThreads, 0, stream>>>(g);
        else gemm_reduce_kernel<Half, false><<<grid, kReduceThreads, 0, stream>>>(g);
    }
    return hipGetLastError();
}

hipError_t launch_gemm_pair(const GemmArgs& x, const GemmArgs& w, bool q_by_k, bool bf16, int bm, hipStream_t stream) {
    return bf16 ? run_pair_any<Bf16>(x, w, q_by_k, bm, stream) : run_pair_any<Half>(x, w, q_by_k, bm, stream);
}

hipError_t launch_grad_tail(GradTail t, bool bf16, hipStream_t stream) {
    t.x_blocks = t.x.splits > 1 ? static_cast<int>(reduce_blocks(t.x)) : 0;
    t.w_blocks = t.w.splits > 1 ? static_cast<int>(reduce_blocks(t.w)) : 0;
    const int grid = t.x_blocks + t.w_blocks + (t.bias_grad ? (t.Z + kSumColumns - 1) / kSumColumns : 0);
    if (grid == 0) return hipSuccess;
    TraceScope trace("moe_linear_reduce", stream);
    if (bf16) grad_tail_kernel<Bf16><<<grid, kReduceThreads, 0, stream>>>(t);
    else grad_tail_kernel<Half><<<grid, kReduceThreads, 0, stream>>>(t);
    return hipGetLastError();
}

hipError_t prepare_gemm_mid() {  // 128-row tiles keep within 64 KB
    hipError_t err = prepare_256<Half>();
    if (err == hipSuccess) err = prepare_256<Bf16>();
    if (err == hipSuccess) err = prepare_bm<Half, 32>();
    if (err == hipSuccess) err = prepare_bm<Half, 64>();
    if (err == hipSuccess) err = prepare_bm<Bf16, 32>();
    if (err == hipSuccess) err = prepare_bm<Bf16, 64>();
    return err;
}

}  // namespace moe
