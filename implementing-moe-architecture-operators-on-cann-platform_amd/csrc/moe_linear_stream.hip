// moe_linear_stream.hip -- the dense product of few rows (serving's single tokens and small batches): weight streaming.
//
// C[m][n] = sum_k P[m][k] Q[n][k], both operands by rows, m <= 64. The weights are read once and bound it: at T = 1 the
// gate and up rows of a dense expert (H = 7168, N = 2048) are 59 MB for 59 MFLOP, 10.7 us (5.5 TB/s). From 16 rows on
// x, which every tile reads again from L2, adds to it. T = 64, N = 7168 takes 11.3, 19.6 and 32.4 us at H = 2048, 4096
// and 8192: weights and x come in at 13.8 TB/s together (59 + 117 MB in the last 12.8 us), and 5 us are the launch, the
// first copies and the sums. T = 16 there: 25.7 us at H = 8192, the weights at 6.2 TB/s in the last 9.4 us.
//   work      a tile is 16 or 32 weight rows (SwiGLU: half gate, half the matching up rows) over the whole k, and its
//             workgroup's waves share k: wave w takes the 64-k pieces w, w + W, ... Their sums meet in LDS, added in
//             wave order, and go through the epilogue: one launch, no partial sums in memory.
//   copies    each wave has its own LDS ring and fills it straight from global memory, 8 rows x 128 bytes an
//             instruction; nobody else reads it, so the main loop has no barrier. Loaded into registers in fragment
//             order (16 rows x 64 bytes an instruction) the same work ran at 4.2 TB/s.
//   persistent  a workgroup per CU walks its tiles and the rings run on across them, so the next tile's weights are in
//             flight while the sums of this one are added.
// Rows past the last and k past the end read zeros without memory traffic.
// 8-bit integers (MoeLinearInt8) take half the bytes: T = 1, H = 7168, N = 2048 SwiGLU, 29 MB, 7.4 us. The products of
// experts with few rows each (GROUPED) are items of 16 rows of an expert by 64 of its weight rows; a workgroup has the
// experts' items in registers, as loads of the offsets between the copies would wait for those.
#include "moe_gemm.h"

#include <type_traits>

namespace moe {

namespace {

constexpr int kBK = 64;                     // k of a piece
constexpr int kBlock = 16 * kBK;            // halfs of 16 rows of a piece
constexpr uint32_t kPastEnd = 0x80000000u;  // a buffer offset past every buffer: the load returns zeros
constexpr int kNonTemporal = 2;             // cache policy of the weights: read once

// QB, MB: blocks of 16 rows of Q and P; DEPTH: pieces of a wave's ring
template <int QB, int MB, int WAVES, int DEPTH>
struct StreamLds {
    static constexpr int kPieceHalfs = (QB + MB) * kBlock;
    static constexpr int kRings = WAVES * DEPTH * kPieceHalfs * 2;
    static constexpr int kPassBlocks = MB < 2 ? MB : 2;  // blocks of P rows whose sums meet at a time
    static constexpr int kSums = WAVES * kPassBlocks * 16 * QB * 16 * 4;
    static constexpr int kBytes = kRings + kSums;
};

template <typename T, int QB, int MB, int WAVES, int DEPTH, bool SWIGLU, bool GROUPED = false>
__global__ __launch_bounds__(WAVES * kWave) void gemm_stream_kernel(GemmArgs g, int tiles) {
    using Lds = StreamLds<QB, MB, WAVES, DEPTH>;
    constexpr int kCopies = 2 * (QB + MB), kCols = QB * (SWIGLU ? 8 : 16);
    extern __shared__ __align__(16) uint16_t lds[];
    float* sums = reinterpret_cast<float*>(lds + Lds::kRings / 2);  // [wave][P row of the pass][Q row]
    const int tid = static_cast<int>(threadIdx.x), lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int row16 = lane & 15, kg = lane >> 4;
    uint16_t* ring = lds + wave * DEPTH * Lds::kPieceHalfs;

    // Copy instruction i of a block: rows 8 i + lane / 8; granule G (8 k) of row r stands at G ^ (r >> 1 & 7)
    const int r8 = lane / 8, gran = (lane % 8) ^ (r8 >> 1);  // of instruction 0; instruction 1: granule ^ 4
    const uint32_t ppitch = static_cast<uint32_t>(g.ldp) * 2, qpitch = static_cast<uint32_t>(g.ldq) * 2;
    const __amdgpu_buffer_rsrc_t pr =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(g.p), 0, 0x7fffffff, 0x00020000);

    // Experts: `tiles` is an expert's, and an item one of them for 16 MB of the expert's rows; items of the same
    // weights are neighbours.
    const int ntiles = tiles;
    GroupItem cgroup{};
    GroupTable table;
    if (GROUPED) {
        table = group_table(g, 16 * MB, ntiles);
        tiles = table.total;
        group_zero_rows(g, table.rows, static_cast<int>(blockIdx.x), static_cast<int>(gridDim.x));
    }
    struct Place {
        int row0, nt;  // first P row, tile of Q rows
    };
    auto place_of = [&](int tile, GroupItem& item) __attribute__((always_inline)) {
        if (!GROUPED) return Place{0, tile};
        item = group_find(table, 16 * MB, ntiles, tile);
        const int passes = (item.row1 - item.row0 + 16 * MB - 1) / (16 * MB);
        const int in = tile - item.first, nt = in / passes;
        return Place{item.row0 + (in - nt * passes) * 16 * MB, nt};
    };

    const int stages = (g.k + kBK - 1) / kBK;
    const int mine = stages > wave ? (stages - wave + WAVES - 1) / WAVES : 0;  // pieces of this wave per tile
    // the wave's pieces of all its tiles in a row: where the next copy is
    int ctile = static_cast<int>(blockIdx.x), cpiece = 0, cslot = 0;
    Place cplace{0, ctile};
    if (GROUPED && ctile < tiles) cplace = place_of(ctile, cgroup);
    auto copy_next = [&]() __attribute__((always_inline)) {
        uint16_t* slot = ring + cslot * Lds::kPieceHalfs;
        const int k0 = (wave + cpiece * WAVES) * kBK;
        const bool live = ctile < tiles && mine > 0;
        const int n0 = (GROUPED ? cplace.nt : ctile) * kCols;
        const uint16_t* qe = GROUPED ? group_q(g, cgroup.expert) : g.q;
#pragma unroll
        for (int i = 0; i < 2 * QB; ++i) {
            const int k = k0 + ((gran ^ (4 * (i & 1))) * 8);
            const int row = 8 * (SWIGLU ? i % QB : i) + r8;
            // SwiGLU: the first QB instructions the gate rows, the others the up rows
            const int64_t first = n0 + (SWIGLU && i >= QB ? static_cast<int64_t>(g.up) : 0);
            const __amdgpu_buffer_rsrc_t qr = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<uint16_t*>(live ? qe + first * g.ldq : g.q), 0, 0x7fffffff, 0x00020000);
            const uint32_t off = static_cast<uint32_t>(row) * qpitch + static_cast<uint32_t>(k) * 2;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                qr, (__attribute__((address_space(3))) void*)(slot + i * 512), 16,
                static_cast<int>(live && n0 + row < g.n && k < g.k ? off : kPastEnd), 0, 0, kNonTemporal);
        }
        const uint16_t* px = g.p + static_cast<int64_t>(cplace.row0) * g.ldp;
        const __amdgpu_buffer_rsrc_t pe =
            GROUPED ? __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(px), 0, 0x7fffffff, 0x00020000) : pr;
        const int rows = GROUPED ? cgroup.row1 - cplace.row0 : g.m;
#pragma unroll
        for (int i = 0; i < 2 * MB; ++i) {
            const int row = 8 * i + r8, k = k0 + ((gran ^ (4 * (i & 1))) * 8);
            const uint32_t off = static_cast<uint32_t>(row) * ppitch + static_cast<uint32_t>(k) * 2;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                pe, (__attribute__((address_space(3))) void*)(slot + QB * kBlock + i * 512), 16,
                static_cast<int>(live && row < rows && k < g.k ? off : kPastEnd), 0, 0, 0);
        }
        cslot = cslot + 1 == DEPTH ? 0 : cslot + 1;
        if (++cpiece >= mine) {
            cpiece = 0;
            ctile += static_cast<int>(gridDim.x);
            if (GROUPED && ctile < tiles) cplace = place_of(ctile, cgroup);
        }
    };
#pragma unroll
    for (int d = 0; d < DEPTH - 1; ++d) copy_next();

    const bool vec = vector_rows(g);
    const int sw = (row16 >> 1) & 7;
    int slot = 0;
    GroupItem group{};
    for (int tile = static_cast<int>(blockIdx.x); tile < tiles; tile += static_cast<int>(gridDim.x)) {
        const Place place = place_of(tile, group);
        const GemmArgs ge = GROUPED ? group_args<SWIGLU>(g, group) : g;
        f32x4 acc[QB][MB];
#pragma unroll
        for (int q = 0; q < QB; ++q)
#pragma unroll
            for (int b = 0; b < MB; ++b) acc[q][b] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int i = 0; i < mine; ++i) {
            // the piece has landed and the slot of the one before it, whose reads are in registers, may be filled again
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_waitcnt(vmcnt_imm((DEPTH - 2) * kCopies) & 0xf0ffu);
            __builtin_amdgcn_sched_barrier(0);
            copy_next();
            const uint16_t* s = ring + slot * Lds::kPieceHalfs;
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                const int at = row16 * kBK + (((kk * 4 + kg) ^ sw) * 8);
                s16x8 a[QB];
#pragma unroll
                for (int q = 0; q < QB; ++q) a[q] = *reinterpret_cast<const s16x8*>(s + q * kBlock + at);
#pragma unroll
                for (int b = 0; b < MB; ++b) {
                    const s16x8 x = *reinterpret_cast<const s16x8*>(s + (QB + b) * kBlock + at);
#pragma unroll
                    for (int q = 0; q < QB; ++q) acc[q][b] = T::mfma(a[q], x, acc[q][b]);
                }
            }
            slot = slot + 1 == DEPTH ? 0 : slot + 1;
        }
        // acc[q][b]: D[Q row 4 kg + r of block q][P row row16 of block b]. Granule G (4 Q rows) of P row r stands at G
        // ^ r.
        constexpr int kGranules = 4 * QB, kRows = 16 * Lds::kPassBlocks;
#pragma unroll
        for (int b0 = 0; b0 < MB; b0 += Lds::kPassBlocks) {
#pragma unroll
            for (int b = 0; b < Lds::kPassBlocks; ++b)
#pragma unroll
                for (int q = 0; q < QB; ++q)
                    *reinterpret_cast<f32x4*>(sums + ((wave * kRows + b * 16 + row16) * kGranules +
                                                      ((q * 4 + kg) ^ (row16 % kGranules))) * 4) = acc[q][b0 + b];
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0); the copies in flight go on
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
            // a thread has 4 columns of one row
            constexpr int kQuads = kCols / 4;
            for (int i = tid; i < kRows * kQuads; i += WAVES * kWave) {
                const int r = i / kQuads, c = i % kQuads, row = place.row0 + b0 * 16 + r;
                if (row >= ge.m) continue;
                f32x4 z = {0.f, 0.f, 0.f, 0.f}, u = z;
#pragma unroll
                for (int w = 0; w < WAVES; ++w) {
                    const float* at = sums + (w * kRows + r) * kGranules * 4;
                    z = T::add(z, *reinterpret_cast<const f32x4*>(at + (c ^ (r % kGranules)) * 4));
                    const float* ups = at + ((kQuads + c) ^ (r % kGranules)) * 4;
                    if (SWIGLU) u = T::add(u, *reinterpret_cast<const f32x4*>(ups));
                }
                store4<T, SWIGLU>(ge, row, place.nt * kCols + c * 4, z, u, vec);
            }
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt(0xc07f);
            __builtin_amdgcn_s_barrier();  // read before the next sums are written
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
        }
    }
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // the surplus copies have landed before the workgroup ends
}

template <int V>
using Int = std::integral_constant<int, V>;

// Rows of P up to 16, 32 and 64: waves and depths whose rings fill a CU's LDS. Four blocks of weight rows: 8-bit
// products of up to 16 rows
constexpr int kWideBlocks = 4;
template <typename F>
hipError_t by_rows(int m, int qb, F&& f) {
    if (qb == kWideBlocks) return f(Int<kWideBlocks>(), Int<1>(), Int<4>(), Int<3>());
    if (qb == 2) {
        if (m <= 16) return f(Int<2>(), Int<1>(), Int<6>(), Int<3>());
        return m <= 32 ? f(Int<2>(), Int<2>(), Int<4>(), Int<4>()) : f(Int<2>(), Int<4>(), Int<4>(), Int<3>());
    }
    if (m <= 16) return f(Int<1>(), Int<1>(), Int<8>(), Int<3>());
    return m <= 32 ? f(Int<1>(), Int<2>(), Int<4>(), Int<4>()) : f(Int<1>(), Int<4>(), Int<4>(), Int<3>());
}

// Blocks of 16 weight rows in a tile. Two halve what a tile reads of x, for 1.45 times the time of a tile of one, so
// they pay where they save rounds of the GPU: T = 64, H = 2048, N = 7168 (2 rounds -> 1) 14.5 -> 11.6 us, H = 18432 100
// -> 71.5; H = 4096, N = 4096 (1 round either way) 13.7 -> 16.6. Up to 16 rows x costs little, and tiles of one keep
// more copies in flight over several rounds: T = 1, N = 16384, H = 4096 (4 rounds -> 2) 23.3 -> 26.5 us; into a single
// round two are as fast or faster there too (T = 16, N = 7168 9.1 -> 8.2 us).
int tile_blocks(int m, int64_t rows) {
    constexpr int64_t kCus = 256;
    const int64_t one = ((rows + 15) / 16 + kCus - 1) / kCus, two = ((rows + 31) / 32 + kCus - 1) / kCus;
    if (m <= 16) return one == 2 && two == 1 ? 2 : 1;
    return 3 * two < 2 * one ? 2 : 1;
}

template <typename T, int QB, int MB, int WAVES, int DEPTH, bool SWIGLU, bool GROUPED = false>
hipError_t run_stream(const GemmArgs& g, hipStream_t stream) {
    auto fn = &gemm_stream_kernel<T, QB, MB, WAVES, DEPTH, SWIGLU, GROUPED>;
    const void* p = reinterpret_cast<const void*>(fn);
    constexpr int kLds = StreamLds<QB, MB, WAVES, DEPTH>::kBytes, kCols = QB * (SWIGLU ? 8 : 16);
    static_assert(kLds <= 160 * 1024);
    const int tiles = (g.n + kCols - 1) / kCols;
    const int resident = resident_workgroups(p, WAVES * kWave, kLds);
    const int64_t most = GROUPED ? static_cast<int64_t>(g.m / (16 * MB) + min(g.experts, g.m)) * tiles : tiles;
    const int grid = static_cast<int>(resident > 0 && resident < most ? resident : most);
    TraceScope trace(T::kInt8 ? "moe_linear_int8_stream" : "moe_linear_stream", stream);
    fn<<<grid, WAVES * kWave, kLds, stream>>>(g, tiles);
    return hipGetLastError();
}

template <typename T, bool GROUPED = false>
hipError_t prepare(int m, int qb) {
    return by_rows(m, qb, [](auto q, auto mb, auto waves, auto depth) {
        constexpr int Q = decltype(q)::value, M = decltype(mb)::value, W = decltype(waves)::value,
                      D = decltype(depth)::value;
        constexpr int kBytes = StreamLds<Q, M, W, D>::kBytes;
        hipError_t err = ensure_lds_limit(
            reinterpret_cast<const void*>(&gemm_stream_kernel<T, Q, M, W, D, true, GROUPED>), kBytes);
        if (err == hipSuccess)
            err = ensure_lds_limit(
                reinterpret_cast<const void*>(&gemm_stream_kernel<T, Q, M, W, D, false, GROUPED>), kBytes);
        return err;
    });
}

template <typename T, bool GROUPED = false>
hipError_t run_stream_any(const GemmArgs& g, int m, int qb, hipStream_t stream) {
    return by_rows(m, qb, [&](auto q, auto mb, auto waves, auto depth) {
        constexpr int Q = decltype(q)::value, M = decltype(mb)::value, W = decltype(waves)::value,
                      D = decltype(depth)::value;
        return g.act == kActSwiglu ? run_stream<T, Q, M, W, D, true, GROUPED>(g, stream)
                                   : run_stream<T, Q, M, W, D, false, GROUPED>(g, stream);
    });
}

int64_t weight_rows(const GemmArgs& g) { return g.act == kActSwiglu ? 2 * static_cast<int64_t>(g.n) : g.n; }

}  // namespace

hipError_t prepare_gemm_stream() {
    for (const int m : {16, 32, 64})
        for (const int qb : {1, 2}) {
            hipError_t err = prepare<Half>(m, qb);
            if (err == hipSuccess) err = prepare<Bf16>(m, qb);
            if (err != hipSuccess) return err;
        }
    return hipSuccess;
}

hipError_t launch_gemm_stream(const GemmArgs& g, bool bf16, hipStream_t stream) {
    const int qb = tile_blocks(g.m, weight_rows(g));
    return bf16 ? run_stream_any<Bf16>(g, g.m, qb, stream) : run_stream_any<Half>(g, g.m, qb, stream);
}

hipError_t prepare_int8_stream() {
    hipError_t err = hipSuccess;
    for (const int m : {16, 32, 64})
        for (const int qb : {1, 2}) {
            if (err == hipSuccess) err = prepare<Int8<Half>>(m, qb);
            if (err == hipSuccess) err = prepare<Int8<Bf16>>(m, qb);
        }
    if (err == hipSuccess) err = prepare<Int8<Half>>(16, kWideBlocks);
    if (err == hipSuccess) err = prepare<Int8<Bf16>>(16, kWideBlocks);
    if (err == hipSuccess) err = prepare<Int8<Half>, true>(16, kWideBlocks);
    if (err == hipSuccess) err = prepare<Int8<Bf16>, true>(16, kWideBlocks);
    return err;
}

// Experts' products go by 64 weight rows for 16 rows of P. E = 64, H = 2048, N = 1408 SwiGLU, 4 rows an expert on
// average: 63 us, 5.6 TB/s of weights (32 weight rows a tile 72, 16 100; tiles for 32 rows of P 80, for 64 107).
hipError_t launch_int8_stream(const GemmArgs& g, bool bf16, hipStream_t stream) {
    if (g.experts)
        return bf16 ? run_stream_any<Int8<Bf16>, true>(g, 16, kWideBlocks, stream)
                    : run_stream_any<Int8<Half>, true>(g, 16, kWideBlocks, stream);
    // Up to 16 rows the widest tile that gives every CU one; us of 16, 32 and 64 weight rows at T = 1, H = 4096: N =
    // 8192 12.7, 11.0, 11.3, N = 16384 19.6, 16.5, 14.9; H = 14336, N = 4096 12.8, 14.7, 24.1
    const int64_t rows = weight_rows(g);
    const int qb = g.m > 16 ? tile_blocks(g.m, rows) : rows >= 64 * 256 ? kWideBlocks : rows >= 32 * 256 ? 2 : 1;
    return bf16 ? run_stream_any<Int8<Bf16>>(g, g.m, qb, stream) : run_stream_any<Int8<Half>>(g, g.m, qb, stream);
}

}  // namespace moe
