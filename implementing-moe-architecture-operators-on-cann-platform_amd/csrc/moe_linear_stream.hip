// moe_linear_stream.hip -- the dense product of few rows (serving's single tokens and small batches): weight streaming.
//
// C[m][n] = sum_k P[m][k] Q[n][k], both operands by rows, m <= 32. The weights are read once and bound it: at T = 1 the
// gate and up rows of a dense expert are 59 MB for 59 MFLOP.
//   work      a tile is 16 weight rows (SwiGLU: 8 gate and the matching 8 up rows) over the whole k, and its workgroup's
//             waves share k: wave w takes the 64-k pieces w, w + W, ... Their sums meet in LDS, added in wave order, and
//             go through the epilogue: one launch, no partial sums in memory.
//   copies    each wave has its own LDS ring and fills it straight from global memory, 8 rows x 128 bytes an instruction;
//             nobody else reads it, so the main loop has no barrier. Loaded into registers in fragment order (16 rows x
//             64 bytes an instruction) the same work ran at 4.2 TB/s.
//   persistent  a workgroup per CU walks its tiles and the rings run on across them, so the next tile's weights are in
//             flight while the sums of this one are added.
// Rows past the last and k past the end read zeros without memory traffic.
#include "moe_gemm.h"

#include <type_traits>

namespace moe {

namespace {

constexpr int kBK = 64;                     // k of a piece
constexpr int kBlock = 16 * kBK;            // halfs of 16 rows of a piece
constexpr uint32_t kPastEnd = 0x80000000u;  // a buffer offset past every buffer: the load returns zeros
constexpr int kNonTemporal = 2;             // cache policy of the weights: read once

// MB: blocks of 16 rows of P; DEPTH: pieces of a wave's ring
template <int MB, int WAVES, int DEPTH>
struct StreamLds {
    static constexpr int kPieceHalfs = (1 + MB) * kBlock;
    static constexpr int kRings = WAVES * DEPTH * kPieceHalfs * 2;
    static constexpr int kSums = WAVES * MB * 16 * 17 * 4;
    static constexpr int kBytes = kRings + kSums;
};

template <typename T, int MB, int WAVES, int DEPTH, bool SWIGLU>
__global__ __launch_bounds__(WAVES * kWave) void gemm_stream_kernel(GemmArgs g, int tiles) {
    using Lds = StreamLds<MB, WAVES, DEPTH>;
    constexpr int kCopies = 2 * (1 + MB);
    extern __shared__ __align__(16) uint16_t lds[];
    float(*sums)[MB * 16][17] = reinterpret_cast<float(*)[MB * 16][17]>(lds + Lds::kRings / 2);  // [wave][P row][Q row]
    const int tid = static_cast<int>(threadIdx.x), lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int row16 = lane & 15, kg = lane >> 4;
    uint16_t* ring = lds + wave * DEPTH * Lds::kPieceHalfs;

    // Copy instruction i of a block: rows 8 i + lane / 8; granule G (8 k) of row r stands at G ^ (r >> 1 & 7)
    const int r8 = lane / 8, gran = (lane % 8) ^ (r8 >> 1);  // of instruction 0; instruction 1: granule ^ 4
    const uint32_t ppitch = static_cast<uint32_t>(g.ldp) * 2, qpitch = static_cast<uint32_t>(g.ldq) * 2;
    const __amdgpu_buffer_rsrc_t pr =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(g.p), 0, 0x7fffffff, 0x00020000);

    const int stages = (g.k + kBK - 1) / kBK;
    const int mine = stages > wave ? (stages - wave + WAVES - 1) / WAVES : 0;  // pieces of this wave per tile
    // the wave's pieces of all its tiles in a row: where the next copy is
    int ctile = static_cast<int>(blockIdx.x), cpiece = 0, cslot = 0;
    auto copy_next = [&]() __attribute__((always_inline)) {
        uint16_t* slot = ring + cslot * Lds::kPieceHalfs;
        const int k0 = (wave + cpiece * WAVES) * kBK;
        const bool live = ctile < tiles && mine > 0;
        const int n0 = ctile * (SWIGLU ? 8 : 16);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int k = k0 + ((gran ^ (4 * i)) * 8);
            const int col = n0 + (SWIGLU ? r8 : 8 * i + r8);
            // SwiGLU: instruction 0 the gate rows, 1 the up rows
            const int64_t first = n0 + (SWIGLU && i == 1 ? static_cast<int64_t>(g.up) : 0);
            const __amdgpu_buffer_rsrc_t qr = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<uint16_t*>(live ? g.q + first * g.ldq : g.q), 0, 0x7fffffff, 0x00020000);
            const uint32_t off = static_cast<uint32_t>(col - n0) * qpitch + static_cast<uint32_t>(k) * 2;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                qr, (__attribute__((address_space(3))) void*)(slot + i * 512), 16,
                static_cast<int>(live && col < g.n && k < g.k ? off : kPastEnd), 0, 0, kNonTemporal);
        }
#pragma unroll
        for (int i = 0; i < 2 * MB; ++i) {
            const int row = 8 * i + r8, k = k0 + ((gran ^ (4 * (i & 1))) * 8);
            const uint32_t off = static_cast<uint32_t>(row) * ppitch + static_cast<uint32_t>(k) * 2;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                pr, (__attribute__((address_space(3))) void*)(slot + kBlock + i * 512), 16,
                static_cast<int>(live && row < g.m && k < g.k ? off : kPastEnd), 0, 0, 0);
        }
        cslot = cslot + 1 == DEPTH ? 0 : cslot + 1;
        if (++cpiece >= mine) {
            cpiece = 0;
            ctile += static_cast<int>(gridDim.x);
        }
    };
#pragma unroll
    for (int d = 0; d < DEPTH - 1; ++d) copy_next();

    const bool vec = vector_rows(g);
    const int sw = (row16 >> 1) & 7;
    int slot = 0;
    for (int tile = static_cast<int>(blockIdx.x); tile < tiles; tile += static_cast<int>(gridDim.x)) {
        f32x4 acc[MB];
#pragma unroll
        for (int b = 0; b < MB; ++b) acc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
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
                const s16x8 a = *reinterpret_cast<const s16x8*>(s + at);
#pragma unroll
                for (int b = 0; b < MB; ++b)
                    acc[b] = T::mfma(a, *reinterpret_cast<const s16x8*>(s + (1 + b) * kBlock + at), acc[b]);
            }
            slot = slot + 1 == DEPTH ? 0 : slot + 1;
        }
        // acc[b]: D[Q row 4 kg + r][P row row16 of block b]
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) sums[wave][b * 16 + row16][kg * 4 + r] = acc[b][r];
        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0); the copies in flight go on
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
        // a thread has 4 columns of one row
        constexpr int kQuads = SWIGLU ? 2 : 4;
        for (int i = tid; i < MB * 16 * kQuads; i += WAVES * kWave) {
            const int row = i / kQuads, c = i % kQuads * 4;
            if (row >= g.m) continue;
            f32x4 z = {0.f, 0.f, 0.f, 0.f}, u = z;
#pragma unroll
            for (int w = 0; w < WAVES; ++w)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    z[r] += sums[w][row][c + r];
                    if (SWIGLU) u[r] += sums[w][row][8 + c + r];
                }
            store4<T, SWIGLU>(g, row, tile * (SWIGLU ? 8 : 16) + c, z, u, vec);
        }
        __builtin_amdgcn_s_waitcnt(0xc07f);
        __builtin_amdgcn_s_barrier();  // read before the next tile's sums are written
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    }
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // the surplus copies have landed before the workgroup ends
}

template <typename T, int MB, int WAVES, int DEPTH, bool SWIGLU>
hipError_t run_stream(const GemmArgs& g, hipStream_t stream) {
    auto fn = &gemm_stream_kernel<T, MB, WAVES, DEPTH, SWIGLU>;
    const void* p = reinterpret_cast<const void*>(fn);
    constexpr int kLds = StreamLds<MB, WAVES, DEPTH>::kBytes;
    const int tiles = (g.n + (SWIGLU ? 7 : 15)) / (SWIGLU ? 8 : 16);
    const int resident = resident_workgroups(p, WAVES * kWave, kLds);
    TraceScope trace("moe_linear_stream", stream);
    fn<<<resident > 0 && resident < tiles ? resident : tiles, WAVES * kWave, kLds, stream>>>(g, tiles);
    return hipGetLastError();
}

template <typename T, int MB, int WAVES, int DEPTH>
hipError_t run_stream_act(const GemmArgs& g, hipStream_t stream) {
    return g.act == kActSwiglu ? run_stream<T, MB, WAVES, DEPTH, true>(g, stream)
                               : run_stream<T, MB, WAVES, DEPTH, false>(g, stream);
}

// rows of P up to 16, 32 and 64
template <typename F>
hipError_t by_rows(int m, F&& f) {
    if (m <= 16) return f(std::integral_constant<int, 1>(), std::integral_constant<int, 8>(), std::integral_constant<int, 3>());
    if (m <= 32) return f(std::integral_constant<int, 2>(), std::integral_constant<int, 4>(), std::integral_constant<int, 4>());
    return f(std::integral_constant<int, 4>(), std::integral_constant<int, 4>(), std::integral_constant<int, 3>());
}

template <typename T>
hipError_t prepare(int m) {
    return by_rows(m, [](auto mb, auto waves, auto depth) {
        constexpr int M = decltype(mb)::value, W = decltype(waves)::value, D = decltype(depth)::value;
        hipError_t err = ensure_lds_limit(reinterpret_cast<const void*>(&gemm_stream_kernel<T, M, W, D, true>),
                                          StreamLds<M, W, D>::kBytes);
        if (err == hipSuccess)
            err = ensure_lds_limit(reinterpret_cast<const void*>(&gemm_stream_kernel<T, M, W, D, false>),
                                   StreamLds<M, W, D>::kBytes);
        return err;
    });
}

template <typename T>
hipError_t run_stream_any(const GemmArgs& g, hipStream_t stream) {
    return by_rows(g.m, [&](auto mb, auto waves, auto depth) {
        return run_stream_act<T, decltype(mb)::value, decltype(waves)::value, decltype(depth)::value>(g, stream);
    });
}

}  // namespace

hipError_t prepare_gemm_stream() {
    for (const int m : {16, 32, 64}) {
        hipError_t err = prepare<Half>(m);
        if (err == hipSuccess) err = prepare<Bf16>(m);
        if (err != hipSuccess) return err;
    }
    return hipSuccess;
}

hipError_t launch_gemm_stream(const GemmArgs& g, bool bf16, hipStream_t stream) {
    return bf16 ? run_stream_any<Bf16>(g, stream) : run_stream_any<Half>(g, stream);
}

}  // namespace moe
