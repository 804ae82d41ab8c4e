// moe_linear_int8.hip -- MoeLinearInt8 for gfx950 on tiles of 32 to 256 rows by 128, and the sum of a split product's
// pieces: y = act((x W^T) x_scale w_scale + b) + r with 8-bit integers x and W.
//
// A 16-byte fragment of v_mfma_i32_16x16x64_i8 has 16 integers of a row where the 16-bit types have 8 values, and takes
// as long, so the kernels of moe_linear_mid.h (and of moe_linear_stream.hip and moe_linear_tiled.hip) move and multiply
// the same bytes at twice the rate. The int32 sums are exact: pieces of k and experts' tiles give the same bits in any
// order. What differs is the epilogue, which converts and scales (moe_gemm.h), and the experts' products: a workgroup
// finds the expert of its tile from the offsets, by all lanes at once.
//   E = 64, T = 768, H = 2048, N = 1408 SwiGLU (tiles of 64 rows): 76 us, 4.9 TB/s of weights
#include "moe_linear_mid.h"

namespace moe {

namespace {

template <typename T, int BM, bool GROUPED>
hipError_t run_int8(const GemmArgs& g, bool direct, hipStream_t stream) {
    if (g.act == kActSwiglu)
        return direct ? run_mid<T, false, false, BM, true, true, GROUPED>(g, stream)
                      : run_mid<T, false, false, BM, true, false, GROUPED>(g, stream);
    return direct ? run_mid<T, false, false, BM, false, true, GROUPED>(g, stream)
                  : run_mid<T, false, false, BM, false, false, GROUPED>(g, stream);
}
template <typename T>
hipError_t run_int8_any(const GemmArgs& g, bool direct, int bm, hipStream_t stream) {
    if (g.experts && bm == 64) return run_int8<T, 64, true>(g, direct, stream);
    if (g.experts)  // operands through registers only
        return g.act == kActSwiglu ? run_mid<T, false, false, 128, true, false, true>(g, stream)
                                   : run_mid<T, false, false, 128, false, false, true>(g, stream);
    if (bm == 256)  // direct operands only
        return g.act == kActSwiglu ? run_mid<T, false, false, 256, true, true>(g, stream)
                                   : run_mid<T, false, false, 256, false, true>(g, stream);
    if (bm == 128) return run_int8<T, 128, false>(g, direct, stream);
    return bm == 64 ? run_int8<T, 64, false>(g, direct, stream) : run_int8<T, 32, false>(g, direct, stream);
}

template <typename T, int BM, bool GROUPED>
hipError_t prepare_int8_bm() {
    for (const void* fn :
         {reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, false, BM, false, true, GROUPED>),
          reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, false, BM, true, true, GROUPED>),
          reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, false, BM, false, false, GROUPED>),
          reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, false, BM, true, false, GROUPED>)}) {
        const hipError_t err = ensure_lds_limit(fn, mid_lds_bytes(BM));
        if (err != hipSuccess) return err;
    }
    return hipSuccess;
}
template <typename T>
hipError_t prepare_int8() {
    hipError_t err = prepare_int8_bm<T, 32, false>();
    if (err == hipSuccess) err = prepare_int8_bm<T, 64, false>();
    if (err == hipSuccess) err = prepare_int8_bm<T, 64, true>();
    for (const void* fn : {reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, false, 256, false, true>),
                           reinterpret_cast<const void*>(&gemm_mid_kernel<T, false, false, 256, true, true>)})
        if (err == hipSuccess) err = ensure_lds_limit(fn, mid_lds_bytes(256));
    return err;
}

}  // namespace

hipError_t launch_int8_mid(const GemmArgs& g, bool bf16, bool direct, int bm, hipStream_t stream) {
    return bf16 ? run_int8_any<Int8<Bf16>>(g, direct, bm, stream) : run_int8_any<Int8<Half>>(g, direct, bm, stream);
}

hipError_t launch_int8_reduce(const GemmArgs& g, bool bf16, hipStream_t stream) {
    const bool swiglu = g.act == kActSwiglu;
    const int grid = static_cast<int>(reduce_blocks(g));
    TraceScope trace("moe_linear_int8_reduce", stream);
    if (bf16) {
        if (swiglu) gemm_reduce_kernel<Int8<Bf16>, true><<<grid, kReduceThreads, 0, stream>>>(g);
        else gemm_reduce_kernel<Int8<Bf16>, false><<<grid, kReduceThreads, 0, stream>>>(g);
    } else {
        if (swiglu) gemm_reduce_kernel<Int8<Half>, true><<<grid, kReduceThreads, 0, stream>>>(g);
        else gemm_reduce_kernel<Int8<Half>, false><<<grid, kReduceThreads, 0, stream>>>(g);
    }
    return hipGetLastError();
}

hipError_t prepare_int8_mid() {  // 128-row tiles keep within 64 KB
    const hipError_t err = prepare_int8<Int8<Half>>();
    return err == hipSuccess ? prepare_int8<Int8<Bf16>>() : err;
}

}  // namespace moe
