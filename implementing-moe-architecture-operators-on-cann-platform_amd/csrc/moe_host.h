// moe_host.h -- what the C-ABI host files (moe_ops.cpp, moe_dense_ops.cpp) share: the error string and argument checks.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "moe_ops.h"

namespace moe {
namespace host {

// Sets the calling thread's error message and returns `st`.
moe_status fail(moe_status st, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
moe_status ok();  // clears it
moe_status hip_fail(hipError_t err, const char* what);
const char* last_error();

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline hipStream_t as_stream(void* s) { return static_cast<hipStream_t>(s); }

constexpr int64_t kMaxExperts = 256;
constexpr int64_t kInt32Max = 2147483647;
// hiddenSize and intermediateSize bound: far above any model's, and small enough that the products of sizes the
// checks form stay within 64 bits
constexpr int64_t kMaxDim = int64_t{1} << 20;

// a * b > limit for a, b >= 0, without forming a product that could overflow
inline bool product_exceeds(int64_t a, int64_t b, int64_t limit) { return b != 0 && a > limit / b; }

}  // namespace host
}  // namespace moe
