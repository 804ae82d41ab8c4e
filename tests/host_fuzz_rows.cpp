// Host-side fuzz driver for the operators on rows and the 8-bit products (include/moe_ops.h), built with
// AddressSanitizer and UBSan on the host side of libmoe_mi355x.so. It launches no kernel: launch calls get null
// pointers, no rows or a workspace one byte short, which their checks reject or return from before any launch. Sizes
// are seeded random and edge cases. It checks statuses and messages, that a workspace holds what a call puts there
// (column sums, ranks, padded copies) and that no query gives room for sizes its call refuses.
// Usage: host_fuzz_rows ITERATIONS
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <random>

#include "moe_ops.h"

namespace {

const int64_t kEdge[] = {INT64_MIN, -(int64_t{1} << 40), -1, 0, 1, 2, 7, 8, 9, 15, 16, 17, 63, 64, 65, 127, 128, 255, 256, 257,
                         1000, 4097, 16384, 16385, 65536, 131071, 131072, 1 << 20, (1 << 20) + 1, int64_t{1} << 27,
                         (int64_t{1} << 31) - 1, int64_t{1} << 31, int64_t{1} << 40, int64_t{1} << 41, INT64_MAX};
int failures = 0;

void expect(bool ok, const char* what, long long a, long long b, long long c, long long d) {
    if (ok) return;
    if (failures++ < 20) std::printf("FAIL %s: %lld %lld %lld %lld\n", what, a, b, c, d);
}

struct Rng {
    std::mt19937_64 g{20250817};
    int64_t below(int64_t n) { return static_cast<int64_t>(g() % static_cast<uint64_t>(n)); }
    int64_t size() {
        if (below(3) == 0) return kEdge[below(sizeof(kEdge) / sizeof(kEdge[0]))];
        return 1 + below(int64_t{1} << (1 + below(18)));
    }
    int32_t type() { return static_cast<int32_t>(below(4) ? (below(2) ? 1 : 27) : below(30)); }
};

bool good(moe_status st) { return st >= MOE_OK && st <= MOE_ERR_HIP && (st == MOE_OK || std::strlen(moe_last_error()) > 0); }
bool refused(moe_status st) { return good(st) && st != MOE_OK; }

}  // namespace

int main(int argc, char** argv) {
    const long n = argc > 1 ? std::atol(argv[1]) : 20000;
    Rng r;
    char* const p = reinterpret_cast<char*>(uintptr_t{4096});  // never read: no call below reaches a launch
    float* const f = reinterpret_cast<float*>(p);
    int8_t* const q = reinterpret_cast<int8_t*>(p);
    int32_t* const ids = reinterpret_cast<int32_t*>(p);
    for (long i = 0; i < n; ++i) {
        const int64_t T = r.size(), H = r.size(), N = r.size(), ld = r.below(2) ? H : r.size();
        const int64_t E = r.below(2) ? r.below(300) : r.size(), K = r.below(2) ? 1 + r.below(16) : r.size();
        const int32_t dt = r.type(), gt = r.below(2) ? dt : r.type(), wt = r.type();
        const float eps = r.below(8) ? 1e-6f : r.below(2) ? 0.0f : -1.0f;
        // null operands: refused, or nothing to do
        moe_status st = moe_add_rms_norm(nullptr, ld, nullptr, ld, nullptr, gt, p, nullptr, nullptr, nullptr, T, H, eps, dt,
                                         nullptr);
        expect(good(st) && (st != MOE_OK || T == 0), "norm of nothing", T, H, dt, st);
        st = moe_quantize(nullptr, ld, q, f, T, H, dt, nullptr);
        expect(good(st) && (st != MOE_OK || T == 0), "quantise nothing", T, H, dt, st);
        const size_t nws = moe_add_rms_norm_grad_workspace_bytes(T, H);
        st = moe_add_rms_norm_grad(p, ld, p, ld, p, gt, nullptr, 0, p, p, p, nws > 0 ? nws - 1 : 0, T, H, eps, dt, nullptr);
        expect(refused(st), "norm gradient without room", T, H, dt, st);
        expect(nws == 0 || nws % (static_cast<size_t>(H) * 4) == 0, "rows of column sums", T, H, dt, nws);
        st = moe_unpermute(nullptr, r.size(), nullptr, p, wt, nullptr, T, H, K, dt, nullptr);
        expect(good(st) && (st != MOE_OK || T == 0), "way back of nothing", T, H, K, st);
        st = moe_unpermute_grad(nullptr, ld, nullptr, nullptr, p, wt, nullptr, nullptr, T, H, K, dt, nullptr);
        expect(good(st) && (st != MOE_OK || T == 0), "its gradient of nothing", T, H, K, st);
        const size_t sws = moe_permute_workspace_bytes(T, E, K);
        st = moe_permute(p, ld, nullptr, ids, p, nullptr, nullptr, ids, p, sws, T, H, E, K, dt, nullptr);
        expect(refused(st), "sorting without offsets", T, E, K, st);
        if (sws > 0) {
            expect(sws >= static_cast<size_t>(T * K) * 4, "room for ranks", T, E, K, sws);
            st = moe_permute(p, ld, nullptr, ids, p, nullptr, ids, ids, p, sws - 1, T, H, E, K, dt, nullptr);
            expect(refused(st), "sorting one byte short", T, E, K, st);
        }
        const int32_t act = static_cast<int32_t>(r.below(8)) - 1;
        const int64_t halves = act == MOE_ACT_SWIGLU ? 2 : 1, ldw = r.below(2) ? H : r.size(), step = r.size();
        const size_t ws = moe_linear_int8_workspace_bytes(T, N, H, E, act);
        st = moe_linear_int8(nullptr, ld, f, q, ldw, step, f, ids, nullptr, nullptr, p, p, ws, T, N, H, E, act, dt, nullptr);
        expect(good(st) && (st != MOE_OK || T == 0), "8-bit product of nothing", T, N, H, st);
        if (ws > 0) {
            st = moe_linear_int8(q, ld, f, q, ldw, step, f, ids, nullptr, nullptr, p, p, ws - 1, T, N, H, E, act, dt, nullptr);
            expect(refused(st), "8-bit product one byte short", T, N, H, st);
            const size_t h16 = static_cast<size_t>((H + 15) / 16 * 16), groups = E > 0 ? E : 1;
            if (H % 16 && T >= (E > 0 ? 32 * E : 256))
                expect(ws >= (static_cast<size_t>(T) + groups * halves * N) * h16, "room for padded rows", T, N, H, E);
        }
    }
    std::printf("%ld iterations, %d failures\n", n, failures);
    return failures == 0 ? 0 : 1;
}
