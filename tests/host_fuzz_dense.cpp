// Host-side fuzz driver for the operators around the routed experts (include/moe_ops.h), built with AddressSanitizer and
// UBSan on the host side of libmoe_mi355x.so. It launches no kernel: launch calls get null pointers, no tokens or a
// workspace one byte short, which their checks reject or return from before any launch. Sizes are seeded random and edge
// cases. It checks statuses and messages, that a workspace holds what a call puts there (dz, and padded copies of rows that
// are no multiple of 16 bytes), and that no query gives room for sizes its call refuses.
// Usage: host_fuzz_dense ITERATIONS
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <random>

#include "moe_ops.h"

namespace {

const int64_t kEdge[] = {-(int64_t{1} << 40), -1, 0, 1, 2, 3, 7, 8, 9, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255,
                         256, 257, 1000, 1056, 4097, 16384, 65536, 1 << 20, (1 << 20) + 1, (int64_t{1} << 27) - 1,
                         int64_t{1} << 27, (int64_t{1} << 31) - 1, int64_t{1} << 31, int64_t{1} << 40, INT64_MAX};
int failures = 0;

void expect(bool ok, const char* what, long long a, long long b, long long c, long long d) {
    if (ok) return;
    if (failures++ < 20) std::printf("FAIL %s: %lld %lld %lld %lld\n", what, a, b, c, d);
}

struct Rng {
    std::mt19937_64 g{20240611};
    int64_t below(int64_t n) { return static_cast<int64_t>(g() % static_cast<uint64_t>(n)); }
    int64_t size() {
        if (below(3) == 0) return kEdge[below(sizeof(kEdge) / sizeof(kEdge[0]))];
        return 1 + below(int64_t{1} << (1 + below(18)));
    }
};

bool good(moe_status st) { return st >= MOE_OK && st <= MOE_ERR_HIP && (st == MOE_OK || std::strlen(moe_last_error()) > 0); }

}  // namespace

int main(int argc, char** argv) {
    const long n = argc > 1 ? std::atol(argv[1]) : 20000;
    Rng r;
    char* const p = reinterpret_cast<char*>(uintptr_t{4096});  // never read: no call below reaches a launch
    for (long i = 0; i < n; ++i) {
        const int64_t T = r.size(), N = r.size(), H = r.size();
        const int32_t act = static_cast<int32_t>(r.below(8)) - 1, dt = r.below(2) ? MOE_DT_FLOAT16 : MOE_DT_BFLOAT16;
        const int64_t halves = act == MOE_ACT_SWIGLU ? 2 : 1;
        const size_t ws = moe_linear_workspace_bytes(T, N, H, act), gws = moe_linear_grad_workspace_bytes(T, N, H, act);
        const bool sized = T > 0 && N > 0 && H > 0 && T < (int64_t{1} << 40) && N <= (1 << 20) && H <= (1 << 20);
        const int64_t ldx = sized ? H + r.below(3) : r.size();
        const int32_t tr = static_cast<int32_t>(r.below(2));
        const int64_t ldw = sized ? (tr ? halves * N : H) + r.below(3) : r.size();
        // null operands: refused, or no tokens
        moe_status st = moe_linear(nullptr, ldx, nullptr, ldw, tr, nullptr, nullptr, nullptr, nullptr, nullptr, 0, T, N, H,
                                   act, dt, dt, nullptr);
        expect(good(st) && (st != MOE_OK || T == 0), "linear of nothing", T, N, H, st);
        if (ws > 0) {
            st = moe_linear(p, ldx, p, ldw, tr, nullptr, nullptr, p, nullptr, p, ws - 1, T, N, H, act, dt, dt, nullptr);
            expect(good(st) && (st != MOE_OK || T == 0), "linear one byte short", T, N, H, st);
            if (sized) expect(st == MOE_ERR_WORKSPACE, "linear workspace", T, N, H, st);
        }
        if (sized && gws > 0) {
            const size_t h8 = (H + 7) / 8 * 8, n8 = (N + 7) / 8 * 8, z8 = (halves * N + 7) / 8 * 8;
            if (H % 8) {
                expect(ws >= T * h8 * 2 + halves * N * h8 * 2, "room for x and the weight", T, N, H, act);
                expect(gws >= T * z8 * 2 + T * h8 * 2 + halves * N * h8 * 2, "room of the gradients", T, N, H, act);
            }
            if (N % 8) expect(ws >= H * halves * n8 * 2, "room for a transposed weight", T, N, H, act);
            expect(gws >= T * z8 * 2, "room for dz", T, N, H, act);
            st = moe_linear_grad(p, N, p, ldx, p, ldw, tr, p, p, p, p, p, gws - 1, T, N, H, act, dt, nullptr);
            expect(st == MOE_ERR_WORKSPACE, "gradient one byte short", T, N, H, st);
        } else if (gws == 0) {  // sizes that the query refuses are refused by the call
            st = moe_linear_grad(p, N, p, ldx, p, ldw, tr, p, p, p, p, p, 0, T, N, H, act, dt, nullptr);
            expect(good(st) && st != MOE_OK, "gradient without room", T, N, H, st);
        }
        st = moe_linear_grad(nullptr, N, nullptr, ldx, nullptr, ldw, tr, nullptr, p, nullptr, nullptr, nullptr, 0, T, N, H,
                             act, dt, nullptr);
        expect(good(st) && (st != MOE_OK || T == 0), "gradient of nothing", T, N, H, st);

        const int64_t E = r.below(2) ? 1 + r.below(300) : r.size(), K = r.below(2) ? 1 + r.below(16) : r.size();
        const int64_t G = r.below(2) ? 1 : r.size(), TG = r.below(2) ? 1 : r.size();
        const int32_t lt = static_cast<int32_t>(r.below(30)), wt = static_cast<int32_t>(r.below(30));
        st = moe_routing_group_topk(nullptr, E, lt, nullptr, nullptr, nullptr, wt, T, E, K, G, TG, 1 + r.below(2),
                                    static_cast<int32_t>(r.below(3)), 1, 1.0f, nullptr);
        expect(good(st) && (st != MOE_OK || T == 0), "routing of nothing", T, E, K, st);
        st = moe_routing_group_topk_grad(nullptr, wt, nullptr, E, lt, nullptr, nullptr, T, E, K,
                                         static_cast<int32_t>(r.below(3)), 1, 1.0f, nullptr);
        expect(good(st) && (st != MOE_OK || T == 0), "routing gradient of nothing", T, E, K, st);
        st = moe_combine_grad(nullptr, nullptr, nullptr, nullptr, nullptr, T, H, K, nullptr);
        expect(good(st) && (st != MOE_OK || T == 0), "combine gradient of nothing", T, H, K, st);
    }
    std::printf("%ld iterations, %d failures\n", n, failures);
    return failures == 0 ? 0 : 1;
}
