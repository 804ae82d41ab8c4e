// moe_dense_ops.cpp -- host side of the operators around the routed experts (include/moe_ops.h): routing from logits,
// the dense product with its epilogue, and the gradients of both and of the combine.
//
// As moe_ops.cpp: nothing here allocates device memory, and every check runs before the first launch.

#include <hip/hip_runtime.h>

#include "moe_gemm.h"
#include "moe_host.h"
#include "moe_launch.h"
#include "moe_ops.h"

using namespace moe::host;

namespace {

bool is_half(int32_t t) { return t == MOE_DT_FLOAT16 || t == MOE_DT_BFLOAT16; }
int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

// ------------------------------------------------------------------------------------------------
// routing from logits
// ------------------------------------------------------------------------------------------------

moe_status check_group_routing(const char* op, int64_t T, int64_t E, int64_t K, int64_t ld, int32_t logits_type,
                               int32_t weights_type, bool grad) {
    if (T < 0 || E <= 0) return fail(MOE_ERR_ARG, "%s: sizes must be T >= 0, E > 0 (T=%lld E=%lld)", op, (long long)T,
                                     (long long)E);
    if (K < 1 || K > E) return fail(MOE_ERR_ARG, "%s: topK=%lld must be in [1, numExperts=%lld]", op, (long long)K,
                                    (long long)E);
    if (E > kMaxExperts)
        return fail(MOE_ERR_UNSUPPORTED, "%s: numExperts=%lld exceeds %lld", op, (long long)E, (long long)kMaxExperts);
    if (T >= int64_t{1} << 27) return fail(MOE_ERR_UNSUPPORTED, "%s: T=%lld too large", op, (long long)T);
    if (ld < E || ld > kInt32Max)
        return fail(MOE_ERR_ARG, "%s: logits rows %lld elements apart hold %lld", op, (long long)ld, (long long)E);
    if (logits_type != MOE_DT_FLOAT32 && !is_half(logits_type))
        return fail(MOE_ERR_ARG, "%s: logits type %d (float32, float16 or bfloat16 expected)", op, logits_type);
    if (weights_type != MOE_DT_FLOAT32 && weights_type != MOE_DT_FLOAT16 && !(grad && weights_type == MOE_DT_BFLOAT16))
        return fail(MOE_ERR_ARG, "%s: weights type %d (float32 or float16%s expected)", op, weights_type,
                    grad ? " or bfloat16" : "");
    return ok();
}

moe_status check_scoring(const char* op, int32_t scoring, float scale) {
    if (scoring != MOE_SCORE_SOFTMAX && scoring != MOE_SCORE_SIGMOID)
        return fail(MOE_ERR_ARG, "%s: scoring %d", op, scoring);
    if (!(scale - scale == 0.0f)) return fail(MOE_ERR_ARG, "%s: scale must be finite", op);
    return ok();
}

// ------------------------------------------------------------------------------------------------
// dense products
// ------------------------------------------------------------------------------------------------

constexpr int kMaxActivation = MOE_ACT_SWIGLU;
constexpr int64_t kMaxTiles = int64_t{1} << 23;  // workgroups of a launch, far below HIP's 2^32 threads

moe_status check_linear(const char* op, int64_t T, int64_t N, int64_t H, int32_t act, int32_t dtype) {
    if (T < 0 || N <= 0 || H <= 0)
        return fail(MOE_ERR_ARG, "%s: sizes must be T >= 0, N > 0, H > 0 (T=%lld N=%lld H=%lld)", op, (long long)T,
                    (long long)N, (long long)H);
    if (act < 0 || act > kMaxActivation) return fail(MOE_ERR_ARG, "%s: activation %d", op, act);
    if (!is_half(dtype)) return fail(MOE_ERR_ARG, "%s: type %d (float16 or bfloat16 expected)", op, dtype);
    if (N > kMaxDim || H > kMaxDim)
        return fail(MOE_ERR_UNSUPPORTED, "%s: N=%lld, H=%lld exceed %lld", op, (long long)N, (long long)H,
                    (long long)kMaxDim);
    // 128 x 128 tiles (64 columns of a SwiGLU) of the forward and of both gradients
    if (T > kInt32Max || ((T + 127) / 128) * ((N > H ? N : H) / 64 + 1) >= kMaxTiles ||
        (N / 64 + 1) * (H / 128 + 1) >= kMaxTiles)
        return fail(MOE_ERR_UNSUPPORTED, "%s: T=%lld N=%lld H=%lld too large", op, (long long)T, (long long)N,
                    (long long)H);
    return ok();
}

moe_status check_pitch(const char* op, const char* what, int64_t rows, int64_t width, int64_t ld) {
    if (rows > 1 && ld < width)
        return fail(MOE_ERR_ARG, "%s: %s rows overlap (%lld elements apart, %lld long)", op, what, (long long)ld,
                    (long long)width);
    if (ld > int64_t{1} << 40 || ld < 0) return fail(MOE_ERR_ARG, "%s: %s stride %lld", op, what, (long long)ld);
    return ok();
}

// How one product runs: weight streaming, tiles of 32 to 256 x 128 (split over k or not), or 256 x 256 tiles
enum class Kernel { kStream, kMid, kTiled };
constexpr double kLaunchSaved = 6.0;  // us of a second launch's start and of the CUs its first round leaves idle

struct ProductPlan {
    Kernel kernel;
    int bm;  // kMid: rows of a tile
    int splits;
    int64_t split_k;
    size_t partial_bytes;
    double us;  // expected, of kMid and kTiled
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Microseconds of a launch by tiles of bm x 128 with `items` workgroups of `stages` 64-k stages. Up to 128 rows two
// workgroups share a CU: a stage takes `one` alone and `two` beside another. At 256 rows a CU has one: `one` with few
// of them, `two` with one on every CU. A launch takes `launch` besides, and each further round of the GPU `round` for
// its first copies and its epilogue. Where P is read by k too, both operands go through transposing reads.
double mid_time(int bm, int64_t items, int64_t stages, bool p_by_k) {
    struct Cost {
        double one, two, launch, round;
    };
    const Cost c = p_by_k      ? (bm == 128 ? Cost{0.70, 0.93, 5.6, 8.8} : Cost{0.89, 0.96, 7.1, 8.4})
                   : bm == 32  ? Cost{0.30, 0.55, 5.5, 3.0}
                   : bm == 64  ? Cost{0.37, 0.65, 5.5, 3.5}
                   : bm == 128 ? Cost{0.56, 0.92, 7.2, 6.0}
                               : Cost{0.75, 0.93, 9.1, 5.6};
    const int64_t slots = bm == 256 ? 256 : 512, rest = items % slots;
    const double tail = rest == 0 ? 0.0
                        : bm == 256 ? c.one + (c.two - c.one) * (rest / 256.0)
                                    : rest <= 256 ? c.one : c.one + (c.two - c.one) * (rest / 256.0 - 1.0);
    return c.launch + c.round * static_cast<double>(ceil_div(items, slots) - 1) +
           stages * (static_cast<double>(items / slots) * c.two + tail);
}
// The same of 256 x 256 tiles: one workgroup a CU, 1.0 us a stage with few tiles up to 1.46 with one on every CU (the
// clock falls), 7 to 10 us of first copies and epilogue a round, of 8-bit products 4 to 5.
double tiled_time(int64_t tiles, int64_t stages, bool p_by_k, bool int8) {
    const double launch = p_by_k ? 7.1 : 5.8, round = p_by_k ? 9.4 : int8 ? 4.5 : 10.2, stage = p_by_k ? 1.59 : 1.46;
    const double few_round = p_by_k ? 7.4 : int8 ? 4.0 : 6.7, few_stage = p_by_k ? 1.2 : 1.01;
    const double more = p_by_k ? 0.43 : 0.41;
    const double f = (tiles % 256) / 256.0;
    const double tail =
        tiles % 256 == 0 ? 0.0 : few_round + (round - few_round) * f + stages * (few_stage + more * f * f);
    return launch + static_cast<double>(tiles / 256) * (round + stage * stages) + tail;
}
// Microseconds of adding a split product's pieces in a launch of its own, their writes counted
double reduce_time(size_t partial, bool p_by_k) {
    return (p_by_k ? 1.7 : 0.1) + 2.0 * static_cast<double>(partial) / (p_by_k ? 6.2e6 : 5.2e6);
}

// The kernel with the least time by those figures, which are fitted to every kernel's times in 306 products (T = 128 ..
// 16384, N and H = 64 .. 12288, in the forward's two layouts and the weight gradient's): of those products the choice
// is the fastest kernel or 0.3 % slower on average, 16 % at worst (T = 16384, N = 256, H = 7168, where all are within
// that). A product by tiles is split over k while that leaves eight stages a piece and at most the workgroups that the
// GPU holds; the pieces' sums then take another launch.
// Few rows stream the weights where both operands are read by rows: T = 16, H = 2048, N = 7168 8.2 us (tiles of 32 rows
// 11.5), T = 64 11.6 (16.0). Above 16 rows that holds between 64 and 512 tiles of 16 weight rows: T = 32, H = 7168, N =
// 256 12.4 us (8.3 split over k), T = 64, H = 4096, N = 16384 35 us (33). Up to 16 rows a call takes 8.3 to 8.9 us from
// N = 8 to 512 and H = 2048 to 8192, the host's time, where two launches take 10.7.
// 8-bit products (k in pairs) take the same times but for the epilogue of their 256 x 256 tiles, and above 16 rows
// stream up to 512 tiles: H = 4096, N = 14336 SwiGLU (1792 tiles) at T = 32 30 us, tiles of 32 rows 24. Of 90 products
// (T = 1 .. 16384) the choice is the fastest kernel or 1 to 2 % slower on average.
// most_rows: the tallest tiles to choose from.
ProductPlan plan_product(int64_t m, int64_t n, int64_t k, bool swiglu, bool p_by_k, bool q_by_k, bool direct,
                         int most_rows = 256, bool int8 = false) {
    ProductPlan best{Kernel::kMid, 128, 1, ceil_div(k > 0 ? k : 1, 64) * 64, 0, 1e30};
    const int64_t stages = ceil_div(k > 0 ? k : 1, 64);
    if (direct && !p_by_k && !q_by_k && m <= 64) {
        const int64_t tiles = ceil_div(n, swiglu ? 8 : 16);
        if (m <= 16 || (tiles >= 64 && ((m <= 32 && !int8) || tiles <= 512))) {
            best.kernel = Kernel::kStream;
            return best;
        }
    }
    for (const int bm : {32, 64, 128, 256}) {
        if (bm == 32 ? m > 32 : bm == 64 ? m <= 32 : bm == 128 ? !p_by_k && m <= 64 : !direct || m <= 128) continue;
        if ((bm < 128 && p_by_k) || bm > most_rows) continue;
        const int64_t tiles = ceil_div(m, bm) * ceil_div(n, swiglu ? 64 : 128);
        int64_t splits = tiles > 0 ? (bm == 256 ? 256 : 512) / tiles : 1;
        if (splits > stages / 8) splits = stages / 8;
        if (splits < 1) splits = 1;
        const int64_t per = ceil_div(stages, splits);
        splits = ceil_div(stages, per);
        const size_t partial =
            splits > 1 ? static_cast<size_t>(splits) * m * moe::part_ld(static_cast<int>(n), swiglu) * 4 : 0;
        const double t = mid_time(bm, tiles * splits, per, p_by_k) + (splits > 1 ? reduce_time(partial, p_by_k) : 0.0);
        if (t < best.us) best = ProductPlan{Kernel::kMid, bm, static_cast<int>(splits), per * 64, partial, t};
    }
    const int64_t tiles = ceil_div(m, 256) * ceil_div(n, swiglu ? 128 : 256);
    const double t = tiled_time(tiles, stages, p_by_k, int8);
    if (direct && m > 64 && most_rows >= 256 && t < best.us)
        best = ProductPlan{Kernel::kTiled, 256, 1, stages * 64, 0, t};
    return best;
}

// The most that a product's partial sums take, whatever its operands' layout and alignment (Q by k: the plan without
// streaming, which needs none). pair: also where it shares a launch with another.
size_t most_partial(int64_t m, int64_t n, int64_t k, bool swiglu, bool p_by_k, bool pair) {
    size_t most = 0;
    auto take = [&](bool direct, int rows) {
        const size_t b = plan_product(m, n, k, swiglu, p_by_k, true, direct, rows).partial_bytes;
        if (b > most) most = b;
    };
    take(false, 256);
    take(true, 256);
    if (pair) take(true, 128);
    return most;
}

// Whether an operand allows 16-byte copies: granules on 16 bytes in every row, tile offsets within 32 bits
bool direct_operand(const void* p, int64_t ld) {
    return aligned16(p) && ld % 8 == 0 && ld <= int64_t{1} << 22;
}
void set_split(moe::GemmArgs& g, const ProductPlan& plan, void* partial) {
    g.partial = static_cast<float*>(partial);
    g.splits = plan.splits;
    g.split_k = static_cast<int>(plan.split_k);
}

// p_padded: P's rows are zero from k up to the next multiple of 8
bool direct_product(const moe::GemmArgs& g, bool p_by_k, bool q_by_k, bool p_padded) {
    return direct_operand(g.p, g.ldp) && direct_operand(g.q, g.ldq) &&
           (g.k % 8 == 0 || (q_by_k && (p_by_k || p_padded))) &&
           !(g.act == moe::kActSwiglu && q_by_k && g.up % 8 != 0);
}

hipError_t run_product(moe::GemmArgs g, void* partial, bool p_by_k, bool q_by_k, bool bf16, hipStream_t stream,
                       bool p_padded = false) {
    const bool direct = direct_product(g, p_by_k, q_by_k, p_padded);
    const ProductPlan plan = plan_product(g.m, g.n, g.k, g.act == moe::kActSwiglu, p_by_k, q_by_k, direct);
    set_split(g, plan, partial);
    if (plan.kernel == Kernel::kStream) return moe::launch_gemm_stream(g, bf16, stream);
    if (plan.kernel == Kernel::kTiled) return moe::launch_gemm_tiled(g, p_by_k, q_by_k, bf16, stream);
    const hipError_t err = moe::launch_gemm_mid(g, p_by_k, q_by_k, bf16, direct, plan.bm, stream);
    return err == hipSuccess && plan.splits > 1 ? moe::launch_gemm_reduce(g, bf16, stream) : err;
}

// The weight's layout that a workspace is for
enum class Layout { kRows, kTransposed, kEither };
Layout layout_of(int32_t weight_transposed) { return weight_transposed ? Layout::kTransposed : Layout::kRows; }

// Room for x and the weight with padded rows (moe_linear_repack.hip), where the sizes alone make them necessary: x and
// a weight [Z, H] where H is no multiple of 8, a transposed weight [H, Z] where Z (a SwiGLU's N) is none.
struct RepackRoom {
    size_t x, w;
};
RepackRoom repack_room(int64_t T, int64_t N, int64_t H, bool swiglu, Layout layout) {
    const int64_t h8 = round_up(H, 8), n8 = round_up(N, 8), halves = swiglu ? 2 : 1;
    RepackRoom r{};
    if (H % 8 != 0) r.x = round_up(T * h8 * 2, 256);
    const int64_t rows = layout != Layout::kTransposed && H % 8 != 0 ? halves * N * h8 * 2 : 0;
    const int64_t cols = layout != Layout::kRows && N % 8 != 0 ? H * halves * n8 * 2 : 0;
    r.w = round_up(rows > cols ? rows : cols, 256);
    return r;
}
moe::Repack repack(const void* src, int64_t ld, int64_t rows, int64_t cols, void* dst, int64_t dst_ld) {
    moe::Repack r{};
    r.src = static_cast<const uint16_t*>(src);
    r.dst = static_cast<uint16_t*>(dst);
    r.src_ld = ld;
    r.dst_ld = dst_ld;
    r.rows = rows;
    r.cols = static_cast<int>(cols);
    r.dst_cols = static_cast<int>(round_up(cols, 8));
    return r;
}

size_t linear_workspace(int64_t T, int64_t N, int64_t H, int32_t act, Layout layout) {
    const bool swiglu = act == MOE_ACT_SWIGLU;
    const RepackRoom room = repack_room(T, N, H, swiglu, layout);
    const size_t padded = H % 8 != 0 ? most_partial(T, N, round_up(H, 8), swiglu, false, false) : 0;
    const size_t partial = most_partial(T, N, H, swiglu, false, false);
    return room.x + room.w + (partial > padded ? partial : padded);
}

// Workspace of the gradients: dz [T, Z rounded up to 8] | column sums of row blocks | x and the weight with padded
// rows, where needed | partial sums of split products | of an fp32 grad_y, the largest values of dz and its scale's
// inverse
struct GradWorkspace {
    int64_t Z, ldz;
    size_t sums_at, x_at, w_at, partial_at, bytes, peaks_at, bytes_f32;
};
GradWorkspace grad_workspace(int64_t T, int64_t N, int64_t H, int32_t act, Layout layout) {
    GradWorkspace g{};
    g.Z = act == MOE_ACT_SWIGLU ? 2 * N : N;
    g.ldz = round_up(g.Z, 8);
    g.sums_at = round_up(T * g.ldz * 2, 256);
    const int64_t row_blocks = moe::act_grad_row_blocks(T, static_cast<int>(g.Z));
    g.x_at = g.sums_at + round_up(row_blocks * g.Z * 4, 256);
    const RepackRoom room = repack_room(T, g.Z, H, false, layout);
    g.w_at = g.x_at + room.x;
    g.partial_at = g.w_at + room.w;
    const size_t x0 = most_partial(T, H, g.Z, false, false, true);
    const size_t x8 = g.ldz != g.Z ? most_partial(T, H, g.ldz, false, false, true) : 0;
    const size_t x = x0 > x8 ? x0 : x8, w = most_partial(g.Z, H, T, false, true, true);
    g.bytes = g.partial_at + round_up(static_cast<int64_t>(x), 256) + w;  // both, for products of one launch
    g.peaks_at = round_up(static_cast<int64_t>(g.bytes), 256);
    g.bytes_f32 = g.peaks_at + (moe::kGradPeaks + 1) * sizeof(float);
    return g;
}

// moe_linear; the workspace has to have what `workspace_for` needs
moe_status linear(const void* x, int64_t x_stride, const void* weight, int64_t weight_stride, int32_t weight_transposed,
                  const void* bias, const void* residual, void* y, void* pre, void* workspace, size_t workspace_bytes,
                  int64_t T, int64_t N, int64_t H, int32_t activation, int32_t dtype, int32_t out_dtype, void* stream,
                  Layout workspace_for) {
    const char* op = "MoeLinear";
    moe_status st = check_linear(op, T, N, H, activation, dtype);
    if (st != MOE_OK) return st;
    if (out_dtype != dtype && out_dtype != MOE_DT_FLOAT32)
        return fail(MOE_ERR_ARG, "%s: result type %d (the operands' or float32 expected)", op, out_dtype);
    const int64_t Z = activation == MOE_ACT_SWIGLU ? 2 * N : N;
    st = check_pitch(op, "x", T, H, x_stride);
    if (st != MOE_OK) return st;
    st = weight_transposed ? check_pitch(op, "weight", H, Z, weight_stride)
                           : check_pitch(op, "weight", Z, H, weight_stride);
    if (st != MOE_OK) return st;
    if (T == 0) return ok();
    if (!x || !weight || !y) return fail(MOE_ERR_NULL, "%s: null tensor pointer", op);
    const size_t need = linear_workspace(T, N, H, activation, workspace_for);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(MOE_ERR_WORKSPACE, "%s: workspace %zu bytes at %p, need %zu", op, workspace_bytes, workspace, need);
    if (need > 0 && !aligned16(workspace))
        return fail(MOE_ERR_UNSUPPORTED, "%s: workspace must be 16-byte aligned", op);
    moe::GemmArgs g{};
    g.p = static_cast<const uint16_t*>(x);
    g.q = static_cast<const uint16_t*>(weight);
    g.ldp = x_stride;
    g.ldq = weight_stride;
    g.m = static_cast<int>(T);
    g.n = static_cast<int>(N);
    g.k = static_cast<int>(H);
    g.out = y;
    g.pre = static_cast<uint16_t*>(pre);
    g.bias = static_cast<const uint16_t*>(bias);
    g.residual = residual;
    g.act = activation;
    g.out_f32 = out_dtype == MOE_DT_FLOAT32;
    g.up = g.n;
    hipError_t err = moe::prepare_linear();
    if (err != hipSuccess) return hip_fail(err, "MoeLinear kernel attributes");
    // rows off 16 bytes by their length: padded copies first
    const bool swiglu = activation == MOE_ACT_SWIGLU, transposed = weight_transposed != 0;
    const RepackRoom room = repack_room(T, N, H, swiglu, layout_of(weight_transposed));
    char* base = static_cast<char*>(workspace);
    moe::RepackArgs pack{};
    const int64_t h8 = round_up(H, 8), n8 = round_up(N, 8);
    bool padded = false;
    if (H % 8 != 0) {
        pack.m[0] = repack(x, x_stride, T, H, base, h8);
        g.p = pack.m[0].dst;
        g.ldp = h8;
        padded = true;
    }
    if (!transposed && H % 8 != 0) {
        pack.m[1] = repack(weight, weight_stride, Z, H, base + room.x, h8);
        g.q = pack.m[1].dst;
        g.ldq = h8;
        g.k = static_cast<int>(h8);  // zeros in both
    } else if (transposed && N % 8 != 0) {
        g.q = reinterpret_cast<uint16_t*>(base + room.x);
        g.ldq = swiglu ? 2 * n8 : n8;
        g.up = static_cast<int>(n8);
        pack.m[1] = repack(weight, weight_stride, H, N, base + room.x, g.ldq);
        if (swiglu)
            pack.m[2] =
                repack(static_cast<const uint16_t*>(weight) + N, weight_stride, H, N, pack.m[1].dst + n8, g.ldq);
    }
    err = moe::launch_repack(pack, as_stream(stream));
    if (err == hipSuccess)
        err = run_product(g, base + room.x + room.w, false, transposed, dtype == MOE_DT_BFLOAT16, as_stream(stream),
                          padded);
    if (err != hipSuccess) return hip_fail(err, "MoeLinear launch");
    return ok();
}
// 8-bit products. In their plans k counts pairs of integers, as the kernels do (moe_gemm.h).
constexpr int64_t kMaxInt8K = 131071;  // 2^14 k < 2^31: no sum leaves 32 bits, -128 included

moe_status check_linear_int8(int64_t T, int64_t N, int64_t H, int64_t E, int32_t act) {
    const char* op = "MoeLinearInt8";
    moe_status st = check_linear(op, T, N, H, act, MOE_DT_FLOAT16);
    if (st != MOE_OK) return st;
    if (H > kMaxInt8K)
        return fail(MOE_ERR_UNSUPPORTED, "%s: H=%lld exceeds %lld, where 32-bit sums end", op, (long long)H,
                    (long long)kMaxInt8K);
    if (E < 0) return fail(MOE_ERR_ARG, "%s: numExperts=%lld", op, (long long)E);
    if (E > kMaxExperts)
        return fail(MOE_ERR_UNSUPPORTED, "%s: numExperts=%lld exceeds %lld", op, (long long)E, (long long)kMaxExperts);
    if (E > 0 && (T / 16 + E) * (N / 8 + 1) > kInt32Max)  // items of 16 rows x 8 columns, the smallest
        return fail(MOE_ERR_UNSUPPORTED, "%s: T=%lld N=%lld too large", op, (long long)T, (long long)N);
    return ok();
}

// Workspace: x and the weights with rows padded to 16 bytes, where H is no multiple of that and the product has rows
// enough for it to pay (T = 8000, H = 4001, N = 4000 429 us through registers; T = 200, H = 2001, N = 2000 20 either
// way) | partial sums of a split product
struct Int8Workspace {
    bool padded;
    size_t w_at, partial_at, bytes;
};
Int8Workspace int8_workspace(int64_t T, int64_t N, int64_t H, int64_t E, int32_t act) {
    const bool swiglu = act == MOE_ACT_SWIGLU;
    const int64_t h16 = round_up(H, 16), groups = E > 0 ? E : 1;
    Int8Workspace w{};
    w.padded = H % 16 != 0 && T >= (E > 0 ? 32 * E : 256);
    if (w.padded) {
        w.w_at = round_up(T * h16, 256);
        w.partial_at = w.w_at + round_up(groups * (swiglu ? 2 : 1) * N * h16, 256);
    }
    w.bytes = w.partial_at;
    if (E > 0) return w;
    size_t most = 0;
    for (const bool direct : {false, true}) {
        const int64_t k = (w.padded ? h16 : H + 1) / 2;
        const ProductPlan plan = plan_product(T, N, k, swiglu, false, false, direct, 256, true);
        if (plan.partial_bytes > most) most = plan.partial_bytes;
    }
    w.bytes += most;
    return w;
}

// Rows of a tile of the experts' products, by their rows on average; 16 streams the weights. us at means of 8, 12, 24
// and 32 rows, of which some experts have three times as many (E = 64, H = 2048, N = 1408 SwiGLU): streaming 68, 80,
// 121, 155; 64 rows 76, 77, 84, 93; 128 rows 76, 89, 91, 93; 256 rows 93, 92, 94, 84, and 90 at 64 rows, where 128 take
// 116. E = 8, H = 4096, N = 14336 152, 185, 300, 358 / 165, 164, 190, 207 / 178, 179, 178, 203 / 200, 199, 201, 190.
// Operands that come through registers have tiles of 64 and 128 rows.
int group_rows(int64_t T, int64_t E, bool direct) {
    const int64_t mean = T / E;
    if (!direct) return mean <= 64 ? 64 : 128;
    return mean <= 10 ? 16 : mean < 32 ? 64 : 256;
}

// moe_linear_grad likewise; grad_y of the operands' type or, with grad_f32, float32
moe_status linear_grad(const void* grad_y, int64_t grad_y_stride, bool grad_f32, const void* x, int64_t x_stride,
                       const void* weight, int64_t weight_stride, int32_t weight_transposed, const void* pre,
                       void* grad_x, void* grad_weight, void* grad_bias, void* workspace, size_t workspace_bytes,
                       int64_t T, int64_t N, int64_t H, int32_t activation, int32_t dtype, void* stream,
                       Layout workspace_for) {
    const char* op = "MoeLinearGrad";
    moe_status st = check_linear(op, T, N, H, activation, dtype);
    if (st != MOE_OK) return st;
    const Layout layout = layout_of(weight_transposed);
    const GradWorkspace ws = grad_workspace(T, N, H, activation, layout);
    const size_t need = grad_f32                  ? ws.bytes_f32
                        : workspace_for == layout ? ws.bytes
                                                  : grad_workspace(T, N, H, activation, workspace_for).bytes;
    st = check_pitch(op, "grad_y", T, N, grad_y_stride);
    if (st != MOE_OK) return st;
    if (grad_weight) st = check_pitch(op, "x", T, H, x_stride);
    if (st != MOE_OK) return st;
    if (grad_x)
        st = weight_transposed ? check_pitch(op, "weight", H, ws.Z, weight_stride)
                               : check_pitch(op, "weight", ws.Z, H, weight_stride);
    if (st != MOE_OK) return st;
    if (!grad_x && !grad_weight && !grad_bias) return ok();
    const bool act = activation != MOE_ACT_NONE;
    if (T > 0 && (!grad_y || (act && !pre) || (grad_weight && !x) || (grad_x && !weight)))
        return fail(MOE_ERR_NULL, "%s: null tensor pointer", op);
    if (T == 0 && !grad_weight && !grad_bias) return ok();
    if (!workspace || workspace_bytes < need)
        return fail(MOE_ERR_WORKSPACE, "%s: workspace %zu bytes at %p, need %zu", op, workspace_bytes, workspace, need);
    if (!aligned16(workspace)) return fail(MOE_ERR_UNSUPPORTED, "%s: workspace must be 16-byte aligned", op);
    const hipStream_t s = as_stream(stream);
    const bool bf16 = dtype == MOE_DT_BFLOAT16;
    char* base = static_cast<char*>(workspace);
    // without an activation dz is grad_y itself, where the products can read that in 16-byte copies
    const bool as_is = !act && !grad_f32 && N % 8 == 0 && direct_operand(grad_y, grad_y_stride);
    const bool need_dz = !as_is && (grad_x || grad_weight) && T > 0;
    const uint16_t* dz = as_is ? static_cast<const uint16_t*>(grad_y) : reinterpret_cast<uint16_t*>(base);
    const int64_t ldz = as_is ? grad_y_stride : ws.ldz;
    hipError_t err = moe::prepare_linear();
    if (err != hipSuccess) return hip_fail(err, "MoeLinearGrad kernel attributes");
    float* sums = reinterpret_cast<float*>(base + ws.sums_at);
    float* peaks = need_dz && grad_f32 && !bf16 ? reinterpret_cast<float*>(base + ws.peaks_at) : nullptr;
    if (need_dz || grad_bias) {
        moe::ActGrad g{};
        g.dy = grad_y;
        g.ldy = grad_y_stride;
        g.pre = act ? static_cast<const uint16_t*>(pre) : nullptr;
        g.dz = need_dz ? reinterpret_cast<uint16_t*>(base) : nullptr;
        g.ldz = ws.ldz;
        g.part = grad_bias ? sums : nullptr;
        g.peaks = peaks;
        g.T = T;
        g.N = static_cast<int>(N);
        g.act = activation;
        g.bf16 = bf16;
        g.dy_f32 = grad_f32;
        err = moe::launch_act_grad(g, s);
    }
    if (err != hipSuccess) return hip_fail(err, "MoeLinearGrad activation launch");
    moe::GradTail tail{};
    moe::GemmArgs &gx = tail.x, &gw = tail.w;
    gx.p = gw.p = dz;
    gx.ldp = gw.ldp = ldz;
    gx.factor = gw.factor = peaks ? peaks + moe::kGradPeaks : nullptr;
    gx.q = static_cast<const uint16_t*>(weight);
    gx.ldq = weight_stride;
    gx.m = gw.k = static_cast<int>(T);
    gx.n = gw.n = static_cast<int>(H);
    gx.k = gw.m = static_cast<int>(ws.Z);
    gx.out = grad_x;
    gw.q = static_cast<const uint16_t*>(x);
    gw.ldq = x_stride;
    gw.out = grad_weight;
    tail.sums = sums;
    tail.bias_grad = static_cast<uint16_t*>(grad_bias);
    tail.Z = static_cast<int>(ws.Z);
    tail.sum_rows = moe::act_grad_row_blocks(T, tail.Z);
    const bool want_x = grad_x && T > 0, by_k = weight_transposed == 0;
    moe::RepackArgs pack{};
    if (grad_weight && T > 0 && H % 8 != 0 && !direct_operand(x, x_stride)) {
        pack.m[0] = repack(x, x_stride, T, H, base + ws.x_at, round_up(H, 8));
        gw.q = pack.m[0].dst;
        gw.ldq = round_up(H, 8);
    }
    if (want_x && (by_k ? H % 8 != 0 && !direct_operand(weight, weight_stride) : ws.Z % 8 != 0)) {
        const int64_t cols = by_k ? H : ws.Z;
        pack.m[1] = repack(weight, weight_stride, by_k ? ws.Z : H, cols, base + ws.w_at, round_up(cols, 8));
        gx.q = pack.m[1].dst;
        gx.ldq = round_up(cols, 8);
        if (!by_k && need_dz) gx.k = static_cast<int>(ws.ldz);  // zeros in both
    }
    err = moe::launch_repack(pack, s);
    if (err != hipSuccess) return hip_fail(err, "MoeLinearGrad launch");
    void* partial = base + ws.partial_at;
    if (want_x && grad_weight && direct_product(gx, false, by_k, need_dz) && direct_product(gw, true, true, false)) {
        // one launch for both by tiles of at most 128 rows, where that costs less than the launch it saves
        const ProductPlan px = plan_product(gx.m, gx.n, gx.k, false, false, by_k, true, 128);
        const ProductPlan pw = plan_product(gw.m, gw.n, gw.k, false, true, true, true, 128);
        const double apart = plan_product(gx.m, gx.n, gx.k, false, false, by_k, true).us +
                             plan_product(gw.m, gw.n, gw.k, false, true, true, true).us;
        if (px.kernel == Kernel::kMid && pw.kernel == Kernel::kMid && px.us + pw.us < apart + kLaunchSaved) {
            set_split(gx, px, partial);
            set_split(gw, pw, static_cast<char*>(partial) + round_up(static_cast<int64_t>(px.partial_bytes), 256));
            err = moe::launch_gemm_pair(gx, gw, by_k, bf16, px.bm, s);
            if (err == hipSuccess) err = moe::launch_grad_tail(tail, bf16, s);
            if (err != hipSuccess) return hip_fail(err, "MoeLinearGrad launch");
            return ok();
        }
    }
    if (want_x) err = run_product(gx, partial, false, by_k, bf16, s, need_dz);
    if (err == hipSuccess && grad_weight) err = run_product(gw, partial, true, true, bf16, s);
    if (err == hipSuccess && grad_bias) {
        gx.splits = gw.splits = 1;
        err = moe::launch_grad_tail(tail, bf16, s);
    }
    if (err != hipSuccess) return hip_fail(err, "MoeLinearGrad launch");
    return ok();
}
}  // namespace

extern "C" {

moe_status moe_routing_group_topk(const void* logits, int64_t logits_stride, int32_t logits_type, const float* bias,
                                  int32_t* expert_ids, void* weights, int32_t weights_type, int64_t T, int64_t E,
                                  int64_t K, int64_t groups, int64_t top_groups, int64_t group_top, int32_t scoring,
                                  int32_t renormalize, float scale, void* stream) {
    const char* op = "MoeRoutingGroupTopK";
    moe_status st = check_group_routing(op, T, E, K, logits_stride, logits_type, weights_type, false);
    if (st != MOE_OK) return st;
    st = check_scoring(op, scoring, scale);
    if (st != MOE_OK) return st;
    if (groups < 1 || groups > E || E % groups != 0)
        return fail(MOE_ERR_ARG, "%s: numGroups=%lld must divide numExperts=%lld", op, (long long)groups, (long long)E);
    if (top_groups < 1 || top_groups > groups)
        return fail(MOE_ERR_ARG, "%s: topGroups=%lld must be in [1, numGroups=%lld]", op, (long long)top_groups,
                    (long long)groups);
    if (group_top != 1 && group_top != 2)
        return fail(MOE_ERR_ARG, "%s: groupTop=%lld must be 1 or 2", op, (long long)group_top);
    if (K > top_groups * (E / groups))
        return fail(MOE_ERR_ARG, "%s: topK=%lld exceeds the %lld experts of %lld groups", op, (long long)K,
                    (long long)(top_groups * (E / groups)), (long long)top_groups);
    if (T == 0) return ok();
    if (!logits || !expert_ids || !weights) return fail(MOE_ERR_NULL, "%s: null tensor pointer", op);
    moe::GroupRouting r{};
    r.logits = logits;
    r.ld = logits_stride;
    r.logits_type = logits_type;
    r.bias = bias;
    r.T = T;
    r.E = static_cast<int>(E);
    r.K = static_cast<int>(K);
    r.groups = static_cast<int>(groups);
    r.top_groups = static_cast<int>(top_groups);
    r.group_top = static_cast<int>(group_top);
    const int size = static_cast<int>(E / groups);
    r.size_inverse = (65536 + size - 1) / size;
    r.sigmoid = scoring == MOE_SCORE_SIGMOID;
    r.renormalize = renormalize != 0;
    r.scale = scale;
    r.weights_type = weights_type;
    const hipError_t err = moe::launch_group_routing(r, expert_ids, weights, as_stream(stream));
    if (err != hipSuccess) return hip_fail(err, "MoeRoutingGroupTopK launch");
    return ok();
}

moe_status moe_routing_group_topk_grad(const void* grad_weights, int32_t weights_type, const void* logits,
                                       int64_t logits_stride, int32_t logits_type, const int32_t* expert_ids,
                                       void* grad_logits, int64_t T, int64_t E, int64_t K, int32_t scoring,
                                       int32_t renormalize, float scale, void* stream) {
    const char* op = "MoeRoutingGroupTopKGrad";
    moe_status st = check_group_routing(op, T, E, K, logits_stride, logits_type, weights_type, true);
    if (st != MOE_OK) return st;
    st = check_scoring(op, scoring, scale);
    if (st != MOE_OK) return st;
    if (T == 0) return ok();
    if (!grad_weights || !logits || !expert_ids || !grad_logits)
        return fail(MOE_ERR_NULL, "%s: null tensor pointer", op);
    moe::GroupRouting r{};
    r.logits = logits;
    r.ld = logits_stride;
    r.logits_type = logits_type;
    r.T = T;
    r.E = static_cast<int>(E);
    r.K = static_cast<int>(K);
    r.sigmoid = scoring == MOE_SCORE_SIGMOID;
    r.renormalize = renormalize != 0;
    r.scale = scale;
    r.weights_type = weights_type;
    const hipError_t err =
        moe::launch_group_routing_grad(r, grad_weights, expert_ids, grad_logits, as_stream(stream));
    if (err != hipSuccess) return hip_fail(err, "MoeRoutingGroupTopKGrad launch");
    return ok();
}

moe_status moe_combine_grad(const uint16_t* grad_y, const uint16_t* expert_out, const uint16_t* weights,
                            uint16_t* grad_expert_out, uint16_t* grad_weights, int64_t T, int64_t H, int64_t K,
                            void* stream) {
    const char* op = "MoeCombineGrad";
    if (T < 0 || H <= 0 || K < 1)
        return fail(MOE_ERR_ARG, "%s: sizes must be T >= 0, H > 0, K >= 1 (T=%lld H=%lld K=%lld)", op, (long long)T,
                    (long long)H, (long long)K);
    if (H % 8 != 0) return fail(MOE_ERR_UNSUPPORTED, "%s: hiddenSize=%lld must be a multiple of 8", op, (long long)H);
    if (H > kMaxDim)
        return fail(MOE_ERR_UNSUPPORTED, "%s: hiddenSize=%lld exceeds %lld", op, (long long)H, (long long)kMaxDim);
    if (product_exceeds(T, K, kInt32Max))
        return fail(MOE_ERR_UNSUPPORTED, "%s: T=%lld K=%lld too large", op, (long long)T, (long long)K);
    if (T == 0) return ok();
    if (!grad_y || !expert_out || !weights || !grad_expert_out || !grad_weights)
        return fail(MOE_ERR_NULL, "%s: null tensor pointer", op);
    if (!aligned16(grad_y) || !aligned16(expert_out) || !aligned16(grad_expert_out))
        return fail(MOE_ERR_UNSUPPORTED, "%s: grad_y, expert_out and grad_expert_out must be 16-byte aligned", op);
    const hipError_t err = moe::launch_combine_grad(grad_y, expert_out, weights, grad_expert_out, grad_weights, T,
                                                    static_cast<int>(H), static_cast<int>(K), as_stream(stream));
    if (err != hipSuccess) return hip_fail(err, "MoeCombineGrad launch");
    return ok();
}

size_t moe_linear_workspace_bytes(int64_t T, int64_t N, int64_t H, int32_t activation) {
    if (check_linear("MoeLinear", T, N, H, activation, MOE_DT_FLOAT16) != MOE_OK) return 0;
    return linear_workspace(T, N, H, activation, Layout::kEither);
}

moe_status moe_linear(const void* x, int64_t x_stride, const void* weight, int64_t weight_stride,
                      int32_t weight_transposed, const void* bias, const void* residual, void* y, void* pre,
                      void* workspace, size_t workspace_bytes, int64_t T, int64_t N, int64_t H, int32_t activation,
                      int32_t dtype, int32_t out_dtype, void* stream) {
    return linear(x, x_stride, weight, weight_stride, weight_transposed, bias, residual, y, pre, workspace,
                  workspace_bytes, T, N, H, activation, dtype, out_dtype, stream, Layout::kEither);
}

size_t moe_linear_layout_workspace_bytes(int64_t T, int64_t N, int64_t H, int32_t activation,
                                         int32_t weight_transposed) {
    if (check_linear("MoeLinear", T, N, H, activation, MOE_DT_FLOAT16) != MOE_OK) return 0;
    return linear_workspace(T, N, H, activation, layout_of(weight_transposed));
}

moe_status moe_linear_layout(const void* x, int64_t x_stride, const void* weight, int64_t weight_stride,
                             int32_t weight_transposed, const void* bias, const void* residual, void* y, void* pre,
                             void* workspace, size_t workspace_bytes, int64_t T, int64_t N, int64_t H,
                             int32_t activation, int32_t dtype, int32_t out_dtype, void* stream) {
    return linear(x, x_stride, weight, weight_stride, weight_transposed, bias, residual, y, pre, workspace,
                  workspace_bytes, T, N, H, activation, dtype, out_dtype, stream, layout_of(weight_transposed));
}

size_t moe_linear_grad_workspace_bytes(int64_t T, int64_t N, int64_t H, int32_t activation) {
    if (check_linear("MoeLinearGrad", T, N, H, activation, MOE_DT_FLOAT16) != MOE_OK) return 0;
    return grad_workspace(T, N, H, activation, Layout::kEither).bytes;
}

moe_status moe_linear_grad(const void* grad_y, int64_t grad_y_stride, const void* x, int64_t x_stride,
                           const void* weight, int64_t weight_stride, int32_t weight_transposed, const void* pre,
                           void* grad_x, void* grad_weight, void* grad_bias, void* workspace, size_t workspace_bytes,
                           int64_t T, int64_t N, int64_t H, int32_t activation, int32_t dtype, void* stream) {
    return linear_grad(grad_y, grad_y_stride, false, x, x_stride, weight, weight_stride, weight_transposed, pre, grad_x,
                       grad_weight, grad_bias, workspace, workspace_bytes, T, N, H, activation, dtype, stream,
                       Layout::kEither);
}

size_t moe_linear_grad_layout_workspace_bytes(int64_t T, int64_t N, int64_t H, int32_t activation,
                                              int32_t weight_transposed) {
    if (check_linear("MoeLinearGrad", T, N, H, activation, MOE_DT_FLOAT16) != MOE_OK) return 0;
    return grad_workspace(T, N, H, activation, layout_of(weight_transposed)).bytes;
}

moe_status moe_linear_grad_layout(const void* grad_y, int64_t grad_y_stride, const void* x, int64_t x_stride,
                                  const void* weight, int64_t weight_stride, int32_t weight_transposed, const void* pre,
                                  void* grad_x, void* grad_weight, void* grad_bias, void* workspace,
                                  size_t workspace_bytes, int64_t T, int64_t N, int64_t H, int32_t activation,
                                  int32_t dtype, void* stream) {
    return linear_grad(grad_y, grad_y_stride, false, x, x_stride, weight, weight_stride, weight_transposed, pre, grad_x,
                       grad_weight, grad_bias, workspace, workspace_bytes, T, N, H, activation, dtype, stream,
                       layout_of(weight_transposed));
}

size_t moe_linear_grad_f32_workspace_bytes(int64_t T, int64_t N, int64_t H, int32_t activation,
                                           int32_t weight_transposed) {
    if (check_linear("MoeLinearGrad", T, N, H, activation, MOE_DT_FLOAT16) != MOE_OK) return 0;
    return grad_workspace(T, N, H, activation, layout_of(weight_transposed)).bytes_f32;
}

moe_status moe_linear_grad_f32(const float* grad_y, int64_t grad_y_stride, const void* x, int64_t x_stride,
                               const void* weight, int64_t weight_stride, int32_t weight_transposed, const void* pre,
                               void* grad_x, void* grad_weight, void* grad_bias, void* workspace,
                               size_t workspace_bytes, int64_t T, int64_t N, int64_t H, int32_t activation,
                               int32_t dtype, void* stream) {
    return linear_grad(grad_y, grad_y_stride, true, x, x_stride, weight, weight_stride, weight_transposed, pre, grad_x,
                       grad_weight, grad_bias, workspace, workspace_bytes, T, N, H, activation, dtype, stream,
                       layout_of(weight_transposed));
}

size_t moe_linear_int8_workspace_bytes(int64_t T, int64_t N, int64_t H, int64_t E, int32_t activation) {
    if (check_linear_int8(T, N, H, E, activation) != MOE_OK) return 0;
    return int8_workspace(T, N, H, E, activation).bytes;
}

moe_status moe_linear_int8(const int8_t* x, int64_t x_stride, const float* x_scale, const int8_t* weight,
                           int64_t weight_stride, int64_t expert_stride, const float* weight_scale,
                           const int32_t* offsets, const void* bias, const void* residual, void* y, void* workspace,
                           size_t workspace_bytes, int64_t T, int64_t N, int64_t H, int64_t E, int32_t activation,
                           int32_t out_dtype, void* stream) {
    const char* op = "MoeLinearInt8";
    moe_status st = check_linear_int8(T, N, H, E, activation);
    if (st != MOE_OK) return st;
    if (out_dtype != MOE_DT_FLOAT32 && !is_half(out_dtype))
        return fail(MOE_ERR_ARG, "%s: result type %d (float32, float16 or bfloat16 expected)", op, out_dtype);
    const bool swiglu = activation == MOE_ACT_SWIGLU;
    const int64_t Z = swiglu ? 2 * N : N;
    st = check_pitch(op, "x", T, H, x_stride);
    if (st == MOE_OK) st = check_pitch(op, "weight", Z, H, weight_stride);
    if (st != MOE_OK) return st;
    if (E > 1 && (expert_stride < (Z - 1) * weight_stride + H || expert_stride > int64_t{1} << 50))
        return fail(MOE_ERR_ARG, "%s: experts' weights %lld elements apart", op, (long long)expert_stride);
    if (T == 0) return ok();
    if (!x || !x_scale || !weight || !weight_scale || !y || (E > 0 && !offsets))
        return fail(MOE_ERR_NULL, "%s: null tensor pointer", op);
    const Int8Workspace room = int8_workspace(T, N, H, E, activation);
    const size_t need = room.bytes;
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(MOE_ERR_WORKSPACE, "%s: workspace %zu bytes at %p, need %zu", op, workspace_bytes, workspace, need);
    if (need > 0 && !aligned16(workspace))
        return fail(MOE_ERR_UNSUPPORTED, "%s: workspace must be 16-byte aligned", op);
    hipError_t err = moe::prepare_linear_int8();
    if (err != hipSuccess) return hip_fail(err, "MoeLinearInt8 kernel attributes");
    const hipStream_t s = as_stream(stream);
    int64_t pitch = T > 1 ? x_stride : 0, weight_pitch = Z > 1 ? weight_stride : 0;
    int64_t step = E > 1 ? expert_stride : 0, k = H;
    if (room.padded) {
        char* base = static_cast<char*>(workspace);
        moe::Repack8 px{}, pw{};
        px.src = reinterpret_cast<const uint8_t*>(x);
        px.dst = reinterpret_cast<uint8_t*>(base);
        px.src_ld = pitch;
        px.rows = T;
        px.cols = pw.cols = static_cast<int>(H);
        pw.src = reinterpret_cast<const uint8_t*>(weight);
        pw.dst = reinterpret_cast<uint8_t*>(base + room.w_at);
        pw.src_ld = weight_pitch;
        pw.group_ld = step;
        pw.rows = Z;
        err = moe::launch_repack8(px, pw, E > 0 ? E : 1, s);
        if (err != hipSuccess) return hip_fail(err, "MoeLinearInt8 launch");
        x = reinterpret_cast<const int8_t*>(px.dst);
        weight = reinterpret_cast<const int8_t*>(pw.dst);
        k = pitch = weight_pitch = round_up(H, 16);
        step = Z * k;
    }
    const bool direct = k % 16 == 0 && aligned16(x) && aligned16(weight) && pitch % 16 == 0 && weight_pitch % 16 == 0 &&
                        step % 16 == 0 && pitch <= int64_t{1} << 23 && weight_pitch <= int64_t{1} << 23;
    const int unit = direct ? 2 : 1;  // bytes that strides and k count
    moe::GemmArgs g{};
    g.p = reinterpret_cast<const uint16_t*>(x);
    g.q = reinterpret_cast<const uint16_t*>(weight);
    g.ldp = pitch / unit;
    g.ldq = weight_pitch / unit;
    g.m = static_cast<int>(T);
    g.n = g.up = static_cast<int>(N);
    g.k = static_cast<int>(k / unit);
    g.out = y;
    g.bias = static_cast<const uint16_t*>(bias);
    g.residual = residual;
    g.act = activation;
    g.out_f32 = out_dtype == MOE_DT_FLOAT32;
    g.splits = 1;
    g.split_k = g.k;
    g.row_scale = x_scale;
    g.col_scale = weight_scale;
    g.experts = static_cast<int>(E);
    g.q_expert = step;
    g.offsets = offsets;
    const bool bf16 = out_dtype == MOE_DT_BFLOAT16;
    if (E > 0) {
        const int rows = group_rows(T, E, direct);
        if (rows == 256) err = moe::launch_int8_tiled(g, bf16, s);
        else if (rows == 16) err = moe::launch_int8_stream(g, bf16, s);
        else err = moe::launch_int8_mid(g, bf16, direct, rows, s);
    } else {
        const ProductPlan plan = plan_product(T, N, (k + 1) / 2, swiglu, false, false, direct, 256, true);
        set_split(g, plan, static_cast<char*>(workspace) + room.partial_at);
        g.split_k = static_cast<int>(plan.split_k * 2 / unit);
        if (plan.kernel == Kernel::kStream) err = moe::launch_int8_stream(g, bf16, s);
        else if (plan.kernel == Kernel::kTiled) err = moe::launch_int8_tiled(g, bf16, s);
        else err = moe::launch_int8_mid(g, bf16, direct, plan.bm, s);
        if (err == hipSuccess && plan.splits > 1) err = moe::launch_int8_reduce(g, bf16, s);
    }
    if (err != hipSuccess) return hip_fail(err, "MoeLinearInt8 launch");
    return ok();
}

}  // extern "C"
