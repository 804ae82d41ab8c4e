/*
 * moe_ops.h -- C ABI of the MI355X (gfx950) MoE operator library libmoe_mi355x.so.
 *
 * Drop-in for the three CANN operators of Lu-Yu-Zhen/Implementing-MoE-Architecture-Operators-on-CANN-Platform:
 *   MoeRoutingTopK -> MoeExpertFFN -> MoeCombine
 * Each CANN operator is one OpDef (prototype) + InferShape + InferDataType + TilingFunc in
 * op_host/moe_ops.cpp, and one kernel entry point in the op_kernel/ sources. Here each becomes a set of plain C
 * functions: *_infer_shape / *_infer_dtype (graph-time), *_plan (launch planning) and the launch itself.
 *
 * Conventions (kept from the reference, op_host/moe_ops.cpp and tests/test_moe.cpp:415-463):
 *   - All tensors are dense row-major ("ND"). fp16 tensors are passed as pointers to IEEE binary16 bit
 *     patterns (uint16_t storage); int32 tensors as int32_t.
 *   - The caller allocates and frees every device buffer, including the workspace; the library never
 *     allocates device memory. Launches are asynchronous and ordered on `stream` (a hipStream_t; NULL means
 *     the default stream); the caller synchronises.
 *   - Shape/argument errors are reported before anything is launched, as a moe_status (the reference's
 *     GRAPH_FAILED + OP_LOGE); moe_last_error() returns the message for the calling thread.
 *   - No host-side state is kept across calls (except the optional tracer in moe_trace.h): calls are
 *     re-entrant and may be issued from several threads on different streams.
 *
 * Expert weight layout (tests/moe_cpu_sim.cpp:174-179,254-260; tests/test_moe.cpp:200-201), per expert e,
 * with I = intermediate size and H = hidden size, in the single tensor expert_weights[E, 3*I, H]:
 *   W_gate[e][i][h] at e*3*I*H +         i*H + h   ([I, H] row-major)
 *   W_up  [e][i][h] at e*3*I*H +   I*H + i*H + h   ([I, H] row-major)
 *   W_down[e][h][i] at e*3*I*H + 2*I*H + h*I + i   ([H, I] row-major)
 * The reference's NPU kernel reads W_down as [I, H] (op_kernel/moe_expert_ffn.cpp:348-375); both of its CPU
 * references use [H, I], and this library follows the CPU references.
 *
 * Limits of the gfx950 kernels (MOE_ERR_UNSUPPORTED otherwise): H % 32 == 0, I % 32 == 0, H and I at most
 * 2^20, 1 <= K <= E <= 256, T*K < 2^31, and 16-byte aligned x, expert_weights, expert_out and y.
 * Calls with many rows per expert (the LDS-tiled schedule, moe_expert_ffn_plan .schedule == 1) also need
 * T*H*2 (x), 3*I*H*2 (one expert's weights) and T*K*4 (the sorted slots) below 2 GiB: the tiled kernels address
 * them with 32-bit buffer offsets. Such calls beyond those bounds are rejected with the reason rather than run
 * on the weight-streaming schedule, which would stream every expert's weights again for each 128 of its rows.
 * The tiled schedule also needs H > 64 and I > 64 (two k-stages of 64); an odd multiple of 32 ends with a
 * 32-column stage.
 */
#ifndef MOE_OPS_H
#define MOE_OPS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum moe_status {
    MOE_OK = 0,
    MOE_ERR_NULL = 1,        /* required pointer is NULL (op_host/moe_ops.cpp:71-74,241-245,412-415)      */
    MOE_ERR_RANK = 2,        /* wrong tensor rank (op_host/moe_ops.cpp:80-85,251-258,421-428)             */
    MOE_ERR_SHAPE = 3,       /* inconsistent dims, e.g. hidden size mismatch (op_host/moe_ops.cpp:86-90)  */
    MOE_ERR_ARG = 4,         /* invalid scalar argument: sizes <= 0, topK outside [1, E]                  */
    MOE_ERR_WORKSPACE = 5,   /* workspace NULL or smaller than moe_expert_ffn_workspace_bytes()           */
    MOE_ERR_UNSUPPORTED = 6, /* valid request outside the gfx950 kernels' limits (see header comment)     */
    MOE_ERR_HIP = 7          /* a HIP runtime call or kernel launch failed                                */
} moe_status;

typedef enum moe_dtype {
    MOE_DT_FLOAT32 = 0,  /* ge::DT_FLOAT   */
    MOE_DT_FLOAT16 = 1,  /* ge::DT_FLOAT16 */
    MOE_DT_INT32 = 3,    /* ge::DT_INT32   */
    MOE_DT_BFLOAT16 = 27 /* ge::DT_BF16    */
} moe_dtype;

/* Human-readable name of a status code. */
const char* moe_status_string(moe_status status);
/* Message describing the last failure on the calling thread ("" if none). */
const char* moe_last_error(void);
/* Library version string. */
const char* moe_version(void);

/* ------------------------------------------------------------------------------------------------------
 * MoeRoutingTopK: x[T, H] fp16, w_gate[H, E] fp16 -> expert_ids[T, K] int32, weights[T, K] fp16.
 *   logits = x @ w_gate (fp32 accumulation), row softmax, top-K experts in descending probability order
 *   (exact ties: lowest expert index first), weights renormalised over the K chosen to sum to 1.
 *   Attr topK (default 2, op_host/moe_ops.cpp:565-567).
 * ---------------------------------------------------------------------------------------------------- */

/* InferShape (op_host/moe_ops.cpp:181-214): expert_ids and weights are [x_dims[0], top_k].
 * top_k <= 0 selects the attr default 2. Checks ranks and x_dims[1] == w_gate_dims[0]
 * (the TilingFunc check, op_host/moe_ops.cpp:80-90). */
moe_status moe_routing_topk_infer_shape(const int64_t* x_dims, int32_t x_rank, const int64_t* w_gate_dims,
                                        int32_t w_gate_rank, int64_t top_k, int64_t expert_ids_dims[2],
                                        int64_t weights_dims[2]);
/* InferDataType (op_host/moe_ops.cpp:219-226): INT32, FLOAT16. */
moe_status moe_routing_topk_infer_dtype(moe_dtype* expert_ids_dtype, moe_dtype* weights_dtype);

/* Launch plan (TilingFunc replacement, op_host/moe_ops.cpp:63-176; TilingData op_host/moe_tiling.h:27-43). */
typedef struct moe_routing_plan {
    int64_t num_tokens, hidden_size, num_experts, top_k;
    int32_t tokens_per_block; /* tokens handled by one workgroup                        */
    int32_t grid;             /* workgroups                                             */
    int32_t block;            /* threads per workgroup                                  */
    int32_t lds_bytes;        /* dynamic LDS per workgroup                              */
    size_t workspace_bytes;   /* always 0, as in the reference (op_host/moe_ops.cpp:164-167) */
} moe_routing_plan;
moe_status moe_routing_topk_plan(int64_t num_tokens, int64_t hidden_size, int64_t num_experts, int64_t top_k,
                                 moe_routing_plan* plan);

/* Kernel entry MoeRoutingTopK(x, wGate, expertIds, weights, tiling) (op_kernel/moe_routing.cpp:434-440). */
moe_status moe_routing_topk(const uint16_t* x, const uint16_t* w_gate, int32_t* expert_ids, uint16_t* weights,
                            int64_t num_tokens, int64_t hidden_size, int64_t num_experts, int64_t top_k,
                            void* stream);

/* ------------------------------------------------------------------------------------------------------
 * MoeExpertFFN: x[T, H] fp16, expert_ids[T, K] int32, weights[T, K] fp16 (not used by the math, kept for
 *   signature parity), expert_weights[E, 3*I, H] fp16 -> expert_out[T, K, H] fp16.
 *   expert_out[t, k, :] = W_down_e @ (silu(W_gate_e @ x_t) * (W_up_e @ x_t)), e = expert_ids[t, k],
 *   fp32 accumulation; the SwiGLU intermediate is kept in fp16 in the workspace.
 *   Ids outside [0, E) are not computed: their expert_out rows are written as zeros.
 *   Attr intermediateSize (default 8192, op_host/moe_ops.cpp:618-620).
 * ---------------------------------------------------------------------------------------------------- */

/* InferShape (op_host/moe_ops.cpp:364-388): expert_out is [x_dims[0], expert_ids_dims[1], x_dims[1]].
 * The intermediate size is expert_weights_dims[1] / 3, overridden by intermediate_size_attr when > 0, as the
 * TilingFunc does (op_host/moe_ops.cpp:264-278); unlike the reference an override that disagrees with
 * expert_weights_dims[1] is rejected (MOE_ERR_SHAPE) instead of reading past the weights.
 * *intermediate_size receives the resolved value. */
moe_status moe_expert_ffn_infer_shape(const int64_t* x_dims, int32_t x_rank, const int64_t* expert_ids_dims,
                                      int32_t expert_ids_rank, const int64_t* expert_weights_dims,
                                      int32_t expert_weights_rank, int64_t intermediate_size_attr,
                                      int64_t expert_out_dims[3], int64_t* intermediate_size);
/* InferDataType (op_host/moe_ops.cpp:393-398): FLOAT16. */
moe_status moe_expert_ffn_infer_dtype(moe_dtype* expert_out_dtype);

/* Workspace bytes for one call (TilingFunc workspace, op_host/moe_ops.cpp:340-349). Holds the expert-sorted
 * slot order, per-expert offsets and the fp16 SwiGLU intermediate [T*K, I]; on the weight-streaming schedule
 * also the split-K partial sums and the slot -> sorted-row map; on the LDS-tiled schedule also up to 64 MiB of
 * fp32 partial tiles for the tiles it splits over k (only when its down tiles fill at most 4 rounds of the
 * GPU). 0 for invalid sizes.
 * Not monotone in num_tokens: a caller that keeps one workspace over its calls takes the largest over every
 * num_tokens it will use. Where the expert weights reach 1 GB and only that takes a size to the tiled schedule, the
 * value covers both schedules, and a call given less than the tiled schedule needs, but enough to stream, streams:
 * its expert_out then differs from that of a call with the whole workspace in fp32 summation order. */
size_t moe_expert_ffn_workspace_bytes(int64_t num_tokens, int64_t hidden_size, int64_t num_experts,
                                      int64_t top_k, int64_t intermediate_size);

typedef struct moe_ffn_plan {
    int64_t num_tokens, hidden_size, num_experts, top_k, intermediate_size;
    int32_t schedule;        /* 0 = weight-streaming (few rows per expert), 1 = LDS-tiled (many rows)    */
    int32_t permute_grid;    /* workgroups of the permute's first launch: one per 1024 slots when it counts */
                             /* (a scatter of as many follows), or one that sorts few slots by itself plus  */
                             /* one per 1024 slots that clear the rows of ids outside [0, E); 0 on the      */
                             /* weight-streaming schedule, whose gate/up kernel finds its rows itself       */
    int32_t gateup_grid;     /* work tiles of the fused gate/up + SwiGLU grouped GEMM (upper bound on its */
                             /* workgroups: the streaming schedule runs a persistent grid of at most as    */
                             /* many workgroups as the GPU holds at once)                                  */
    int32_t down_grid;       /* work tiles of the down-projection grouped GEMM (same convention)           */
    int32_t block;           /* threads per workgroup of the GEMMs                                         */
    int32_t rows_per_tile;   /* token rows per GEMM tile                                                   */
    size_t workspace_bytes;  /* == moe_expert_ffn_workspace_bytes(...)                                    */
} moe_ffn_plan;
moe_status moe_expert_ffn_plan(int64_t num_tokens, int64_t hidden_size, int64_t num_experts, int64_t top_k,
                               int64_t intermediate_size, moe_ffn_plan* plan);

/* Kernel entry MoeExpertFFN(x, expertIds, weights, expertWeights, expertOut, workspace, tiling)
 * (op_kernel/moe_expert_ffn.cpp:613-621). */
moe_status moe_expert_ffn(const uint16_t* x, const int32_t* expert_ids, const uint16_t* weights,
                          const uint16_t* expert_weights, uint16_t* expert_out, void* workspace,
                          size_t workspace_bytes, int64_t num_tokens, int64_t hidden_size, int64_t num_experts,
                          int64_t top_k, int64_t intermediate_size, void* stream);

/* ------------------------------------------------------------------------------------------------------
 * MoeCombine: expert_out[T, K, H] fp16, expert_ids[T, K] int32 (not used by the math), weights[T, K] fp16
 *   -> y[T, H] fp16, y[t, :] = sum_k weights[t, k] * expert_out[t, k, :] accumulated in fp32 in ascending k
 *   (the reference kernel accumulates in fp16, op_kernel/moe_combine.cpp:87-106; its CPU references in fp32).
 *   Attr topK (default 2, op_host/moe_ops.cpp:665-667); K is taken from expert_out's dim 1.
 * ---------------------------------------------------------------------------------------------------- */

/* InferShape (op_host/moe_ops.cpp:495-515): y is [expert_out_dims[0], expert_out_dims[2]]. expert_ids_dims
 * may be NULL; when given it must be [T, K] (the TilingFunc rank check, op_host/moe_ops.cpp:425-428). */
moe_status moe_combine_infer_shape(const int64_t* expert_out_dims, int32_t expert_out_rank,
                                   const int64_t* expert_ids_dims, int32_t expert_ids_rank, int64_t y_dims[2]);
/* InferDataType (op_host/moe_ops.cpp:520-525): FLOAT16. */
moe_status moe_combine_infer_dtype(moe_dtype* y_dtype);

typedef struct moe_combine_plan {
    int64_t num_tokens, hidden_size, top_k;
    int32_t grid, block;
    int32_t elems_per_thread;
    size_t workspace_bytes; /* always 0 (op_host/moe_ops.cpp:477-481) */
} moe_combine_plan;
moe_status moe_combine_plan_for(int64_t num_tokens, int64_t hidden_size, int64_t top_k, moe_combine_plan* plan);

/* Kernel entry MoeCombine(expertOut, expertIds, weights, y, tiling) (op_kernel/moe_combine.cpp:136-143).
 * expert_ids may be NULL. */
moe_status moe_combine(const uint16_t* expert_out, const int32_t* expert_ids, const uint16_t* weights, uint16_t* y,
                       int64_t num_tokens, int64_t hidden_size, int64_t top_k, void* stream);

/* MoeExpertFFN that allocates nothing and takes no workspace. It has no counterpart in the reference. It is for
 * callers that cannot allocate device memory: code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc.
 * The workspace is a fixed per-GPU device array inside the library (64 MiB, held by every GPU the library runs
 * on until the process ends). Sizes whose workspace exceeds it return MOE_ERR_UNSUPPORTED before anything is
 * launched (e.g. T*K*I*2 > ~60 MiB). The LDS-tiled schedule runs its down projection without the split
 * leftover round here, so expert_out can differ from moe_expert_ffn's in fp32 summation order on that schedule.
 * The weight-streaming schedule is bit-identical, except that an H above 2272 whose split gate/up partial sums
 * (splits x T*K x 2I x 4 bytes) do not fit runs gate/up unsplit (16-row passes, or the tiled schedule when H
 * exceeds 4568), with the same difference in summation order.
 * Every call on a GPU shares that GPU's array: calls that overlap on one GPU (two streams or threads) race.
 * The first call on each device looks up that device's array address and sets the kernels' LDS limits: make it
 * outside graph capture (one eager call per device); later calls may be captured and replayed.
 * Arguments, errors and outputs otherwise as moe_expert_ffn. */
moe_status moe_expert_ffn_no_alloc(const uint16_t* x, const int32_t* expert_ids, const uint16_t* weights,
                                   const uint16_t* expert_weights, uint16_t* expert_out, int64_t num_tokens,
                                   int64_t hidden_size, int64_t num_experts, int64_t top_k,
                                   int64_t intermediate_size, void* stream);

/* ------------------------------------------------------------------------------------------------------
 * Optional fast path: MoeExpertFFN followed by MoeCombine in one call. It has no single counterpart in the
 * reference; it chains the kernel entries MoeExpertFFN (op_kernel/moe_expert_ffn.cpp:613-621) and MoeCombine
 * (op_kernel/moe_combine.cpp:136-143), which stay the contract. expert_out is written exactly as
 * moe_expert_ffn writes it, and y is bit-identical to moe_combine(expert_out, expert_ids, weights, y, ...).
 * When the weight-streaming schedule splits the down projection over K, the split reduce produces y as well,
 * saving the combine pass over expert_out; otherwise the combine kernel runs after the FFN. Deterministic (no
 * global atomics). Workspace as for moe_expert_ffn. Sizes and errors as moe_expert_ffn plus moe_combine's checks.
 * ---------------------------------------------------------------------------------------------------- */
moe_status moe_expert_ffn_combine(const uint16_t* x, const int32_t* expert_ids, const uint16_t* weights,
                                  const uint16_t* expert_weights, uint16_t* expert_out, uint16_t* y,
                                  void* workspace, size_t workspace_bytes, int64_t num_tokens, int64_t hidden_size,
                                  int64_t num_experts, int64_t top_k, int64_t intermediate_size, void* stream);

/* ------------------------------------------------------------------------------------------------------
 * Optional fast path: the whole layer, MoeRoutingTopK -> MoeExpertFFN -> MoeCombine, in one call. It has no
 * single counterpart in the reference, whose harness chains the three operators (tests/test_moe.cpp:520-612:
 * routing, FFN, combine on one stream); the three operators stay the contract. On the LDS-tiled schedule the
 * routing kernel also ranks each token block's (token, k) slots by expert, so the FFN's permute is a single
 * scatter launch after it (the per-expert id scan of op_kernel/moe_expert_ffn.cpp:182-195, done once); on the
 * weight-streaming schedule it is routing (for T <= 16 and E > 64 spread over 4 * E / 32 workgroups, whose fp32
 * sums pass through the workspace) followed by moe_expert_ffn_combine. expert_ids, weights, expert_out and y are
 * bit-identical to the three calls' (each with the workspace of its own query). Deterministic (no global atomics;
 * nothing depends on timing).
 * The workspace is moe_layer_workspace_bytes() (>= moe_expert_ffn_workspace_bytes()); 0 = unsupported sizes; not
 * monotone in num_tokens and covering both schedules, as moe_expert_ffn_workspace_bytes().
 * Sizes and errors as the three operators' checks together.
 * ---------------------------------------------------------------------------------------------------- */
size_t moe_layer_workspace_bytes(int64_t num_tokens, int64_t hidden_size, int64_t num_experts, int64_t top_k,
                                 int64_t intermediate_size);
moe_status moe_layer(const uint16_t* x, const uint16_t* w_gate, const uint16_t* expert_weights,
                     int32_t* expert_ids, uint16_t* weights, uint16_t* expert_out, uint16_t* y, void* workspace,
                     size_t workspace_bytes, int64_t num_tokens, int64_t hidden_size, int64_t num_experts,
                     int64_t top_k, int64_t intermediate_size, void* stream);

/* ======================================================================================================
 * Operators around the routed experts. The reference has none of them: they are what a layer with scored and
 * grouped routing, a dense expert beside the routed ones, or a training step of its router needs next to the
 * three operators above. Tensors, streams, workspaces and errors as there.
 * ==================================================================================================== */

typedef enum moe_scoring { MOE_SCORE_SOFTMAX = 0, MOE_SCORE_SIGMOID = 1 } moe_scoring;

typedef enum moe_activation {
    MOE_ACT_NONE = 0,
    MOE_ACT_RELU = 1,
    MOE_ACT_GELU = 2,      /* z/2 (1 + erf(z / sqrt 2))                              */
    MOE_ACT_GELU_TANH = 3, /* z/2 (1 + tanh(sqrt(2 / pi) (z + 0.044715 z^3)))        */
    MOE_ACT_SILU = 4,      /* z / (1 + exp(-z))                                      */
    MOE_ACT_SWIGLU = 5     /* silu(gate) * up: 2 N weight rows, the N gate rows first */
} moe_activation;

/* ------------------------------------------------------------------------------------------------------
 * MoeRoutingGroupTopK: logits[T, E] (float32, float16 or bfloat16, rows logits_stride >= E elements apart),
 *   bias[E] float32 or NULL -> expert_ids[T, K] int32, weights[T, K] (float16 or float32).
 *   s = softmax or sigmoid of a row, c = s + bias. The groups are E / groups consecutive experts; a group's score is
 *   its best c (group_top 1) or the sum of its two best (group_top 2), and only the top_groups best groups stay (equal
 *   scores: the lower group). expert_ids are the K best c of the experts that stay, in descending order (equal
 *   c: the lower index). weights = scale * s, divided by the sum of the K chosen s where renormalize is set
 *   (the ratios hold where the scores themselves would underflow). bias only steers the choice.
 *   c is compared beyond fp32: without a bias by the logits, which order the scores, with one in float64. An expert
 *   whose logit or c is NaN or -infinity is not available; where a row has fewer than K available ones the picks left
 *   are id -1 and weight 0, which moe_expert_ffn computes as zero rows. 1 <= K <= top_groups * E / groups, E <= 256.
 * ---------------------------------------------------------------------------------------------------- */
moe_status moe_routing_group_topk(const void* logits, int64_t logits_stride, int32_t logits_type, const float* bias,
                                  int32_t* expert_ids, void* weights, int32_t weights_type, int64_t num_tokens,
                                  int64_t num_experts, int64_t top_k, int64_t groups, int64_t top_groups,
                                  int64_t group_top, int32_t scoring, int32_t renormalize, float scale, void* stream);

/* Its gradient: grad_weights[T, K] (float32, float16 or bfloat16), the same logits and the expert_ids it chose ->
 * grad_logits[T, E] contiguous, of logits_type. The choice itself has no gradient, so bias has none. Ids outside
 * [0, E) and unavailable experts receive nothing; an id that a row holds twice receives both. Any K in [1, E]. */
moe_status moe_routing_group_topk_grad(const void* grad_weights, int32_t weights_type, const void* logits,
                                       int64_t logits_stride, int32_t logits_type, const int32_t* expert_ids,
                                       void* grad_logits, int64_t num_tokens, int64_t num_experts, int64_t top_k,
                                       int32_t scoring, int32_t renormalize, float scale, void* stream);

/* ------------------------------------------------------------------------------------------------------
 * MoeCombineGrad: grad_y[T, H], expert_out[T, K, H], weights[T, K] fp16 -> grad_expert_out[T, K, H] =
 *   weights * grad_y, grad_weights[T, K] = <grad_y, expert_out> (fp32 sums), both fp16. H a multiple of 8.
 * ---------------------------------------------------------------------------------------------------- */
moe_status moe_combine_grad(const uint16_t* grad_y, const uint16_t* expert_out, const uint16_t* weights,
                            uint16_t* grad_expert_out, uint16_t* grad_weights, int64_t num_tokens,
                            int64_t hidden_size, int64_t top_k, void* stream);

/* ------------------------------------------------------------------------------------------------------
 * MoeLinear: x[T, H], weight[N, H] (SwiGLU: [2N, H]) -> y[T, N] = act(x weight^T + bias) + residual, fp32 sums, rounded
 *   once. x and weight are float16 or bfloat16 (dtype); x rows lie x_stride elements apart. weight's rows lie
 *   weight_stride apart; with weight_transposed set it is stored [H, N] with weight_stride between the H rows, as
 *   MoeRoutingTopK's w_gate. bias[N] (SwiGLU: [2N]) of dtype, or NULL; residual[T, N] of out_dtype, or NULL; out_dtype
 *   is dtype or float32. pre, if not NULL, receives the sums before the activation, [T, N] (SwiGLU: [T, 2N]) of dtype,
 *   which moe_linear_grad takes. Any sizes from 1; N, H <= 2^20.
 *   Any strides and alignment. 16-byte aligned operands whose strides are multiples of 8 run at full speed. Where H (of
 *   a transposed weight N) is no multiple of 8, x and the weight are first copied with padded rows; other operands that
 *   16-byte copies cannot read go through registers, at a fraction of the speed. residual may be y itself.
 *   The workspace (moe_linear_workspace_bytes, either layout's; 0 where none is needed; 16-byte aligned) holds fp32
 *   partial sums of a product split over H and those copies; calls in flight at the same time, captured graphs among
 *   them, need one each. Deterministic: the order of every sum depends on the sizes, strides and alignment alone.
 * ---------------------------------------------------------------------------------------------------- */
size_t moe_linear_workspace_bytes(int64_t num_tokens, int64_t n, int64_t hidden_size, int32_t activation);
moe_status moe_linear(const void* x, int64_t x_stride, const void* weight, int64_t weight_stride,
                      int32_t weight_transposed, const void* bias, const void* residual, void* y, void* pre,
                      void* workspace, size_t workspace_bytes, int64_t num_tokens, int64_t n, int64_t hidden_size,
                      int32_t activation, int32_t dtype, int32_t out_dtype, void* stream);

/* moe_linear with the workspace that the weight's layout needs alone: copies of a weight stored [H, N] need room only
 * where weight_transposed is set. T = 1, N = 50257, H = 8192 by rows: none, where moe_linear wants 823 MB. */
size_t moe_linear_layout_workspace_bytes(int64_t num_tokens, int64_t n, int64_t hidden_size, int32_t activation,
                                         int32_t weight_transposed);
moe_status moe_linear_layout(const void* x, int64_t x_stride, const void* weight, int64_t weight_stride,
                             int32_t weight_transposed, const void* bias, const void* residual, void* y, void* pre,
                             void* workspace, size_t workspace_bytes, int64_t num_tokens, int64_t n,
                             int64_t hidden_size, int32_t activation, int32_t dtype, int32_t out_dtype, void* stream);

/* MoeLinearGrad: grad_y[T, N] of dtype (rows grad_y_stride apart) and what moe_linear had -> grad_x[T, H],
 * grad_weight[N, H] (SwiGLU: [2N, H]) and grad_bias, contiguous, of dtype; each may be NULL (not wanted). pre is
 * moe_linear's (not read without an activation). dz = grad_y * act'(pre) is rounded to dtype for the two products
 * grad_x = dz weight and grad_weight = dz^T x (with float16 values above 65504 become infinite, below 2^-25 zero);
 * grad_bias sums it before that. residual's gradient is grad_y.
 * With T = 0 grad_weight and grad_bias are zeros. The workspace holds dz, column sums, copies with padded rows and
 * partial sums: always needed, by the same rules. */
size_t moe_linear_grad_workspace_bytes(int64_t num_tokens, int64_t n, int64_t hidden_size, int32_t activation);
moe_status moe_linear_grad(const void* grad_y, int64_t grad_y_stride, const void* x, int64_t x_stride,
                           const void* weight, int64_t weight_stride, int32_t weight_transposed, const void* pre,
                           void* grad_x, void* grad_weight, void* grad_bias, void* workspace, size_t workspace_bytes,
                           int64_t num_tokens, int64_t n, int64_t hidden_size, int32_t activation, int32_t dtype,
                           void* stream);

/* moe_linear_grad with the workspace that the weight's layout needs alone, as moe_linear_layout. */
size_t moe_linear_grad_layout_workspace_bytes(int64_t num_tokens, int64_t n, int64_t hidden_size, int32_t activation,
                                              int32_t weight_transposed);
moe_status moe_linear_grad_layout(const void* grad_y, int64_t grad_y_stride, const void* x, int64_t x_stride,
                                  const void* weight, int64_t weight_stride, int32_t weight_transposed,
                                  const void* pre, void* grad_x, void* grad_weight, void* grad_bias, void* workspace,
                                  size_t workspace_bytes, int64_t num_tokens, int64_t n, int64_t hidden_size,
                                  int32_t activation, int32_t dtype, void* stream);

/* The same for the gradient of a float32 result: grad_y is float32, the gradients of dtype. dz is rounded to dtype for
 * the products, with float16 after a multiplication by the power of two that takes its largest finite value to
 * [2^14, 2^15), which the sums are divided by: dz does not overflow, and what vanishes is below 2^-39 of its largest
 * value.
 * grad_y of any alignment (4 bytes) and row stride. */
size_t moe_linear_grad_f32_workspace_bytes(int64_t num_tokens, int64_t n, int64_t hidden_size, int32_t activation,
                                           int32_t weight_transposed);
moe_status moe_linear_grad_f32(const float* grad_y, int64_t grad_y_stride, const void* x, int64_t x_stride,
                               const void* weight, int64_t weight_stride, int32_t weight_transposed, const void* pre,
                               void* grad_x, void* grad_weight, void* grad_bias, void* workspace,
                               size_t workspace_bytes, int64_t num_tokens, int64_t n, int64_t hidden_size,
                               int32_t activation, int32_t dtype, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MOE_OPS_H */
