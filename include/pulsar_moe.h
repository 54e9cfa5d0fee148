/* pulsar_moe.h - C ABI of the MI355X (gfx950) quantized expert-matvec library.
 *
 * Every entry point keeps the name, argument order, argument meaning and
 * return convention of the reference kernel library it replaces, so the
 * reference's Rust FFI block (crates/kernels/src/lib.rs:78-194) binds this
 * library unchanged:
 *   - return 1 on success, 0 on failure (invalid arguments or a launch error);
 *     the reason is printed as "pulsar-kernels: <what>: <error>" on stderr
 *     (crates/kernels/cuda/pulsar_kernels.cu:25-29);
 *   - every pointer argument except the self-tests' is a DEVICE pointer the
 *     caller owns; the library allocates nothing on these paths;
 *   - launches are asynchronous on the calling thread's per-thread default
 *     stream (hipStreamPerThread), the stream the reference's
 *     --default-stream=per-thread build launches on
 *     (crates/kernels/build.rs:42-48), so a thread-local graph capture begun
 *     on it records them; pulsar_set_stream selects another stream. Nothing
 *     here synchronises.
 *   - one axis of a launch holds fewer than 2^32 threads, and the runtime leaves
 *     out what is past them without an error: calls that go by values or rows
 *     take two axes (up to 2^31 - 1 blocks: of 256 values, of 4 q8_K blocks, of
 *     an f32 product's row and two tokens, of a routed token), the MoE stages
 *     refuse the rows of an expert that one does not hold (fewer than 2^24 always
 *     go). f32 rows have at most 2^32 - 256 values.
 *
 * Byte layouts are the GGUF/ggml ones (crates/gguf/src/lib.rs:145-180):
 *   Q2_K 84 B / 256, Q4_K 144 B / 256, Q6_K 210 B / 256, IQ2_XXS 66 B / 256,
 *   MXFP4 17 B / 32 (rows pack whole 32-value blocks, not super-blocks),
 *   q8_K 292 B / 256.
 */
#ifndef PULSAR_MOE_H
#define PULSAR_MOE_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Quant codes (crates/kernels/src/lib.rs:55-73; pulsar_kernels.cu:2649-2668),
 * every one the reference defines. Bytes per 256 values: Q2_K 84, IQ2_XXS 66,
 * Q4_K 144, Q5_K 176, Q6_K 210, Q3_K 110, IQ2_XS 74, IQ3_XXS 98, Q4_0 8 x 18,
 * Q5_1 8 x 24, Q8_0 8 x 34, IQ4_XS 136, MXFP4 8 x 17, IQ4_NL 8 x 18, IQ3_S
 * 110, IQ2_S 82, IQ1_S 50, NVFP4 4 x 36 (crates/gguf/src/lib.rs:145-172). */
#define PULSAR_QUANT_Q2_K     0u
#define PULSAR_QUANT_IQ2_XXS  1u
#define PULSAR_QUANT_Q4_K     2u
#define PULSAR_QUANT_Q5_K     3u
#define PULSAR_QUANT_Q6_K     4u
#define PULSAR_QUANT_Q3_K     5u
#define PULSAR_QUANT_IQ2_XS   6u
#define PULSAR_QUANT_IQ3_XXS  7u
#define PULSAR_QUANT_Q4_0     8u
#define PULSAR_QUANT_Q5_1     9u
#define PULSAR_QUANT_Q8_0    10u
#define PULSAR_QUANT_IQ4_XS  11u
#define PULSAR_QUANT_MXFP4   12u
#define PULSAR_QUANT_IQ4_NL  13u
#define PULSAR_QUANT_IQ3_S   14u
#define PULSAR_QUANT_IQ2_S   15u
#define PULSAR_QUANT_IQ1_S   16u
#define PULSAR_QUANT_NVFP4   17u
/* OR'd into `quant` by callers that permit W4A4 (crates/kernels/src/lib.rs:51-55);
 * accepted and ignored here (it only selects an NVFP4 path in the reference). */
#define PULSAR_QUANT_A4_OK   0x80000000u

/* act_op codes of the gated combine (pulsar_kernels.cu:114-141) */
#define PULSAR_ACT_SILU        0u /* silu(g) * u */
#define PULSAR_ACT_SWIGLU_OAI  2u /* gpt-oss: clamp 7, alpha 1.702, (u + 1) */

/* act codes of the dense product's epilogue (pulsar_matmul_kq_fused) */
#define PULSAR_EPI_NONE    0u
#define PULSAR_EPI_SILU    1u /* v / (1 + exp(-v)) */
#define PULSAR_EPI_GELU    2u /* v / 2 (1 + tanh(sqrt(2 / pi) (v + 0.044715 v^3))) */
#define PULSAR_EPI_RELU    3u /* max(v, 0) */
#define PULSAR_EPI_SIGMOID 4u /* 1 / (1 + exp(-v)) */

/* scores of pulsar_router_select_groups */
#define PULSAR_SCORE_SIGMOID 0u
#define PULSAR_SCORE_SOFTMAX 1u

/* element types of the rows that pulsar_rms_norm_q8, pulsar_quantize_i8 and
 * pulsar_matmul_i8 read or write (every other call's rows are f32) */
#define PULSAR_TYPE_F32  0u
#define PULSAR_TYPE_F16  1u
#define PULSAR_TYPE_BF16 2u

/* 8-bit rows that pulsar_rms_norm_q8 writes */
#define PULSAR_ROWS_Q8_K 0u /* q8_K blocks */
#define PULSAR_ROWS_I8   1u /* int8 values, one f32 scale a row */

#define PULSAR_QK_K 256u

/* q8_K activation block (pulsar_kernels.cu:1492-1496; lane Q8KRow,
 * crates/quant/src/cpu_dot.rs:19-23): d at byte 0, qs at 4, bsums at 260. */
typedef struct pulsar_block_q8_K {
    float d;
    int8_t qs[256];
    int16_t bsums[16];
} pulsar_block_q8_K;

/* Per-(token, slot) expert pointers (pulsar_kernels.cu:2555-2564;
 * crates/kernels/src/lib.rs:21-49). A NULL gate or up makes the pair stage
 * write 0 for that slot; a NULL down makes the down stage skip it; NULL
 * biases are skipped. gate_b/up_b hold mid_dim floats, down_b out_dim. */
typedef struct pulsar_expert_ptrs {
    const void *gate;
    const void *up;
    const void *down;
    const float *gate_b;
    const float *up_b;
    const float *down_b;
} pulsar_expert_ptrs;

#ifdef __cplusplus
static_assert(sizeof(pulsar_block_q8_K) == 292, "block_q8_K is 292 bytes");
static_assert(sizeof(pulsar_expert_ptrs) == 48, "pulsar_expert_ptrs is 48 bytes");
#else
_Static_assert(sizeof(pulsar_block_q8_K) == 292, "block_q8_K is 292 bytes");
_Static_assert(sizeof(pulsar_expert_ptrs) == 48, "pulsar_expert_ptrs is 48 bytes");
#endif

/* f32 rows [n_rows][in_dim] -> q8_K rows [n_rows][ceil(in_dim/256)].
 * Algorithm of the CPU lane (crates/quant/src/cpu_dot.rs:26-50): d = amax/127,
 * q = clamp(round_half_away(x * (127/amax)), -127, 127), bsums = 16-sums;
 * elements past in_dim in the tail block quantize to 0 (pulsar_kernels.cu:1499-1501).
 * Replaces pulsar_quantize_q8_K (pulsar_kernels.cu:1552). */
int pulsar_quantize_q8_K(void *out, const void *x, uint32_t in_dim, uint32_t n_rows);

/* out[t][r] = sum_b dot(w row r block b, xq[t] block b), fp32 [n_tok][out_dim].
 * quant: the reference's dense list (pulsar_kernels.cu:5090-5142) - Q2_K,
 * IQ2_XXS, Q4_K, Q5_K, Q6_K, Q3_K, IQ4_XS, IQ4_NL, NVFP4 (the expert-only
 * formats return 0, as there); in_dim % 256 == 0. Chunks of 5 or more tokens
 * run on the int8 matrix cores (IQ4_NL and the smallest chunks of the formats
 * without a 16-row kernel excepted). xq may start at any byte, here and in the
 * grouped stages; rows on a 4-byte boundary run fastest.
 * Replaces pulsar_matmul_kq (pulsar_kernels.cu:4895). */
int pulsar_matmul_kq(void *out, const void *w, const void *xq, uint32_t in_dim,
                     uint32_t out_dim, uint32_t n_tok, uint64_t row_bytes,
                     uint32_t quant);

/* ---- 8-bit rows with a scale each, and what a layer makes them of (no reference
 * counterpart: the reference runs its norms in kernels of their own and quantizes
 * their f32 rows) ----
 *
 * Codes of 8 bits, in all of these: of values v with the largest size A = max |v|
 * (of the row, or of a q8_K block), q = 127 v / A to the nearest integer, halves away
 * from 0, decided as it stands in 64 bits (an argument nearer than 2^-40 to a half
 * counts as on it); the scale is A / 127, rounded to f32. A row of zeros has codes and
 * scale 0. Where a row (block) holds a NaN its scale is NaN, where it holds an infinity
 * the scale is infinite (in the norm, where a row's infinity makes the root 0, NaN; one
 * of the two where a gain is not finite); the codes of what is not finite are 0. Strides count elements (bytes in int8 rows), 0 stands for
 * packed rows; what lies between rows is left as it is. */

/* s = x + residual (NULL: x), rounded to `type`; y = s * gain / sqrt(mean(s^2) + eps)
 * and its 8-bit form, in one pass:
 *   sum       s, rows of `type` (NULL: left out); may be x or residual itself, at the
 *             same stride
 *   y         packed rows of `type` (NULL: left out)
 *   q         format PULSAR_ROWS_Q8_K: q8_K [n_rows][ceil(dim / 256)], as
 *             pulsar_matmul_kq and the routed stages read them, values past dim 0;
 *             scales NULL, q_stride 0. PULSAR_ROWS_I8: int8 rows q_stride apart, scales
 *             f32 [n_rows], as pulsar_matmul_i8 reads them. NULL: left out
 * gain f32 [dim]. The codes are those of s * gain, which the root does not change, so
 * they are not off by y's rounding: pulsar_quantize_q8_K of y, which decides in f32,
 * gives another code for about one value in 10^5, by 1. Sums of squares are kept in 64
 * bits and do not overflow. A row of zeros gives zeros with eps 0 too; eps >= 0. y or q
 * has to be there. dim <= 2^24, n_rows < 2^31, strides < 2^32. Outputs over an input or another
 * output are refused, but for sum as above. */
int pulsar_rms_norm_q8(void *q, void *scales, void *y, void *sum, const void *x,
                       const void *residual, const void *gain, uint32_t dim, uint32_t n_rows,
                       float eps, uint32_t type, uint32_t format, uint64_t x_stride,
                       uint64_t res_stride, uint64_t sum_stride, uint64_t q_stride);

/* Rows of `type` to int8 rows with a scale each (f32 [n_rows]): of v = x, or where up
 * is given of v = glu(x, up, act_op), the gated combine of pulsar_moe_pair_swiglu in 64
 * bits (SWIGLU_OAI's alpha: 1.702). Gates far below 0 count as they stand, under
 * e^gate's end of the normal numbers too (the scale is 0 there); where it is below 2^-1074
 * for the whole row, about -745, the row is one of zeros. up NULL: act_op 0. gate and up
 * may be columns of one array. dim <= 2^24, n_rows < 2^31, strides < 2^32. q or scales over
 * an input or one another are refused. */
int pulsar_quantize_i8(void *q, void *scales, const void *x, const void *up, uint32_t dim,
                       uint32_t n_rows, uint32_t act_op, uint32_t type, uint64_t x_stride,
                       uint64_t up_stride, uint64_t q_stride);

/* out[t][r] = act(x_scales[t] w_scales[r] sum_i x[t][i] w[r][i] + bias[r]) + residual[t][r]
 * int8 x [n_tok] and w [out_dim] rows of in_dim values, x_stride and w_stride bytes apart;
 * f32 x_scales [n_tok], w_scales [out_dim], bias [out_dim] (NULL: none); residual (NULL:
 * none) and out rows of `type`, res_stride and out_stride elements apart; act: a
 * PULSAR_EPI_* code. The sums are exact in 32 bits (in_dim <= 131071: 2^14 a product);
 * sum, times the token's scale, times the channel's: a rounding to f32 each, as for bias,
 * activation and residual; one to `type` at the end. residual may be out itself, at the
 * same stride; any other overlap of out with an operand is refused. x_stride and w_stride
 * <= 2^23, out_stride and res_stride < 2^32, n_tok and out_dim < 2^31 (2^31 tiles of 128
 * tokens x 128 channels are refused). Rows of whole 16 bytes on 16-byte boundaries (base,
 * stride and in_dim) run fastest. */
int pulsar_matmul_i8(void *out, const void *w, const void *w_scales, const void *x,
                     const void *x_scales, const void *bias, const void *residual,
                     uint32_t in_dim, uint32_t out_dim, uint32_t n_tok, uint32_t act,
                     uint32_t type, uint64_t w_stride, uint64_t x_stride, uint64_t out_stride,
                     uint64_t res_stride);

/* pulsar_matmul_kq with its epilogue in the same launch (no reference
 * counterpart: the reference runs the bias, the activation and the residual
 * add as kernels of their own):
 *   out[t][r] = act(dot(w row r, xq[t]) + bias[r]) + residual[t][r]
 * bias f32 [out_dim] and residual f32 rows are left out where NULL; act: a
 * PULSAR_EPI_* code. Row t of out starts at t * out_stride floats, of residual
 * at t * res_stride (0: out_dim, the packed rows; never less than out_dim);
 * floats between the rows are left as they are. residual may be out itself, at
 * the same stride (each element is read before it is written); any other
 * overlap of out with an operand is refused. Formats and limits are
 * pulsar_matmul_kq's, and so are the dots, but short chunks run a kernel of their
 * own, which adds a row's super-blocks in another order. That kernel is 1.36 times
 * as fast on average, so a chunk of 2 to some 500 tokens is worth this call without
 * an epilogue too (bias and residual NULL, PULSAR_EPI_NONE); where both calls run
 * the same kernel, this one takes 4% longer. */
int pulsar_matmul_kq_fused(void *out, const void *w, const void *xq, const void *bias,
                           const void *residual, uint32_t in_dim, uint32_t out_dim,
                           uint32_t n_tok, uint64_t row_bytes, uint32_t quant, uint32_t act,
                           uint64_t out_stride, uint64_t res_stride);

/* mid[t][s][r] = glu(gate_r . x_t + gate_b[r], up_r . x_t + up_b[r], act_op) * weights[t][s].
 * ptrs: pulsar_expert_ptrs[n_tok][n_used]; weights: f32 [n_tok][n_used];
 * xq: q8_K [n_tok][ceil(in_dim/256)]. Replaces pulsar_moe_pair_swiglu
 * (pulsar_kernels.cu:5149). */
int pulsar_moe_pair_swiglu(void *mid, const void *ptrs, const void *weights,
                           const void *xq, uint32_t in_dim, uint32_t mid_dim,
                           uint32_t n_used, uint32_t n_tok, uint64_t row_bytes,
                           uint32_t quant, uint32_t act_op);

/* out[t][r] = sum_s down_r(slot s) . midq[t][s], fp32 [n_tok][out_dim];
 * midq: q8_K [n_tok][n_used][ceil(mid_dim/256)]. Replaces pulsar_moe_down
 * (pulsar_kernels.cu:5289). */
int pulsar_moe_down(void *out, const void *ptrs, const void *midq,
                    uint32_t mid_dim, uint32_t out_dim, uint32_t n_used,
                    uint32_t n_tok, uint64_t row_bytes, uint32_t quant);

/* Grouped (CSR by expert) pair stage: gptrs [n_group], starts [n_group+1],
 * pairs [starts[n_group]] packing token << 4 | slot (n_used <= 16).
 * Writes mid[t][s][r] for every listed pair. Replaces
 * pulsar_moe_pair_swiglu_grouped (pulsar_kernels.cu:3483). */
int pulsar_moe_pair_swiglu_grouped(void *mid, const void *gptrs, const void *starts,
                                   const void *pairs, const void *weights,
                                   const void *xq, uint32_t in_dim, uint32_t mid_dim,
                                   uint32_t n_used, uint32_t n_group,
                                   uint64_t row_bytes, uint32_t quant,
                                   uint32_t act_op);

/* Grouped down stage: partial[t][s][r] = down_r(group of (t,s)) . midq[t][s]
 * for every listed pair; unlisted (t, s) are left untouched, so the caller
 * zeroes partial before every layer (crates/engine/src/lib.rs:8481-8482):
 * pulsar_moe_slot_sum reads every slot. Replaces pulsar_moe_down_grouped
 * (pulsar_kernels.cu:3537). */
int pulsar_moe_down_grouped(void *partial, const void *gptrs, const void *starts,
                            const void *pairs, const void *midq, uint32_t mid_dim,
                            uint32_t out_dim, uint32_t n_used, uint32_t n_group,
                            uint64_t row_bytes, uint32_t quant);

/* The two grouped calls for a caller that knows how many pairs its CSR lists
 * at most (the capacity of `pairs`; starts[n_group] - starts[0] <= max_pairs).
 * The calls above do not: where the tile may take the stage they launch two
 * kernels, each of which works or ends at once by the groups' mean on the
 * device. These leave the second out where max_pairs / n_group shows the
 * groups short. The same rows. */
int pulsar_moe_pair_swiglu_grouped_bounded(void *mid, const void *gptrs, const void *starts,
                                           const void *pairs, const void *weights,
                                           const void *xq, uint32_t in_dim, uint32_t mid_dim,
                                           uint32_t n_used, uint32_t n_group,
                                           uint64_t row_bytes, uint32_t quant,
                                           uint32_t act_op, uint32_t max_pairs);
int pulsar_moe_down_grouped_bounded(void *partial, const void *gptrs, const void *starts,
                                    const void *pairs, const void *midq, uint32_t mid_dim,
                                    uint32_t out_dim, uint32_t n_used, uint32_t n_group,
                                    uint64_t row_bytes, uint32_t quant, uint32_t max_pairs);

/* out[t][r] = sum_s partial[t][s][r] in slot order. Replaces
 * pulsar_moe_slot_sum (pulsar_kernels.cu:3651). */
int pulsar_moe_slot_sum(void *out, const void *partial, uint32_t out_dim,
                        uint32_t n_used, uint32_t n_tok);

/* out[t][r] += sum_s weights[t][s] * down_b(slot s)[r] (slots with a NULL
 * down_b skipped; nothing added where the sum is 0). Replaces
 * pulsar_moe_down_bias (pulsar_kernels.cu:3640). */
int pulsar_moe_down_bias(void *out, const void *ptrs, const void *weights,
                         uint32_t out_dim, uint32_t n_used, uint32_t n_tok);

/* Router top-k (pulsar_kernels.cu:938-1050): selected int32 and weights f32
 * [n_tok][k_used(+n_shexp)] from logits f32 [n_tok][n_expert(+n_shexp)].
 * mode 0 sigmoid + bias, normalised; mode 1 softmax over the k winners
 * (selection on raw logit + bias); mode 2 sigmoid+bias selection with the
 * shared "sink" logits appended, weights softmax(logsigmoid). Ties go to the
 * lower expert index. n_expert(+n_shexp) <= 1024. Replaces
 * pulsar_router_select (pulsar_kernels.cu:1052). */
int pulsar_router_select(void *selected, void *weights, const void *logits,
                         const void *bias, uint32_t n_expert, uint32_t k_used,
                         float weight_scale, uint32_t n_tok, uint32_t softmax_mode,
                         uint32_t n_shexp);

/* Routing with expert groups (no reference counterpart). Per token, of its
 * logits f32 [n_expert]:
 *   score s: PULSAR_SCORE_SIGMOID 1 / (1 + exp(-l)), PULSAR_SCORE_SOFTMAX the
 *     softmax over the token's experts; +-inf beyond f32 counts as the largest
 *     finite value
 *   choice c = s + bias[e] (bias f32 [n_expert], NULL: s alone). A logit or
 *     bias of NaN or -inf takes its expert out of the choice (the logit out of
 *     the softmax too)
 *   groups: n_group groups of n_expert / n_group neighbouring experts; a group
 *     stands with the sum of its group_top (1 or 2) largest c (with one alone
 *     if it has no other); the topk_group best groups are kept, ties to the
 *     lower group. n_group = 1: every expert
 *   selected int32 [n_tok][k_used]: the largest c of the kept groups in
 *     falling order, ties to the lower id, each expert once; -1 with weight 0
 *     where fewer than k_used are left
 *   weights f32 [n_tok][k_used]: the winners' s (without the bias); renorm != 0:
 *     over their sum (sigmoid: at least 2^-14, as pulsar_router_select; softmax:
 *     all 0 where every winner's s is 0 in 64 bits); times weight_scale
 * Ids are decided as c stands in 64 bits, whatever f32 would round it to.
 * n_expert <= 1024, a multiple of n_group <= 64; k_used <= 64 and <= the
 * experts of topk_group groups; n_tok <= 2^25. selected and weights over one
 * another, the logits or the bias are refused. */
int pulsar_router_select_groups(void *selected, void *weights, const void *logits,
                                const void *bias, uint32_t n_expert, uint32_t k_used,
                                uint32_t n_group, uint32_t topk_group, uint32_t group_top,
                                uint32_t score, uint32_t renorm, float weight_scale,
                                uint32_t n_tok);

/* out[t][o] = sum_i w[o][i] * x[t][i] in fp32 (router logits). Replaces
 * pulsar_matmul_f32 (pulsar_kernels.cu:6526). */
int pulsar_matmul_f32(void *out, const void *w, const void *x, uint32_t in_dim,
                      uint32_t out_dim, uint32_t n_tok);

/* x[r][i] += bias[i] for rows rows of dim floats. Replaces
 * pulsar_add_bias_rows (pulsar_kernels.cu:3631). */
int pulsar_add_bias_rows(void *x, const void *bias, uint32_t dim, uint32_t rows);

/* ---- device-side routing (no counterpart entry point in the reference) ----
 * The reference builds the per-(token, slot) pointer array and the grouped
 * CSR on the host after reading the router's ids back
 * (crates/engine/src/lib.rs:7663-7670, 8255-8344, 8357-8392). These two
 * entry points do the same on the device, so a layer needs no host round
 * trip. */

/* One resident expert bank per projection: expert e's matrix starts at
 * base + e * stride bytes; its bias (NULL base = none) at b_base + e * b_stride
 * floats. Passed by host pointer, read at launch. */
typedef struct pulsar_expert_bank {
    const void *gate;
    const void *up;
    const void *down;
    const float *gate_b;
    const float *up_b;
    const float *down_b;
    uint64_t gate_stride;
    uint64_t up_stride;
    uint64_t down_stride;
    uint64_t gate_b_stride;
    uint64_t up_b_stride;
    uint64_t down_b_stride;
} pulsar_expert_bank;

/* ptrs[t][s] / slot_weights[t][s] for s < k_used from the router's
 * selected ids and weights ([n_tok][k_used]); an id outside [0, n_expert)
 * gives a NULL slot. Then n_shared always-on slots (s = k_used + i) with
 * pointers shared[i] (host array) and weight 1. Row stride of both outputs
 * is k_used + n_shared. Replaces the host pointer build at
 * crates/engine/src/lib.rs:8255-8344. */
int pulsar_moe_route_ptrs(void *ptrs, void *slot_weights, const void *selected,
                          const void *router_weights, const pulsar_expert_bank *bank,
                          uint32_t n_expert, const pulsar_expert_ptrs *shared,
                          uint32_t n_shared, uint32_t n_tok, uint32_t k_used);

/* Groups the (token, slot) pairs of ptrs [n_tok][n_used] by expert (equal
 * gate pointer, groups in order of first appearance, members in (token,
 * slot) order; NULL gates skipped), as crates/engine/src/lib.rs:8357-8392
 * does on the host. Writes gptrs [max_groups], starts [max_groups + 1] and
 * pairs (token << 4 | slot); group slots past the real count get NULL
 * pointers and empty ranges, so the grouped kernels can always be launched
 * with n_group = max_groups (which must be at least the number of distinct
 * experts, e.g. min(n_expert, n_tok * n_used)). n_used <= 16,
 * n_tok * n_used <= 2048. */
int pulsar_moe_group_csr(void *gptrs, void *starts, void *pairs, const void *ptrs,
                         uint32_t n_tok, uint32_t n_used, uint32_t max_groups);

/* The CSR by expert of a chunk of any length, straight from the router's ids
 * (pulsar_moe_group_csr takes at most 2048 pairs): group e < n_expert is bank
 * expert e, its pairs (token << 4 | slot) in (token, slot) order, empty for an
 * expert nothing selects; group n_expert + i is shared slot k_used + i of every
 * token. Writes gptrs [n_expert + n_shared], starts [n_expert + n_shared + 1]
 * and pairs [starts[n_expert + n_shared]] (room for n_tok * (k_used + n_shared);
 * what lies behind the last pair is left as it is), for the grouped stages with
 * n_group = n_expert + n_shared and n_used = k_used + n_shared. Those have a fast
 * path for long groups up to n_group = 1024: behind 1024 experts, call them once on
 * the first 1024 groups and once on the shared slots' (gptrs and starts + 1024,
 * n_group = n_shared, the same pairs), which writes the same rows, to the rounding
 * for Q3_K and IQ4_XS, whose long groups run on another kernel. 8192 tokens of 8 +
 * 1 slots, 2048 x 512 values: gate / up 0.9 ms in two calls, 12.4 in one for Q4_K,
 * 81 for IQ4_XS. selected int32 [n_tok][k_used]; ids outside [0, n_expert) get no
 * pair, so the caller zeroes partial as for any CSR. slot_weights f32 [n_tok][k_used
 * + n_shared], left out where NULL: router_weights [n_tok][k_used], then 1 for the
 * shared slots. n_expert <= 1024, k_used + n_shared <= 16, n_shared <= 4, n_tok <=
 * 2^28, n_tok * (k_used + n_shared) < 2^31; bank and shared are host pointers read
 * at launch. An output over an input or another output is refused, but for
 * slot_weights that are router_weights themselves where n_shared is 0. gptrs and
 * starts are working memory too while the call runs: two calls that may run at
 * once take buffers of their own. */
int pulsar_moe_group_ids(void *gptrs, void *starts, void *pairs, void *slot_weights,
                         const void *selected, const void *router_weights,
                         const pulsar_expert_bank *bank, uint32_t n_expert,
                         const pulsar_expert_ptrs *shared, uint32_t n_shared, uint32_t n_tok,
                         uint32_t k_used);

/* pulsar_router_select (softmax_mode 0 or 1, no sink slots) +
 * pulsar_moe_route_ptrs + pulsar_moe_group_csr in one launch (no reference
 * counterpart: the reference selects on the device, then builds pointers
 * and the CSR on the host, crates/engine/src/lib.rs:7663-7670,
 * 8255-8392). Outputs equal those three calls': selected / weights
 * [n_tok][k_used], ptrs / slot_weights [n_tok][k_used + n_shared], gptrs,
 * starts, pairs. k_used + n_shared <= 16, n_tok * (k_used + n_shared) <=
 * 2048, k_used <= n_expert <= 1024; bank and shared are host pointers read
 * at launch. */
int pulsar_moe_route_group(void *selected, void *weights, void *ptrs, void *slot_weights,
                           void *gptrs, void *starts, void *pairs, const void *logits,
                           const void *router_bias, uint32_t n_expert, uint32_t k_used,
                           float weight_scale, uint32_t softmax_mode,
                           const pulsar_expert_bank *bank, const pulsar_expert_ptrs *shared,
                           uint32_t n_shared, uint32_t n_tok, uint32_t max_groups);

/* pulsar_router_select (softmax_mode 0 or 1, no sink slots) +
 * pulsar_moe_route_ptrs in one launch (no reference counterpart: the
 * reference selects on the device and builds the pointers on the host,
 * crates/engine/src/lib.rs:7663-7670, 8255-8344). Outputs equal those two
 * calls': selected / weights [n_tok][k_used], ptrs / slot_weights
 * [n_tok][k_used + n_shared]. It also writes active, uint32 [2 + n_expert]
 * (the grouped stages below may read all of it): active[0] = the number of
 * distinct experts the chunk selects,
 * active[1] = the number of NULL slots (ids outside [0, n_expert)),
 * active[2 ..] = the selected expert ids in order of first appearance in
 * (token, slot) order; the expert-indexed grouped stages below read it.
 * k_used + n_shared <= 16, k_used <= n_expert <= 1024, n_tok * (k_used +
 * n_shared) <= 2048; bank and shared are host pointers read at launch. */
int pulsar_moe_route(void *selected, void *weights, void *ptrs, void *slot_weights, void *active,
                     const void *logits, const void *router_bias, uint32_t n_expert, uint32_t k_used,
                     float weight_scale, uint32_t softmax_mode, const pulsar_expert_bank *bank,
                     const pulsar_expert_ptrs *shared, uint32_t n_shared, uint32_t n_tok);

/* The grouped stages with one group per expert the chunk selects, found
 * on the device from pulsar_moe_route's selected and active outputs
 * instead of a CSR (no reference counterpart: the reference groups on the
 * host, crates/engine/src/lib.rs:8357-8392). Each routed (token, slot)
 * pair runs in the group of its expert, shared slot i (s = k_used + i,
 * weight 1) of every token in a group of its own, exactly as
 * pulsar_moe_pair_swiglu_grouped / pulsar_moe_down_grouped would for the
 * same pairs, so the rows they write are bit-identical to those calls',
 * whatever the sizes of the groups. One exception: stages that the lane
 * kernels run where groups are short (Q3_K, IQ4_XS: below about 2 pairs per
 * group; rows of more than 13568 values: below 2 to 3). Each call goes by its
 * own groups' mean; where one is short and the other is not, a row's
 * super-blocks are added in another order and its last bits may differ.
 * Slots whose id is outside [0, n_expert) get rows of 0 in mid (partial),
 * so every row of mid [n_tok][k_used + n_shared][mid_dim] (partial
 * [..][out_dim]) is written and partial needs no zeroing. slot_weights
 * [n_tok][k_used + n_shared]. k_used + n_shared <= 16, n_tok * (k_used +
 * n_shared) <= 2048, n_expert <= 1024; bank and shared are host pointers. */
int pulsar_moe_pair_swiglu_experts(void *mid, const void *selected, const void *active,
                                   const void *slot_weights, const void *xq, const pulsar_expert_bank *bank,
                                   uint32_t n_expert, const pulsar_expert_ptrs *shared, uint32_t n_shared,
                                   uint32_t n_tok, uint32_t k_used, uint32_t in_dim, uint32_t mid_dim,
                                   uint64_t row_bytes, uint32_t quant, uint32_t act_op);
int pulsar_moe_down_experts(void *partial, const void *selected, const void *active, const void *midq,
                            const pulsar_expert_bank *bank, uint32_t n_expert, const pulsar_expert_ptrs *shared,
                            uint32_t n_shared, uint32_t n_tok, uint32_t k_used, uint32_t mid_dim,
                            uint32_t out_dim, uint64_t row_bytes, uint32_t quant);

/* pulsar_moe_slot_sum + pulsar_moe_down_bias in one launch (no reference
 * counterpart; the same sums in the same order, bit-identical to the two
 * calls). */
int pulsar_moe_slot_sum_bias(void *out, const void *partial, const void *ptrs,
                             const void *weights, uint32_t out_dim, uint32_t n_used,
                             uint32_t n_tok);

/* Self-checks: small device runs of the entry points compared with host
 * mirrors (q8_K bit-exact; every stage of the MoE path for Q2_K, IQ2_XXS,
 * Q4_K, Q6_K and MXFP4; router modes 0, 1 and 2). They allocate and
 * synchronise, print one line per case to stderr and return 1 when all pass.
 * Replace pulsar_kernels.cu:6421-6460 and 1271-1285. */
int pulsar_moe_selftest(void);
int pulsar_router_selftest(void);

/* ---- fused decode layer (no reference counterpart: the reference runs
 * these steps as separate launches with a host round trip in between,
 * crates/engine/src/lib.rs:7663-7670, 8416-8510). Each call produces
 * exactly the bytes of the separate calls it replaces. */

/* pulsar_matmul_f32(logits, w_r, x) [+ pulsar_add_bias_rows(logits, bias)
 * when bias != NULL] + pulsar_quantize_q8_K(xq, x, in_dim, n_tok), one
 * launch. */
int pulsar_router_logits_q8(void *logits, void *xq, const void *x, const void *w_r,
                            const void *bias, uint32_t in_dim, uint32_t n_expert,
                            uint32_t n_tok);

/* pulsar_router_select (softmax_mode 0 or 1, no sink slots) +
 * pulsar_moe_route_ptrs + pulsar_moe_pair_swiglu, one launch: every block
 * routes its token itself. Writes selected / weights [n_tok][k_used],
 * ptrs / slot_weights [n_tok][k_used + n_shared] and mid
 * [n_tok][k_used + n_shared][mid_dim]. k_used + n_shared <= 64,
 * n_shared <= 4; bank and shared are host pointers read at launch. */
int pulsar_moe_pair_routed(void *mid, void *ptrs, void *slot_weights, void *selected,
                           void *weights, const void *logits, const void *router_bias,
                           uint32_t n_expert, uint32_t k_used, float weight_scale,
                           uint32_t softmax_mode, const pulsar_expert_bank *bank,
                           const pulsar_expert_ptrs *shared, uint32_t n_shared,
                           const void *xq, uint32_t in_dim, uint32_t mid_dim, uint32_t n_tok,
                           uint64_t row_bytes, uint32_t quant, uint32_t act_op);

/* pulsar_quantize_q8_K(midq, mid, mid_dim, n_tok * n_used) +
 * pulsar_moe_down(out, ptrs, midq, ...) [+ pulsar_moe_down_bias(out, ptrs,
 * slot_weights) when add_bias], one launch; mid is f32
 * [n_tok][n_used][mid_dim]. The token's staged q8_K rows must fit 64 KiB
 * (n_used * ceil(mid_dim / 256) <= 215). */
int pulsar_moe_down_f32(void *out, const void *ptrs, const void *slot_weights, const void *mid,
                        uint32_t mid_dim, uint32_t out_dim, uint32_t n_used, uint32_t n_tok,
                        uint64_t row_bytes, uint32_t quant, uint32_t add_bias);

/* pulsar_moe_down + pulsar_moe_down_bias(out, ptrs, weights), one launch. */
int pulsar_moe_down_biased(void *out, const void *ptrs, const void *weights, const void *midq,
                           uint32_t mid_dim, uint32_t out_dim, uint32_t n_used, uint32_t n_tok,
                           uint64_t row_bytes, uint32_t quant);

/* Selects the stream every later launch from the calling thread goes to
 * (NULL restores the per-thread default stream, the default). No
 * counterpart in the reference, whose launches always use the per-thread
 * default stream (crates/kernels/build.rs:42-48); it lets a caller capture
 * the path into a graph on a stream of its own. Returns 1. */
int pulsar_set_stream(void *stream);

/* Streaming-read probe: reads `bytes` (a multiple of 16) from buf through
 * the compute units; `sink` receives nothing unless the data sums to an
 * impossible value. Replaces pulsar_bw_read (pulsar_kernels.cu:4889). */
int pulsar_bw_read(void *buf, uint64_t bytes, void *sink);

#ifdef __cplusplus
}
#endif

#endif /* PULSAR_MOE_H */
