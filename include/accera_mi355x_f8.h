/*
 * accera_mi355x_f8.h -- C ABI of the feed-forward operators in 8-bit floating point (MI355X, gfx950), in the same library as
 * accera_mi355x_gemm.h: quantising to e4m3 with block scales, the block-scaled matrix product, routing to experts, and the
 * experts' products.
 *
 * Values are OCP e4m3 (ACC950_F8: 1 sign, 4 exponent, 3 mantissa bits, largest 448, no infinity).  The sum of a product runs over
 * blocks of 128: every row of A has one fp32 scale for each block, B has one for each block and 128 (or each single) column.
 *
 * The conventions are those of accera_mi355x_gemm.h: DEVICE pointers, element strides that are 64-bit and not negative, an
 * asynchronous launch on `stream` (a hipStream_t, or NULL for the default stream), an ACC950_* status and
 * acc950_last_error() for its text.  No call allocates device memory or waits for the device, so all may be captured into a graph
 * (after one call outside it: the first launch of a kernel loads its code).  Scratch memory is the caller's; a call that takes
 * some says how much in the function beside it, and calls that may run at the same time (on two streams) take a piece each.  Arguments come in a
 * struct, read before the function returns.
 * None of these has a counterpart in the reference, whose tensorized plans end at 16-bit and int8 inputs
 * (accera/python/accera/Targets.py:796-821).
 */
#ifndef ACCERA_MI355X_F8_H
#define ACCERA_MI355X_F8_H

#include "accera_mi355x_gemm.h"

#if defined(__cplusplus)
extern "C" {
#endif

#define ACC950_F8 6         /* e4m3, an input type of the products below */
#define ACC950_F8_BLOCK 128 /* elements of the product's sum that share a scale */

/* what is done to an input before it is quantised (in fp32) */
#define ACC950_ACT_NONE 0
#define ACC950_ACT_RELU 1
#define ACC950_ACT_SILU_MUL 2 /* x holds [gate | up], 2 * cols wide: gate / (1 + exp(-gate)) * up */

/*
 * q, scale = e4m3 of act(x), a rows x cols matrix of in_type F32 / F16 / BF16.  q is rows x cols, or with `transpose` cols x rows;
 * groups of 128 run along q's rows (its last axis) and group_rows (1 or 128) rows of q share a scale.
 *   s = max(largest |v| of the group / 448, 2^-126)   (power_of_two: the smallest power of two that is not below that)
 *   q = v * (1 / s), rounded to nearest even;  scale = s
 * An infinity or NaN makes its whole group stand for NaN, behind a ReLU too (which keeps a NaN, unlike the product's).  q's elements are contiguous along its last axis.
 * scale[i, b] (i: group of rows, b: block) lies at i * s_row_stride + b * s_block_stride.  Activations go with transpose = 0.
 */
typedef struct acc950_f8_quantize_call {
    int64_t in_type, rows, cols;
    const void* x;
    int64_t x_row_stride, x_col_stride;
    int64_t activation, transpose, group_rows, power_of_two;
    void* q;
    int64_t q_row_stride;
    void* scale;
    int64_t s_row_stride, s_block_stride;
    void* stream;
} acc950_f8_quantize_call;
int acc950_f8_quantize(const acc950_f8_quantize_call* call);

/*
 * C[i, j] = epilogue(sum over blocks b of a_scale[i, b] * b_scale[b, j / group_cols] * sum over k in b of A[i, k] * B[k, j]),
 * out_type F32 / F16 / BF16; epilogue ACC950_EPILOGUE_NONE or _RELU (v > 0 ? v : 0: a NaN gives 0, as everywhere in this library); group_cols 128 or 1.
 * Sums: blocks are added in fp32, always.  Inside a block, F32 results have fp32 sums throughout.  F16 and BF16 ones are left to the e4m3 matrix
 * instruction, twice as fast, which adds its products eight at a time and drops what lies below 2^-13 of the largest of them (2^16 + 2^2 gives 2^16): 2^-16 of a sum
 * of random terms, but 2^-13 of its largest terms where they cancel.  For fp32 sums take an F32 result, or one of the variants that name them below.
 * With B = W^T for a weight W quantised in 128 x 128 blocks this is a layer's forward product; with W quantised transposed the
 * gradient of its input; with both operands quantised transposed and group_cols 1 the gradient of W.
 * Any sizes, strides and alignments; fast where A and B are contiguous along K and their rows start on 16-byte boundaries.  Where they are not, they
 * are laid out anew in `workspace` first, if it holds them; otherwise every element is a load of its own.
 * `variant`: ACC950_VARIANT_AUTO, or ACC950_F8_VARIANT_*; one that does not take the problem returns ACC950_UNSUPPORTED.
 * K may go in slices whose fp32 sums meet in `workspace` (16-byte aligned, or NULL) and are added in their order by a second kernel: small results
 * with a long sum.  acc950_f8_gemm_workspace says how many bytes a call takes for all that; a smaller workspace is right too with ACC950_VARIANT_AUTO, or none (NULL).
 * k_slices: 0 = the library decides, n = at most n slices of a named tile variant (4 * M * (N rounded up to 4) bytes each), which is refused where the workspace
 * does not hold them: a named variant is what the caller asked for, and what is said above of smaller workspaces goes for ACC950_VARIANT_AUTO.
 */
typedef struct acc950_f8_gemm_call {
    int64_t out_type, M, N, K;
    const void* A;
    int64_t a_row_stride, a_col_stride;
    const void* a_scale;
    int64_t as_row_stride, as_block_stride;
    const void* B;
    int64_t b_row_stride, b_col_stride;
    const void* b_scale;
    int64_t bs_block_stride, bs_col_stride, group_cols;
    void* C;
    int64_t c_row_stride, c_col_stride;
    int64_t epilogue, variant, k_slices;
    void* workspace;
    int64_t workspace_bytes;
    void* stream;
} acc950_f8_gemm_call;
int acc950_f8_gemm(const acc950_f8_gemm_call* call);
int64_t acc950_f8_gemm_workspace(const acc950_f8_gemm_call* call); /* (reads no memory but the call's) */
#define ACC950_F8_VARIANT_ANY 0  /* 64x64 tiles, element by element: any strides and alignments; fp32 sums throughout */
#define ACC950_F8_VARIANT_TILE 1 /* + i: LDS tiles of 256x256, 128x128, 64x64, 64x64 (fewer stages) (i = 0 .. 3) on the e4m3 instruction; + 4: with
                                    * fp32 sums throughout (i > 0; 256x256 takes group_cols 128 only) */
#define ACC950_F8_VARIANT_FEW 16 /* + i: kernels for few rows (i = 0, 1: 16 or 128 columns to a workgroup), B streamed into registers; + 2: with fp32 sums throughout */

/* scores of acc950_route; how several experts of a group make the group's score */
#define ACC950_SCORE_SOFTMAX 0
#define ACC950_SCORE_SIGMOID 1
#define ACC950_GROUP_BEST 0
#define ACC950_GROUP_BEST_TWO 1 /* the sum of the two best */

/*
 * Routing: p = softmax or sigmoid of a token's logits (F32 / F16 / BF16, tokens x experts), choice = p + bias (bias: fp32 per
 * expert, or NULL).  Of `groups` equal groups of neighbouring experts the top_groups with the best scores stay open; the top_k best
 * choices of their experts are taken, best first, ties to the lowest number.  weights = route_scale * p, with `renormalise` of
 * p / (sum of the p taken), also where these are too small for fp32.  ids (int32) and weights (fp32) are tokens x top_k, contiguous.
 * An expert whose logit or bias is -infinity is never taken; where too few are left, the last ids are -1 and their weights 0.
 * NaN ranks above everything (and its weight is NaN).  Up to 1024 experts, top_k up to 64.
 * acc950_route_backward: gradient of the logits (their type, contiguous rows grad_row_stride apart) from the gradient of the
 * weights; the choice itself has none, and neither has the bias.
 */
typedef struct acc950_route_call {
    int64_t in_type, tokens, experts, top_k;
    const void* logits;
    int64_t l_row_stride;
    const void* bias;
    int64_t score, groups, top_groups, group_score, renormalise;
    double route_scale;
    void* ids;
    void* weights;
    void* stream;
} acc950_route_call;
int acc950_route(const acc950_route_call* call);

typedef struct acc950_route_backward_call {
    int64_t in_type, tokens, experts, top_k;
    const void* logits;
    int64_t l_row_stride;
    const void* ids;
    const void* dweights;
    int64_t score, renormalise;
    double route_scale;
    void* dlogits;
    int64_t grad_row_stride;
    void* stream;
} acc950_route_backward_call;
int acc950_route_backward(const acc950_route_backward_call* call);

/*
 * Order of the tokens * top_k (token, slot) pairs by expert, those of one expert in their own order, pairs without an expert
 * (-1, or any number outside 0 .. experts - 1) last: order[r] = pair of sorted row r, position[pair] = its row (-1: none), offsets[e] = first row of
 * expert e (experts + 1 of them; the last is the number of rows).  All int32.  `workspace` holds acc950_expert_plan_workspace bytes,
 * which acc950_expert_plan takes on trust and acc950_expert_plan_within checks.
 */
typedef struct acc950_expert_plan_call {
    const void* ids;
    int64_t tokens, top_k, experts;
    void* order;
    void* position;
    void* offsets;
    void* workspace;
    void* stream;
} acc950_expert_plan_call;
int acc950_expert_plan(const acc950_expert_plan_call* call);
int acc950_expert_plan_within(const acc950_expert_plan_call* call, int64_t workspace_bytes);
int64_t acc950_expert_plan_workspace(int64_t tokens, int64_t top_k, int64_t experts);

/*
 * C[r, j] = (product as acc950_f8_gemm, its sums too; group_cols 128) of A's row for sorted row r and the matrix of r's expert.  `rows` is the
 * number of (token, slot) pairs; `order` and `offsets` are a plan's.  A's row is order[r] / top_k with gather = 1 (A by token) and
 * r with gather = 0.  B[e] starts at e * b_expert_stride, its scales at e * bs_expert_stride.  row_weights: NULL, or one
 * fp32 factor per pair (by pair, not by sorted row), applied before C is rounded.  Rows of C behind offsets[experts] are not written.
 */
typedef struct acc950_f8_expert_gemm_call {
    int64_t out_type, rows, N, K, experts, top_k, gather;
    const void* order;
    const void* offsets;
    const void* A;
    int64_t a_row_stride;
    const void* a_scale;
    int64_t as_row_stride, as_block_stride;
    const void* B;
    int64_t b_expert_stride, b_col_stride;
    const void* b_scale;
    int64_t bs_expert_stride, bs_block_stride, bs_col_stride;
    const void* row_weights;
    void* C;
    int64_t c_row_stride;
    int64_t variant;
    void* stream;
} acc950_f8_expert_gemm_call;
int acc950_f8_expert_gemm(const acc950_f8_expert_gemm_call* call);

/* y[t] = sum over the slots of t, in their order, of weights[t, slot] * x[position[t, slot]] (weights NULL: of 1), fp32 sums; a slot
 * without a row adds nothing.  x and y of `type` F32 / F16 / BF16, rows contiguous. */
typedef struct acc950_expert_combine_call {
    int64_t type, tokens, top_k, cols;
    const void* x;
    int64_t x_row_stride;
    const void* position;
    const void* weights;
    void* y;
    int64_t y_row_stride;
    void* stream;
} acc950_expert_combine_call;
int acc950_expert_combine(const acc950_expert_combine_call* call);

/*
 * A routed feed-forward layer: y[t] = sum over slots of weights[t, slot] * W2[e] * q(silu(W1[e] q(x[t])) * (W3[e] q(x[t]))), where q quantises rows
 * with power-of-two scales and e = ids[t, slot].  x and y: tokens x hidden of `type` F16 / BF16.  w13: (experts, 2, inner, hidden) e4m3 -- gate
 * and up --, scales (experts, 2, ceil(inner / 128), ceil(hidden / 128)); w2: (experts, hidden, inner), scales
 * (experts, ceil(hidden / 128), ceil(inner / 128)); all contiguous, w13 and w2 from 16-byte boundaries on.
 * Numerics: up to 16 rows for each expert (tokens * top_k <= 16 * experts) all sums are fp32 and rounded once, to `type`.  With more, the sums of the down product, and for BF16 those of
 * the gate and up product, are the e4m3 instruction's (see acc950_f8_gemm: about 1 in 5000 of the inner codes is its neighbour then); and for BF16 a token's rows, the terms of its
 * weighted sum, are kept in 16 bits: fp16 with a power of two for each 32 or 64 columns, 2^-12 of a value beside the result's 2^-9.  The weighted sum itself is fp32.
 * `workspace` holds acc950_f8_expert_ffn_workspace bytes, 256-byte aligned;
 * acc950_f8_expert_ffn takes that on trust, acc950_f8_expert_ffn_within checks it.  It needs no clearing and may be used again by calls that follow each other on
 * a stream, but not by two that may run at the same time: steps' results and the counters that hand out tiles lie there.
 */
typedef struct acc950_f8_expert_ffn_call {
    int64_t type, tokens, hidden, inner, experts, top_k;
    const void* x;
    int64_t x_row_stride;
    const void* ids;
    const void* weights;
    const void* w13;
    const void* w13_scale;
    const void* w2;
    const void* w2_scale;
    void* y;
    int64_t y_row_stride;
    void* workspace;
    void* stream;
} acc950_f8_expert_ffn_call;
int acc950_f8_expert_ffn(const acc950_f8_expert_ffn_call* call);
int acc950_f8_expert_ffn_within(const acc950_f8_expert_ffn_call* call, int64_t workspace_bytes);
int64_t acc950_f8_expert_ffn_workspace(int64_t tokens, int64_t hidden, int64_t inner, int64_t experts, int64_t top_k);

#if defined(__cplusplus)
}
#endif
#endif /* ACCERA_MI355X_F8_H */
