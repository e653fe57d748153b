/* C ABI of what an MoE layer does around its grouped products (libggemm_vark.so): routing tokens to
 * experts, ordering the choices by expert, copying the tokens' rows into that order and summing the
 * experts' rows back per token, with the backward passes. Return codes, strerror and the ABI version
 * are those of ggemm_vark.h. There is no counterpart inside the reference tree, whose harness makes
 * its group offsets on the host (reference bench.py:196-209).
 *
 * All pointers are device pointers; sizes and strides in elements unless they say bytes. Launches are
 * asynchronous on `stream`; no allocation, no synchronization, no state between calls; results do not
 * depend on the order in which the hardware runs anything.
 *
 * T tokens take top_k experts each. A choice is token * top_k + j. `slots[choice]` is the row of that
 * choice in expert order, or -1: rows of expert g are group_offs[g] .. group_offs[g + 1] - 1, in the
 * order of their tokens; choices whose expert is not in [0, G) have no row.
 */
#ifndef GGEMM_MOE_H
#define GGEMM_MOE_H

#include <stdint.h>

#include "ggemm_vark.h"

#ifdef __cplusplus
extern "C" {
#endif

/* element types (the codes of ggemm_quant.h) */
#ifndef GGEMM_IN_BF16
#define GGEMM_IN_BF16 0
#define GGEMM_IN_F32 1
#endif

#define GGEMM_MOE_SOFTMAX 0
#define GGEMM_MOE_SIGMOID 1

#define GGEMM_MOE_MAX_EXPERTS 1024   /* of a router */
#define GGEMM_MOE_MAX_TOP_K 64
#define GGEMM_MOE_MAX_GROUPS 2047    /* of a plan, as the grouped products take */
#define GGEMM_MOE_PLAN_ALONE 2048    /* choices that one workgroup orders by itself */

/* The top_k experts of each token and their weights, from router logits [T, E] (bf16 or fp32, row
 * stride `stride` >= E).
 *   score p = softmax over the E logits, or sigmoid of each; in fp32.
 *   key: p + bias[e] where a bias (fp32 [E], may be NULL) is given, p where there are groups, else the
 *     logit itself (the same order, without the scores' rounding).
 *   num_groups > 1: the experts are num_groups groups of consecutive E / num_groups; a group's value is
 *     the sum of its group_best (1 or 2) largest keys, and only experts of the top_groups groups of the
 *     largest values are taken.
 *   experts [T, top_k] int32: the experts with the largest keys, the largest first, equal keys by the
 *     lower index; NaN is larger than any number. An expert whose logit or key is -inf is never taken:
 *     where fewer than top_k are left, the last experts are -1 with weight 0.
 *   weights [T, top_k] fp32: scale * p, or with renormalize scale * p / sum of the token's taken p
 *     (softmax: softmax over the taken logits; sigmoid: the sum at least 1e-20). */
int ggemm_moe_route(const void* logits, int32_t dtype, int64_t T, int32_t E, int64_t stride, int32_t top_k,
                    int32_t score, const float* bias, int32_t num_groups, int32_t top_groups, int32_t group_best,
                    int32_t renormalize, float scale, float* weights, int32_t* experts, void* stream);

/* Gradient of the weights by the logits: dlogits [T, E] contiguous, of the logits' type, every element
 * written. experts as ggemm_moe_route gave them (entries outside [0, E) are skipped); the choice itself
 * and its bias have no gradient. */
int ggemm_moe_route_backward(const float* dweights, const void* logits, int32_t dtype, int64_t T, int32_t E,
                             int64_t stride, int32_t top_k, int32_t score, int32_t renormalize, float scale,
                             const int32_t* experts, void* dlogits, void* stream);

/* group_offs [G + 1] int64 and slots [n] int32 of n choices' experts (int32). workspace:
 * ggemm_moe_plan_workspace(n, G) 32-bit words; none (it may be NULL) up to GGEMM_MOE_PLAN_ALONE choices. n < 2^31 - 256. */
int ggemm_moe_plan(const int32_t* experts, int64_t n, int32_t G, int64_t* group_offs, int32_t* slots,
                   int32_t* workspace, void* stream);
int64_t ggemm_moe_plan_workspace(int64_t n, int32_t G);

/* rows[slots[c]] = x[c / top_k] for every choice c with 0 <= slots[c] < M; rows [group_offs[G], M) become
 * zero. Rows of row_bytes bytes whatever their type, strides in bytes. */
int ggemm_moe_dispatch(const void* x, int64_t row_bytes, int64_t x_stride, int64_t T, int32_t top_k,
                       const int32_t* slots, const int64_t* group_offs, int32_t G, void* rows, int64_t rows_stride,
                       int64_t M, void* stream);

/* out[t] = residual[t] + sum over j of weights[t, j] * y[slots[t, j]], j in order, in fp32, rounded once.
 * Choices with a slot outside [0, M) have no term. weights fp32 [T, top_k] or NULL (ones); residual NULL for
 * none; y [M, H], residual and out [T, H] of `dtype`, H up to 2^28. */
int ggemm_moe_combine(const void* y, int32_t dtype, int64_t y_stride, int64_t M, const int32_t* slots, int64_t T,
                      int32_t top_k, const float* weights, const void* residual, int64_t residual_stride, int32_t H,
                      void* out, int64_t out_stride, void* stream);

/* Its gradients: dy[slots[c]] = weights[c] * dout[c / top_k] (ones without weights), rows
 * [group_offs[G], M) zero; dweights[c] = dot of dout[c / top_k] and y[slots[c]] in fp32, 0 without a row. Either of
 * dy and dweights may be NULL; y is read for dweights only. */
int ggemm_moe_combine_backward(const void* dout, int32_t dtype, int64_t dout_stride, const void* y, int64_t y_stride,
                               int64_t M, const int32_t* slots, int64_t T, int32_t top_k, const float* weights,
                               const int64_t* group_offs, int32_t G, int32_t H, void* dy, int64_t dy_stride,
                               float* dweights, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* GGEMM_MOE_H */
