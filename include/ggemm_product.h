/* C ABI of the grouped FP8 product with bias, activation and residual in its epilogue, and of the
 * gradient of bias and activation (libggemm_vark.so). Return codes, strerror and the ABI version are
 * those of ggemm_vark.h. The reference's products end at the scaled bf16 result (reference
 * bench.py:238-247); what follows them there is the framework's.
 *
 *   z[r, :]   = a_scale * b_scale * A[r, :] @ B[g]^T + bias[g, :]      for offs[g] <= r < offs[g+1]
 *   out[r, :] = act(z[r, :]) + residual[r, :]
 *
 * in fp32, rounded once to bf16. act: identity, silu z / (1 + e^-z), gelu z (1 + erf(z / sqrt 2)) / 2, or the
 * gated swiglu over pairs of columns, out[:, i] = g / (1 + e^(-slope g)) * (u + shift) with
 * g = min(z[:, 2i], limit) and u = z[:, 2i + 1] clamped to +-limit: out and residual are N / 2 wide then.
 *
 * All pointers are device pointers; sizes and strides in elements. Launches are asynchronous on `stream`;
 * no allocation, no synchronization, no state between calls.
 */
#ifndef GGEMM_PRODUCT_H
#define GGEMM_PRODUCT_H

#include <stdint.h>

#include "ggemm_vark.h"

#ifdef __cplusplus
extern "C" {
#endif

#ifndef GGEMM_IN_BF16
#define GGEMM_IN_BF16 0
#define GGEMM_IN_F32 1
#endif

#define GGEMM_ACT_NONE 0
#define GGEMM_ACT_SILU 1
#define GGEMM_ACT_GELU 2
#define GGEMM_ACT_SWIGLU 3

#define GGEMM_PRODUCT_MAX_GROUPS 2047

/* a: e4m3 [M_total, K], b: e4m3 [G, N, K], scales, group_offs and their strides as for
 * ggemm_persistent_fp8 (ggemm_persistent.h), with its requirements.
 *   out: bf16 [M_total, N or N / 2], row stride a multiple of 8, 16-byte aligned;
 *   pre: bf16 [M_total, N] or NULL: z, rounded to bf16, for the backward pass; as out;
 *   bias: [G, N] contiguous of bias_dtype (GGEMM_IN_*) or NULL, 16-byte aligned;
 *   residual: bf16, as wide as out, or NULL; row stride a multiple of 8, 16-byte aligned. It may be out.
 *   slope, limit, shift: of swiglu (others ignore them); limit > 0, INFINITY for none.
 * Rows of out and pre outside [0, offs[G]) are not written, or rows from offs[G] on become zero with
 * zero_tail != 0. */
int ggemm_product_fp8_bias_act(const void* a, const void* b, void* out, void* pre, const float* a_scale,
                               const float* b_scale, const void* bias, int32_t bias_dtype, const void* residual,
                               const int64_t* group_offs, int32_t G, int32_t N, int32_t K, int32_t stride_am,
                               int32_t stride_bg, int32_t stride_bn, int32_t stride_out, int32_t stride_pre,
                               int32_t stride_res, int32_t act, float slope, float limit, float shift,
                               int64_t M_total, int32_t zero_tail, void* stream);

/* Rows of the output tiles of the kernel that such a call runs on a device of num_cus CUs: 16 (few rows), 64 or 128
 * (mid tiles), 192 (the 512-thread kernel) or 256 (wide tiles). stride_pre 0: no pre; residual: whether there is one.
 * Each kernel sums a row's products in an order of its own, so a row's last bit can depend on G and M_total. */
int32_t ggemm_product_tile_rows(int32_t G, int32_t N, int32_t K, int32_t stride_am, int32_t stride_bn,
                                int32_t stride_out, int32_t stride_pre, int32_t act, int32_t residual, int64_t M_total,
                                int32_t num_cus);

/* dpre[r, :] = dout[r, :] * act'(pre[r, :]) (bf16, from fp32) and dbias[g, :] = sum over the group's rows of it, before
 * its rounding (fp32 [G, N] contiguous, or NULL). dout: bf16 [M_total, N or N / 2]; pre, dpre: bf16 [M_total, N]; rows of
 * dpre outside the groups become zero. act NONE: dpre may be NULL (it is dout). N a multiple of 16, row strides of 8,
 * addresses 16-byte aligned. With dbias, workspace: ggemm_product_act_workspace(...) floats, 16-byte aligned; sums are
 * made in an order that depends on the sizes and group_offs alone. Where swiglu clamps, the gradient is zero. */
int ggemm_product_act_backward(const void* dout, const void* pre, const int64_t* group_offs, int32_t G, int32_t N,
                               int32_t stride_dout, int32_t stride_pre, int32_t act, float slope, float limit,
                               float shift, int64_t M_total, void* dpre, int32_t stride_dpre, float* dbias,
                               float* workspace, void* stream);
int64_t ggemm_product_act_workspace(int64_t M_total, int32_t G, int32_t N);

#ifdef __cplusplus
}
#endif
#endif /* GGEMM_PRODUCT_H */
