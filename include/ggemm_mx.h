/* C ABI of microscaled (MX) rows: their quantization and restoration, the grouped product of 4-bit weights,
 * and the value before an activation kept in 8 bits between a product and its gradient (libggemm_vark.so).
 * Return codes, strerror and the ABI version are those of ggemm_vark.h; GGEMM_IN_*, GGEMM_ACT_* and the activations
 * those of ggemm_product.h. The reference has no microscaled form: its products take per-tensor scales (reference
 * bench.py:238-247).
 *
 * A row of `cols` values, a multiple of 16, is blocks of 32 (the last one may be 16 long). A block's values share a
 * power of two 2^X, held as the byte X + 127 (e8m0; 255 is NaN):
 *   e2m1   4 bits a value, two to a byte, the even column in the low half: 0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives
 *   e4m3   8 bits a value
 *
 * All pointers are device pointers. Strides of quantized values and of scales are in bytes, others in elements.
 * Launches are asynchronous on `stream`; no allocation, no synchronization, no state between calls.
 */
#ifndef GGEMM_MX_H
#define GGEMM_MX_H

#include <stdint.h>

#include "ggemm_product.h"

#ifdef __cplusplus
extern "C" {
#endif

#define GGEMM_MX_E4M3 0
#define GGEMM_MX_E2M1 1

/* q = values of fmt nearest to x 2^-X, ties to the even code, and X + 127 for every block. X is the smallest exponent,
 * -127 at least, at which the block's largest value, rounded as though the format went on past its own largest (6 or
 * 448), stays within it: amax = m 2^e gives e - 2, one more from m = 1.75 on (e2m1), or e - 8, one more from m = 1.8125
 * on (e4m3). A block of zeros has X = 0; one that holds an infinity or NaN the byte 255 and values 0.
 *   x: [rows, cols] of dtype (GGEMM_IN_*), rows `stride` apart, a multiple of 8 (bf16) or 4, 16-byte aligned;
 *   q: rows q_stride bytes apart, a multiple of 8 (e4m3) or 4, aligned so; scales: [rows, ceil(cols / 32)], rows
 *   scale_stride apart. */
int ggemm_mx_quantize(const void* x, int32_t dtype, int64_t rows, int32_t cols, int64_t stride, int32_t fmt, void* q,
                      int64_t q_stride, uint8_t* scales, int64_t scale_stride, void* stream);

/* out = q 2^X, in dtype: exact, but for what the type does not hold (bf16 below 2^-133, 2^128 and more). Scales of
 * row r and block b at scales[r * scale_row + b * scale_block]; out as x above. */
int ggemm_mx_dequantize(const void* q, int32_t fmt, int64_t rows, int32_t cols, int64_t q_stride, const uint8_t* scales,
                        int64_t scale_row, int64_t scale_block, void* out, int32_t dtype, int64_t out_stride,
                        void* stream);

/* z[r, :] = A[r, :] @ B[g]^T + bias[g, :] for offs[g] <= r < offs[g + 1], out[r, :] = act(z[r, :]) + residual[r, :], as
 * ggemm_product_fp8_bias_act, on blocks: A is a_fmt [M_total, K], B e2m1 [G, N, K], K a multiple of 32, N of 16.
 * Rows of A, B and of both scales start on multiples of 16 bytes, and a row of scales is ceil(K / 512) * 16 bytes that
 * may be read (those past K / 32 are not used). Offsets count as the largest one so far, within [0, M_total]: groups
 * never overlap. Rows of no group are not written, or rows from offs[G] on become zero with zero_tail != 0.
 * tile: rows of the output tiles, 16, 32, 64, 128 or 256, or 0 for the library's choice. Each kernel sums a row's products in
 * an order of its own, so a row's last bit can depend on G and M_total. */
int ggemm_mx_product(const void* a, int32_t a_fmt, const uint8_t* a_scales, const void* b, const uint8_t* b_scales,
                     void* out, const void* bias, int32_t bias_dtype, const void* residual, const int64_t* group_offs,
                     int32_t G, int32_t N, int32_t K, int64_t stride_a, int64_t stride_as, int64_t stride_bg,
                     int64_t stride_bn, int64_t stride_bsg, int64_t stride_bsn, int32_t stride_out, int32_t stride_res,
                     int32_t act, float slope, float limit, float shift, int64_t M_total, int32_t zero_tail,
                     int32_t tile, void* stream);

/* The tile that such a call takes by itself on a device of num_cus CUs. */
int32_t ggemm_mx_tile_rows(int32_t a_fmt, int32_t G, int32_t N, int32_t K, int64_t M_total, int32_t num_cus);

/* ggemm_product_fp8_bias_act (ggemm_product.h) with z kept in 8 bits for the backward pass instead of bf16: quantized from
 * fp32 as by ggemm_mx_quantize. Without an activation (GGEMM_E_FORMAT) z is the result and nothing is kept.
 *   q: e4m3 [M_total, N], rows stride_q bytes apart, a multiple of 16, 16-byte aligned;
 *   scales: of row r and block b at scales[b * scale_block + r], scale_block >= M_total.
 * Rows outside [0, offs[G]) are not written, or rows from offs[G] on become zero (scale 127) with zero_tail != 0. */
int ggemm_mx_keep_product(const void* a, const void* b, void* out, void* q, uint8_t* scales, const float* a_scale,
                          const float* b_scale, const void* bias, int32_t bias_dtype, const void* residual,
                          const int64_t* group_offs, int32_t G, int32_t N, int32_t K, int32_t stride_am, int32_t stride_bg,
                          int32_t stride_bn, int32_t stride_out, int32_t stride_q, int64_t scale_block, int32_t stride_res,
                          int32_t act, float slope, float limit, float shift, int64_t M_total, int32_t zero_tail,
                          void* stream);

/* Rows of the output tiles of the kernel that such a call runs, as ggemm_product_tile_rows. */
int32_t ggemm_mx_keep_tile_rows(int32_t G, int32_t N, int32_t K, int32_t stride_am, int32_t stride_bn, int32_t stride_out,
                                int32_t stride_q, int32_t act, int32_t residual, int64_t M_total, int32_t num_cus);

/* ggemm_product_act_backward (ggemm_product.h) from such a z: q and scales as above, or of any strides (scale of row r and
 * block b at scales[r * scale_row + b * scale_block]); stride_q a multiple of 8, q 8-byte aligned. The gradient is
 * that of the values that were kept; a block with scale 255 gives NaN. With dbias, workspace:
 * ggemm_mx_act_workspace(...) floats, 16-byte aligned. */
int ggemm_mx_act_backward(const void* dout, const void* q, const uint8_t* scales, const int64_t* group_offs, int32_t G,
                          int32_t N, int32_t stride_dout, int32_t stride_q, int64_t scale_row, int64_t scale_block,
                          int32_t act, float slope, float limit, float shift, int64_t M_total, void* dpre,
                          int32_t stride_dpre, float* dbias, float* workspace, void* stream);

/* Floats of workspace that ggemm_mx_act_backward needs, whatever group_offs holds. */
int64_t ggemm_mx_act_workspace(int64_t M_total, int32_t G, int32_t N);

#ifdef __cplusplus
}
#endif
#endif /* GGEMM_MX_H */
