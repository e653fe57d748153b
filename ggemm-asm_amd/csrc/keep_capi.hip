// extern "C" launchers of the value before an activation kept in 8 bits: the product that writes it and the gradient that
// reads it (include/ggemm_mx.h), part of libggemm_vark.so. Arguments are validated on the host; nothing is launched on a
// validation error.
#include "../../include/ggemm_mx.h"
#include "product_launch.h"

extern "C" {

int ggemm_mx_keep_product(const void* a, const void* b, void* out, void* q, uint8_t* scales, const float* a_scale,
                          const float* b_scale, const void* bias, int32_t bias_dtype, const void* residual,
                          const int64_t* group_offs, int32_t G, int32_t N, int32_t K, int32_t stride_am, int32_t stride_bg,
                          int32_t stride_bn, int32_t stride_out, int32_t stride_q, int64_t scale_block, int32_t stride_res,
                          int32_t act, float slope, float limit, float shift, int64_t M_total, int32_t zero_tail,
                          void* stream) {
  const nt::Args x{(const uint8_t*)a, (const uint8_t*)b, (uint16_t*)out, a_scale, b_scale, group_offs, G, N, K,
                   stride_am, stride_bg, stride_bn, stride_out, 1, M_total, zero_tail};
  const epi::Args e{nullptr, 0, bias, bias_dtype == GGEMM_IN_F32, (const uint16_t*)residual, stride_res, slope, limit,
                    shift, slope * -epi::kLog2e, (uint8_t*)q, stride_q, scales, scale_block};
  if (!q || !scales) return GGEMM_E_NULL;
  if (act == GGEMM_ACT_NONE) return GGEMM_E_FORMAT;
  int rc = validate(x, e, act, bias_dtype);
  if (rc) return rc;
  if (stride_q < N || stride_q % 16 || scale_block < M_total) return GGEMM_E_STRIDE;
  if (!aligned(q, 16)) return GGEMM_E_ALIGN;
  if (scale_block > INT32_MAX || (int64_t)stride_q * ggemm::kTileM >= nt::kOob) return GGEMM_E_SHAPE;
  int cus = 0;
  rc = device_cus(&cus);
  if (rc) return rc;
  if (M_total == 0) return GGEMM_OK;
  return launch_product<epi::kKeepMx>(x, e, act, cus, (hipStream_t)stream);
}

int32_t ggemm_mx_keep_tile_rows(int32_t G, int32_t N, int32_t K, int32_t stride_am, int32_t stride_bn, int32_t stride_out,
                                int32_t stride_q, int32_t act, int32_t residual, int64_t M_total, int32_t num_cus) {
  nt::Args x{};
  x.G = G, x.N = N, x.K = K, x.stride_am = stride_am, x.stride_bn = stride_bn, x.stride_cm = stride_out;
  x.m_total = M_total;
  epi::Args e{};
  uint16_t there = 0;                                  // stands for a tensor: never read
  e.q8 = (uint8_t*)&there, e.stride_q = stride_q, e.residual = residual ? &there : nullptr;
  const int rows[] = {16, 16, 64, 128, ggemm::kTileM, ggemm::pw::kTM};
  return rows[(int)choose(x, e, act, num_cus).kernel];
}

int64_t ggemm_mx_act_workspace(int64_t M_total, int32_t G, int32_t N) {
  if (M_total < 0 || M_total > nt::kMaxRow || G <= 0 || G > ag::kMaxGroups || N <= 0) return 0;
  return units_of(M_total, G, N, true) * N;
}

int ggemm_mx_act_backward(const void* dout, const void* q, const uint8_t* scales, const int64_t* group_offs, int32_t G,
                          int32_t N, int32_t stride_dout, int32_t stride_q, int64_t scale_row, int64_t scale_block,
                          int32_t act, float slope, float limit, float shift, int64_t M_total, void* dpre,
                          int32_t stride_dpre, float* dbias, float* workspace, void* stream) {
  if (act == GGEMM_ACT_NONE) return GGEMM_E_FORMAT;
  int rc = act_code(act, limit);
  if (rc) return rc;
  if (!dout || !q || !scales || !group_offs || !dpre || (dbias && !workspace)) return GGEMM_E_NULL;
  if (G <= 0 || G > ag::kMaxGroups || N <= 0 || N % 16 || M_total < 0 || M_total > nt::kMaxRow) return GGEMM_E_SHAPE;
  const int width = act == GGEMM_ACT_SWIGLU ? N / 2 : N;
  if (stride_dout < width || stride_dout % 8 || stride_q < N || stride_q % 8 || stride_dpre < N || stride_dpre % 8 ||
      scale_row < 0 || scale_block < 0)
    return GGEMM_E_STRIDE;
  if (!aligned(dout, 16) || !aligned(q, 8) || !aligned(dpre, 16) || !aligned(dbias, 16) || !aligned(workspace, 16))
    return GGEMM_E_ALIGN;
  int cus = 0;
  rc = device_cus(&cus);
  if (rc) return rc;
  const ag::Args a{(const uint16_t*)dout, nullptr, group_offs, G, N, stride_dout, stride_q,
                   epi::Args{nullptr, 0, nullptr, 0, nullptr, 0, slope, limit, shift, slope * -epi::kLog2e}, M_total, 0, 0, 0, 0,
                   (uint16_t*)dpre, stride_dpre, dbias, workspace, (const uint8_t*)q, scales, scale_row, scale_block};
  return launch_act_backward<true>(a, act, (hipStream_t)stream);
}

}  // extern "C"
