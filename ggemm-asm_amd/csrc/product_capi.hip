// extern "C" launchers of the grouped FP8 product with an epilogue and of the gradient of bias and
// activation (include/ggemm_product.h), part of libggemm_vark.so. Arguments are validated on the host;
// nothing is launched on a validation error.
#include "product_launch.h"

static_assert(GGEMM_PRODUCT_MAX_GROUPS == ggemm::nt::kMaxGroups && GGEMM_PRODUCT_MAX_GROUPS == ggemm::ag::kMaxGroups &&
                  GGEMM_ACT_SILU == ggemm::epi::kSilu && GGEMM_ACT_GELU == ggemm::epi::kGelu &&
                  GGEMM_ACT_SWIGLU == ggemm::epi::kSwiglu,
              "header and kernels agree");

extern "C" {

int ggemm_product_fp8_bias_act(const void* a, const void* b, void* out, void* pre, const float* a_scale,
                               const float* b_scale, const void* bias, int32_t bias_dtype, const void* residual,
                               const int64_t* group_offs, int32_t G, int32_t N, int32_t K, int32_t stride_am,
                               int32_t stride_bg, int32_t stride_bn, int32_t stride_out, int32_t stride_pre,
                               int32_t stride_res, int32_t act, float slope, float limit, float shift,
                               int64_t M_total, int32_t zero_tail, void* stream) {
  int cus = 0;
  const nt::Args x{(const uint8_t*)a, (const uint8_t*)b, (uint16_t*)out, a_scale, b_scale, group_offs, G, N, K,
             stride_am, stride_bg, stride_bn, stride_out, 1, M_total, zero_tail};
  const epi::Args e{(uint16_t*)pre, stride_pre, bias, bias_dtype == GGEMM_IN_F32, (const uint16_t*)residual,
                    stride_res, slope, limit, shift, slope * -epi::kLog2e};
  int rc = validate(x, e, act, bias_dtype);
  if (rc) return rc;
  rc = device_cus(&cus);
  if (rc) return rc;
  if (M_total == 0) return GGEMM_OK;
  return launch_product<0>(x, e, act, cus, (hipStream_t)stream);
}

int32_t ggemm_product_tile_rows(int32_t G, int32_t N, int32_t K, int32_t stride_am, int32_t stride_bn,
                                int32_t stride_out, int32_t stride_pre, int32_t act, int32_t residual, int64_t M_total,
                                int32_t num_cus) {
  nt::Args x{};
  x.G = G, x.N = N, x.K = K, x.stride_am = stride_am, x.stride_bn = stride_bn, x.stride_cm = stride_out;
  x.m_total = M_total;
  epi::Args e{};
  uint16_t there = 0;                                  // stands for a tensor: never read
  e.pre = stride_pre ? &there : nullptr, e.stride_pre = stride_pre, e.residual = residual ? &there : nullptr;
  const int rows[] = {16, 16, 64, 128, ggemm::kTileM, ggemm::pw::kTM};
  return rows[(int)choose(x, e, act, num_cus).kernel];
}

int64_t ggemm_product_act_workspace(int64_t M_total, int32_t G, int32_t N) {
  if (M_total < 0 || M_total > nt::kMaxRow || G <= 0 || G > ag::kMaxGroups || N <= 0) return 0;
  return units_of(M_total, G, N, false) * N;
}

int ggemm_product_act_backward(const void* dout, const void* pre, const int64_t* group_offs, int32_t G, int32_t N,
                               int32_t stride_dout, int32_t stride_pre, int32_t act, float slope, float limit,
                               float shift, int64_t M_total, void* dpre, int32_t stride_dpre, float* dbias,
                               float* workspace, void* stream) {
  int rc = act_code(act, limit);
  if (rc) return rc;
  if (!dout || !group_offs || (act != GGEMM_ACT_NONE && (!pre || !dpre)) || (dbias && !workspace)) return GGEMM_E_NULL;
  if (G <= 0 || G > ag::kMaxGroups || N <= 0 || N % 16 || M_total < 0 || M_total > nt::kMaxRow) return GGEMM_E_SHAPE;
  const int width = act == GGEMM_ACT_SWIGLU ? N / 2 : N;
  if (stride_dout < width || stride_dout % 8 || (pre && (stride_pre < N || stride_pre % 8)) ||
      (dpre && (stride_dpre < N || stride_dpre % 8)))
    return GGEMM_E_STRIDE;
  if (!aligned(dout, 16) || !aligned(pre, 16) || !aligned(dpre, 16) || !aligned(dbias, 16) || !aligned(workspace, 16))
    return GGEMM_E_ALIGN;
  int cus = 0;
  rc = device_cus(&cus);
  if (rc) return rc;
  const ag::Args a{(const uint16_t*)dout, (const uint16_t*)pre, group_offs, G, N, stride_dout, stride_pre,
                   epi::Args{nullptr, 0, nullptr, 0, nullptr, 0, slope, limit, shift, slope * -epi::kLog2e}, M_total, 0, 0, 0, 0,
                   (uint16_t*)dpre, stride_dpre, dbias, workspace};
  return launch_act_backward<false>(a, act, (hipStream_t)stream);
}

}  // extern "C"
