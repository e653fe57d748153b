// extern "C" launchers of the grouped FP8 product with an epilogue and of the gradient of bias and
// activation (include/ggemm_product.h), part of libggemm_vark.so. Arguments are validated on the host;
// nothing is launched on a validation error.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "../../include/ggemm_product.h"
#include "act_kernel.h"
#include "capi_common.h"
#include "mid_choice.h"

static_assert(GGEMM_PRODUCT_MAX_GROUPS == ggemm::nt::kMaxGroups && GGEMM_PRODUCT_MAX_GROUPS == ggemm::ag::kMaxGroups &&
                  GGEMM_ACT_SILU == ggemm::epi::kSilu && GGEMM_ACT_GELU == ggemm::epi::kGelu &&
                  GGEMM_ACT_SWIGLU == ggemm::epi::kSwiglu,
              "header and kernels agree");

namespace {

using ggemm::host::aligned;
using ggemm::host::device_cus;
using ggemm::host::mid_preferred;
using ggemm::host::mid_tiles;
namespace nt = ggemm::nt;
namespace epi = ggemm::epi;
namespace ag = ggemm::ag;

// What follows the last group's rows becomes zero in out and pre.
template <int kAct>
__device__ __forceinline__ void clear_tails(const nt::Args& a, const epi::Args& e) {
  if (!a.zero_tail) return;
  nt::clear_tail_rows(a.c, a.stride_cm, kAct == epi::kSwiglu ? a.N / 2 : a.N, a.group_offs, a.G, a.m_total);
  if (e.pre != nullptr) nt::clear_tail_rows(e.pre, e.stride_pre, a.N, a.group_offs, a.G, a.m_total);
}

template <int kAct, int kBM>
__global__ __launch_bounds__(ggemm::mid::kNT, 2) void product_mid_kernel(nt::Args a, epi::Args e) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[ggemm::mid::GemmCfg<kBM>::LdsBytes];
  ggemm::mid::gemm_body<false, kBM, 1 + kAct>(nt::without_tail(a), (GG_LDS uint8_t*)lds, e);
  clear_tails<kAct>(a, e);
}

template <int kAct>
__global__ __launch_bounds__(ggemm::kThreads) void product_512_kernel(nt::Args a, epi::Args e) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t ggemm_product_lds[];
  nt::persistent_entry<false, 1 + kAct>(nt::without_tail(a), (GG_LDS uint8_t*)ggemm_product_lds, e);
  clear_tails<kAct>(a, e);
}

// The wide tiles, one workgroup to a CU (persistent_wide.h): bias alone, or swiglu with or without z kept.
template <int kMode>
__global__ __launch_bounds__(ggemm::pw::kNT) __attribute__((amdgpu_waves_per_eu(1, 1)))
void product_wide_kernel(nt::Args a, epi::Args e) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[ggemm::pw::kLdsBytes];
  ggemm::persistent_wide_body<false, kMode>(nt::without_tail(a), (GG_LDS uint8_t*)lds, e);
  clear_tails<kMode == ggemm::pw::kBias ? epi::kNone : epi::kSwiglu>(a, e);
}

// f(activation) with the code as a constant.
template <typename F>
int with_act(int act, F f) {
  using std::integral_constant;
  switch (act) {
    case GGEMM_ACT_SILU: return f(integral_constant<int, epi::kSilu>{});
    case GGEMM_ACT_GELU: return f(integral_constant<int, epi::kGelu>{});
    case GGEMM_ACT_SWIGLU: return f(integral_constant<int, epi::kSwiglu>{});
    default: return f(integral_constant<int, epi::kNone>{});
  }
}

int act_code(int act, float limit) {
  if (act < GGEMM_ACT_NONE || act > GGEMM_ACT_SWIGLU) return GGEMM_E_FORMAT;
  return act == GGEMM_ACT_SWIGLU && !(limit > 0.f) ? GGEMM_E_SHAPE : GGEMM_OK;
}

int validate(const nt::Args& a, const epi::Args& e, int act, int bias_dtype) {
  if (!a.a || !a.b || !a.c || !a.a_scale || !a.b_scale || !a.group_offs) return GGEMM_E_NULL;
  if (e.bias && bias_dtype != GGEMM_IN_BF16 && bias_dtype != GGEMM_IN_F32) return GGEMM_E_FORMAT;
  const int rc = act_code(act, e.limit);
  if (rc) return rc;
  if (a.G <= 0 || a.G > nt::kMaxGroups || a.N <= 0 || a.K <= 0 || a.N % 16 || a.K % 16) return GGEMM_E_SHAPE;
  if (a.m_total < 0 || a.m_total > nt::kMaxRow) return GGEMM_E_SHAPE;
  if ((a.m_total / ggemm::kTileM + a.G) * (int64_t)((a.N + 319) / 320) > nt::kMaxTiles) return GGEMM_E_SHAPE;
  const int out = act == GGEMM_ACT_SWIGLU ? a.N / 2 : a.N;
  if (a.stride_am < a.K || a.stride_bn < a.K || a.stride_am % 16 || a.stride_bn % 16 || a.stride_bg % 16)
    return GGEMM_E_STRIDE;
  if ((int64_t)a.stride_bg < (int64_t)(a.N - 1) * a.stride_bn + a.K) return GGEMM_E_STRIDE;
  if (a.stride_cm < out || a.stride_cm % 8) return GGEMM_E_STRIDE;
  if (e.pre && (e.stride_pre < a.N || e.stride_pre % 8)) return GGEMM_E_STRIDE;
  if (e.residual && (e.stride_res < out || e.stride_res % 8)) return GGEMM_E_STRIDE;
  // 32-bit buffer offsets of a stage: 192 A rows, up to 384 B rows
  if ((int64_t)a.stride_am * ggemm::kTileM >= nt::kOob || (int64_t)a.stride_bn * 384 >= nt::kOob) return GGEMM_E_SHAPE;
  if (!aligned(a.a, 16) || !aligned(a.b, 16) || !aligned(a.c, 16) || !aligned(e.pre, 16) || !aligned(e.bias, 16) ||
      !aligned(e.residual, 16))
    return GGEMM_E_ALIGN;
  return GGEMM_OK;
}

// The wide kernel's epilogue for this launch, 0 where it has none: shapes as for the plain product (32-bit offsets of
// a stage's rows and of a tile's rows of C and z), no residual, and of the activations none, without a z of its own,
// or swiglu.
int wide_mode(const nt::Args& a, const epi::Args& e, int act) {
  auto rows_fit = [](int64_t stride) { return stride * 2 * ggemm::pw::kTM < nt::kOob; };
  if (!ggemm::pw::fits(a.N, a.K) || (int64_t)a.stride_am * ggemm::pw::kTM >= nt::kOob ||
      (int64_t)a.stride_bn * ggemm::pw::kTN >= nt::kOob || !rows_fit(a.stride_cm) || e.residual)
    return 0;
  if (act == GGEMM_ACT_NONE) return e.pre ? 0 : ggemm::pw::kBias;
  if (act != GGEMM_ACT_SWIGLU) return 0;
  return !e.pre ? ggemm::pw::kGate : rows_fit(e.stride_pre) ? ggemm::pw::kGateKeep : 0;
}

// Rows of a unit of the gradient: few enough that the units fill the chip, 64 at most (131072 x 5760: 256 rows 810 us, 64
// 795: more rounds of workgroups even out), but for launches of more units than a grid takes.
constexpr int64_t kMaxUnits = 1 << 22;
int strips_of(int N) { return (N / 8 + ag::kThreads - 1) / ag::kThreads; }
int unit_rows(int64_t M, int N) {
  const int strips = strips_of(N);
  int64_t rows = 64;
  while (rows > 16 && M / rows * strips < 2048) rows /= 2;
  while (M / rows * strips > kMaxUnits) rows *= 2;
  return (int)rows;
}
int64_t units_of(int64_t M, int G, int N) { return std::max<int64_t>(1, M / unit_rows(M, N) + std::min<int64_t>(G, M)); }

}  // namespace

extern "C" {

int ggemm_product_fp8_bias_act(const void* a, const void* b, void* out, void* pre, const float* a_scale,
                               const float* b_scale, const void* bias, int32_t bias_dtype, const void* residual,
                               const int64_t* group_offs, int32_t G, int32_t N, int32_t K, int32_t stride_am,
                               int32_t stride_bg, int32_t stride_bn, int32_t stride_out, int32_t stride_pre,
                               int32_t stride_res, int32_t act, float slope, float limit, float shift,
                               int64_t M_total, int32_t zero_tail, void* stream) {
  int cus = 0;
  nt::Args x{(const uint8_t*)a, (const uint8_t*)b, (uint16_t*)out, a_scale, b_scale, group_offs, G, N, K,
             stride_am, stride_bg, stride_bn, stride_out, 1, M_total, zero_tail};
  const epi::Args e{(uint16_t*)pre, stride_pre, bias, bias_dtype == GGEMM_IN_F32, (const uint16_t*)residual,
                    stride_res, slope, limit, shift};
  int rc = validate(x, e, act, bias_dtype);
  if (rc) return rc;
  rc = device_cus(&cus);
  if (rc) return rc;
  if (M_total == 0) return GGEMM_OK;
  const int wide = wide_mode(x, e, act);
  const int mid = mid_preferred(G, N, K, stride_out, M_total, wide != 0, cus);
  if (!mid && wide) {
    x.num_wg = cus;
    auto kern = wide == ggemm::pw::kBias   ? product_wide_kernel<ggemm::pw::kBias>
                : wide == ggemm::pw::kGate ? product_wide_kernel<ggemm::pw::kGate>
                                           : product_wide_kernel<ggemm::pw::kGateKeep>;
    hipLaunchKernelGGL(kern, dim3(cus), dim3(ggemm::pw::kNT), 0, (hipStream_t)stream, x, e);
    return (int)hipGetLastError();
  }
  return with_act(act, [&](auto code) {
    constexpr int kAct = decltype(code)::value;
    if (mid) {
      const int64_t tiles = mid_tiles(mid, G, N, M_total), run = ggemm::kXcds * ggemm::mid::kXcdRun;
      hipLaunchKernelGGL((mid == 64 ? product_mid_kernel<kAct, 64> : product_mid_kernel<kAct, 128>),
                         dim3((uint32_t)((tiles + run - 1) / run * run)), dim3(ggemm::mid::kNT), 0, (hipStream_t)stream,
                         x, e);
    } else {
      x.num_wg = cus;
      hipLaunchKernelGGL(product_512_kernel<kAct>, dim3(cus), dim3(ggemm::kThreads), ggemm::kDynLdsBytes,
                         (hipStream_t)stream, x, e);
    }
    return (int)hipGetLastError();
  });
}

int64_t ggemm_product_act_workspace(int64_t M_total, int32_t G, int32_t N) {
  if (M_total < 0 || M_total > nt::kMaxRow || G <= 0 || G > ag::kMaxGroups || N <= 0) return 0;
  return units_of(M_total, G, N) * N;
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
  const int strips = strips_of(N);
  const int64_t units = units_of(M_total, G, N);
  if (units * strips > 2 * kMaxUnits) return GGEMM_E_SHAPE;
  const ag::Args a{(const uint16_t*)dout, (const uint16_t*)pre, group_offs, G, N, stride_dout, stride_pre,
                   epi::Args{nullptr, 0, nullptr, 0, nullptr, 0, slope, limit, shift}, M_total, unit_rows(M_total, N),
                   (int)units, strips, (N / 8 + strips - 1) / strips, (uint16_t*)dpre, stride_dpre, dbias, workspace};
  if (M_total > 0 && (dpre || dbias)) {
    rc = with_act(act, [&](auto code) {
      hipLaunchKernelGGL(ag::act_backward_kernel<decltype(code)::value>, dim3((uint32_t)(units * strips)),
                         dim3(ag::kThreads), 0, (hipStream_t)stream, a);
      return (int)hipGetLastError();
    });
    if (rc) return rc;
  }
  if (dbias) {
    hipLaunchKernelGGL(ag::bias_sum_kernel, dim3((uint32_t)((N + 63) / 64), (uint32_t)G),
                       dim3(ag::kThreads), 0, (hipStream_t)stream, a);
    rc = (int)hipGetLastError();
  }
  return rc;
}

}  // extern "C"
