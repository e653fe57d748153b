// Kernels and the choice between them of the grouped FP8 product with an epilogue and of the gradient of bias and activation,
// for the entry points that launch them (product_capi.hip; keep_capi.hip, where z is kept in 8 bits).
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "../../include/ggemm_product.h"
#include "act_kernel.h"
#include "capi_common.h"
#include "few_rows.h"
#include "mid_choice.h"

namespace {

using ggemm::host::aligned;
using ggemm::host::device_cus;
using ggemm::host::mid_preferred;
using ggemm::host::mid_tiles;
namespace nt = ggemm::nt;
namespace epi = ggemm::epi;
namespace ag = ggemm::ag;

// What follows the last group's rows becomes zero in out and in the z that is kept.
template <int kAct>
__device__ __forceinline__ void clear_tails(const nt::Args& a, const epi::Args& e) {
  if (!a.zero_tail) return;
  nt::clear_tail_rows(a.c, a.stride_cm, epi::act_of(kAct) == epi::kSwiglu ? a.N / 2 : a.N, a.group_offs, a.G, a.m_total);
  if constexpr ((kAct & epi::kKeepMx) != 0) {
    nt::clear_tail_rows((uint16_t*)e.q8, e.stride_q / 2, a.N / 2, a.group_offs, a.G, a.m_total);
    int64_t r0 = a.group_offs[a.G];
    r0 = r0 < 0 ? 0 : r0;
    for (int64_t r = r0 + blockIdx.x; r < a.m_total; r += gridDim.x)
      for (int b = threadIdx.x; b < (a.N + 31) / 32; b += blockDim.x) e.scales[b * e.scale_block + r] = 127;
  } else if (e.pre != nullptr) nt::clear_tail_rows(e.pre, e.stride_pre, a.N, a.group_offs, a.G, a.m_total);
}

template <int kAct, int kBM>
__global__ __launch_bounds__(ggemm::mid::kNT, 2) void product_mid_kernel(nt::Args a, epi::Args e) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[ggemm::mid::GemmCfg<kBM>::LdsBytes];
  ggemm::mid::gemm_body<false, kBM, 1 + kAct>(nt::without_tail(a), (GG_LDS uint8_t*)lds, e);
  clear_tails<kAct>(a, e);
}

template <int kAct, int NB>
__global__ __launch_bounds__(ggemm::few::kNT) void product_few_kernel(nt::Args a, epi::Args e) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[ggemm::few::Cfg<NB>::LdsBytes];
  ggemm::few::body<kAct, NB>(nt::without_tail(a), (GG_LDS uint8_t*)lds, e);
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
  clear_tails<kMode == ggemm::pw::kBias       ? epi::kNone
              : kMode == ggemm::pw::kGateKeep8 ? epi::kSwiglu + epi::kKeepMx
                                               : epi::kSwiglu>(a, e);
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
  if (e.q8) return (int64_t)e.stride_q * ggemm::pw::kTM < nt::kOob ? ggemm::pw::kGateKeep8 : 0;
  return !e.pre ? ggemm::pw::kGate : rows_fit(e.stride_pre) ? ggemm::pw::kGateKeep : 0;
}

enum class Kernel { kFew16, kFew32, kMid64, kMid128, k512, kWide };
struct Choice {
  Kernel kernel;
  int wide;                // its epilogue, of the wide kernel
  int64_t workgroups;      // of the kernels that take a tile each: whole runs over the XCDs
};

// Few rows (few_rows.h): on average at most eight to a group, so that nearly every group is one row tile, and too few
// mid tiles to fill the chip's two per CU, where those wait out the latency of each stage in turn; with short rows of K
// only while all workgroups fit on the chip at once. 16 columns for each as long as that is so. Measured (us, mid tiles ->
// this; N = 5760, K = 2880 but as said): 1 row of 1 expert 12.9 -> 6.7, 2 rows of 2 13.2 -> 8.8, 4 of 4 16.8 ->
// 14.0, 8 of 8 26.8 -> 25.7, 64 of 8 30.3 -> 29.8, 128 of 8 30.0 -> 38.5 (stays), 32 of 22 63.2 -> 67.2 (stays);
// 128 of 16, N = K = 4096 61.8 -> 52.8; 16 of 15, N = 1536, K = 1024 8.6 -> 9.5 (stays).
constexpr int64_t kFewPerCu = 3;                         // workgroups of either width that a CU holds
bool few_preferred(const nt::Args& a, int64_t g, int64_t cus) {
  return a.G <= ggemm::mid::kMaxGroups && a.m_total <= 8 * (g + 1) && g * ((a.N + 127) / 128) <= 2 * cus &&
         (a.K >= 2048 || g * ((a.N + 31) / 32) <= kFewPerCu * cus / 2);
}

// The others. Against the estimates of the plain product: the large tiles' epilogue takes 3 us a tile, 12 with z
// kept, while the mid tiles' runs beside other workgroups' products; and 64 rows have to be 10 % better. Of 70 drawn
// launches (1 to 40 groups, 16 to 131072 rows, features 64 to 5760) with bias, swiglu, swiglu and z, gelu and residual,
// the choice was 1.012, 1.009, 1.008 and 1.016 times the best of the three kernels in the mean, 1.028, 1.020, 1.044 and
// 1.023 by the plain product's numbers. With z in 8 bits the 512-thread kernel's tiles are 384 columns wide and cost 6 us each:
// of 140 drawn launches, 110 of them near the line, the choice was 1.016 times the best (1.019 by 12 us and bf16 z's tiles);
// 14998 rows of 8 groups, 1040 x 3696, swiglu 73 us (101 on 128-row tiles).
Choice choose(const nt::Args& a, const epi::Args& e, int act, int cus) {
  const int64_t run = ggemm::kXcds * ggemm::mid::kXcdRun, g = std::min<int64_t>(a.G, a.m_total);
  auto runs = [&](int64_t tiles) { return (tiles + run - 1) / run * run; };
  if (few_preferred(a, g, cus)) {
    const bool narrow = g * ((a.N + 15) / 16) <= kFewPerCu * cus && !e.q8;   // a scale is of 32 columns
    const int64_t row_tiles = a.m_total / 16 + g, bn = narrow ? 16 : 32;
    return {narrow ? Kernel::kFew16 : Kernel::kFew32, 0, runs(row_tiles * ((a.N + bn - 1) / bn))};
  }
  const int wide = wide_mode(a, e, act);
  const int extra = e.q8 && !wide ? 6 : e.pre || e.q8 ? 12 : 3;
  const int mid = mid_preferred(a.G, a.N, a.K, a.stride_cm, a.m_total, wide != 0, cus, extra, 0.9, e.q8 != nullptr);
  if (mid) return {mid == 64 ? Kernel::kMid64 : Kernel::kMid128, 0, runs(mid_tiles(mid, a.G, a.N, a.m_total))};
  return {wide ? Kernel::kWide : Kernel::k512, wide, 0};
}

// The launch of checked arguments; kKeep: 0, or epi::kKeepMx.
template <int kKeep>
int launch_product(nt::Args x, const epi::Args& e, int act, int cus, hipStream_t stream) {
  x.num_wg = cus;
  const Choice k = choose(x, e, act, cus);
  if (k.kernel == Kernel::kWide) {
    auto launch = [&](auto kern) { hipLaunchKernelGGL(kern, dim3(cus), dim3(ggemm::pw::kNT), 0, stream, x, e); };
    if constexpr (kKeep != 0)
      launch(product_wide_kernel<ggemm::pw::kGateKeep8>);
    else
      launch(k.wide == ggemm::pw::kBias   ? product_wide_kernel<ggemm::pw::kBias>
             : k.wide == ggemm::pw::kGate ? product_wide_kernel<ggemm::pw::kGate>
                                          : product_wide_kernel<ggemm::pw::kGateKeep>);
    return (int)hipGetLastError();
  }
  return with_act(act, [&](auto code) {
    constexpr int kAct = decltype(code)::value + kKeep;
    const dim3 grid((uint32_t)k.workgroups);
    if constexpr (kAct == epi::kKeepMx) {
      return (int)GGEMM_E_FORMAT;                            // refused before: without an activation z is the result
    } else {
      switch (k.kernel) {
        case Kernel::kFew16:
          if constexpr (kKeep == 0)
            hipLaunchKernelGGL((product_few_kernel<kAct, 1>), grid, dim3(ggemm::few::kNT), 0, stream, x, e);
          break;
        case Kernel::kFew32:
          hipLaunchKernelGGL((product_few_kernel<kAct, 2>), grid, dim3(ggemm::few::kNT), 0, stream, x, e);
          break;
        case Kernel::kMid64:
          hipLaunchKernelGGL((product_mid_kernel<kAct, 64>), grid, dim3(ggemm::mid::kNT), 0, stream, x, e);
          break;
        case Kernel::kMid128:
          hipLaunchKernelGGL((product_mid_kernel<kAct, 128>), grid, dim3(ggemm::mid::kNT), 0, stream, x, e);
          break;
        default:
          hipLaunchKernelGGL(product_512_kernel<kAct>, dim3(cus), dim3(ggemm::kThreads), ggemm::kDynLdsBytes, stream, x, e);
      }
      return (int)hipGetLastError();
    }
  });
}

// Rows of a unit of the gradient: few enough that the units fill the chip, 64 at most (131072 x 5760: 256 rows 810 us, 64
// 795: more rounds of workgroups even out), but for launches of more units than a grid takes. Of 8-bit z, eight rows of which
// a thread has in flight at once, eight at least: 5003 x 1424 14.6 us, 16.4 with sixteen.
constexpr int64_t kMaxUnits = 1 << 22;
int strips_of(int N) { return (N / 8 + ag::kThreads - 1) / ag::kThreads; }
int unit_rows(int64_t M, int N, int least) {
  const int strips = strips_of(N);
  int64_t rows = 64;
  while (rows > least && M / rows * strips < 2048) rows /= 2;
  while (M / rows * strips > kMaxUnits) rows *= 2;
  return (int)rows;
}
constexpr int least_rows(bool mx) { return mx ? 8 : 16; }
int64_t units_of(int64_t M, int G, int N, bool mx) {
  return std::max<int64_t>(1, M / unit_rows(M, N, least_rows(mx)) + std::min<int64_t>(G, M));
}

// Both launches of the gradient on checked arguments; kMx: z from its 8-bit checkpoint.
template <bool kMx>
int launch_act_backward(ag::Args a, int act, hipStream_t stream) {
  const int strips = strips_of(a.N);
  const int64_t units = units_of(a.m_total, a.G, a.N, kMx);
  if (units * strips > 2 * kMaxUnits) return GGEMM_E_SHAPE;
  a.rows = unit_rows(a.m_total, a.N, least_rows(kMx));
  a.units = (int)units;
  a.strips = strips;
  a.lanes = ((a.N / 8 + strips - 1) / strips + 3) / 4 * 4;      // whole blocks of 32 columns
  const bool few = a.G < ag::kThreads * ag::kPerFew;             // and the last offset
  const dim3 grid((uint32_t)(units * strips)), sums((uint32_t)((a.N + 63) / 64), (uint32_t)a.G);
  if (a.m_total > 0 && (a.dpre || a.dbias)) {
    const int rc = with_act(act, [&](auto code) {
      constexpr int kAct = decltype(code)::value;
      if constexpr (kMx && kAct == epi::kNone)
        return (int)GGEMM_E_FORMAT;                          // refused before: nothing is read
      else if (few)
        hipLaunchKernelGGL((ag::act_backward_kernel<kAct, kMx, ag::kPerFew>), grid, dim3(ag::kThreads), 0, stream, a);
      else
        hipLaunchKernelGGL((ag::act_backward_kernel<kAct, kMx, ag::kPerMost>), grid, dim3(ag::kThreads), 0, stream, a);
      return (int)hipGetLastError();
    });
    if (rc) return rc;
  }
  if (a.dbias && few)
    hipLaunchKernelGGL(ag::bias_sum_kernel<ag::kPerFew>, sums, dim3(ag::kThreads), 0, stream, a);
  else if (a.dbias)
    hipLaunchKernelGGL(ag::bias_sum_kernel<ag::kPerMost>, sums, dim3(ag::kThreads), 0, stream, a);
  return (int)hipGetLastError();
}

}  // namespace

