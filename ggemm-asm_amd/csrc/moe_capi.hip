// extern "C" launchers of expert routing and of the rows' way to the experts and back
// (include/ggemm_moe.h), part of libggemm_vark.so. Arguments are validated on the host; nothing is
// launched on a validation error.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "../../include/ggemm_moe.h"
#include "capi_common.h"
#include "exchange_kernel.h"
#include "route_kernel.h"

static_assert(GGEMM_MOE_MAX_EXPERTS == ggemm::rt::kMaxExperts && GGEMM_MOE_MAX_TOP_K == ggemm::rt::kMaxTopK &&
                  GGEMM_MOE_MAX_GROUPS == ggemm::ex::kMaxGroups && GGEMM_MOE_PLAN_ALONE == ggemm::ex::kPlanAlone,
              "header and kernels agree");

namespace {

using ggemm::host::aligned;
using ggemm::host::device_cus;
namespace rt = ggemm::rt;
namespace ex = ggemm::ex;

constexpr int kMaxWidth = 1 << 28;                       // elements of a row: 32-bit byte offsets
constexpr int64_t kMaxRows = (int64_t(1) << 31) - 256;   // rows and choices: 32-bit numbers

int check_logits(const void* logits, int dtype, int64_t T, int E, int64_t stride, int k, int score) {
  if (!logits) return GGEMM_E_NULL;
  if (dtype != GGEMM_IN_BF16 && dtype != GGEMM_IN_F32) return GGEMM_E_FORMAT;
  if (score != GGEMM_MOE_SOFTMAX && score != GGEMM_MOE_SIGMOID) return GGEMM_E_FORMAT;
  if (T < 0 || E <= 0 || E > rt::kMaxExperts || k <= 0 || k > rt::kMaxTopK || k > E) return GGEMM_E_SHAPE;
  if (T > kMaxRows || T * k > kMaxRows) return GGEMM_E_SHAPE;
  if (stride < E) return GGEMM_E_STRIDE;
  if (!aligned(logits, dtype == GGEMM_IN_BF16 ? 2 : 4)) return GGEMM_E_ALIGN;
  return GGEMM_OK;
}

// f(L, V) of the smallest layout that holds E experts: four per lane, from eight lanes to a wave; then more per lane.
template <typename F>
int with_layout(int E, F f) {
  using std::integral_constant;
#define GGEMM_RT(L, V) \
  if (E <= (L) * (V)) return f(integral_constant<int, L>{}, integral_constant<int, V>{})
  GGEMM_RT(8, 1);
  GGEMM_RT(8, 2);
  GGEMM_RT(8, 4);
  GGEMM_RT(16, 4);
  GGEMM_RT(32, 4);
  GGEMM_RT(64, 4);
  GGEMM_RT(64, 8);
  GGEMM_RT(64, 16);
#undef GGEMM_RT
  return GGEMM_E_SHAPE;
}

// Bytes that every address and stride here is a multiple of: 16, 4, 2 or 1.
int common_bytes(uint64_t all) { return all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : all % 2 == 0 ? 2 : 1; }
uint64_t bits(const void* p) { return (uint64_t)reinterpret_cast<uintptr_t>(p); }

// Whether a lane's V elements of every row are one aligned access (of at most 16 bytes each).
bool one_load(int V, int item, int E, int64_t stride, const void* p) {
  return E % V == 0 && stride % V == 0 && aligned(p, (uintptr_t)std::min(V * item, 16));
}

// Workgroups of four waves, a wave per row, at most eight to a CU.
int row_grid(int64_t rows, int cus) {
  return (int)std::max<int64_t>(1, std::min<int64_t>((rows + ex::kWaves - 1) / ex::kWaves, (int64_t)cus * 8));
}

int check_slots(const int32_t* slots, int64_t T, int k, int64_t M) {
  if (!slots) return GGEMM_E_NULL;
  if (T < 0 || k <= 0 || M < 0 || T > kMaxRows || M > kMaxRows || T * k > kMaxRows) return GGEMM_E_SHAPE;
  return aligned(slots, 4) ? GGEMM_OK : GGEMM_E_ALIGN;
}

int plan_blocks(int64_t n, int G, int* per) {
  if (n <= ex::kPlanAlone) {
    *per = (int)std::max<int64_t>(ex::kThreads, (n + ex::kThreads - 1) / ex::kThreads * ex::kThreads);
    return 1;
  }
  const int most = ex::plan_blocks_most(G);
  int64_t p = std::max<int64_t>(ex::kPlanEntries, (n + most - 1) / most);
  p = (p + ex::kThreads - 1) / ex::kThreads * ex::kThreads;
  *per = (int)p;
  return (int)((n + p - 1) / p);
}

}  // namespace

extern "C" {

int ggemm_moe_route(const void* logits, int32_t dtype, int64_t T, int32_t E, int64_t stride, int32_t top_k,
                    int32_t score, const float* bias, int32_t num_groups, int32_t top_groups, int32_t group_best,
                    int32_t renormalize, float scale, float* weights, int32_t* experts, void* stream) {
  int rc = check_logits(logits, dtype, T, E, stride, top_k, score);
  if (rc) return rc;
  if (!weights || !experts) return GGEMM_E_NULL;
  if (num_groups < 1 || E % num_groups || top_groups < 1 || top_groups > num_groups) return GGEMM_E_SHAPE;
  if (group_best < 1 || group_best > 2 || (num_groups > 1 && E / num_groups < group_best)) return GGEMM_E_SHAPE;
  if (!aligned(weights, 4) || !aligned(experts, 4) || !aligned(bias, 4)) return GGEMM_E_ALIGN;
  int cus = 0;
  rc = device_cus(&cus);
  if (rc) return rc;
  if (T == 0) return GGEMM_OK;
  rt::Args a{logits, T, stride, E, top_k, score, bias, num_groups, top_groups, group_best, renormalize, scale, weights,
             experts, false};
  const int item = dtype == GGEMM_IN_BF16 ? 2 : 4;
  return with_layout(E, [&](auto l, auto v) {
    constexpr int L = decltype(l)::value, V = decltype(v)::value;
    const dim3 grid((uint32_t)((T + rt::kThreads / L - 1) / (rt::kThreads / L)));
    const int lds = rt::route_lds(L, E, top_k, num_groups);
    a.vec = one_load(V, item, E, stride, logits);
    if (dtype == GGEMM_IN_BF16)
      hipLaunchKernelGGL((rt::route_kernel<uint16_t, L, V>), grid, dim3(rt::kThreads), lds, (hipStream_t)stream, a);
    else
      hipLaunchKernelGGL((rt::route_kernel<float, L, V>), grid, dim3(rt::kThreads), lds, (hipStream_t)stream, a);
    return (int)hipGetLastError();
  });
}

int ggemm_moe_route_backward(const float* dweights, const void* logits, int32_t dtype, int64_t T, int32_t E,
                             int64_t stride, int32_t top_k, int32_t score, int32_t renormalize, float scale,
                             const int32_t* experts, void* dlogits, void* stream) {
  int rc = check_logits(logits, dtype, T, E, stride, top_k, score);
  if (rc) return rc;
  if (!dweights || !experts || !dlogits) return GGEMM_E_NULL;
  if (!aligned(dweights, 4) || !aligned(experts, 4) || !aligned(dlogits, dtype == GGEMM_IN_BF16 ? 2 : 4))
    return GGEMM_E_ALIGN;
  int cus = 0;
  rc = device_cus(&cus);
  if (rc) return rc;
  if (T == 0) return GGEMM_OK;
  rt::BackArgs a{dweights, logits, T, stride, E, top_k, score, renormalize, scale, experts, dlogits, false, false};
  const int item = dtype == GGEMM_IN_BF16 ? 2 : 4;
  return with_layout(E, [&](auto l, auto v) {
    constexpr int L = decltype(l)::value, V = decltype(v)::value;
    const dim3 grid((uint32_t)((T + rt::kThreads / L - 1) / (rt::kThreads / L)));
    const int lds = rt::route_back_lds(L, E, top_k);
    a.vec = one_load(V, item, E, stride, logits);
    a.vec_out = one_load(V, item, E, E, dlogits);
    if (dtype == GGEMM_IN_BF16)
      hipLaunchKernelGGL((rt::route_backward_kernel<uint16_t, L, V>), grid, dim3(rt::kThreads), lds,
                         (hipStream_t)stream, a);
    else
      hipLaunchKernelGGL((rt::route_backward_kernel<float, L, V>), grid, dim3(rt::kThreads), lds, (hipStream_t)stream,
                         a);
    return (int)hipGetLastError();
  });
}

int64_t ggemm_moe_plan_workspace(int64_t n, int32_t G) {
  if (n < 0 || n > kMaxRows || G <= 0 || G > ex::kMaxGroups) return 0;
  int per = 0;
  const int blocks = plan_blocks(n, G, &per);
  return blocks > 1 ? (int64_t)blocks * G : 0;
}

int ggemm_moe_plan(const int32_t* experts, int64_t n, int32_t G, int64_t* group_offs, int32_t* slots,
                   int32_t* workspace, void* stream) {
  if (!group_offs || (n > ex::kPlanAlone && !workspace) || (n > 0 && (!experts || !slots))) return GGEMM_E_NULL;
  if (n < 0 || n > kMaxRows || G <= 0 || G > ex::kMaxGroups) return GGEMM_E_SHAPE;
  if (!aligned(experts, 4) || !aligned(slots, 4) || !aligned(workspace, 4) || !aligned(group_offs, 8))
    return GGEMM_E_ALIGN;
  int cus = 0;
  const int rc = device_cus(&cus);
  if (rc) return rc;
  ex::PlanArgs a{experts, n, G, 0, group_offs, slots, workspace};
  const int blocks = plan_blocks(n, G, &a.per);
  if (blocks > 1) {
    hipLaunchKernelGGL(ex::plan_count_kernel, dim3(blocks), dim3(ex::kThreads), 4 * G, (hipStream_t)stream, a);
    const int e = (int)hipGetLastError();
    if (e) return e;
  }
  hipLaunchKernelGGL(ex::plan_kernel, dim3(blocks), dim3(ex::kThreads), ex::plan_lds(G), (hipStream_t)stream, a);
  return (int)hipGetLastError();
}

int ggemm_moe_dispatch(const void* x, int64_t row_bytes, int64_t x_stride, int64_t T, int32_t top_k,
                       const int32_t* slots, const int64_t* group_offs, int32_t G, void* rows, int64_t rows_stride,
                       int64_t M, void* stream) {
  int rc = check_slots(slots, T, top_k, M);
  if (rc) return rc;
  if (!x || !rows || !group_offs) return GGEMM_E_NULL;
  if (row_bytes <= 0 || row_bytes > INT32_MAX || G <= 0 || G > ex::kMaxGroups) return GGEMM_E_SHAPE;
  if (x_stride < row_bytes || rows_stride < row_bytes) return GGEMM_E_STRIDE;
  if (!aligned(group_offs, 8)) return GGEMM_E_ALIGN;
  int cus = 0;
  rc = device_cus(&cus);
  if (rc) return rc;
  if (M == 0) return GGEMM_OK;
  const ex::CopyArgs a{(const uint8_t*)x, row_bytes, x_stride, T, top_k, slots, group_offs, G, (uint8_t*)rows,
                       rows_stride, M};
  const bool lines = (bits(rows) | (uint64_t)rows_stride) % 128 == 0;
  auto kern = ex::dispatch_kernel<1, false>;
  switch (common_bytes(bits(x) | bits(rows) | (uint64_t)(row_bytes | x_stride | rows_stride))) {
    case 16: kern = lines ? ex::dispatch_kernel<16, true> : ex::dispatch_kernel<16, false>; break;
    case 4: kern = ex::dispatch_kernel<4, false>; break;
    case 2: kern = ex::dispatch_kernel<2, false>; break;
  }
  hipLaunchKernelGGL(kern, dim3(row_grid(std::max(T, M / 8), cus)), dim3(ex::kThreads), 0, (hipStream_t)stream, a);
  return (int)hipGetLastError();
}

int ggemm_moe_combine(const void* y, int32_t dtype, int64_t y_stride, int64_t M, const int32_t* slots, int64_t T,
                      int32_t top_k, const float* weights, const void* residual, int64_t residual_stride, int32_t H,
                      void* out, int64_t out_stride, void* stream) {
  int rc = check_slots(slots, T, top_k, M);
  if (rc) return rc;
  if (!y || !out) return GGEMM_E_NULL;
  if (dtype != GGEMM_IN_BF16 && dtype != GGEMM_IN_F32) return GGEMM_E_FORMAT;
  if (H <= 0 || H > kMaxWidth) return GGEMM_E_SHAPE;
  if (y_stride < H || out_stride < H || (residual && residual_stride < H)) return GGEMM_E_STRIDE;
  const int item = dtype == GGEMM_IN_BF16 ? 2 : 4;
  if (!aligned(y, item) || !aligned(out, item) || !aligned(residual, item) || !aligned(weights, 4))
    return GGEMM_E_ALIGN;
  int cus = 0;
  rc = device_cus(&cus);
  if (rc) return rc;
  if (T == 0) return GGEMM_OK;
  ex::CombineArgs a{y, y_stride, M, slots, T, top_k, weights, residual, residual_stride, H, out, out_stride, 1};
  const bool lines = (bits(out) | (uint64_t)(item * out_stride)) % 128 == 0;
  const uint64_t all = bits(y) | bits(out) | bits(residual) |
                       (uint64_t)item * (uint64_t)(y_stride | out_stride | (residual ? residual_stride : 0) | H);
  const bool wide = common_bytes(all) == 16;
  auto pick = [&](auto narrow, auto whole, auto shared) { return !wide ? narrow : lines ? whole : shared; };
  auto kern = dtype == GGEMM_IN_BF16
                  ? pick(ex::combine_kernel<uint16_t, 1, false>, ex::combine_kernel<uint16_t, 8, true>,
                         ex::combine_kernel<uint16_t, 8, false>)
                  : pick(ex::combine_kernel<float, 1, false>, ex::combine_kernel<float, 4, true>,
                         ex::combine_kernel<float, 4, false>);
  // a token's columns go to as many waves as they have steps while that fills no more than a wave per SIMD: one token of
  // 2880 takes one round trip to memory then, not six
  const int steps = (H + 64 * (wide ? 16 / item : 1) - 1) / (64 * (wide ? 16 / item : 1));
  a.parts = (int)std::min<int64_t>(steps, std::max<int64_t>(1, (int64_t)cus * 4 / T));
  hipLaunchKernelGGL(kern, dim3(row_grid(T * a.parts, cus)), dim3(ex::kThreads), 0, (hipStream_t)stream, a);
  return (int)hipGetLastError();
}

int ggemm_moe_combine_backward(const void* dout, int32_t dtype, int64_t dout_stride, const void* y, int64_t y_stride,
                               int64_t M, const int32_t* slots, int64_t T, int32_t top_k, const float* weights,
                               const int64_t* group_offs, int32_t G, int32_t H, void* dy, int64_t dy_stride,
                               float* dweights, void* stream) {
  int rc = check_slots(slots, T, top_k, M);
  if (rc) return rc;
  if (!dout || !group_offs || (dweights && !y)) return GGEMM_E_NULL;
  if (dtype != GGEMM_IN_BF16 && dtype != GGEMM_IN_F32) return GGEMM_E_FORMAT;
  if (H <= 0 || H > kMaxWidth || G <= 0 || G > ex::kMaxGroups) return GGEMM_E_SHAPE;
  if (dout_stride < H || (dweights && y_stride < H) || (dy && dy_stride < H)) return GGEMM_E_STRIDE;
  const int item = dtype == GGEMM_IN_BF16 ? 2 : 4;
  if (!aligned(dout, item) || !aligned(y, item) || !aligned(dy, item) || !aligned(weights, 4) ||
      !aligned(dweights, 4) || !aligned(group_offs, 8))
    return GGEMM_E_ALIGN;
  int cus = 0;
  rc = device_cus(&cus);
  if (rc) return rc;
  if ((!dy && !dweights) || (T == 0 && M == 0)) return GGEMM_OK;
  const ex::CombineBackArgs a{dout, dout_stride, y,          y_stride, M, slots, T,         top_k,
                              weights, group_offs, G, H, dy, dy_stride, dweights};
  const bool lines = (bits(dy) | (uint64_t)(item * dy_stride)) % 128 == 0;
  const uint64_t all = bits(dout) | (dweights ? bits(y) : 0) | bits(dy) |
                       (uint64_t)item * (uint64_t)(dout_stride | (dweights ? y_stride : 0) | (dy ? dy_stride : 0) | H);
  const bool wide = common_bytes(all) == 16;
  auto pick = [&](auto narrow, auto whole, auto shared) { return !wide ? narrow : lines ? whole : shared; };
  auto kern = dtype == GGEMM_IN_BF16
                  ? pick(ex::combine_backward_kernel<uint16_t, 1, false>, ex::combine_backward_kernel<uint16_t, 8, true>,
                         ex::combine_backward_kernel<uint16_t, 8, false>)
                  : pick(ex::combine_backward_kernel<float, 1, false>, ex::combine_backward_kernel<float, 4, true>,
                         ex::combine_backward_kernel<float, 4, false>);
  hipLaunchKernelGGL(kern, dim3(row_grid(std::max(T, M / 8), cus)), dim3(ex::kThreads), 0, (hipStream_t)stream, a);
  return (int)hipGetLastError();
}

}  // extern "C"
