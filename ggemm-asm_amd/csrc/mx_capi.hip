// extern "C" launchers of microscaled rows (include/ggemm_mx.h), part of libggemm_vark.so. Arguments are validated on
// the host; nothing is launched on a validation error.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "../../include/ggemm_mx.h"
#include "capi_common.h"
#include "mx_gemm.h"
#include "mx_quant.h"

namespace {

using ggemm::host::aligned;
using ggemm::host::device_cus;
namespace epi = ggemm::epi;
namespace mx = ggemm::mx;
namespace mxq = ggemm::mxq;
namespace nt = ggemm::nt;

static_assert(GGEMM_ACT_SILU == epi::kSilu && GGEMM_ACT_GELU == epi::kGelu && GGEMM_ACT_SWIGLU == epi::kSwiglu &&
                  GGEMM_PRODUCT_MAX_GROUPS == mx::kMaxGroups,
              "header and kernels agree");

// ------------------------------------------------------------------------------ quantization

constexpr int64_t kUnit = mxq::kThreads * mxq::kUnroll;    // units of a workgroup
constexpr int64_t kMaxUnits = (int64_t(1) << 31) - kUnit;  // of a launch: 31-bit indices

int check_rows(const mxq::Args& a, int dtype, int fmt, const void* x, const void* q) {
  if (!x || !q || !a.scales) return GGEMM_E_NULL;
  if ((dtype != GGEMM_IN_BF16 && dtype != GGEMM_IN_F32) || (fmt != GGEMM_MX_E4M3 && fmt != GGEMM_MX_E2M1))
    return GGEMM_E_FORMAT;
  if (a.rows < 0 || a.cols <= 0 || a.cols % 16) return GGEMM_E_SHAPE;
  const int64_t bytes = fmt == GGEMM_MX_E4M3 ? a.cols : a.cols / 2, unit = fmt == GGEMM_MX_E4M3 ? 8 : 4;
  if (a.stride < a.cols || a.stride % (dtype == GGEMM_IN_BF16 ? 8 : 4) || a.q_stride < bytes || a.q_stride % unit)
    return GGEMM_E_STRIDE;
  if (!aligned(x, 16) || !aligned(q, (uintptr_t)unit)) return GGEMM_E_ALIGN;
  return GGEMM_OK;
}

// kernel(dtype, format)(a) over all rows, as many at a time as 31 bits index.
template <typename F>
int over_rows(mxq::Args a, int dtype, F launch) {
  int cus = 0;
  const int rc = device_cus(&cus);
  if (rc) return rc;
  const int64_t per = 4 * ((a.cols + 31) / 32), most = std::max<int64_t>(1, kMaxUnits / per), rows = a.rows;
  if (per > kMaxUnits) return GGEMM_E_SHAPE;
  a.per = mxq::Divisor::of((uint32_t)per);
  for (int64_t r = 0; r < rows; r += most) {
    a.rows = std::min(most, rows - r);
    launch(a, dim3((uint32_t)((a.rows * per + kUnit - 1) / kUnit)));
    const int err = (int)hipGetLastError();
    if (err) return err;
    a.x = (const uint8_t*)a.x + a.rows * a.stride * (dtype == GGEMM_IN_BF16 ? 2 : 4);
    a.q += a.rows * a.q_stride;
    a.scales += a.rows * a.scale_row;
  }
  return GGEMM_OK;
}

// ------------------------------------------------------------------------------ the product

// Slots of a stage: as many as LDS has room for, but three for what the small tiles gain by (two workgroups to a CU).
template <bool kA8>
using Tile256 = mx::Cfg<kA8, 256, 256, 4, 2, kA8 ? 128 : 256, 2, true>;
template <bool kA8>
using Tile128 = mx::Cfg<kA8, 128, 128, 2, 2, kA8 ? 128 : 256, kA8 ? 3 : 2, false>;
template <bool kA8>
using Tile64 = mx::Cfg<kA8, 64, 128, 1, 4, 256, kA8 ? 2 : 3, false>;
template <bool kA8>
using Tile32 = mx::Cfg<kA8, 32, 128, 1, 4, 256, 3, false>;

__device__ __forceinline__ void clear_tail(int kAct, const mx::Args& a) {
  if (a.zero_tail)
    nt::clear_tail_rows(a.out, a.stride_out, kAct == epi::kSwiglu ? a.N / 2 : a.N, a.group_offs, a.G, a.m_total);
}

template <int kAct, bool kA8, typename C>
__global__ __launch_bounds__(C::NT) __attribute__((amdgpu_waves_per_eu(2, 2)))
void mx_product_kernel(mx::Args a, epi::Args e, int grid, int blocks) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[C::LdsBytes];
  mx::gemm_body<kAct, kA8, C>(a, (GG_LDS uint8_t*)lds, e, grid, blocks);
  clear_tail(kAct, a);
}

template <int kAct, bool kA8, int NB>
__global__ __launch_bounds__(mx::few::kNT) void mx_few_kernel(mx::Args a, epi::Args e) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[mx::few::kWaves * NB * 1024];
  mx::few::body<kAct, kA8, NB>(a, (GG_LDS uint8_t*)lds, e);
  clear_tail(kAct, a);
}

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

int64_t tiles_of(int64_t M, int64_t g, int N, int bm, int bn) { return (M / bm + g) * ((N + bn - 1) / bn); }

// Rows of the output tiles of the fastest kernel. Few rows go to few::body while its tiles of 16 columns are what fills the chip: up
// to 16 rows to a group in the mean and 160 tiles of 32 x 128. Measured (us, 32-row tiles -> it; weights not in a
// cache): N = 5760, K = 2880, e4m3: 1 row of 1 expert 10.2 -> 6.3, 16 of 2 10.7 -> 9.5, 4 of 4 13.0 -> 13.4 (stays),
// 64 of 32 55.8 -> 70.0 (stays); 2 of 2, N = K = 2880 9.7 -> 5.9; 2 of 1, N = K = 4096 11.6 -> 6.1.
// The others by an estimate in us, c + rounds (e + s K / 1000), where a round is as many tiles as the chip holds at once; where
// workgroups walk over their tiles, the last round is a whole one.
// The numbers are a fit to 32 launches of each format, of 32 to 35149 rows, 1 to 32 groups, N 512 to 5760, K 512 to 4096:
// single times are off by up to 0.5 to 1.4, the choice by 3.0 % (e4m3) and 1.6 % (e2m1) in the mean, 19 % and 17 % at most.
struct Fit {
  int rows, cols, per_cu;
  double c, e, s;
};
constexpr Fit kFits[2][4] = {{{32, 128, 2, 0.7, 3.9, 3.08}, {64, 128, 2, -1.8, 4.9, 4.42},
                              {128, 128, 2, -7.0, 11.6, 5.48}, {256, 256, 1, -0.5, 9.1, 10.4}},
                             {{32, 128, 2, 0.0, 4.7, 2.31}, {64, 128, 2, -4.6, 9.5, 2.09},
                              {128, 128, 2, -8.9, 14.0, 3.09}, {256, 256, 1, -0.3, 9.3, 5.72}}};
int choose(int fmt, int G, int N, int K, int64_t M, int cus) {
  const int64_t g = std::min<int64_t>(G, M);
  if (M <= 16 * g && g * ((N + 127) / 128) <= 5 * cus / 8) return 16;
  int best = 0;
  double least = 0;
  for (const Fit& f : kFits[fmt == GGEMM_MX_E2M1]) {
    const double tiles = std::max<double>(g, (double)M / f.rows + g / 2.0) * ((N + f.cols - 1) / f.cols);
    const double part = std::max(1.0, tiles / (f.per_cu * cus)), rounds = f.per_cu == 1 ? std::ceil(part) : part;
    const double t = f.c + rounds * (f.e + f.s * K / 1000);
    if (best == 0 || t < least) best = f.rows, least = t;
  }
  return best;
}

// Whole runs of tiles over the XCDs (mid_common.h).
uint32_t grid_of(int64_t tiles) {
  const int64_t run = ggemm::kXcds * ggemm::mid::kXcdRun;
  return (uint32_t)((tiles + run - 1) / run * run);
}

template <int kAct, bool kA8>
int launch(const mx::Args& a, const epi::Args& e, int tile, int cus, hipStream_t stream) {
  const int64_t g = std::min<int64_t>(a.G, a.m_total);
  auto tiles = [&](int bm, int bn) { return grid_of(tiles_of(a.m_total, g, a.N, bm, bn)); };
  auto run = [&](auto cfg) {
    using C = decltype(cfg);
    const uint32_t blocks = tiles(C::BM, C::BN);
    const uint32_t grid = C::kWalk && a.K > C::KS ? mx::walk_grid((int)blocks, cus) : blocks;
    hipLaunchKernelGGL((mx_product_kernel<kAct, kA8, C>), dim3(grid), dim3(C::NT), 0, stream, a, e, (int)grid, (int)blocks);
  };
  if (tile == 16) {
    if (tiles_of(a.m_total, g, a.N, 16, 16) <= 3 * cus)
      hipLaunchKernelGGL((mx_few_kernel<kAct, kA8, 1>), dim3(tiles(16, 16)), dim3(mx::few::kNT), 0, stream, a, e);
    else
      hipLaunchKernelGGL((mx_few_kernel<kAct, kA8, 2>), dim3(tiles(16, 32)), dim3(mx::few::kNT), 0, stream, a, e);
  } else if (tile == 32) {
    run(Tile32<kA8>{});
  } else if (tile == 64) {
    run(Tile64<kA8>{});
  } else if (tile == 128) {
    run(Tile128<kA8>{});
  } else {
    run(Tile256<kA8>{});
  }
  return (int)hipGetLastError();
}

int validate(const mx::Args& a, const epi::Args& e, int fmt, int act, int bias_dtype, const int64_t (&strides)[6]) {
  if (!a.a || !a.a_scales || !a.b || !a.b_scales || !a.out || !a.group_offs) return GGEMM_E_NULL;
  if (fmt != GGEMM_MX_E4M3 && fmt != GGEMM_MX_E2M1) return GGEMM_E_FORMAT;
  if (e.bias && bias_dtype != GGEMM_IN_BF16 && bias_dtype != GGEMM_IN_F32) return GGEMM_E_FORMAT;
  if (act < GGEMM_ACT_NONE || act > GGEMM_ACT_SWIGLU) return GGEMM_E_FORMAT;
  if (act == GGEMM_ACT_SWIGLU && !(e.limit > 0.f)) return GGEMM_E_SHAPE;
  if (a.G <= 0 || a.G > mx::kMaxGroups || a.N <= 0 || a.K <= 0 || a.N % 16 || a.K % 32) return GGEMM_E_SHAPE;
  if (a.m_total < 0 || a.m_total > nt::kMaxRow) return GGEMM_E_SHAPE;
  if ((a.m_total / 16 + a.G) * (int64_t)((a.N + 15) / 16) > nt::kMaxTiles * 2) return GGEMM_E_SHAPE;
  const int64_t chunk = (int64_t)(a.K + 511) / 512 * 16, bytes_a = fmt == GGEMM_MX_E4M3 ? a.K : a.K / 2;
  const int64_t sa = strides[0], sas = strides[1], sbg = strides[2], sbn = strides[3], sbsg = strides[4], sbsn = strides[5];
  if (sa < bytes_a || sas < chunk || sbn < a.K / 2 || sbsn < chunk) return GGEMM_E_STRIDE;
  if (a.G > 1 && (sbg < (a.N - 1) * sbn + a.K / 2 || sbsg < (a.N - 1) * sbsn + chunk)) return GGEMM_E_STRIDE;
  for (int64_t s : strides)
    if (s % 16) return GGEMM_E_STRIDE;
  // 32-bit buffer offsets of a tile's 256 rows
  for (int64_t s : {sa, sas, sbn, sbsn})
    if (s * 256 >= (int64_t)nt::kOob) return GGEMM_E_SHAPE;
  if ((int64_t)a.stride_out * 2 * 256 >= (int64_t)nt::kOob) return GGEMM_E_SHAPE;
  const int width = act == GGEMM_ACT_SWIGLU ? a.N / 2 : a.N;
  if (a.stride_out < width || a.stride_out % 8) return GGEMM_E_STRIDE;
  if (e.residual && (e.stride_res < width || e.stride_res % 8)) return GGEMM_E_STRIDE;
  for (const void* p : {(const void*)a.a, (const void*)a.a_scales, (const void*)a.b, (const void*)a.b_scales,
                        (const void*)a.out, (const void*)e.bias, (const void*)e.residual})
    if (!aligned(p, 16)) return GGEMM_E_ALIGN;
  return GGEMM_OK;
}

}  // namespace

extern "C" {

int ggemm_mx_quantize(const void* x, int32_t dtype, int64_t rows, int32_t cols, int64_t stride, int32_t fmt, void* q,
                      int64_t q_stride, uint8_t* scales, int64_t scale_stride, void* stream) {
  const mxq::Args a{x, rows, stride, cols, {}, (uint8_t*)q, q_stride, scales, scale_stride, 1};
  const int rc = check_rows(a, dtype, fmt, x, q);
  if (rc) return rc;
  if (scale_stride < (cols + 31) / 32) return GGEMM_E_STRIDE;
  const bool f32 = dtype == GGEMM_IN_F32, e4m3 = fmt == GGEMM_MX_E4M3;
  return over_rows(a, dtype, [&](const mxq::Args& part, dim3 grid) {
    auto kernel = f32 ? (e4m3 ? mxq::quantize_kernel<true, true> : mxq::quantize_kernel<true, false>)
                      : (e4m3 ? mxq::quantize_kernel<false, true> : mxq::quantize_kernel<false, false>);
    hipLaunchKernelGGL(kernel, grid, dim3(mxq::kThreads), 0, (hipStream_t)stream, part);
  });
}

int ggemm_mx_dequantize(const void* q, int32_t fmt, int64_t rows, int32_t cols, int64_t q_stride, const uint8_t* scales,
                        int64_t scale_row, int64_t scale_block, void* out, int32_t dtype, int64_t out_stride,
                        void* stream) {
  const mxq::Args a{out, rows, out_stride, cols, {}, (uint8_t*)q, q_stride, (uint8_t*)scales, scale_row, scale_block};
  const int rc = check_rows(a, dtype, fmt, out, q);
  if (rc) return rc;
  if (scale_row < 0 || scale_block < 0) return GGEMM_E_STRIDE;
  const bool f32 = dtype == GGEMM_IN_F32, e4m3 = fmt == GGEMM_MX_E4M3;
  return over_rows(a, dtype, [&](const mxq::Args& part, dim3 grid) {
    auto kernel = f32 ? (e4m3 ? mxq::dequantize_kernel<true, true> : mxq::dequantize_kernel<true, false>)
                      : (e4m3 ? mxq::dequantize_kernel<false, true> : mxq::dequantize_kernel<false, false>);
    hipLaunchKernelGGL(kernel, grid, dim3(mxq::kThreads), 0, (hipStream_t)stream, part);
  });
}

int32_t ggemm_mx_tile_rows(int32_t a_fmt, int32_t G, int32_t N, int32_t K, int64_t M_total, int32_t num_cus) {
  return choose(a_fmt, G, N, K, M_total, num_cus);
}

int ggemm_mx_product(const void* a, int32_t a_fmt, const uint8_t* a_scales, const void* b, const uint8_t* b_scales,
                     void* out, const void* bias, int32_t bias_dtype, const void* residual, const int64_t* group_offs,
                     int32_t G, int32_t N, int32_t K, int64_t stride_a, int64_t stride_as, int64_t stride_bg,
                     int64_t stride_bn, int64_t stride_bsg, int64_t stride_bsn, int32_t stride_out, int32_t stride_res,
                     int32_t act, float slope, float limit, float shift, int64_t M_total, int32_t zero_tail,
                     int32_t tile, void* stream) {
  const mx::Args x{(const uint8_t*)a, a_scales, (const uint8_t*)b, b_scales, (uint16_t*)out, group_offs, G, N, K,
                   (int)stride_a, (int)stride_as, (int)stride_bn, (int)stride_bsn, stride_out, stride_bg, stride_bsg,
                   M_total, zero_tail};
  const epi::Args e{nullptr, 0, bias, bias_dtype == GGEMM_IN_F32, (const uint16_t*)residual, stride_res, slope, limit,
                    shift, slope * -epi::kLog2e};
  int rc = validate(x, e, a_fmt, act, bias_dtype, {stride_a, stride_as, stride_bg, stride_bn, stride_bsg, stride_bsn});
  if (rc) return rc;
  if (tile != 0 && tile != 16 && tile != 32 && tile != 64 && tile != 128 && tile != 256) return GGEMM_E_SHAPE;
  int cus = 0;
  rc = device_cus(&cus);
  if (rc) return rc;
  if (M_total == 0) return GGEMM_OK;
  if (tile == 0) tile = choose(a_fmt, G, N, K, M_total, cus);
  return with_act(act, [&](auto code) {
    constexpr int kAct = decltype(code)::value;
    return a_fmt == GGEMM_MX_E4M3 ? launch<kAct, true>(x, e, tile, cus, (hipStream_t)stream)
                                  : launch<kAct, false>(x, e, tile, cus, (hipStream_t)stream);
  });
}

}  // extern "C"
