// Gradient of bias and activation for gfx950:
//
//   dpre[r, :] = dout[r, :] act'(pre[r, :]);   dbias[g, :] = sum over the rows r of group g of dpre[r, :]
//
// Bound by HBM: pre and dout are read once and dpre written once, the sums made on the way. A unit is up to
// `rows` consecutive rows of one group; a workgroup takes a unit and a strip of columns, each thread eight
// columns down the unit's rows, and leaves the unit's sums in a row of the workspace, which a second kernel
// adds up per group in unit order: no atomics, so the sums do not depend on what ran first. 131072 x 5760 with
// swiglu: 761 us, 5.0 TB/s, and 16 for the second kernel.
//
// With z in 8 bits (kMx) a quarter less is read and written in all: 629 us, 4.8 TB/s, where the bf16 form takes 761. Its waves
// wait for memory 0.62 of their cycles and yet it stays under the 6.1 TB/s that the quantizer streams; why is not found. A
// row's eight values are 8 bytes, half of what the bf16 form loads, so eight rows are in flight and not four (700 us
// against 686 with the scales read alike), and scales are read two rows to a lane (row_scales). 16 columns to a thread,
// one load each of z and dout, store in halves of lines: 870 us, 1228 past the caches.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fused_epilogue.h"

namespace ggemm {
namespace ag {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMaxGroups = 2047;
// Group offsets a thread holds: one of up to 255 groups, else all that there may be. (5003 x 1424 of 7 groups: 14.7 us with one,
// 16.4 with eight, and the second kernel 4.0 and 4.7.)
constexpr int kPerFew = 1, kPerMost = (kMaxGroups + 1) / kThreads;

struct Args {
  const uint16_t* dout;
  const uint16_t* pre;
  const int64_t* group_offs;
  int G, N, stride_dout, stride_pre;
  epi::Args act;           // slope, limit, shift
  int64_t m_total;
  int rows;                // of a unit
  int units;               // of the launch, at least as many as the groups have
  int strips, lanes;       // strips of columns, the threads of one, eight columns each
  uint16_t* dpre;
  int stride_dpre;
  float* dbias;
  float* partial;          // [units][N]
  const uint8_t* q8 = nullptr;   // z in 8 bits instead of pre: e4m3 values (rows stride_pre bytes apart) and the scale of
  const uint8_t* scales = nullptr;   // row r and block of 32 columns b at [r scale_row + b scale_block]
  int64_t scale_row = 0, scale_block = 0;
};

// Group g has rows start[g] .. start[g + 1] - 1 and units pre[g] .. pre[g + 1] - 1. Offsets are clamped to
// [0, m_total] and to the largest one before them, so groups never overlap and there are at most
// m_total / rows + G units whatever group_offs holds.
template <int kPer>
struct Table {
  int start[kThreads * kPer];
  int pre[kThreads * kPer];
  int scan[2 * kWaves];
};

template <int kPer>
__device__ __forceinline__ void group_table(const Args& a, Table<kPer>& t) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int o[kPer + 1], mx = 0;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int64_t v = a.group_offs[min(tid * kPer + k, a.G)];
    o[k] = (int)(v < 0 ? 0 : v > a.m_total ? a.m_total : v);
    mx = max(mx, o[k]);
    o[k] = mx;
  }
  int incl = mx;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int v = __shfl_up(incl, d, 64);
    if (lane >= d) incl = max(incl, v);
  }
  if (lane == 63) t.scan[wave] = incl;
  __syncthreads();
  int before = __shfl_up(incl, 1, 64);
  if (lane == 0) before = 0;
  for (int w = 0; w < wave; ++w) before = max(before, t.scan[w]);
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    o[k] = max(o[k], before);
    t.start[tid * kPer + k] = o[k];        // entries past G repeat the last offset
  }
  __syncthreads();
  o[kPer] = tid == kThreads - 1 ? o[kPer - 1] : t.start[(tid + 1) * kPer];
  int units[kPer], sum = 0;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    // unsigned: 2^31 - 256 rows and a unit's 512 are more than 31 bits hold
    units[k] = (int)(((uint32_t)(o[k + 1] - o[k]) + (uint32_t)a.rows - 1u) / (uint32_t)a.rows);
    sum += units[k];
  }
  int acc = sum;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int v = __shfl_up(acc, d, 64);
    if (lane >= d) acc += v;
  }
  if (lane == 63) t.scan[kWaves + wave] = acc;
  __syncthreads();
  int run = acc - sum;
  for (int w = 0; w < wave; ++w) run += t.scan[kWaves + w];
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    t.pre[tid * kPer + k] = run;
    run += units[k];
  }
  __syncthreads();
}

template <int kAct>
__device__ __forceinline__ void grad8(const float (&z)[8], const v4i& d8, const epi::Args& e, float (&out)[8]) {
  float d[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    d[2 * i] = epi::from_bf16(d8[i]);
    d[2 * i + 1] = __uint_as_float(d8[i] & 0xffff0000u);
  }
  if constexpr (kAct == epi::kSwiglu) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float g = epi::at_most(z[2 * i], e.limit), u = epi::within(z[2 * i + 1], e.limit);
      const float s = epi::sigmoid2(e.nslope * g), gs = g * s;
      const float dg = d[i] * ((u + e.shift) * (s + e.slope * gs * (1.f - s)));   // a closed gate closes before d
      out[2 * i] = z[2 * i] > e.limit ? 0.f : dg;
      out[2 * i + 1] = fabsf(z[2 * i + 1]) > e.limit ? 0.f : d[i] * gs;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (kAct == epi::kSilu) {
        const float s = epi::sigmoid(z[i]);
        out[i] = d[i] * (s + z[i] * s * (1.f - s));
      } else if constexpr (kAct == epi::kGelu) {
        float gauss;
        const float cdf = epi::normal_cdf_fp32(z[i], &gauss);
        out[i] = d[i] * (cdf + z[i] * gauss * 0.398942280401433f);
      } else {
        out[i] = d[i];
      }
    }
  }
}

// The scales of eight rows and a block of columns, in the four lanes that hold its columns: lane k has those of rows 2 k
// and 2 k + 1, low byte first. A byte a row and lane takes 16 us more of 645 (131072 x 5760, swiglu; silu on 2880 columns: 47
// of 415): by blocks, as the product leaves them, a wave's bytes of a row lie in 16 lines.
__device__ __forceinline__ uint32_t row_scales(const Args& a, int64_t r, int64_t r1, int n) {
  const uint8_t* s = a.scales + (int64_t)(n / 32) * a.scale_block;
  const int64_t k = r + 2 * (threadIdx.x & 3);
  uint32_t v = 0;
  if (k < r1) v = s[k * a.scale_row];
  if (k + 1 < r1) v |= (uint32_t)s[(k + 1) * a.scale_row] << 16;
  return v;
}

// Row u's of them, as 2^X.
template <int u>
__device__ __forceinline__ float row_scale(uint32_t v) {
  const uint32_t b = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, u / 2 * 0x55, 0xf, 0xf, true);
  return __uint_as_float(u & 1 ? b >> 16 << 23 : (b & 0xff) << 23);
}

// grid: units x strips; kMx: z from its 8-bit checkpoint
template <int kAct, bool kMx, int kPer>
__global__ __launch_bounds__(kThreads) void act_backward_kernel(Args a) {
  __shared__ Table<kPer> t;
  group_table(a, t);
  const int unit = (int)blockIdx.x / a.strips, strip = (int)blockIdx.x % a.strips;
  const int n = 8 * (strip * a.lanes + (int)threadIdx.x), no = kAct == epi::kSwiglu ? n / 2 : n;
  // four lanes hold a block's columns and read its scales for each other: they go together, the last two of a half block idle
  if ((int)threadIdx.x >= a.lanes || (kMx ? n & ~31 : n) >= a.N) return;
  const bool live = !kMx || n < a.N;
  if (live && a.dpre != nullptr) {                    // rows of no group
    for (int64_t r = unit; r < t.start[0]; r += a.units) *(v4i*)(a.dpre + r * a.stride_dpre + n) = v4i{0, 0, 0, 0};
    for (int64_t r = t.start[a.G] + (int64_t)unit; r < a.m_total; r += a.units)
      *(v4i*)(a.dpre + r * a.stride_dpre + n) = v4i{0, 0, 0, 0};
  }
  if (unit >= t.pre[a.G]) return;
  int lo = 0, hi = a.G - 1;                           // the last group whose units begin at or before this one
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.pre[mid] <= unit) lo = mid; else hi = mid - 1;
  }
  const int64_t r0 = t.start[lo] + (int64_t)(unit - t.pre[lo]) * a.rows;
  const int64_t r1 = min(r0 + a.rows, (int64_t)t.start[lo + 1]);
  float sum[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) sum[i] = 0.f;
  constexpr int kUnroll = kMx ? 8 : 4;                // rows a thread has in flight
  for (int64_t r = r0; r < r1; r += kUnroll) {
    v4i z[kUnroll], d[kUnroll];
    uint32_t scales = 0;
    if constexpr (kMx) scales = row_scales(a, r, r1, n);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      z[u] = d[u] = v4i{0, 0, 0, 0};
      if (!live || r + u >= r1) continue;
      if constexpr (kMx) {
        const v2i h = __builtin_nontemporal_load((const v2i*)(a.q8 + (r + u) * a.stride_pre + n));
        z[u][0] = h[0];
        z[u][1] = h[1];
      } else if constexpr (kAct != epi::kNone) z[u] = __builtin_nontemporal_load((const v4i*)(a.pre + (r + u) * a.stride_pre + n));
      if constexpr (kAct == epi::kSwiglu) {
        const v2i h = __builtin_nontemporal_load((const v2i*)(a.dout + (r + u) * a.stride_dout + no));
        d[u][0] = h[0];
        d[u][1] = h[1];
      } else {
        d[u] = __builtin_nontemporal_load((const v4i*)(a.dout + (r + u) * a.stride_dout + no));
      }
    }
    float power[kUnroll];
    if constexpr (kMx) {
      power[0] = row_scale<0>(scales), power[1] = row_scale<1>(scales), power[2] = row_scale<2>(scales);
      power[3] = row_scale<3>(scales), power[4] = row_scale<4>(scales), power[5] = row_scale<5>(scales);
      power[6] = row_scale<6>(scales), power[7] = row_scale<7>(scales);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (!live || r + u >= r1) continue;
      float x[8], v[8];
      if constexpr (kMx) {
        mxq::restore_f32<true>(mxq::v2u{(unsigned)z[u][0], (unsigned)z[u][1]}, power[u], v);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[2 * i] = epi::from_bf16(z[u][i]);
          v[2 * i + 1] = __uint_as_float(z[u][i] & 0xffff0000u);
        }
      }
      grad8<kAct>(v, d[u], a.act, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] += x[i];
      if (a.dpre != nullptr) {
        store_c16(a.dpre + (r + u) * a.stride_dpre + n,
                  v4i{epi::pack(x[0], x[1]), epi::pack(x[2], x[3]), epi::pack(x[4], x[5]), epi::pack(x[6], x[7])});
      }
    }
  }
  if (live && a.dbias != nullptr) {
    float* p = a.partial + (int64_t)unit * a.N + n;
    *(v4f*)p = v4f{sum[0], sum[1], sum[2], sum[3]};
    *(v4f*)(p + 4) = v4f{sum[4], sum[5], sum[6], sum[7]};
  }
}

// dbias[g, n] over the group's units; grid (columns / 64, G): a wave takes 64 columns and every kWaves-th unit, eight
// of them in flight, and the waves' sums are added in their order.
template <int kPer>
__global__ __launch_bounds__(kThreads) void bias_sum_kernel(Args a) {
  __shared__ Table<kPer> t;
  __shared__ float s_sum[kThreads];
  group_table(a, t);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = blockIdx.x * 64 + lane, g = blockIdx.y;
  float s = 0.f;
  if (n < a.N)
    for (int u = t.pre[g] + wave; u < t.pre[g + 1]; u += 8 * kWaves) {
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = u + i * kWaves < t.pre[g + 1] ? a.partial[(int64_t)(u + i * kWaves) * a.N + n] : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s += p[i];
    }
  s_sum[threadIdx.x] = s;
  __syncthreads();
  if (wave == 0 && n < a.N) {
    for (int w = 1; w < kWaves; ++w) s += s_sum[64 * w + lane];
    a.dbias[(int64_t)g * a.N + n] = s;
  }
}

}  // namespace ag
}  // namespace ggemm
