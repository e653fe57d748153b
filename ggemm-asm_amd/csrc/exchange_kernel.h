// Rows of tokens into expert order and back, for gfx950: the order itself (a stable counting sort of the
// choices by expert), the copy of each token's row to its experts' rows, and the weighted sum back, with
// its gradients.
//
// All but the sort are streams of rows, bound by HBM. They go by token: a token's row is read once and
// written to its rows (or its rows read and summed in registers), so no inverse of the order is kept, no
// two waves write one element and no sum depends on the order in which waves run.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ggemm {
namespace ex {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMaxGroups = 2047;
// Workgroups of a plan: each 1024 choices or more, at most 256 and fewer the more experts there are, since each reads all
// workgroups' counts of each. Measured (us, at most 64 -> 128 -> 256): 131072 choices of 32 experts 8.9, 8.1, 8.7; 2^20 of 64
// 40.8, 24.8, 18.5; 131072 of 256 14.3, 17.5, 26.6.
constexpr int kPlanEntries = 1024;
inline int plan_blocks_most(int G) { return 16384 / G > 256 ? 256 : 16384 / G < 64 ? 64 : 16384 / G; }
constexpr int kPlanAlone = 2048;             // choices that one workgroup orders by itself
typedef unsigned int v4u __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------------------------ the order

struct PlanArgs {
  const int* experts;
  int64_t n;
  int G;
  int per;                 // choices per workgroup, a multiple of kThreads
  int64_t* group_offs;
  int* slots;
  int* hist;               // [workgroups][G]: choices of each expert (plan_count_kernel)
};

// The experts of kAhead choices from i on, `step` apart, all loads in flight; at or past end, and of no group, negative.
constexpr int kAhead = 8;
__device__ __forceinline__ void groups_of(const PlanArgs& a, int64_t i, int64_t end, int step, int (&g)[kAhead]) {
#pragma unroll
  for (int u = 0; u < kAhead; ++u) {
    const int64_t at = i + (int64_t)u * step;
    g[u] = at < end ? a.experts[at] : -1;
  }
#pragma unroll
  for (int u = 0; u < kAhead; ++u) g[u] = g[u] < a.G ? g[u] : -1;
}

__global__ __launch_bounds__(kThreads) void plan_count_kernel(PlanArgs a) {
  extern __shared__ int s_cnt[];
  for (int g = threadIdx.x; g < a.G; g += kThreads) s_cnt[g] = 0;
  __syncthreads();
  const int64_t lo = (int64_t)blockIdx.x * a.per, end = min(lo + a.per, a.n);
  for (int64_t i = lo + threadIdx.x; i < end; i += kAhead * kThreads) {
    int g[kAhead];
    groups_of(a, i, end, kThreads, g);
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (g[u] >= 0) atomicAdd(&s_cnt[g[u]], 1);
  }
  __syncthreads();
  for (int g = threadIdx.x; g < a.G; g += kThreads) a.hist[(int64_t)blockIdx.x * a.G + g] = s_cnt[g];
}

// Rows of this workgroup's choices: first row of the expert (a scan over the experts' totals), plus its
// choices in the workgroups before, in the waves before, and in the wave before. A wave takes consecutive
// choices, 64 at a time; lanes of one expert find each other by a ballot for each bit of its number. Bound by the
// latency of its phases: 131072 choices of 32 experts 4.8 + 5.5 us with the counts, eight choices alone 2.9.
inline int plan_lds(int G) { return 4 * ((kWaves + 2) * G + kWaves); }

__global__ __launch_bounds__(kThreads) void plan_kernel(PlanArgs a) {
  extern __shared__ int s_pl[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, G = a.G;
  int* s_wave = s_pl;                        // [kWaves][G]: counts, then each wave's next row
  int* s_all = s_pl + kWaves * G;            // [G]: choices of each expert
  int* s_before = s_all + G;                 // [G]: those in the workgroups before this one
  int* s_scan = s_before + G;                // [kWaves]
  for (int g = tid; g < (kWaves + 2) * G; g += kThreads) s_pl[g] = 0;
  __syncthreads();
  const int64_t lo = (int64_t)blockIdx.x * a.per, end = min(lo + a.per, a.n);
  const int each = a.per / kWaves;           // a multiple of 64
  const int64_t wlo = lo + wave * each, wend = min(wlo + each, end);
  int first[kAhead];                         // the wave's choices, or the first of them
  groups_of(a, wlo + lane, wend, 64, first);
#pragma unroll
  for (int u = 0; u < kAhead; ++u)
    if (first[u] >= 0) atomicAdd(&s_wave[wave * G + first[u]], 1);
  for (int64_t i = wlo + lane + 64 * kAhead; i < wend; i += 64 * kAhead) {
    int g[kAhead];
    groups_of(a, i, wend, 64, g);
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (g[u] >= 0) atomicAdd(&s_wave[wave * G + g[u]], 1);
  }
  const int blocks = gridDim.x;
  if (blocks > 1) {
    const int parts = max(1, kThreads / G);  // threads that share an expert's column
    for (int u = tid; u < G * parts; u += kThreads) {
      const int g = u % G;
      int before = 0, all = 0;
      for (int b0 = u / G; b0 < blocks; b0 += 8 * parts) {
        int c[8];                            // eight rows in flight
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = b0 + i * parts < blocks ? a.hist[(int64_t)(b0 + i * parts) * G + g] : 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          all += c[i];
          before += b0 + i * parts < (int)blockIdx.x ? c[i] : 0;
        }
      }
      atomicAdd(&s_all[g], all);
      atomicAdd(&s_before[g], before);
    }
  }
  __syncthreads();
  const int span = (G + kThreads - 1) / kThreads, g0 = min(tid * span, G), g1 = min(g0 + span, G);
  int sum = 0;
  for (int g = g0; g < g1; ++g) {
    if (blocks == 1)
      for (int w = 0; w < kWaves; ++w) s_all[g] += s_wave[w * G + g];
    sum += s_all[g];
  }
  int incl = sum;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(incl, d, 64);
    if (lane >= d) incl += o;
  }
  if (lane == 63) s_scan[wave] = incl;
  __syncthreads();
  int run = incl - sum;
  for (int w = 0; w < wave; ++w) run += s_scan[w];
  for (int g = g0; g < g1; ++g) {
    if (blockIdx.x == 0) a.group_offs[g] = run;
    int start = run + s_before[g];
    for (int w = 0; w < kWaves; ++w) {
      const int c = s_wave[w * G + g];
      s_wave[w * G + g] = start;
      start += c;
    }
    run += s_all[g];
  }
  if (blockIdx.x == 0 && tid == kThreads - 1) a.group_offs[G] = run;
  __syncthreads();
  const int bits = 32 - __builtin_clz(G);    // of expert numbers below G
  int* next = s_wave + wave * G;
  for (int64_t i0 = wlo; i0 < wend; i0 += 64 * kAhead) {
    int gs[kAhead];
    if (i0 == wlo) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) gs[u] = first[u];
    } else {
      groups_of(a, i0 + lane, wend, 64, gs);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t i = i0 + 64 * u;
      if (i >= wend) break;
      const int g = gs[u];
      uint64_t same = __ballot(g >= 0);
      for (int b = 0; b < bits; ++b) {
        const bool bit = (g >> b) & 1;
        const uint64_t with = __ballot(bit);
        same &= bit ? with : ~with;
      }
      int row = -1;
      if (g >= 0) row = next[g] + __popcll(same & ((1ull << lane) - 1));
      if (i + lane < wend) a.slots[i + lane] = row;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (g >= 0 && __builtin_ctzll(same) == lane) next[g] = row + __popcll(same);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  }
}

// ------------------------------------------------------------------------------------ the rows

struct CopyArgs {
  const uint8_t* x;
  int64_t bytes, x_stride, T;   // bytes of a row
  int k;
  const int* slots;
  const int64_t* group_offs;
  int G;
  uint8_t* rows;
  int64_t rows_stride, M;
};

template <int kBytes> struct Word;
template <> struct Word<16> { typedef v4u type; };
template <> struct Word<4> { typedef uint32_t type; };
template <> struct Word<2> { typedef uint16_t type; };
template <> struct Word<1> { typedef uint8_t type; };

// Rows from the end of the last group to M become zero, dealt to the grid's waves.
template <typename W>
__device__ __forceinline__ void clear_rows(uint8_t* rows, int64_t stride, int64_t bytes, const int64_t* group_offs,
                                           int G, int64_t M, int64_t wave, int64_t waves, int lane) {
  int64_t r = group_offs[G];
  r = (r < 0 ? 0 : r) + wave;
  for (; r < M; r += waves)
    for (int64_t c = lane * (int64_t)sizeof(W); c < bytes; c += 64 * sizeof(W)) *(W*)(rows + r * stride + c) = W{};
}

// What is written once and next read by another launch: past the caches where rows are whole lines (131072 fp8 rows of 2880 in
// 2944 from 32768 tokens 125 -> 106 us); else through them, which put together the lines that two stores share (30018 bf16
// rows of 1424: 19.2 us, 21.8 past them).
template <bool kLines, typename W>
__device__ __forceinline__ void store_once(W w, W* p) {
  if constexpr (kLines) __builtin_nontemporal_store(w, p);
  else *p = w;
}

// A wave per token: kUnroll words of the row in each lane, stored k times. Bound by its writes: 131072 fp8 rows of 2880
// from 32768 tokens 73 us, 6.5 TB/s with x in the memory-side cache.
// kLines: rows start on 128-byte lines.
template <int kBytes, bool kLines>
__global__ __launch_bounds__(kThreads) void dispatch_kernel(CopyArgs a) {
  using W = typename Word<kBytes>::type;
  constexpr int kUnroll = 4;
  const int lane = threadIdx.x & 63;
  const int64_t wave = (int64_t)blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t waves = (int64_t)gridDim.x * kWaves;
  for (int64_t t = wave; t < a.T; t += waves) {
    const uint8_t* src = a.x + t * a.x_stride;
    const int* slots = a.slots + t * a.k;
    for (int64_t c0 = lane * kBytes; c0 < a.bytes; c0 += 64 * kBytes * kUnroll) {
      W v[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (c0 + 64 * kBytes * u < a.bytes) v[u] = *(const W*)(src + c0 + 64 * kBytes * u);
      for (int j = 0; j < a.k; ++j) {
        const int s = slots[j];
        if (s < 0 || s >= a.M) continue;
        uint8_t* dst = a.rows + s * a.rows_stride;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
          if (c0 + 64 * kBytes * u < a.bytes) store_once<kLines>(v[u], (W*)(dst + c0 + 64 * kBytes * u));
      }
    }
  }
  clear_rows<W>(a.rows, a.rows_stride, a.bytes, a.group_offs, a.G, a.M, wave, waves, lane);
}

// Two values rounded to bf16 (nearest even), the first in the low half.
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
  typedef float v2f __attribute__((ext_vector_type(2)));
  typedef __bf16 v2b __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{a, b}, v2b));
}

// N elements of a row in fp32.
template <typename T, int N>
struct Vec {
  float f[N];
  typedef typename Word<N * sizeof(T)>::type Raw;
  __device__ __forceinline__ void set(Raw w) {
    if constexpr (N == 1) {
      f[0] = __uint_as_float(sizeof(T) == 2 ? (uint32_t)w << 16 : (uint32_t)w);
    } else {
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f[2 * i] = __uint_as_float(w[i] << 16);
          f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
      }
    }
  }
  template <bool kLines>
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (N == 1) {
      if constexpr (sizeof(T) == 2) *(uint16_t*)p = __builtin_bit_cast(uint16_t, (__bf16)f[0]);
      else *(float*)p = f[0];
    } else {
      v4u w;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if constexpr (sizeof(T) == 2) w[i] = bf16_pair(f[2 * i], f[2 * i + 1]);
        else w[i] = __float_as_uint(f[i]);
      store_once<kLines>(w, (v4u*)p);
    }
  }
};

// A row that may be there or not, as a buffer: loads from none give zeros, so that the loads of several rows are issued
// without a branch between them. Non-temporal: a row is read by one wave.
struct Row {
  __amdgpu_buffer_rsrc_t r;
  __device__ __forceinline__ Row(const void* p, int bytes)
      : r(__builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00020000)) {}
  // kBytes = 16, 4 or 2 at byte `at` of the row
  template <int kBytes>
  __device__ __forceinline__ typename Word<kBytes>::type load(int at) const {
    if constexpr (kBytes == 16) return __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 2));
    if constexpr (kBytes == 4) return __builtin_amdgcn_raw_buffer_load_b32(r, at, 0, 2);
    if constexpr (kBytes == 2) return __builtin_amdgcn_raw_buffer_load_b16(r, at, 0, 2);
  }
};

struct CombineArgs {
  const void* y;
  int64_t y_stride, M;
  const int* slots;
  int64_t T;
  int k;
  const float* weights;
  const void* residual;
  int64_t residual_stride;
  int H;
  void* out;
  int64_t out_stride;
  int parts;               // waves that share a token's columns
};

// A wave per token and part of its columns, N elements of the row per lane and step; the rows of four choices are loaded
// before the first is added. Non-temporal loads and stores: each byte passes once (131072 bf16 rows of 2880 into 32768
// tokens with a residual: 235 us with ordinary ones, 223 with ordinary loads, 217; with buffer loads, which need no
// branches, 209, 5.4 TB/s).
template <typename T, int N, bool kLines>
__global__ __launch_bounds__(kThreads) void combine_kernel(CombineArgs a) {
  constexpr int kJ = 4;
  const int lane = threadIdx.x & 63;
  const int64_t wave = (int64_t)blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t waves = (int64_t)gridDim.x * kWaves;
  using V = Vec<T, N>;
  constexpr int kBytes = N * sizeof(T);
  const int bytes = a.H * (int)sizeof(T);
  for (int64_t u = wave; u < a.T * a.parts; u += waves) {
    const int64_t t = a.parts == 1 ? u : u / a.parts;
    const int part = (int)(u - t * a.parts);
    const int* slots = a.slots + t * a.k;
    const Row res(a.residual ? (const T*)a.residual + t * a.residual_stride : (const T*)a.y, a.residual ? bytes : 0);
    for (int c = (64 * part + lane) * N; c < a.H; c += 64 * N * a.parts) {
      const typename V::Raw first = res.load<kBytes>(c * (int)sizeof(T));
      float acc[N];
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] = 0.f;
      for (int j0 = 0; j0 < a.k; j0 += kJ) {
        typename V::Raw raw[kJ];
        float w[kJ];
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
          const int s = j0 + j < a.k ? slots[j0 + j] : -1;
          const bool use = s >= 0 && s < a.M;
          w[j] = !use ? 0.f : a.weights ? a.weights[t * a.k + j0 + j] : 1.f;
          raw[j] = Row((const T*)a.y + (use ? s : 0) * a.y_stride, use ? bytes : 0).load<kBytes>(c * (int)sizeof(T));
        }
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
          V v;
          v.set(raw[j]);
#pragma unroll
          for (int i = 0; i < N; ++i) acc[i] = fmaf(w[j], v.f[i], acc[i]);
        }
      }
      V r;
      r.set(first);
#pragma unroll
      for (int i = 0; i < N; ++i) r.f[i] += acc[i];
      r.template store<kLines>((T*)a.out + t * a.out_stride + c);
    }
  }
}

struct CombineBackArgs {
  const void* dout;
  int64_t dout_stride;
  const void* y;
  int64_t y_stride, M;
  const int* slots;
  int64_t T;
  int k;
  const float* weights;
  const int64_t* group_offs;
  int G, H;
  void* dy;
  int64_t dy_stride;
  float* dweights;
};

// A wave per token, eight choices at a time: their rows are loaded before the first is used, the token's gradient once
// for all eight. Bound by memory: 30018 bf16 rows of 1424 from 5003 tokens 43 us, 4.3 TB/s, rows that start inside lines.
template <typename T, int N, bool kLines>
__global__ __launch_bounds__(kThreads) void combine_backward_kernel(CombineBackArgs a) {
  constexpr int kJ = 8;
  const int lane = threadIdx.x & 63;
  const int64_t wave = (int64_t)blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t waves = (int64_t)gridDim.x * kWaves;
  using V = Vec<T, N>;
  constexpr int kBytes = N * sizeof(T);
  const int bytes = a.H * (int)sizeof(T);
  for (int64_t t = wave; t < a.T; t += waves) {
    const Row dout((const T*)a.dout + t * a.dout_stride, bytes);
    for (int j0 = 0; j0 < a.k; j0 += kJ) {
      int slot[kJ];
      float w[kJ], dot[kJ];
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        const int s = j0 + j < a.k ? a.slots[t * a.k + j0 + j] : -1;
        slot[j] = s < a.M ? s : -1;
        w[j] = a.weights && j0 + j < a.k ? a.weights[t * a.k + j0 + j] : 1.f;
        dot[j] = 0.f;
      }
      for (int c = lane * N; c < a.H; c += 64 * N) {
        const typename V::Raw rd = dout.load<kBytes>(c * (int)sizeof(T));
        typename V::Raw ry[kJ];
#pragma unroll
        for (int j = 0; j < kJ; ++j)
          ry[j] = (slot[j] >= 0 && a.dweights ? Row((const T*)a.y + slot[j] * a.y_stride, bytes) : Row(a.dout, 0))
                      .load<kBytes>(c * (int)sizeof(T));
        V d;
        d.set(rd);
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
          V y;
          y.set(ry[j]);
#pragma unroll
          for (int i = 0; i < N; ++i) dot[j] = fmaf(d.f[i], y.f[i], dot[j]);
          if (a.dy && slot[j] >= 0) {
            V g;
#pragma unroll
            for (int i = 0; i < N; ++i) g.f[i] = w[j] * d.f[i];
            g.template store<kLines>((T*)a.dy + slot[j] * a.dy_stride + c);
          }
        }
      }
      if (a.dweights) {
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
          if (j0 + j >= a.k) continue;
#pragma unroll
          for (int d = 32; d > 0; d >>= 1) dot[j] += __shfl_xor(dot[j], d, 64);
          if (lane == 0) a.dweights[t * a.k + j0 + j] = slot[j] >= 0 ? dot[j] : 0.f;
        }
      }
    }
  }
  if (a.dy) {
    if constexpr (N > 1)
      clear_rows<v4u>((uint8_t*)a.dy, a.dy_stride * sizeof(T), (int64_t)a.H * sizeof(T), a.group_offs, a.G, a.M, wave,
                      waves, lane);
    else
      clear_rows<T>((uint8_t*)a.dy, a.dy_stride * sizeof(T), (int64_t)a.H * sizeof(T), a.group_offs, a.G, a.M, wave,
                    waves, lane);
  }
}

}  // namespace ex
}  // namespace ggemm
