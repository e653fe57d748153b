// Routing of tokens to experts for gfx950: the top-k experts of each token from its router logits, their
// weights, and the logits' gradient.
//
//   p = softmax(l) or sigmoid(l);  key = l, p or p + bias;  experts = top-k by key, first index first;
//   w_j = scale * p_j  or  scale * p_j / sum_i p_i over the taken experts.
//
// Reads T E logits and writes T k pairs: bound by latency below some thousand tokens, by instruction
// issue above (32 experts, 4 taken: 298 vector instructions a wave for
// eight tokens, 0.73 of the SIMDs' cycles while the CUs run). One token of 32 experts takes
// 3.2 us, 131072 tokens with bf16 logits and 4 taken 12.6 (1.0 TB/s of logits and pairs); 16384 of 256 with fp32
// logits, a bias, 8 groups and 8 taken 21.4, the gradient 10.8.
//
// L lanes hold a token's experts, V consecutive ones each, in registers; 64 / L tokens per wave. A round
// of the top-k takes the largest key over the lanes (a DPP max of one 32-bit word per step: keys are the
// floats' bits mapped to unsigned order), the lowest lane that holds it and in that lane the first
// expert, which is then struck out. Equal keys are thus taken by the lower index.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ggemm {
namespace rt {

constexpr int kThreads = 256;
constexpr int kMaxExperts = 1024, kMaxTopK = 64;
constexpr uint32_t kDead = 0x007fffffu;   // key of -inf: at or below it an expert is never taken

struct Args {
  const void* logits;
  int64_t T, stride;
  int E, k, score;                // score: 0 softmax, 1 sigmoid
  const float* bias;
  int groups, top_groups, group_best;
  int renorm;
  float scale;
  float* weights;
  int* experts;
  bool vec;                       // a lane's logits are one aligned load
};

struct BackArgs {
  const float* dweights;
  const void* logits;
  int64_t T, stride;
  int E, k, score, renorm;
  float scale;
  const int* experts;
  void* dlogits;
  bool vec, vec_out;              // a lane's logits, and its part of dlogits, are one aligned access
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
__device__ __forceinline__ void from_f32(float f, float* p) { *p = f; }
__device__ __forceinline__ void from_f32(float f, uint16_t* p) {
  *p = __builtin_bit_cast(uint16_t, (__bf16)f);
}

// Floats as unsigned integers of the same order: -inf is kDead, zeros are equal, NaN is the largest.
__device__ __forceinline__ uint32_t key_of(float f) {
  const uint32_t u = __float_as_uint(f + 0.0f);   // -0 becomes +0
  const uint32_t k = u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
  return (u & 0x7fffffffu) > 0x7f800000u ? 0xffffffffu : k;
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}

// x of lane ^ 1, ^ 2, mirrored in 8, mirrored in 16, ^ 16, ^ 32: six steps combine a wave, the first
// log2(L) of them groups of L lanes, with the same result in every lane of a group.
template <int kStep>
__device__ __forceinline__ uint32_t partner(uint32_t x) {
  if constexpr (kStep == 0) return __builtin_amdgcn_mov_dpp((int)x, 0xB1, 0xf, 0xf, true);
  if constexpr (kStep == 1) return __builtin_amdgcn_mov_dpp((int)x, 0x4E, 0xf, 0xf, true);
  if constexpr (kStep == 2) return __builtin_amdgcn_mov_dpp((int)x, 0x141, 0xf, 0xf, true);
  if constexpr (kStep == 3) return __builtin_amdgcn_mov_dpp((int)x, 0x140, 0xf, 0xf, true);
  if constexpr (kStep == 4) return __shfl_xor((int)x, 16, 64);
  return __shfl_xor((int)x, 32, 64);
}
template <int L, int kStep = 0, typename F>
__device__ __forceinline__ uint32_t reduce(uint32_t x, F f) {
  if constexpr ((1 << kStep) < L) return reduce<L, kStep + 1>(f(x, partner<kStep>(x)), f);
  return x;
}
template <int L>
__device__ __forceinline__ uint32_t max_u32(uint32_t x) {
  return reduce<L>(x, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
template <int L>
__device__ __forceinline__ float max_f32(float x) {
  return __uint_as_float(reduce<L>(__float_as_uint(x), [](uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}
template <int L>
__device__ __forceinline__ float sum_f32(float x) {
  return __uint_as_float(reduce<L>(__float_as_uint(x), [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}

// The two largest keys of groups of `lanes` lanes (a power of two), in each of their lanes.
template <int L, int kStep = 0>
__device__ __forceinline__ void merge_best(uint32_t& b0, uint32_t& b1, int lanes) {
  if constexpr ((1 << kStep) < L) {
    if ((1 << kStep) >= lanes) return;               // the same for the whole launch
    const uint32_t o0 = partner<kStep>(b0), o1 = partner<kStep>(b1);
    b1 = max(max(b1, o1), min(b0, o0));
    b0 = max(b0, o0);
    merge_best<L, kStep + 1>(b0, b1, lanes);
  }
}

// Logits of the lane's V experts e0 .. e0 + V - 1 (-inf past E). vec: E is a multiple of V and every row starts on a
// multiple of V elements, so a lane's logits are one load.
template <typename T, int V>
__device__ __forceinline__ void load_logits(const T* row, int e0, int E, bool vec, float (&x)[V]) {
  if (V > 1 && vec) {
    struct alignas(V * sizeof(T) < 16 ? V * sizeof(T) : 16) Pack {
      T v[V];
    };
    if (e0 < E) {
      const Pack p = *(const Pack*)(row + e0);
#pragma unroll
      for (int v = 0; v < V; ++v) x[v] = to_f32(p.v[v]);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) x[v] = -INFINITY;
    }
    return;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) x[v] = e0 + v < E ? to_f32(row[e0 + v]) : -INFINITY;
}

// Orders this wave's LDS accesses for the compiler (the hardware runs them in order): what the lanes of a token
// hand each other never leaves their wave.
__device__ __forceinline__ void lds_order() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// max and sum of exp(l - max) over a token's logits; the max of a token with every expert masked as 0.
template <int L, int V>
__device__ __forceinline__ void softmax_stats(const float (&x)[V], float* m, float* sum) {
  float mx = x[0];
#pragma unroll
  for (int v = 1; v < V; ++v) mx = fmaxf(mx, x[v]);
  mx = max_f32<L>(mx);
  if (mx == -INFINITY) mx = 0.f;
  float s = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v) s += expf(x[v] - mx);   // NaN and +inf make the sum NaN
  *m = mx;
  *sum = sum_f32<L>(s);
}

__device__ __forceinline__ float sigmoid(float x) { return 1.f / (1.f + expf(-x)); }

// Bytes of dynamic LDS: the taken experts and their values for each token; with groups the keys, the
// groups' values and whether they stay.
inline int route_lds(int L, int E, int k, int groups) {
  return kThreads / L * (8 * k + (groups > 1 ? 4 * (E + 2 * groups) : 0));
}

template <typename T, int L, int V>
__global__ __launch_bounds__(kThreads) void route_kernel(Args a) {
  extern __shared__ uint32_t s_rt[];
  constexpr int kTokens = kThreads / L;
  const int tid = threadIdx.x, l = tid % L, tok = tid / L;
  const int64_t t = (int64_t)blockIdx.x * kTokens + tok;
  const bool real = t < a.T;
  int* s_idx = (int*)s_rt + tok * a.k;
  float* s_val = (float*)s_rt + kTokens * a.k + tok * a.k;

  float x[V];
  load_logits<T, V>((const T*)a.logits + (real ? t : 0) * a.stride, l * V, a.E, a.vec, x);
  // p[v]: the score where keys or weights need it, else the logit
  const bool by_logit = a.bias == nullptr && a.groups <= 1;
  const bool scored = a.score == 1 || !a.renorm || !by_logit;
  float m = 0.f, sum = 1.f;
  if (a.score == 0 && scored) softmax_stats<L, V>(x, &m, &sum);
  uint32_t key[V];
  float val[V];   // what the weights are made of: the score, or the logit where they are a softmax of the taken
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = l * V + v;
    const float p = !scored ? x[v] : a.score == 1 ? sigmoid(x[v]) : expf(x[v] - m) / sum;
    val[v] = a.score == 0 && a.renorm ? x[v] : p;
    const float f = by_logit ? x[v] : a.bias ? p + (e < a.E ? a.bias[e] : 0.f) : p;
    key[v] = e >= a.E ? 0u : x[v] == -INFINITY ? kDead : key_of(f);
  }

  const int lane = tid & 63, seg = lane / L * L;
  if (a.groups > 1) {
    const int gs = a.E / a.groups, lg = gs / V;
    if (gs % V == 0 && (lg & (lg - 1)) == 0) {
      // a group is the V experts each of lg = 1, 2, 4 .. lanes: their two largest keys merged over those lanes,
      // then every group's value read from its first lane
      uint32_t b0 = 0, b1 = 0;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        b1 = max(b1, min(b0, key[v]));
        b0 = max(b0, key[v]);
      }
      merge_best<L>(b0, b1, lg);
      const uint32_t mine = a.group_best == 2 ? key_of(value_of(b0) + value_of(b1)) : b0;
      const int group = l / lg;
      int before = 0;
      for (int h = 0; h < a.groups; ++h) {
        const uint32_t other = L == 64 ? (uint32_t)__builtin_amdgcn_readlane((int)mine, h * lg)
                                       : (uint32_t)__shfl((int)mine, seg + h * lg, 64);
        before += other > mine || (other == mine && h < group);
      }
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (key[v] != 0 && before >= a.top_groups) key[v] = kDead;
    } else {
      uint32_t* s_key = s_rt + 2 * kTokens * a.k + tok * a.E;
      uint32_t* s_grp = s_rt + kTokens * (2 * a.k + a.E) + tok * a.groups;
      uint32_t* s_keep = s_rt + kTokens * (2 * a.k + a.E + a.groups) + tok * a.groups;
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (l * V + v < a.E) s_key[l * V + v] = key[v];
      lds_order();
      for (int g = l; g < a.groups; g += L) {
        uint32_t b0 = 0, b1 = 0;
        for (int i = 0; i < gs; ++i) {
          const uint32_t k = s_key[g * gs + i];
          b1 = max(b1, min(b0, k));
          b0 = max(b0, k);
        }
        s_grp[g] = a.group_best == 2 ? key_of(value_of(b0) + value_of(b1)) : b0;
      }
      lds_order();
      for (int g = l; g < a.groups; g += L) {
        const uint32_t mine = s_grp[g];
        int before = 0;
        for (int h = 0; h < a.groups; ++h) before += s_grp[h] > mine || (s_grp[h] == mine && h < g);
        s_keep[g] = before < a.top_groups;
      }
      lds_order();
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int e = l * V + v;
        if (e < a.E && !s_keep[e / gs]) key[v] = kDead;
      }
    }
  }

  for (int j = 0; j < a.k; ++j) {
    uint32_t best = key[0];
#pragma unroll
    for (int v = 1; v < V; ++v) best = max(best, key[v]);
    const uint32_t top = max_u32<L>(best);
    const uint64_t holds = __ballot(best == top) >> seg;
    const int owner = __builtin_ctzll(holds);        // this token's lanes are the low L bits
    if (top <= kDead) {
      if (l == 0) s_idx[j] = -1, s_val[j] = 0.f;
    } else if (l == owner) {
      bool found = false;
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (!found && key[v] == top) {
          found = true;
          s_idx[j] = l * V + v;
          s_val[j] = val[v];
          key[v] = 0;
        }
    }
  }
  lds_order();
  // weights: lane l takes places l, l + L, .. of the token; max and sum over the lanes
  const bool over_taken = a.score == 0 && a.renorm;
  float base = 0.f, total = 1.f;
  if (over_taken) {
    base = -INFINITY;
    for (int j = l; j < a.k; j += L) base = s_idx[j] >= 0 ? fmaxf(base, s_val[j]) : base;
    base = max_f32<L>(base);
  }
  if (a.renorm) {
    total = 0.f;
    for (int j = l; j < a.k; j += L) {
      if (over_taken) s_val[j] = s_idx[j] >= 0 ? expf(s_val[j] - base) : 0.f;
      total += s_val[j];
    }
    total = sum_f32<L>(total);
    if (!over_taken && total < 1e-20f) total = 1e-20f;
  }
  if (!real) return;
  for (int j = l; j < a.k; j += L) {
    const int e = s_idx[j];
    a.weights[t * a.k + j] = e >= 0 ? s_val[j] / total * a.scale : 0.f;
    a.experts[t * a.k + j] = e;
  }
}

// dlogits, one token to L lanes again. Per taken expert d = scale * dweight; with renormalised weights
// d -= sum_i d_i q_i (q = weight / scale), and sigmoid divides by the sum of scores. Then
//   softmax of the taken: d q;  softmax of all: d p [taken] - p sum_i d_i p_i;  sigmoid: d p (1 - p).
// Of the row k values are not zero but for a softmax of all: the taken experts' terms are put into a row of LDS, which the
// lanes write whole. Only a softmax of all reads the other experts' logits. Bound by instruction issue: 16384
// tokens of 256 experts in fp32, eight taken, a token to a wave, are 255 vector instructions a wave, 0.86 of the SIMDs'
// cycles while the CUs run: 10.8 us, 17 MB written at 1.6 TB/s.
inline int route_back_lds(int L, int E, int k) { return kThreads / L * 4 * (E + 3 * k); }

template <typename T, int L, int V>
__global__ __launch_bounds__(kThreads) void route_backward_kernel(BackArgs a) {
  extern __shared__ uint32_t s_rt[];
  constexpr int kTokens = kThreads / L;
  const int tid = threadIdx.x, l = tid % L, tok = tid / L;
  const int64_t t = (int64_t)blockIdx.x * kTokens + tok;
  const bool real = t < a.T;
  float* s_row = (float*)s_rt + tok * a.E;
  int* s_idx = (int*)s_rt + kTokens * a.E + tok * a.k;
  float* s_val = (float*)s_rt + kTokens * (a.E + a.k) + tok * a.k;
  float* s_d = (float*)s_rt + kTokens * (a.E + 2 * a.k) + tok * a.k;
  const T* row = (const T*)a.logits + (real ? t : 0) * a.stride;
  const bool over_all = a.score == 0 && !a.renorm;

  float x[V], m = 0.f, sum = 1.f;
  if (over_all) {
    load_logits<T, V>(row, l * V, a.E, a.vec, x);
    softmax_stats<L, V>(x, &m, &sum);
  }
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (l * V + v < a.E) s_row[l * V + v] = 0.f;
  float base = -INFINITY;
  for (int j = l; j < a.k; j += L) {
    int e = real ? a.experts[t * a.k + j] : -1;
    e = e >= 0 && e < a.E ? e : -1;
    const float lj = e >= 0 ? to_f32(row[e]) : -INFINITY;
    s_idx[j] = e;
    s_val[j] = lj;
    s_d[j] = e >= 0 ? a.dweights[t * a.k + j] * a.scale : 0.f;
    base = fmaxf(base, lj);
  }
  lds_order();
  base = max_f32<L>(base);
  // s_val becomes the score, or with a softmax of the taken its numerator
  float total = 0.f, dot = 0.f;
  for (int j = l; j < a.k; j += L) {
    const float p = s_idx[j] < 0      ? 0.f
                    : a.score == 1    ? sigmoid(s_val[j])
                    : over_all        ? expf(s_val[j] - m) / sum
                                      : expf(s_val[j] - base);
    s_val[j] = p;
    total += p;
    dot += s_d[j] * p;
  }
  total = sum_f32<L>(total);
  dot = sum_f32<L>(dot);
  if (a.renorm) {
    const bool small = a.score == 1 && total < 1e-20f;   // the sum's floor: the weights are p / 1e-20
    total = small ? 1e-20f : total;
    dot = small ? 0.f : dot / total;
  }
  for (int j = l; j < a.k; j += L) {
    const int e = s_idx[j];
    if (e < 0) continue;
    const float p = s_val[j], d = s_d[j];
    s_row[e] = over_all      ? d * p
               : a.score == 0 ? (d - dot) * (p / total)
                              : (a.renorm ? (d - dot) / total : d) * p * sigmoid(-to_f32(row[e]));
  }
  lds_order();
  if (!real) return;
  float g[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = l * V + v;
    g[v] = e < a.E ? s_row[e] : 0.f;
    if (over_all) g[v] = e < a.E && x[v] == -INFINITY ? 0.f : g[v] - dot * (expf(x[v] - m) / sum);
  }
  T* out = (T*)a.dlogits + t * a.E + l * V;
  if (V > 1 && a.vec_out) {
    struct alignas(V * sizeof(T) < 16 ? V * sizeof(T) : 16) Pack {
      T v[V];
    } p;
#pragma unroll
    for (int v = 0; v < V; ++v) from_f32(g[v], &p.v[v]);
    if (l * V < a.E) *(Pack*)out = p;
    return;
  }
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (l * V + v < a.E) from_f32(g[v], out + v);
}

}  // namespace rt
}  // namespace ggemm
