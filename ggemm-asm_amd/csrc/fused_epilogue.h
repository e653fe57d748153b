// Epilogue of the grouped FP8 products with bias, activation and residual:
//
//   z = alpha acc + bias[g];  out = act(z) + residual   (fp32, rounded once to bf16)
//
// for the kernels whose waves hold C as blocks of 16 x 16 from v_mfma_f32_16x16x128 (mid_gemm.h,
// persistent_kernel.h): lane 16 q + s holds row s, columns 4 q .. 4 q + 3 of a block, so the gate and the
// value of a swiglu pair (columns 2 i, 2 i + 1) are neighbours in one lane, and its output is half as
// wide as the product.
#pragma once

#include "vark_kernel.h"

namespace ggemm {
namespace epi {

constexpr int kNone = 0, kSilu = 1, kGelu = 2, kSwiglu = 3;

struct Args {
  uint16_t* pre;           // z in bf16, or null
  int stride_pre;
  const void* bias;        // [G, N] fp32 or bf16, or null
  int bias_f32;
  const uint16_t* residual;
  int stride_res;
  float slope, limit, shift;
  float nslope;            // -log2(e) slope: sigmoid(slope g) = 1 / (1 + 2^(nslope g))
};

// 1 / (1 + 2^x). The hardware's exp2 and reciprocal, each within an ulp; the rounding of x = -log2(e) y adds |y| 2^-24:
// against the 2^-8 of the bf16 results, and 2e-7 in the fp32 sums of the bias' gradient.
constexpr float kLog2e = 1.44269504088896f;
__device__ __forceinline__ float sigmoid2(float x) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x)); }
__device__ __forceinline__ float sigmoid(float x) { return sigmoid2(x * -kLog2e); }

// The normal distribution's cdf and e^(-x^2 / 2). With y = |x| / sqrt 2, erfc(y) e^(y^2) is smooth and falls like 1 / y: it
// is fitted as t P(t), t = 1 / (1 + 0.44 y), P of degree 7 with the least largest relative error over y = 0 .. 10.5, 1.8e-7
// (the coefficients hold the half of cdf(-|x|) = erfc(y) / 2). In fp32 the cdf of x < 0 is off by at most 5 units of 2^-23 of
// its own value and, by the exponent's rounding, x^2 / 2 more (7.4e-6 at -12.5); of x > 0 by 3.2e-7. An instruction more
// than an approximation that is bounded by 1.5e-7 of one, which is all error far below zero. Degree 9 (2.7e-9) took two
// more: 131072 x 5760 x 2880 with gelu and a residual 2.352 ms, 2.330 so, 2.331 with the former.
__device__ __forceinline__ float normal_cdf(float x, float* gauss) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.311126977f, fabsf(x), 1.f));
  float p = fmaf(t, 0.0356666967f, -0.139214039f);
  p = fmaf(t, p, 0.148778901f);
  p = fmaf(t, p, -0.0105133327f);
  p = fmaf(t, p, 0.108143263f);
  p = fmaf(t, p, 0.108580425f);
  p = fmaf(t, p, 0.124448597f);
  p = fmaf(t, p, 0.124109574f);
  *gauss = __builtin_amdgcn_exp2f(x * x * -0.721347520444482f);
  const float below = t * p * *gauss;
  return x > 0.f ? 1.f - below : below;
}
__device__ __forceinline__ float gelu_cdf(float x) {
  float gauss;
  return normal_cdf(x, &gauss);
}

// The same for sums that are kept in fp32: up to |x| = 1.25 the cdf as 1/2 + x Q(x^2), whose error is that of its last
// rounding (Q of degree 5 with the least largest error of x Q, 2.1e-9): 4e-8, 8e-8 past it.
__device__ __forceinline__ float normal_cdf_fp32(float x, float* gauss) {
  const float far = normal_cdf(x, gauss), h = x * x;
  float q = fmaf(h, -6.64485742e-06f, 0.000110327448f);
  q = fmaf(h, q, -0.00118270959f);
  q = fmaf(h, q, 0.00997150037f);
  q = fmaf(h, q, -0.0664899871f);
  q = fmaf(h, q, 0.398942262f);
  return h < 1.5625f ? fmaf(x, q, 0.5f) : far;
}

// NaN stays NaN in both.
__device__ __forceinline__ float at_most(float x, float m) { return __builtin_elementwise_minimum(x, m); }
__device__ __forceinline__ float within(float x, float m) {
  return __builtin_elementwise_maximum(__builtin_elementwise_minimum(x, m), -m);
}

__device__ __forceinline__ float swiglu(float g, float u, const Args& e) {
  g = at_most(g, e.limit);
  return g * sigmoid2(e.nslope * g) * (within(u, e.limit) + e.shift);
}

__device__ __forceinline__ float from_bf16(uint32_t low) { return __uint_as_float(low << 16); }

__device__ __forceinline__ v4f unpack4(const v2i& w) {
  return v4f{from_bf16(w[0]), __uint_as_float(w[0] & 0xffff0000u), from_bf16(w[1]), __uint_as_float(w[1] & 0xffff0000u)};
}

// The activations that are not gated.
template <int kAct>
__device__ __forceinline__ v4f activation(v4f z) {
  if constexpr (kAct == kSilu || kAct == kGelu) {
#pragma unroll
    for (int c = 0; c < 4; ++c) z[c] *= kAct == kSilu ? sigmoid(z[c]) : gelu_cdf(z[c]);
  }
  return z;
}

__device__ __forceinline__ v4f load_bias(const Args& e, int64_t i) {
  if (e.bias == nullptr) return v4f{0.f, 0.f, 0.f, 0.f};
  if (e.bias_f32) return *(const v4f*)((const float*)e.bias + i);
  return unpack4(*(const v2i*)((const uint16_t*)e.bias + i));
}

typedef float v2f __attribute__((ext_vector_type(2)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));

// Two values rounded to nearest even, one v_cvt_pk_bf16_f32.
__device__ __forceinline__ int pack(float a, float b) {
  return __builtin_bit_cast(int, __builtin_convertvector(v2f{a, b}, v2b));
}

// LDS that a wave stages 32 rows of NB blocks in, rows 16 bytes apart so that 16 of them start on different banks.
template <int NB>
constexpr int kRegion = 32 * (32 * NB + 16);

// 32 staged rows of kChunks 16-byte chunks to dst (row 0), the first `rows` of them; chunk c is stored where c < chunks.
template <int kChunks>
__device__ __forceinline__ void store_rows(const GG_LDS uint8_t* reg, uint16_t* dst, int64_t stride, int rows,
                                           int chunks, int lane) {
  constexpr int kPitch = 16 * kChunks + 16;
#pragma unroll
  for (int k = 0; k < (32 * kChunks + 63) / 64; ++k) {
    const int f = 64 * k + lane, r = f / kChunks, c = f - r * kChunks;
    if (r < rows && r < 32 && c < chunks) store_c16(dst + r * stride + 8 * c, *(const GG_LDS v4i*)(reg + r * kPitch + 16 * c));
  }
}

// A wave's block of 16 MB x 16 NB: rows row0 .. of the launch (the first `rows` of them exist), columns n0 .. of
// group g's product. reg: this wave's kRegion<NB> bytes of LDS.
template <int kAct, int MB, int NB>
__device__ __forceinline__ void store(const v4f (&acc)[MB][NB], float alpha, const Args& e, uint16_t* out,
                                      int stride_out, int g, int N, int64_t row0, int rows, int n0,
                                      GG_LDS uint8_t* reg, int lane) {
  static_assert(MB % 2 == 0, "two blocks of rows per pass");
  constexpr bool kGated = kAct == kSwiglu, kRoom = MB * NB <= 16;   // registers for a pass's residual beside acc
  const int q = lane >> 4, s = lane & 15;
  const int blocks = min(NB, (N - n0 + 15) / 16);      // N is a multiple of 16; none past it
  v4f bias[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j)
    bias[j] = j < blocks ? load_bias(e, (int64_t)g * N + n0 + 16 * j + 4 * q) : v4f{0.f, 0.f, 0.f, 0.f};
  constexpr int kOutChunks = kGated ? NB : 2 * NB;
  const int o0 = kGated ? n0 / 2 : n0;
#pragma unroll
  for (int p = 0; p < MB / 2; ++p) {
    const int64_t prow = row0 + 32 * p;
    const int prows = rows - 32 * p;
    if (prows <= 0) return;                            // uniform in the wave
    // the pass's residual, in flight while z is staged; by row blocks where it would take the last registers (the
    // 512-thread kernel, 131072 x 5760 x 2880 with gelu and a residual: 2.59 ms
    // with the whole pass, 2.50 so)
    v2i res[2][NB];
    auto load_residual = [&](int i) {
      if (e.residual == nullptr) return;
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        res[i][j] = v2i{0, 0};
        if (16 * i + s >= prows || j >= blocks) continue;
        const uint16_t* at = e.residual + (prow + 16 * i + s) * e.stride_res + o0 + (kGated ? 8 * j + 2 * q : 16 * j + 4 * q);
        if constexpr (kGated) res[i][j][0] = *(const int*)at;
        else res[i][j] = *(const v2i*)at;
      }
    };
    load_residual(0);
    if constexpr (kRoom) load_residual(1);
    if (e.pre != nullptr) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          const v4f z = acc[2 * p + i][j] * alpha + bias[j];
          *(GG_LDS v2i*)(reg + (16 * i + s) * (32 * NB + 16) + 32 * j + 8 * q) = v2i{pack(z[0], z[1]), pack(z[2], z[3])};
        }
      store_rows<2 * NB>(reg, e.pre + prow * e.stride_pre + n0, e.stride_pre, prows, 2 * blocks, lane);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 16 * i + s;
      if constexpr (!kRoom)
        if (i == 1) load_residual(1);
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const v4f z = acc[2 * p + i][j] * alpha + bias[j];
        GG_LDS uint8_t* at = reg + r * (16 * kOutChunks + 16);
        if constexpr (kGated) {
          float x = swiglu(z[0], z[1], e), y = swiglu(z[2], z[3], e);
          if (e.residual != nullptr) {
            const uint32_t w = res[i][j][0];
            x += from_bf16(w);
            y += __uint_as_float(w & 0xffff0000u);
          }
          *(GG_LDS int*)(at + 16 * j + 4 * q) = pack(x, y);
        } else {
          v4f x = activation<kAct>(z);
          if (e.residual != nullptr) x += unpack4(res[i][j]);
          *(GG_LDS v2i*)(at + 32 * j + 8 * q) = v2i{pack(x[0], x[1]), pack(x[2], x[3])};
        }
      }
    }
    store_rows<kOutChunks>(reg, out + prow * stride_out + o0, stride_out, prows, kGated ? blocks : 2 * blocks, lane);
  }
}

}  // namespace epi
}  // namespace ggemm
