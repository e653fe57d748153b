// Microscaled (MX) rows for gfx950: blocks of 32 values along a row share a power of two 2^X, the values are e2m1
// (4 bits) or e4m3 (8 bits).
//
//   amax = max |x| over a block = m 2^e (1 <= m < 2);  X = e - emax, one more from m = `kUp` on;  q = rne(x 2^-X)
//
// emax is the exponent of the format's largest value (6 = 1.5 2^2, 448 = 1.75 2^8) and kUp half a step above its
// mantissa: from there on the largest value would round past the format, so nothing saturates by more than half a
// step, what any other value is rounded by. A power of two is taken off without a rounding, so a value is rounded once.
//
// Bound by HBM: x is read once. A thread holds eight values, four lanes a block: the block's maximum is two DPP
// steps, the conversion one instruction for two values (v_cvt_scalef32_pk, which divides by the power itself). Weights of
// 32 x 5760 x 2880 bf16 to e2m1 and back: 215 and 216 us, 6.2 TB/s each way.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ggemm {
namespace mxq {

constexpr int kThreads = 256, kUnroll = 4;      // units of eight values that a thread has in flight

typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef short v2s __attribute__((ext_vector_type(2)));
typedef unsigned short v2us __attribute__((ext_vector_type(2)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));

// n / d for n < 2^31 and d >= 2, by a multiplication.
struct Divisor {
  uint32_t mul, shift, d;
  static Divisor of(uint32_t d) {
    uint32_t l = 1;
    while ((uint64_t(1) << l) < d) ++l;
    return {(uint32_t)((uint64_t(1) << (31 + l)) / d + 1), l - 1, d};
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return __umulhi(n, mul) >> shift; }
};

// The scale byte of a block from its largest |x|, given as fp32 bits.
template <bool kE4M3>
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax) {
  constexpr uint32_t kCarry = kE4M3 ? 0x180000u : 0x200000u;   // 2 - 1.8125, 2 - 1.75: m from kUp on carries into e
  const int e = (int)((amax + kCarry) >> 23) - (kE4M3 ? 8 : 2);
  return amax >= 0x7f800000u ? 255u : amax == 0u ? 127u : (uint32_t)max(e, 0);
}

__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true));   // lane ^ 1
  return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true));   // lane ^ 2
}

struct Args {
  const void* x;
  int64_t rows, stride;
  int cols;
  Divisor per;                     // units of a row: four to a block
  uint8_t* q;
  int64_t q_stride;
  uint8_t* scales;
  int64_t scale_row, scale_block;
};

template <bool kF32, bool kE4M3>
__global__ __launch_bounds__(kThreads) void quantize_kernel(Args a) {
  constexpr int kW = kF32 ? 2 : 1;
  v4u w[kUnroll][kW];
  uint32_t row[kUnroll], c[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint32_t n = (blockIdx.x * kUnroll + u) * kThreads + threadIdx.x;
    row[u] = a.per(n);
    c[u] = n - row[u] * a.per.d;
    const bool live = row[u] < a.rows && 8 * c[u] < (uint32_t)a.cols;
#pragma unroll
    for (int k = 0; k < kW; ++k) w[u][k] = v4u{0, 0, 0, 0};
    if (live) {
      const v4u* p = (const v4u*)((const uint8_t*)a.x + ((int64_t)row[u] * a.stride + 8 * c[u]) * (kF32 ? 4 : 2));
#pragma unroll
      for (int k = 0; k < kW; ++k) w[u][k] = __builtin_nontemporal_load(p + k);
    }
    row[u] = live ? row[u] : ~0u;
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    uint32_t m;
    if constexpr (kF32) {
      m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, w[u][i / 4][i % 4] & 0x7fffffffu);
    } else {
      // pairs of 16-bit patterns order like the values
      v2us p = __builtin_bit_cast(v2us, w[u][0][0] & 0x7fff7fffu);
#pragma unroll
      for (int i = 1; i < 4; ++i) p = __builtin_elementwise_max(p, __builtin_bit_cast(v2us, w[u][0][i] & 0x7fff7fffu));
      m = (uint32_t)max(p[0], p[1]) << 16;
    }
    const uint32_t byte = scale_byte<kE4M3>(quad_max(m));
    const float scale = __uint_as_float(byte << 23);           // the conversions take 2^X as its exponent field
    if (row[u] == ~0u) continue;
    if ((c[u] & 3u) == 0u) a.scales[(int64_t)row[u] * a.scale_row + (int64_t)(c[u] / 4) * a.scale_block] = (uint8_t)byte;
    uint8_t* q = a.q + (int64_t)row[u] * a.q_stride + (kE4M3 ? 8 : 4) * c[u];
    auto pair = [&](int i) {
      const uint32_t both = w[u][0][i];                        // a cast of the element itself takes the first one
      return __builtin_bit_cast(v2b, both);
    };
    auto at = [&](int i) { return __uint_as_float(w[u][i / 4][i % 4]); };
    if constexpr (kE4M3) {
      v2s lo{}, hi{};
      if constexpr (kF32) {
        lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, at(0), at(1), scale, false);
        lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, at(2), at(3), scale, true);
        hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, at(4), at(5), scale, false);
        hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, at(6), at(7), scale, true);
      } else {
        lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(lo, pair(0), scale, false);
        lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(lo, pair(1), scale, true);
        hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(hi, pair(2), scale, false);
        hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(hi, pair(3), scale, true);
      }
      v2u v{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
      if (byte == 255u) v = v2u{0, 0};
      __builtin_nontemporal_store(v, (v2u*)q);
    } else {
      uint32_t v = 0;
      if constexpr (kF32) {
        v = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(v, at(0), at(1), scale, 0);
        v = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(v, at(2), at(3), scale, 1);
        v = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(v, at(4), at(5), scale, 2);
        v = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(v, at(6), at(7), scale, 3);
      } else {
        v = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(v, pair(0), scale, 0);
        v = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(v, pair(1), scale, 1);
        v = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(v, pair(2), scale, 2);
        v = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(v, pair(3), scale, 3);
      }
      __builtin_nontemporal_store(byte == 255u ? 0u : v, (uint32_t*)q);
    }
  }
}

// Eight values of a unit times their scale, as four words of bf16 pairs or eight fp32.
template <bool kE4M3>
__device__ __forceinline__ v4u restore_bf16(v2u q, float scale) {
  v4u r;
  if constexpr (kE4M3) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      r[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[i], scale, false));
      r[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[i], scale, true));
    }
  } else {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q[0], scale, 0));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q[0], scale, 1));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q[0], scale, 2));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q[0], scale, 3));
  }
  return r;
}

template <bool kE4M3>
__device__ __forceinline__ void restore_f32(v2u q, float scale, float (&x)[8]) {
  v2f p[4];
  if constexpr (kE4M3) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      p[2 * i] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(q[i], scale, false);
      p[2 * i + 1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(q[i], scale, true);
    }
  } else {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[0], scale, 0);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[0], scale, 1);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[0], scale, 2);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[0], scale, 3);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = p[i / 2][i % 2];
}

// Args as above: x is written, q and scales read.
template <bool kF32, bool kE4M3>
__global__ __launch_bounds__(kThreads) void dequantize_kernel(Args a) {
  v2u q[kUnroll];
  uint32_t row[kUnroll], c[kUnroll], byte[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint32_t n = (blockIdx.x * kUnroll + u) * kThreads + threadIdx.x;
    row[u] = a.per(n);
    c[u] = n - row[u] * a.per.d;
    q[u] = v2u{0, 0};
    byte[u] = 0;
    if (row[u] < a.rows && 8 * c[u] < (uint32_t)a.cols) {
      const uint8_t* p = a.q + (int64_t)row[u] * a.q_stride + (kE4M3 ? 8 : 4) * c[u];
      if constexpr (kE4M3) q[u] = __builtin_nontemporal_load((const v2u*)p);
      else q[u][0] = __builtin_nontemporal_load((const uint32_t*)p);
      byte[u] = a.scales[(int64_t)row[u] * a.scale_row + (int64_t)(c[u] / 4) * a.scale_block];
    } else {
      row[u] = ~0u;
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    if (row[u] == ~0u) continue;
    const float scale = __uint_as_float(byte[u] << 23);
    v4u* p = (v4u*)((uint8_t*)a.x + ((int64_t)row[u] * a.stride + 8 * c[u]) * (kF32 ? 4 : 2));
    if constexpr (kF32) {
      float x[8];
      restore_f32<kE4M3>(q[u], scale, x);
#pragma unroll
      for (int k = 0; k < 2; ++k)
        __builtin_nontemporal_store(v4u{__float_as_uint(x[4 * k]), __float_as_uint(x[4 * k + 1]),
                                        __float_as_uint(x[4 * k + 2]), __float_as_uint(x[4 * k + 3])}, p + k);
    } else {
      __builtin_nontemporal_store(restore_bf16<kE4M3>(q[u], scale), p);
    }
  }
}

}  // namespace mxq
}  // namespace ggemm
