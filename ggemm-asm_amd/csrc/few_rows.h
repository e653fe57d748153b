// Grouped FP8 product with an epilogue for few rows per group (decoding), gfx950, library only:
//
//   z[r, :] = s_a s_b A[r, :] @ B[g]^T + bias[g, :];  out = act(z) + residual     (fused_epilogue.h)
//
// Such a launch is bound by reading the weights once, so nothing but loads in flight counts: a workgroup
// takes 16 rows of one group and 16 NB columns, and its four waves share the K axis, wave w the 128-byte
// steps w, w + 4, ..: a row's consecutive lines are asked for at once, by different waves, and a wave of
// K = 2880 has its whole part, 12 KiB per 16 columns, in flight before its first MFMA. No LDS stages and no barrier before
// the end, where the waves' sums are added in their order through LDS. 4 rows of 4 experts, 5760 x 2880 (66 MB of
// weights), take 14.2 us, 4.7 TB/s; 16.8 on the 64-row tiles.
//
// v_mfma_f32_16x16x128 with 16 weight rows (columns of C) on the A side and 16 activation rows on the B
// side: lane 16 q + s feeds row s of either, bytes 16 q .. + 15 and 64 + 16 q .. + 15 of a step (any
// assignment of K to operand bytes that both sides share gives the sum), and ends with row s, columns
// 4 q .. 4 q + 3.
#pragma once

#include "fused_epilogue.h"
#include "mid_common.h"
#include "persistent_kernel.h"

namespace ggemm {
namespace few {

constexpr int kNT = 256, kWaves = 4;
constexpr int kBatch = 6;            // steps a wave has in flight: all of its share of up to 24

template <int NB>
struct Cfg {
  static constexpr int BM = 16, BN = 16 * NB;
  static constexpr int LdsBytes = kWaves * NB * 1024;
};

template <int kAct, int NB>
__device__ __forceinline__ void body(const nt::Args& a, GG_LDS uint8_t* lds, const epi::Args& e) {
  using C = Cfg<NB>;
  constexpr bool kGated = epi::act_of(kAct) == epi::kSwiglu;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n_tn = (a.N + C::BN - 1) / C::BN;

  // ---- this workgroup's tile, row tiles fastest: those of one group share its weights' columns
  const int t = mid::tile_of_block(blockIdx.x);
  bool negative;
  const mid::Groups gr = mid::load_groups(a.group_offs, a.G, a.m_total, lane, &negative);
  if (negative) return;
  int cnt[4], sum = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    cnt[k] = (gr.len[k] + C::BM - 1) / C::BM * n_tn;
    sum += cnt[k];
  }
  const int incl = mid::wave_scan(sum, lane);
  const uint64_t past = __ballot(incl > t);
  if (past == 0) return;                                     // more workgroups than tiles
  const int gl = __builtin_ctzll(past);
  int in_g = t - __builtin_amdgcn_readlane(incl - sum, gl), gx = 0;
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const int c = __builtin_amdgcn_readlane(cnt[k], gl);
    if (gx == k && in_g >= c) {
      in_g -= c;
      gx = k + 1;
    }
  }
  const int row_base = mid::pick(gr.start, gl, gx), len = mid::pick(gr.len, gl, gx);
  const int g = 4 * gl + gx;
  const int n_tm = (len + C::BM - 1) / C::BM;
  const int tn = in_g / n_tm, m0 = (in_g - tn * n_tm) * C::BM, n0 = tn * C::BN;
  const int rows = min(C::BM, len - m0), cols = min(C::BN, a.N - n0);

  // ---- the wave's steps: rows past the tile and chunks past K read as zero
  const int q = lane >> 4, s = lane & 15;
  const auto ra = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(a.a) + (int64_t)(row_base + m0) * a.stride_am, 0, (rows - 1) * a.stride_am + a.K, kRsrcWord3);
  const auto rb = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(a.b) + (int64_t)g * a.stride_bg + (int64_t)n0 * a.stride_bn, 0,
      (cols - 1) * a.stride_bn + a.K, kRsrcWord3);
  v4f acc[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) acc[j] = v4f{0.f, 0.f, 0.f, 0.f};
  const int nsteps = (a.K + 127) / 128;
  auto load = [&](__amdgpu_buffer_rsrc_t r, int row, int stride, int k) {
    v8i x;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = k + 64 * h + 16 * q;
      const v4i w = __builtin_bit_cast(
          v4i, __builtin_amdgcn_raw_buffer_load_b128(r, at < a.K ? row * stride + at : (int)nt::kOob, 0, 0));
#pragma unroll
      for (int c = 0; c < 4; ++c) x[4 * h + c] = w[c];
    }
    return x;
  };
  for (int s0 = wave; s0 < nsteps; s0 += kWaves * kBatch) {
    v8i w[kBatch][NB], x[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int k = 128 * (s0 + kWaves * u);                 // at or past K: zeros
#pragma unroll
      for (int j = 0; j < NB; ++j) w[u][j] = load(rb, 16 * j + s, a.stride_bn, k);
      x[u] = load(ra, s, a.stride_am, k);
    }
    __builtin_amdgcn_sched_barrier(0);                       // every load before the first use
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
#pragma unroll
      for (int j = 0; j < NB; ++j)
        acc[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[u][j], x[u], acc[j], 0, 0, 0, 0, 0, 0);
  }

  // ---- the waves' sums, block b of the tile finished by wave b % 4
  GG_LDS v4f* s_acc = (GG_LDS v4f*)lds;                      // [wave][block][lane]
#pragma unroll
  for (int j = 0; j < NB; ++j) s_acc[(wave * NB + j) * 64 + lane] = acc[j];
  __syncthreads();
  const float alpha = *a.a_scale * *a.b_scale;
  const int64_t row = (int64_t)row_base + m0 + s;
  auto value = [&](int b) {
    v4f z = s_acc[b * 64 + lane];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) z += s_acc[(w * NB + b) * 64 + lane];
    return z;
  };
  auto finish = [&](int b, const v4f& z) {
    const int n = n0 + 16 * b + 4 * q;
    if constexpr (kGated) {
      float x = epi::swiglu(z[0], z[1], e), y = epi::swiglu(z[2], z[3], e);
      if (e.residual != nullptr) {
        const uint32_t h = *(const uint32_t*)(e.residual + row * e.stride_res + n / 2);
        x += epi::from_bf16(h);
        y += __uint_as_float(h & 0xffff0000u);
      }
      *(int*)(a.c + row * a.stride_cm + n / 2) = epi::pack(x, y);
    } else {
      v4f x = epi::activation<epi::act_of(kAct)>(z);
      if (e.residual != nullptr) x += epi::unpack4(*(const v2i*)(e.residual + row * e.stride_res + n));
      *(v2i*)(a.c + row * a.stride_cm + n) = v2i{epi::pack(x[0], x[1]), epi::pack(x[2], x[3])};
    }
  };
  if constexpr ((kAct & epi::kKeepMx) != 0) {
    static_assert(NB == 2, "a block of 32 columns");
    if (wave != 0) return;                                   // one wave holds a block's scale
    const bool whole = n0 + 16 < a.N;                        // else the block's second half is past N
    v4f z[2];
#pragma unroll
    for (int b = 0; b < 2; ++b)
      z[b] = b == 0 || whole ? value(b) * alpha + epi::load_bias(e, (int64_t)g * a.N + n0 + 16 * b + 4 * q) : v4f{0.f, 0.f, 0.f, 0.f};
    int w[2];
    const uint32_t byte = epi::quantize32(z[0], z[1], w);
    if (s >= rows) return;
    if (q == 0) e.scales[(int64_t)(n0 / 32) * e.scale_block + row] = (uint8_t)byte;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      if (b == 1 && !whole) break;
      *(int*)(e.q8 + row * e.stride_q + n0 + 16 * b + 4 * q) = w[b];
      finish(b, z[b]);
    }
  } else {
    for (int b = wave; b < NB; b += kWaves) {
      const int n = n0 + 16 * b + 4 * q;
      if (s >= rows || n >= a.N) continue;
      const v4f z = value(b) * alpha + epi::load_bias(e, (int64_t)g * a.N + n);
      if (e.pre != nullptr) *(v2i*)(e.pre + row * e.stride_pre + n) = v2i{epi::pack(z[0], z[1]), epi::pack(z[2], z[3])};
      finish(b, z);
    }
  }
}

}  // namespace few
}  // namespace ggemm
