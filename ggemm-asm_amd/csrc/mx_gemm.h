// Grouped product of microscaled rows for gfx950 (blocks of 32 along K share a power of two):
//
//   z[r, :] = A[r, :] @ B[g]^T + bias[g];  out = act(z) + residual         for offs[g] <= r < offs[g + 1]
//
// B e2m1, A e2m1 or e4m3, on v_mfma_scale_f32_32x32x64_f8f6f4: the scales go into the matrix instruction, which sums a
// block's products and multiplies by both powers. Two e2m1 sides run at twice the rate of fp8; with e4m3 on one side at
// fp8's.
//
// One tile of BM rows of one group x BN columns for each workgroup of four waves. A stage is 128 bytes of every A row
// (256 values of e2m1, 128 of e4m3) and as many values of every B row, loaded by LDS-DMA into one of S slots. The
// scales are 1/16 of the bytes, but rows far apart: 16 bytes of a row, 512 values, come at once and serve two or four
// stages, since one more request for each row and stage would double the requests of the load path.
//
// Which K bytes a lane feeds is free as long as both sides and the scales agree: lane half h takes blocks 4 h .. 4 h +
// 3 of a stage's eight (e2m1) or 2 h, 2 h + 1 of its four (e4m3), one to a step, so that its scales of a whole stage
// are one word, whose byte the instruction picks, and its operands neighbouring chunks of 16 bytes.
//
// The operands of step t + 1 are read while step t multiplies; the barrier that frees a stage's slot stands before its
// last step, whose operands are in registers by then, so that the next stage's first reads run beside its products.
#pragma once

#include "fused_epilogue.h"
#include "mid_common.h"
#include "persistent_kernel.h"

namespace ggemm {
namespace mx {

constexpr int kNT = 256;
constexpr int kMaxGroups = 2047;
using nt::kOob;

struct Args {
  const uint8_t* a;
  const uint8_t* a_scales;
  const uint8_t* b;
  const uint8_t* b_scales;
  uint16_t* out;
  const int64_t* group_offs;
  int G, N, K;
  int stride_a, stride_as, stride_bn, stride_bsn, stride_out;
  int64_t stride_bg, stride_bsg;
  int64_t m_total;
  int zero_tail;
};

// What the tiles of a launch with zero_tail see: rows from offs[G] on are the clearing's alone.
__device__ __forceinline__ int64_t tile_rows_end(const Args& a) {
  if (!a.zero_tail) return a.m_total;
  return clamp_off(a.group_offs[a.G], a.m_total);
}

// Tile t of a launch whose groups hold ceil(rows / BM) n_tn tiles each. Offsets count as the largest one so far, in
// [0, m_total]. Lane l sums up ceil(G / 64) consecutive groups; a scan finds the lane, a walk over its groups the tile.
struct Tile {
  int g, start, len, in_g;          // group, its first row and rows, the tile's index in it; g < 0: none
};
template <int BM>
__device__ __forceinline__ Tile find_tile(const int64_t* offs, int G, int64_t m, int n_tn, int t, int lane) {
  const int per = (G + 63) >> 6, g0 = min(lane * per, G), g1 = min(g0 + per, G);
  auto row = [&](int g) { return (int)clamp_off(offs[g], m); };
  int top = 0;
  for (int g = g0; g < g1; ++g) top = max(top, row(g));
  int before = top;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int v = __shfl_up(before, d, 64);
    if (lane >= d) before = max(before, v);
  }
  before = __shfl_up(before, 1, 64);
  if (lane == 0) before = 0;
  int sum = 0, run = before;
  for (int g = g0; g < g1; ++g) {
    run = max(run, row(g));
    sum += (max(run, row(g + 1)) - run + BM - 1) / BM * n_tn;
  }
  const int incl = mid::wave_scan(sum, lane);
  const uint64_t past = __ballot(incl > t);
  if (past == 0) return {-1, 0, 0, 0};
  const int gl = __builtin_ctzll(past);
  int in_g = t - __builtin_amdgcn_readlane(incl - sum, gl), start = __builtin_amdgcn_readlane(before, gl);
  for (int g = gl * per;; ++g) {                              // ends in the lane's groups: in_g is below their sum
    start = max(start, row(g));
    const int len = max(start, row(g + 1)) - start, n = (len + BM - 1) / BM * n_tn;
    if (in_g < n || g + 1 >= G) return {g, start, len, in_g};
    in_g -= n;
  }
}

template <bool kA8, int kBM, int kBN, int kWM, int kWN, int kStages>
struct Cfg {
  static constexpr int BM = kBM, BN = kBN, WM = kWM, WN = kWN, S = kStages;
  static constexpr int KS = kA8 ? 128 : 256;                    // values of K in a stage
  static constexpr int RowA = 128, RowB = kA8 ? 64 : 128;       // bytes of a row in it
  static constexpr int T = KS / 64;                             // steps of a stage
  static constexpr int Super = 512 / KS;                        // stages that a row's 16 scale bytes serve
  static constexpr int ABytes = BM * RowA, BBytes = BN * RowB, Slot = ABytes + BBytes;
  static constexpr int PA = ABytes / 4096, PB = BBytes / 4096;  // LDS-DMA instructions for each wave and stage
  static constexpr int SA = (BM + 63) / 64, SB = (BN + 63) / 64;   // of scales for the workgroup, 64 rows each
  static constexpr int ScaleOff = S * Slot, ScaleBytes = 1024 * (SA + SB);
  static constexpr int LdsBytes = ScaleOff + 2 * ScaleBytes;
  static constexpr int MB = BM / WM / 32, NB = BN / WN / 32;    // 32-wide blocks of a wave
  static constexpr int Region = 32 * (64 * NB + 16);            // a wave's staged rows of results
  static constexpr int BandN = 8;                               // column tiles of a band, row tiles walked inside
  static_assert(WM * WN == 4 && MB >= 1 && NB >= 1 && BM % (32 * WM) == 0 && BN % (32 * WN) == 0, "waves");
  static_assert(ABytes % 4096 == 0 && BBytes % 4096 == 0, "uniform LDS-DMA split");
  static_assert(S >= 2 && S <= Super + 1, "a scale buffer is free when its next chunk is asked for");
  static_assert(4 * Region <= LdsBytes && LdsBytes <= 160 * 1024, "LDS");
};

template <int kSel, bool kA8>
__device__ __forceinline__ v16f mma(const v4i& w, const v4i& lo, const v4i& hi, v16f c, int sw, int sx) {
  const v8i a{w[0], w[1], w[2], w[3], 0, 0, 0, 0};
  if constexpr (kA8) {
    const v8i b{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 4, 0, kSel, sw, kSel, sx);
  } else {
    const v8i b{lo[0], lo[1], lo[2], lo[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 4, 4, kSel, sw, kSel, sx);
  }
}

// Products have no side effects, so the compiler would move those of a whole stage past the branch before its last step
// and leave the reads that they hide in front of them. An empty statement that takes the sums keeps a step in its place.
template <int MB, int NB>
__device__ __forceinline__ void keep_here(v16f (&acc)[MB][NB]) {
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      if constexpr (MB * NB >= 16) asm volatile("" : "+a"(acc[i][j]));
      else asm volatile("" : "+v"(acc[i][j]));
    }
}

// A wave's MB x NB blocks of 32 x 32: lane 32 h + s holds row s, columns 8 g + 4 h .. + 3 of a block in accumulators
// 4 g .. 4 g + 3. Rows row0 .. of the launch (the first `rows` of them exist), columns n0 .. of group g's product; reg:
// the wave's Region of LDS, through which the rows leave as 16-byte chunks.
template <int kAct, int MB, int NB>
__device__ __forceinline__ void store(const v16f (&acc)[MB][NB], const epi::Args& e, uint16_t* out, int stride_out, int g,
                                      int N, int64_t row0, int rows, int n0, GG_LDS uint8_t* reg, int lane) {
  constexpr bool kGated = kAct == epi::kSwiglu;
  constexpr int kChunks = kGated ? 2 * NB : 4 * NB;
  const int h = lane >> 5, s = lane & 31;
  const int cols = min(32 * NB, N - n0);                       // a multiple of 16; none where not positive
  if (cols <= 0) return;
  v4f bias[NB][4];
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int n = 32 * j + 8 * c + 4 * h;
      bias[j][c] = n < cols ? epi::load_bias(e, (int64_t)g * N + n0 + n) : v4f{0.f, 0.f, 0.f, 0.f};
    }
  const int o0 = kGated ? n0 / 2 : n0;
  GG_LDS uint8_t* at = reg + s * (16 * kChunks + 16);
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    const int prows = rows - 32 * i;
    if (prows <= 0) return;                                    // uniform in the wave
    const int64_t prow = row0 + 32 * i;
    const uint16_t* res = e.residual == nullptr ? nullptr : e.residual + (prow + s) * e.stride_res + o0;
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int n = 32 * j + 8 * c + 4 * h;
        const bool live = res != nullptr && s < prows && n < cols;
        v4f z = bias[j][c];
#pragma unroll
        for (int k = 0; k < 4; ++k) z[k] += acc[i][j][4 * c + k];
        if constexpr (kGated) {
          float x = epi::swiglu(z[0], z[1], e), y = epi::swiglu(z[2], z[3], e);
          if (live) {
            const uint32_t w = *(const uint32_t*)(res + n / 2);
            x += epi::from_bf16(w);
            y += __uint_as_float(w & 0xffff0000u);
          }
          *(GG_LDS int*)(at + n) = epi::pack(x, y);
        } else {
          v4f x = epi::activation<kAct>(z);
          if (live) x += epi::unpack4(*(const v2i*)(res + n));
          *(GG_LDS v2i*)(at + 2 * n) = v2i{epi::pack(x[0], x[1]), epi::pack(x[2], x[3])};
        }
      }
    epi::store_rows<kChunks>(reg, out + prow * stride_out + o0, stride_out, prows, kGated ? cols / 16 : cols / 8, lane);
  }
}

template <int kAct, bool kA8, typename C>
__device__ __forceinline__ void gemm_body(const Args& a, GG_LDS uint8_t* lds, const epi::Args& e) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n_tn = (a.N + C::BN - 1) / C::BN;
  const Tile w = find_tile<C::BM>(a.group_offs, a.G, tile_rows_end(a), n_tn, mid::tile_of_block(blockIdx.x), lane);
  if (w.g < 0) return;                                         // more workgroups than tiles
  const int g = __builtin_amdgcn_readfirstlane(w.g), start = __builtin_amdgcn_readfirstlane(w.start);
  const int len = __builtin_amdgcn_readfirstlane(w.len), in_g = __builtin_amdgcn_readfirstlane(w.in_g);
  const int n_tm = (len + C::BM - 1) / C::BM;
  const int band = in_g / (n_tm * C::BandN), r = in_g - band * n_tm * C::BandN;
  const int bw = min(C::BandN, n_tn - band * C::BandN), tm = r / bw;
  const int m0 = tm * C::BM, n0 = (band * C::BandN + r - tm * bw) * C::BN;
  const int rows = min(C::BM, len - m0), cols = min(C::BN, a.N - n0);
  const int64_t row0 = (int64_t)start + m0;

  const uint8_t* pa = a.a + row0 * a.stride_a;
  const uint8_t* pb = a.b + (int64_t)g * a.stride_bg + (int64_t)n0 * a.stride_bn;
  const v4i ras = make_rsrc(a.a_scales + row0 * a.stride_as, rows * a.stride_as);
  const v4i rbs = make_rsrc(a.b_scales + (int64_t)g * a.stride_bsg + (int64_t)n0 * a.stride_bsn, cols * a.stride_bsn);
  const int rec_a = rows * a.stride_a, rec_b = cols * a.stride_bn;
  const int bytes_a = kA8 ? a.K : a.K / 2, bytes_b = a.K / 2;

  // ---- loads: rows of 128 bytes as in persistent_kernel.h; of 64 bytes chunk c of row r at c ^ ((r >> 2) & 3)
  const int lca = (lane & 7) ^ (lane >> 3) ^ (wave & 1);
  const int va = (8 * wave + (lane >> 3)) * a.stride_a + 16 * lca;
  const int lcb = kA8 ? (lane & 3) ^ (lane >> 4) : lca;
  const int vb = kA8 ? (16 * wave + (lane >> 2)) * a.stride_bn + 16 * lcb : (8 * wave + (lane >> 3)) * a.stride_bn + 16 * lcb;
  constexpr int kRowsB = kA8 ? 64 : 32;                        // B rows of the four waves' instructions
  const uint32_t base = lds_u32(lds);
  auto issue = [&](int st, int slot) {
    if (st % C::Super == 0) {
      const int u = st / C::Super;
      const uint32_t at = base + C::ScaleOff + (u & 1) * C::ScaleBytes;
#pragma unroll
      for (int k = 0; k < (C::SA + C::SB + 3) / 4; ++k) {
        const int i = wave + 4 * k;                            // uniform
        if (i < C::SA)
          dma16(ras, at + 1024 * i, (64 * i + lane) * a.stride_as + 16 * u);
        else if (i < C::SA + C::SB)
          dma16(rbs, at + 1024 * i, (64 * (i - C::SA) + lane) * a.stride_bsn + 16 * u);
      }
    }
    const int ka = st * C::RowA, kb = st * C::RowB;
    const v4i ra = make_rsrc(pa + ka, rec_a - ka), rb = make_rsrc(pb + kb, rec_b - kb);
    const bool dead_a = 16 * lca >= bytes_a - ka, dead_b = 16 * lcb >= bytes_b - kb;   // chunks past K read as zero
    const uint32_t at = base + slot * C::Slot + 1024 * wave;
#pragma unroll
    for (int j = 0; j < C::PA; ++j) dma16(ra, at + 4096 * j, dead_a ? (int)kOob : va + 32 * j * a.stride_a);
#pragma unroll
    for (int j = 0; j < C::PB; ++j)
      dma16(rb, at + C::ABytes + 4096 * j, dead_b ? (int)kOob : vb + kRowsB * j * a.stride_bn);
  };

  // ---- operand reads
  const int wm = wave % C::WM, wn = wave / C::WM;
  const int h = lane >> 5, s = lane & 31;
  const int ra0 = (32 * C::MB * wm + s) * C::RowA, rb0 = C::ABytes + (32 * C::NB * wn + s) * C::RowB;
  const int sws = nt::swz(s), swb = kA8 ? (s >> 2) & 3 : sws;
  const int sa0 = C::ScaleOff + 16 * (32 * C::MB * wm + s) + (kA8 ? 2 : 4) * h;
  const int sb0 = C::ScaleOff + 1024 * C::SA + 16 * (32 * C::NB * wn + s) + (kA8 ? 2 : 4) * h;
  const int blocks = a.K / 32;
  v4i xl[2][C::MB], xh[2][C::MB], wt[2][C::NB];
  int sx[C::MB], sw[C::NB], nsx[C::MB], nsw[C::NB];
  auto read = [&](auto set, int slot, int t) {
    constexpr int k = decltype(set)::value;
    const GG_LDS uint8_t* p = lds + slot * C::Slot;
    const int ca = kA8 ? 2 * t + h : 4 * h + t, cb = kA8 ? 2 * h + t : 4 * h + t;
#pragma unroll
    for (int j = 0; j < C::NB; ++j) wt[k][j] = *(const GG_LDS v4i*)(p + rb0 + 32 * C::RowB * j + 16 * (cb ^ swb));
#pragma unroll
    for (int i = 0; i < C::MB; ++i) {
      xl[k][i] = *(const GG_LDS v4i*)(p + ra0 + 32 * C::RowA * i + 16 * (ca ^ sws));
      if constexpr (kA8) xh[k][i] = *(const GG_LDS v4i*)(p + ra0 + 32 * C::RowA * i + 16 * ((ca + 4) ^ sws));
    }
  };
  // a lane's scales of a stage, those of blocks past K as zero: what follows them in a row is not looked at
  auto read_scales = [&](int st) {
    const GG_LDS uint8_t* p = lds + (st / C::Super & 1) * C::ScaleBytes + (kA8 ? 4 * (st & 3) : 8 * (st & 1));
    const int left = blocks - (kA8 ? 4 * st + 2 * h : 8 * st + 4 * h);
    const uint32_t mask = left >= 4 ? ~0u : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
#pragma unroll
    for (int j = 0; j < C::NB; ++j) {
      const GG_LDS uint8_t* q = p + sb0 + 512 * j;
      nsw[j] = (int)((kA8 ? (uint32_t)*(const GG_LDS uint16_t*)q : *(const GG_LDS uint32_t*)q) & mask);
    }
#pragma unroll
    for (int i = 0; i < C::MB; ++i) {
      const GG_LDS uint8_t* q = p + sa0 + 512 * i;
      nsx[i] = (int)((kA8 ? (uint32_t)*(const GG_LDS uint16_t*)q : *(const GG_LDS uint32_t*)q) & mask);
    }
  };
  v16f acc[C::MB][C::NB];
#pragma unroll
  for (int i = 0; i < C::MB; ++i)
#pragma unroll
    for (int j = 0; j < C::NB; ++j)
#pragma unroll
      for (int k = 0; k < 16; ++k) acc[i][j][k] = 0.f;

  const int nst = (a.K + C::KS - 1) / C::KS;
  constexpr int kPer = C::PA + C::PB;
#pragma unroll
  for (int st = 0; st < C::S; ++st)
    if (st < nst) issue(st, st);
  if (nst >= C::S) wait_vmcnt<(C::S - 1) * kPer>(); else wait_vmcnt<0>();
  lds_barrier();
  read(std::integral_constant<int, 0>{}, 0, 0);
  read_scales(0);
  int cur = 0;
  for (int st = 0; st < nst; ++st) {
#pragma unroll
    for (int j = 0; j < C::NB; ++j) sw[j] = nsw[j];
#pragma unroll
    for (int i = 0; i < C::MB; ++i) sx[i] = nsx[i];
    const int nxt = cur + 1 == C::S ? 0 : cur + 1;
    static_for<C::T>([&](auto step) {
      constexpr int t = decltype(step)::value;
      if constexpr (t + 1 < C::T) {
        read(std::integral_constant<int, (t + 1) & 1>{}, cur, t + 1);
      } else if (st + 1 < nst) {
        // stage st + 1 has landed for this wave (those after it may be in flight), then for all; every wave holds
        // its last operands of stage st, whose slot is free
        if (st + C::S <= nst) wait_vmcnt<(C::S - 2) * kPer>(); else wait_vmcnt<0>();
        lds_barrier();
        if (st + C::S < nst) issue(st + C::S, cur);
        read(std::integral_constant<int, 0>{}, nxt, 0);
        read_scales(st + 1);
      }
      __builtin_amdgcn_sched_barrier(0);                       // the reads go out before the products
#pragma unroll
      for (int j = 0; j < C::NB; ++j)
#pragma unroll
        for (int i = 0; i < C::MB; ++i)
          acc[i][j] = mma<t, kA8>(wt[t & 1][j], xl[t & 1][i], xh[t & 1][i], acc[i][j], sw[j], sx[i]);
      keep_here(acc);
    });
    cur = nxt;
  }

  lds_barrier();                                               // every wave is past its reads: the slots are free
  store<kAct, C::MB, C::NB>(acc, e, a.out, a.stride_out, g, a.N, row0 + 32 * C::MB * wm, rows - 32 * C::MB * wm,
                            n0 + 32 * C::NB * wn, lds + wave * C::Region, lane);
}

// Few rows (decoding): bound by reading the weights once, so nothing but loads in flight counts. A workgroup takes 16
// rows of one group and 16 NB columns; its four waves share K, wave w the pairs of steps w, w + 4, .. of 256 values:
// 128 bytes of a weight row, a whole line. No LDS stages; the waves' sums are added in their order at the end.
// v_mfma_scale_f32_16x16x128, weights as rows: lane 16 q + s feeds row s of either side, blocks 2 q and 2 q + 1 of
// the pair's eight, one to a step, its scales two neighbouring bytes.
namespace few {
constexpr int kWaves = 4, kBatch = 3;    // pairs a wave has in flight: all of its share of up to 12

template <int kSel, bool kA8>
__device__ __forceinline__ v4f mma(const v4i& w, const v4i& lo, const v4i& hi, v4f c, int sw, int sx) {
  const v8i a{w[0], w[1], w[2], w[3], 0, 0, 0, 0};
  if constexpr (kA8) {
    const v8i b{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 0, kSel, sw, kSel, sx);
  } else {
    const v8i b{lo[0], lo[1], lo[2], lo[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 4, kSel, sw, kSel, sx);
  }
}

template <int kAct, bool kA8, int NB>
__device__ __forceinline__ void body(const Args& a, GG_LDS uint8_t* lds, const epi::Args& e) {
  constexpr bool kGated = kAct == epi::kSwiglu;
  constexpr int BN = 16 * NB, kX = kA8 ? 2 : 1;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n_tn = (a.N + BN - 1) / BN;
  const Tile at = find_tile<16>(a.group_offs, a.G, tile_rows_end(a), n_tn, mid::tile_of_block(blockIdx.x), lane);
  if (at.g < 0) return;
  const int g = __builtin_amdgcn_readfirstlane(at.g), start = __builtin_amdgcn_readfirstlane(at.start);
  const int len = __builtin_amdgcn_readfirstlane(at.len), in_g = __builtin_amdgcn_readfirstlane(at.in_g);
  const int n_tm = (len + 15) / 16;                            // row tiles fastest: those of one group share its columns
  const int tn = in_g / n_tm, m0 = (in_g - tn * n_tm) * 16, n0 = tn * BN;
  const int rows = min(16, len - m0), cols = min(BN, a.N - n0);
  const int64_t row0 = (int64_t)start + m0;

  const int q = lane >> 4, s = lane & 15;
  auto rsrc = [](const uint8_t* p, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, bytes, kRsrcWord3);
  };
  const auto ra = rsrc(a.a + row0 * a.stride_a, rows * a.stride_a);
  const auto rb = rsrc(a.b + (int64_t)g * a.stride_bg + (int64_t)n0 * a.stride_bn, cols * a.stride_bn);
  const auto ras = rsrc(a.a_scales + row0 * a.stride_as, rows * a.stride_as);
  const auto rbs = rsrc(a.b_scales + (int64_t)g * a.stride_bsg + (int64_t)n0 * a.stride_bsn, cols * a.stride_bsn);
  const int bytes_a = kA8 ? a.K : a.K / 2, bytes_b = a.K / 2, blocks = a.K / 32;
  auto load = [](__amdgpu_buffer_rsrc_t r, int row, int at, int end) {       // chunks past K read as zero
    return __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(r, at < end ? row + at : (int)kOob, 0, 0));
  };
  auto load_scales = [&](__amdgpu_buffer_rsrc_t r, int row, int pair) {
    const int left = blocks - 8 * pair - 2 * q;
    const uint32_t w = __builtin_amdgcn_raw_buffer_load_b16(r, left > 0 ? row + 8 * pair + 2 * q : (int)kOob, 0, 0);
    return (int)(left >= 2 ? w & 0xffffu : w & 0xffu);
  };
  v4f acc[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) acc[j] = v4f{0.f, 0.f, 0.f, 0.f};
  const int npairs = (a.K + 255) / 256;
  for (int p0 = wave; p0 < npairs; p0 += kWaves * kBatch) {
    v4i w[kBatch][NB][2], x[kBatch][2][kX];
    int sw[kBatch][NB], sx[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int p = p0 + kWaves * u;                           // at or past K: zeros
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        sw[u][j] = load_scales(rbs, (16 * j + s) * a.stride_bsn, p);
#pragma unroll
        for (int t = 0; t < 2; ++t) w[u][j][t] = load(rb, (16 * j + s) * a.stride_bn, 128 * p + 32 * q + 16 * t, bytes_b);
      }
      sx[u] = load_scales(ras, s * a.stride_as, p);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if constexpr (kA8) {
          // the instruction's block b is 2 b + t of the pair; its bytes 0 - 15 hold half q & 1 of block q / 2, its
          // bytes 16 - 31 that of block 2 + q / 2
          const int at = 256 * p + 32 * (2 * (q >> 1) + t) + 16 * (q & 1);
          x[u][t][0] = load(ra, s * a.stride_a, at, bytes_a);
          x[u][t][1] = load(ra, s * a.stride_a, at + 128, bytes_a);
        } else {
          x[u][t][0] = load(ra, s * a.stride_a, 128 * p + 32 * q + 16 * t, bytes_a);
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);                         // every load before the first use
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        acc[j] = mma<0, kA8>(w[u][j][0], x[u][0][0], x[u][0][kX - 1], acc[j], sw[u][j], sx[u]);
        acc[j] = mma<1, kA8>(w[u][j][1], x[u][1][0], x[u][1][kX - 1], acc[j], sw[u][j], sx[u]);
      }
  }

  GG_LDS v4f* s_acc = (GG_LDS v4f*)lds;                        // [wave][block][lane]
#pragma unroll
  for (int j = 0; j < NB; ++j) s_acc[(wave * NB + j) * 64 + lane] = acc[j];
  __syncthreads();
  for (int b = wave; b < NB; b += kWaves) {
    const int n = n0 + 16 * b + 4 * q;
    if (s >= rows || n >= a.N) continue;
    v4f z = s_acc[b * 64 + lane];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) z += s_acc[(w * NB + b) * 64 + lane];
    z += epi::load_bias(e, (int64_t)g * a.N + n);
    const int64_t row = row0 + s;
    if constexpr (kGated) {
      float x = epi::swiglu(z[0], z[1], e), y = epi::swiglu(z[2], z[3], e);
      if (e.residual != nullptr) {
        const uint32_t v = *(const uint32_t*)(e.residual + row * e.stride_res + n / 2);
        x += epi::from_bf16(v);
        y += __uint_as_float(v & 0xffff0000u);
      }
      *(int*)(a.out + row * a.stride_out + n / 2) = epi::pack(x, y);
    } else {
      v4f x = epi::activation<kAct>(z);
      if (e.residual != nullptr) x += epi::unpack4(*(const v2i*)(e.residual + row * e.stride_res + n));
      *(v2i*)(a.out + row * a.stride_out + n) = v2i{epi::pack(x[0], x[1]), epi::pack(x[2], x[3])};
    }
  }
}
}  // namespace few

}  // namespace mx
}  // namespace ggemm
