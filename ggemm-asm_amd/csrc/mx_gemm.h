// Grouped product of microscaled rows for gfx950 (blocks of 32 along K share a power of two):
//
//   z[r, :] = A[r, :] @ B[g]^T + bias[g];  out = act(z) + residual         for offs[g] <= r < offs[g + 1]
//
// B e2m1, A e2m1 or e4m3, on v_mfma_scale_f32_32x32x64_f8f6f4: the scales go into the matrix instruction, which sums a
// block's products and multiplies by both powers. Two e2m1 sides run at twice the rate of fp8; with e4m3 on one side at
// fp8's.
//
// A tile is BM rows of one group x BN columns. A stage is 128 bytes of every A row (256 values of e2m1, 128 of e4m3) and as
// many values of every B row, loaded by LDS-DMA into one of S slots. The scales are 1/16 of the bytes, but rows far
// apart: 16 bytes of a row, 512 values, come at once and serve two or four stages, since one more request for each row
// and stage would double the requests of the load path.
//
// Which K bytes a lane feeds is free as long as both sides and the scales agree: lane half h takes blocks 4 h .. 4 h +
// 3 of a stage's eight (e2m1) or 2 h, 2 h + 1 of its four (e4m3), one to a step, so that its scales of a whole stage
// are one word, whose byte the instruction picks, and its operands neighbouring chunks of 16 bytes.
//
// The operands of step t + 1 are read while step t multiplies; the barrier that frees a stage's slot stands in its
// last step, whose operands are in registers by then, so that the next stage's loads and first reads run beside its products.
//
// Tiles (mx_capi.hip): 256 x 256 by eight waves of 64 x 128, two stages of 64 or 48 KB, one workgroup to a CU that walks over its
// tiles, the next one's first stages in flight during an epilogue. Waves of 128 x 128 would read a quarter less of LDS, but
// with all 256 accumulation registers taken the compiler moves them back and forth (11 ms for the 1.6 of then); 256 x 192 and
// 256 x 128 tiles take 7 and 11 % more. 128, 64 and 32 rows x 128 columns by four waves, two workgroups to a CU, for launches
// with fewer rows.
//
// The large ones are bound by power and by the epilogue, which no product runs beside: 131072 x 5760 x 2880 with swiglu takes
// 1307 us with e2m1 rows, 3.33 PFLOP/s (a library's plain fp4 product of 16384^3 reaches 3.41, instructions alone on random
// operands 6.26; matrix units busy 0.48 of the time at 1.66 GHz), and 1886 us, 2.31, with e4m3 (instructions alone 3.79), 1.1 times
// what fp8 weights take (1700-1750): with e4m3 rows 4 bits pay up to some ten thousand rows, where weights are read. Random
// codes as operands, whose sums toggle more: 1555 and 2105 us, without the results' stores 1310 and 1818. The small ones
// read weights: 256 rows of 32 experts, e4m3, 56 us, 5.0 TB/s.
#pragma once

#include "fused_epilogue.h"
#include "mid_common.h"
#include "persistent_kernel.h"

namespace ggemm {
namespace mx {

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

// Inclusive maximum or sum over a wave's lanes of values that are not negative, by DPP: lanes 1, 2, 4 and 8 to the left in a
// row of 16, then the last lane of a row to the next ones. (Shuffles go through LDS: twelve in turn are a microsecond.)
template <int kCtrl, int kRows>
__device__ __forceinline__ int dpp(int v) {
  return __builtin_amdgcn_update_dpp(0, v, kCtrl, kRows, 0xF, false);
}
template <typename F>
__device__ __forceinline__ int scan(int v, F f) {
  v = f(v, dpp<0x111, 0xF>(v));
  v = f(v, dpp<0x112, 0xF>(v));
  v = f(v, dpp<0x114, 0xF>(v));
  v = f(v, dpp<0x118, 0xF>(v));
  v = f(v, dpp<0x142, 0xA>(v));
  return f(v, dpp<0x143, 0xC>(v));
}
struct Max {
  __device__ int operator()(int a, int b) const { return max(a, b); }
};
struct Sum {
  __device__ int operator()(int a, int b) const { return a + b; }
};

// The groups of a launch as tiles: lane l holds ceil(G / 64) consecutive ones. Offsets count as the largest one so far, in
// [0, m_total].
struct Groups {
  const int64_t* offs;
  int64_t m;
  int G, per;
  int first, len;                   // the lane's first group: first row, rows
  int sum, incl;                    // tiles of the lane's groups, and of those up to it
  __device__ __forceinline__ int row(int g) const { return (int)clamp_off(offs[g], m); }
};
template <int BM>
__device__ __forceinline__ Groups load_groups(const int64_t* offs, int G, int64_t m, int n_tn, int lane) {
  Groups r{offs, m, G, (G + 63) >> 6, 0, 0, 0, 0};
  const int g0 = min(lane * r.per, G), g1 = min(g0 + r.per, G);
  const int begin = r.row(g0);                                // lanes past the last group: offs[G], of no group
  int end = r.row(min(g0 + 1, G)), top = max(begin, 0);
  if (r.per > 1)
    for (int g = g0 + 1; g < g1; ++g) top = max(top, r.row(g));
  top = scan(top, Max{});
  const int before = dpp<0x138, 0xF>(top);                    // of the lane to the left; 0 for the first
  r.first = max(before, begin);
  r.len = g0 < g1 ? max(r.first, end) - r.first : 0;
  r.sum = (r.len + BM - 1) / BM * n_tn;
  if (r.per > 1)
    for (int g = g0 + 1, run = r.first + r.len; g < g1; ++g) {
      run = max(run, r.row(g));
      r.sum += (max(run, r.row(g + 1)) - run + BM - 1) / BM * n_tn;
    }
  r.incl = scan(r.sum, Sum{});
  return r;
}

struct Tile {
  int g, start, len, in_g;          // group, its first row and rows, the tile's index in it; g < 0: none
};
template <int BM>
__device__ __forceinline__ Tile find_tile(const Groups& r, int n_tn, int t) {
  const uint64_t past = __ballot(r.incl > t);
  if (past == 0) return {-1, 0, 0, 0};
  const int gl = __builtin_ctzll(past);
  int in_g = t - __builtin_amdgcn_readlane(r.incl - r.sum, gl);
  int start = __builtin_amdgcn_readlane(r.first, gl), len = __builtin_amdgcn_readlane(r.len, gl);
  for (int g = gl * r.per;;) {                                // ends in the lane's groups: in_g is below their sum
    const int n = (len + BM - 1) / BM * n_tn;
    if (in_g < n || ++g >= r.G) return {g, start, len, in_g};
    in_g -= n;
    start += len;
    start = max(start, __builtin_amdgcn_readfirstlane(r.row(g)));
    len = max(start, __builtin_amdgcn_readfirstlane(r.row(g + 1))) - start;
  }
}

// kWalk: one workgroup on a CU, which walks over its tiles; else two, with a tile each.
template <bool kA8, int kBM, int kBN, int kWM, int kWN, int kKS, int kStages, bool kWalk_>
struct Cfg {
  static constexpr int BM = kBM, BN = kBN, WM = kWM, WN = kWN, W = WM * WN, NT = 64 * W;   // waves and threads
  static constexpr bool kWalk = kWalk_;
  static constexpr int KS = kKS, S = kStages;                   // values of K in a stage, and slots
  static constexpr int RowA = kA8 ? KS : KS / 2, RowB = KS / 2; // bytes of a row in it
  static constexpr int Blocks = KS / 32;                        // and blocks
  static constexpr int T = KS / 64;                             // steps of a stage
  static constexpr int Super = 512 / KS;                        // stages that a row's 16 scale bytes serve
  static constexpr int ABytes = BM * RowA, BBytes = BN * RowB, Slot = ABytes + BBytes;
  static constexpr int PA = ABytes / 1024 / W, PB = BBytes / 1024 / W;   // LDS-DMA instructions for each wave and stage
  static constexpr int SA = (BM + 63) / 64, SB = (BN + 63) / 64;   // of scales for the workgroup, 64 rows each
  static constexpr int ScaleOff = S * Slot, ScaleBytes = 1024 * (SA + SB);
  static constexpr int MB = BM / WM / 32, NB = BN / WN / 32;    // 32-wide blocks of a wave
  // Where results are put together, Line bytes of 32 rows of each wave, and a wave's columns of the bias (in the place of its
  // lines where those are not whole). No Line where LDS has no room or a wave's rows are short.
  static constexpr int LineOff = ScaleOff + 2 * ScaleBytes, Room = (kWalk ? 160 : 80) * 1024;
  static constexpr int Line = NB % 2 ? 0 : LineOff + 5120 * W <= Room ? 128 : LineOff + 2048 * W <= Room ? 64 : 0;
  static constexpr int BiasOff = Line == 128 ? LineOff + 4096 * W : LineOff, BiasBytes = Line == 128 ? 1024 : 2048;
  static constexpr int LdsBytes = LineOff + 32 * Line * W + (Line == 128 ? 1024 * W : 0);
  static constexpr int BandN = 8;                               // column tiles of a band, row tiles walked inside
  static_assert(W % 2 == 0 && MB >= 1 && NB >= 1 && BM % (32 * WM) == 0 && BN % (32 * WN) == 0, "waves");
  static_assert(ABytes % (1024 * W) == 0 && BBytes % (1024 * W) == 0, "uniform LDS-DMA split");
  static_assert(S >= 2 && (kWalk ? S == 2 : S <= Super + 1), "a buffer of scales is read out when its next chunk is asked for");
  static_assert(LdsBytes <= Room, "LDS");
};

// Chunk c of row r, `row` bytes a stage, lies at c ^ swizzle: 16 rows' equal chunks on 16 different groups of banks. Rows that
// are a multiple of 16 apart have the same one, and so have the rows of a wave's load instructions.
__device__ __forceinline__ constexpr int swizzle(int row, int r) {
  return row == 256 ? r & 15 : row == 128 ? (r & 7) ^ ((r >> 3) & 1) : (r >> 2) & 3;
}

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
    for (int j = 0; j < NB; ++j) asm volatile("" : "+v"(acc[i][j]));
}

// x and y of lanes l and l + 32 to (x of both) and (y of both): lane half 0 holds x's, half 1 y's. Its own inverse.
__device__ __forceinline__ void by_half(int& x, int& y) {
  const auto r = __builtin_amdgcn_permlane32_swap((unsigned)x, (unsigned)y, false, false);
  x = (int)r[0];
  y = (int)r[1];
}

// A wave's MB x NB blocks of 32 x 32: lane 32 h + s holds row s, columns 8 g + 4 h .. + 3 of a block in accumulators
// 4 g .. 4 g + 3. Rows row0 .. of the launch (the first `rows` of them exist), columns n0 .. of group g's product. The halves
// of a row's columns change places between lanes s and s + 32, so that a lane holds (and reads of a residual) 16 bytes at a
// time. kLine = 0: it stores them as they are. Else they go through 32 kLine bytes of the wave's LDS (`lines`) and are stored
// kLine bytes of a row to neighbouring lanes, and the bias lies in LDS too (`bias_at`, raw, this wave's columns): a load's
// wait would drain the stores before it and the next tile's loads. 32768 x 2880 x 2880, e4m3, with a
// bias: 343-350 us without, 259-263 so, even and skewed groups alike; 131072 x 5760 x 2880, e2m1, swiglu: 1434 and 1307;
// 128-row tiles, 4096 x 5760 x 2880, e2m1, swiglu: 90 and 84.
template <int kAct, int MB, int NB, int kLine>
__device__ __forceinline__ void store(const v16f (&acc)[MB][NB], const epi::Args& e, uint16_t* out, int stride_out, int g,
                                      int N, int64_t row0, int rows, int n0, int lane, GG_LDS uint8_t* lines,
                                      GG_LDS uint8_t* bias_at) {
  constexpr bool kGated = kAct == epi::kSwiglu;
  constexpr int kParts = kGated ? 1 : 2;                       // 16-byte chunks of a lane and block
  // or what follows from them is kept from tile to tile
  if constexpr (kLine != 0) asm volatile("" : "+s"(stride_out));
  if constexpr (kLine == 128) asm volatile("" : "+v"(lane));
  const int h = lane >> 5, s = lane & 31;
  const int width = kGated ? N / 2 : N;
  // block (i, j): chunk p of the lane has columns 16 h (gated: of z 16 h .. + 15; else 16 h + 8 p .. + 7)
  auto block = [&](int i, int j, const v4f (&bias)[4], int (&w)[kParts][4]) {
    const int nj = n0 + 32 * j, o0 = (kGated ? nj / 2 : nj) + (kGated ? 8 : 16) * h;
    if (e.residual != nullptr) {
      const int64_t row = row0 + 32 * i + s;
      const bool live = 16 * h < min(32, N - nj) && 32 * i + s < rows;
#pragma unroll
      for (int p = 0; p < kParts; ++p) {
        const v4i r = live ? *(const v4i*)(e.residual + row * e.stride_res + o0 + 8 * p) : v4i{0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < 4; ++k) w[p][k] = r[k];
        // gated: words (0, 1) of a lane are column groups 2 h and, its other half, ..; else groups 2 h + p
        by_half(w[p][0], w[p][kGated ? 1 : 2]);
        by_half(w[p][kGated ? 2 : 1], w[p][3]);
      }
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      v4f z = bias[c];
#pragma unroll
      for (int k = 0; k < 4; ++k) z[k] += acc[i][j][4 * c + k];
      // group c: the two lanes' halves end up in lane half c / 2
      if constexpr (kGated) {
        int& at = w[0][2 * (c & 1) + (c >> 1)];
        float x = epi::swiglu(z[0], z[1], e), y = epi::swiglu(z[2], z[3], e);
        if (e.residual != nullptr) {
          x += epi::from_bf16((uint32_t)at);
          y += __uint_as_float((uint32_t)at & 0xffff0000u);
        }
        at = epi::pack(x, y);
      } else {
        int &lo = w[c & 1][2 * (c >> 1)], &hi = w[c & 1][2 * (c >> 1) + 1];
        v4f x = epi::activation<kAct>(z);
        if (e.residual != nullptr) x += epi::unpack4(v2i{lo, hi});
        lo = epi::pack(x[0], x[1]);
        hi = epi::pack(x[2], x[3]);
      }
    }
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
      by_half(w[p][0], w[p][kGated ? 1 : 2]);
      by_half(w[p][kGated ? 2 : 1], w[p][3]);
    }
  };
  auto load_bias = [&](int j, v4f (&bias)[4]) {
    const int nj = n0 + 32 * j, cols = N - nj;                 // a multiple of 16
#pragma unroll
    for (int c = 0; c < 4; ++c)
      bias[c] = 8 * c < cols ? epi::load_bias(e, (int64_t)g * N + nj + 8 * c + 4 * h) : v4f{0.f, 0.f, 0.f, 0.f};
  };
  if constexpr (kLine != 0) {
    constexpr int kRow = kLine / (32 * kParts), kChunks = kLine / 16;   // blocks and chunks of a piece
    constexpr bool kOwn = kLine == 128;                        // the bias has a place of its own
    static_assert(NB % 2 == 0 && NB % kRow == 0, "whole pieces");
    float own[NB / 2] = {};                                    // bias of columns 64 k + `lane`
    if (!kOwn && e.bias != nullptr)
#pragma unroll
      for (int k = 0; k < NB / 2; ++k)
        own[k] = e.bias_f32 ? *(const GG_LDS float*)(bias_at + 4 * (64 * k + lane))
                            : __uint_as_float((uint32_t)*(const GG_LDS uint16_t*)(bias_at + 2 * (64 * k + lane)) << 16);
    auto read_bias = [&](int j, bool f32, v4f (&bias)[4]) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int at = 32 * j + 8 * c + 4 * h;
        bias[c] = e.bias == nullptr ? v4f{0.f, 0.f, 0.f, 0.f}
                  : f32             ? *(const GG_LDS v4f*)(bias_at + 4 * at)
                                    : epi::unpack4(v2i(*(const GG_LDS v2i*)(bias_at + 2 * at)));
      }
    };
#pragma unroll
    for (int j = 0; j < NB; j += kRow) {
      const int nj = n0 + 32 * j, c = lane & (kChunks - 1), oj = kGated ? nj / 2 : nj;
      if (nj >= N) return;                                     // uniform in the wave, as all but the rows
      v4f bias[kRow][4];
      if constexpr (!kOwn) {
        if (e.bias != nullptr) {
#pragma unroll
          for (int k = 0; k < NB / 2; ++k) *(GG_LDS float*)(bias_at + 4 * (64 * k + lane)) = own[k];
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
#pragma unroll
        for (int k = 0; k < kRow; ++k) read_bias(j + k, true, bias[k]);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      }
      // rows that do not exist are out of the buffer's range, and so are columns by their offset
      const auto rsrc =
          __builtin_amdgcn_make_buffer_rsrc(out + row0 * stride_out + oj, 0, 2 * max(rows, 0) * stride_out, kRsrcWord3);
      const int to = 8 * c < width - oj ? 2 * (lane / kChunks * stride_out + 8 * c) : (int)kOob;
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        if (rows <= 32 * i) break;
#pragma unroll
        for (int k = 0; k < kRow; ++k) {
          int w[kParts][4];
          if constexpr (kOwn) read_bias(j + k, e.bias_f32, bias[k]);
          block(i, j + k, bias[k], w);
#pragma unroll
          for (int p = 0; p < kParts; ++p)
            *(GG_LDS v4i*)(lines + kLine * s + 16 * ((2 * kParts * k + kParts * h + p) ^ (s & (kChunks - 1)))) =
                v4i{w[p][0], w[p][1], w[p][2], w[p][3]};
          __builtin_amdgcn_sched_barrier(0);                   // one block's values (and bias) in registers at a time
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int q = 0; q < kChunks / 2; ++q) {
          const int r = 64 / kChunks * q + lane / kChunks;
          const v4i v = *(const GG_LDS v4i*)(lines + kLine * r + 16 * (c ^ (r & (kChunks - 1))));
          // whole lines past the caches, 33 us of what the epilogue gains at 32768 x 2880 x 2880 (e4m3); halves through them
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(mid::v4u32, v), rsrc,
                                                 to + 2 * (32 * i + 64 / kChunks * q) * stride_out, 0, kLine == 128 ? 2 : 0);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int nj = n0 + 32 * j, o0 = (kGated ? nj / 2 : nj) + (kGated ? 8 : 16) * h;
    if (nj >= N) return;
    v4f bias[4];
    load_bias(j, bias);
#pragma unroll
    for (int i = 0; i < MB; ++i) {
      if (rows <= 32 * i) break;
      int w[kParts][4];
      block(i, j, bias, w);
      if (16 * h < min(32, N - nj) && 32 * i + s < rows)
#pragma unroll
        for (int p = 0; p < kParts; ++p)
          *(v4i*)(out + (row0 + 32 * i + s) * stride_out + o0 + 8 * p) = v4i{w[p][0], w[p][1], w[p][2], w[p][3]};
    }
  }
}

// Workgroups of a launch whose tiles are walked over, of `blocks` with one for each: as many as CUs, but a multiple of the XCDs,
// so that the tiles of block, block + grid, .. rise (tile_of_block) and a walk may end at the first that is not there.
__host__ __device__ constexpr int walk_grid(int blocks, int cus) {
  const int even = cus < kXcds ? kXcds : cus - cus % kXcds;
  return blocks < even ? blocks : even;
}

// grid: workgroups of the launch; blocks: what it would have with one for each tile. A grid of fewer (walk_grid) needs tiles of
// two stages at least: loads are asked for two stages ahead, which may not reach past the next tile.
template <int kAct, bool kA8, typename C>
__device__ __forceinline__ void gemm_body(const Args& a, GG_LDS uint8_t* lds, const epi::Args& e, int grid, int blocks) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n_tn = (a.N + C::BN - 1) / C::BN;
  const Groups groups = load_groups<C::BM>(a.group_offs, a.G, tile_rows_end(a), n_tn, lane);
  struct At {
    int g, rows, n0;                // rows 0: no tile
    int64_t row0;
  };
  auto tile_at = [&](int block) {
    Tile w{-1, 0, 0, 0};
    if (block < blocks) w = find_tile<C::BM>(groups, n_tn, mid::tile_of_block(block));
    if (w.g < 0) return At{0, 0, 0, 0};
    const int n_tm = (w.len + C::BM - 1) / C::BM;
    const int band = w.in_g / (n_tm * C::BandN), r = w.in_g - band * n_tm * C::BandN;
    const int bw = min(C::BandN, n_tn - band * C::BandN), tm = r / bw;
    return At{w.g, min(C::BM, w.len - tm * C::BM), (band * C::BandN + r - tm * bw) * C::BN, (int64_t)w.start + tm * C::BM};
  };
  int block = blockIdx.x;
  At tile = tile_at(block);
  if (tile.rows == 0) return;                                  // more workgroups than tiles
  block += grid;
  At next = C::kWalk ? tile_at(block) : At{0, 0, 0, 0};

  // ---- loads, S stages ahead of the products, across the end of a tile
  const int bytes_a = kA8 ? a.K : a.K / 2, bytes_b = a.K / 2, all_blocks = a.K / 32;
  const int nst = (a.K + C::KS - 1) / C::KS;
  // the row of a wave's first instruction that this lane loads, and its chunk of it
  auto lane_row = [&](int row) { return row == 256 ? 4 * wave + (lane >> 4) : row == 128 ? 8 * wave + (lane >> 3) : 16 * wave + (lane >> 2); };
  auto lane_chunk = [&](int row) { return (lane & (row / 16 - 1)) ^ swizzle(row, lane_row(row)); };
  const int lca = lane_chunk(C::RowA), lcb = lane_chunk(C::RowB);
  const int va = lane_row(C::RowA) * a.stride_a + 16 * lca, vb = lane_row(C::RowB) * a.stride_bn + 16 * lcb;
  const int step_a = 1024 * C::W / C::RowA * a.stride_a, step_b = 1024 * C::W / C::RowB * a.stride_bn;   // the waves' rows
  constexpr int kPer = C::PA + C::PB;
  const uint32_t base = lds_u32(lds);
  int ahead = 0, ahead_chunk = 0;                              // the stage in its tile, the chunk of scales
  const uint8_t *pa, *pb;                                      // at the stage
  int left_a, left_b;                                          // bytes of the tile's rows from there on
  v4i ra, rb, ras, rbs;
  bool dead_a, dead_b;
  auto load_from = [&](const At& t) {
    const int cols = min(C::BN, a.N - t.n0), live = t.rows > 0;   // no tile: everything is out of range and reads as zero
    pa = a.a + t.row0 * a.stride_a;
    pb = a.b + (int64_t)t.g * a.stride_bg + (int64_t)t.n0 * a.stride_bn;
    left_a = t.rows * a.stride_a;
    left_b = live * cols * a.stride_bn;
    ras = make_rsrc(a.a_scales + t.row0 * a.stride_as, t.rows * a.stride_as);
    rbs = make_rsrc(a.b_scales + (int64_t)t.g * a.stride_bsg + (int64_t)t.n0 * a.stride_bsn, live * cols * a.stride_bsn);
  };
  // what instructions of a stage share: its resources, and whether this lane's chunk lies past K (and reads as zero)
  auto begin_stage = [&] {
    if (ahead == nst) {                                        // asked for once `next` follows the tile of the products
      ahead = 0;
      load_from(next);
    }
    ra = make_rsrc(pa, max(left_a, 0));                        // of no tile nothing is left: never a negative count
    rb = make_rsrc(pb, max(left_b, 0));
    dead_a = 16 * lca >= bytes_a - ahead * C::RowA;
    dead_b = 16 * lcb >= bytes_b - ahead * C::RowB;
    if (ahead % C::Super == 0 && left_b > 0) {                 // the rows' 16 scale bytes from here on; none of no tile, whose
                                                               // place a scale of this one may still have
      const uint32_t at = base + C::ScaleOff + (ahead_chunk++ & 1) * C::ScaleBytes;
      const int u = 16 * (ahead / C::Super);
#pragma unroll
      for (int k = 0; k < (C::SA + C::SB + C::W - 1) / C::W; ++k) {
        const int i = wave + C::W * k;                            // uniform
        if (i < C::SA)
          dma16(ras, at + 1024 * i, (64 * i + lane) * a.stride_as + u);
        else if (i < C::SA + C::SB)
          dma16(rbs, at + 1024 * i, (64 * (i - C::SA) + lane) * a.stride_bsn + u);
      }
    }
  };
  auto issue_one = [&](int slot, int j) {                      // of this wave's PA + PB
    const uint32_t at = base + slot * C::Slot + 1024 * wave;
    if (j < C::PA) dma16(ra, at + 1024 * C::W * j, dead_a ? (int)kOob : va + j * step_a);
    else dma16(rb, at + C::ABytes + 1024 * C::W * (j - C::PA), dead_b ? (int)kOob : vb + (j - C::PA) * step_b);
  };
  auto end_stage = [&] {
    pa += C::RowA, left_a -= C::RowA;
    pb += C::RowB, left_b -= C::RowB;
    ++ahead;
  };

  // ---- operand reads
  const int wm = wave % C::WM, wn = wave / C::WM;
  const int h = lane >> 5, s = lane & 31;
  const int ra0 = (32 * C::MB * wm + s) * C::RowA, rb0 = C::ABytes + (32 * C::NB * wn + s) * C::RowB;
  const int swa = swizzle(C::RowA, s), swb = swizzle(C::RowB, s);
  const int sa0 = C::ScaleOff + 16 * (32 * C::MB * wm + s) + C::Blocks / 2 * h;
  const int sb0 = C::ScaleOff + 1024 * C::SA + 16 * (32 * C::NB * wn + s) + C::Blocks / 2 * h;
  v4i xl[2][C::MB], xh[2][C::MB], wt[2][C::NB];
  int sx[C::MB], sw[C::NB], nsx[C::MB], nsw[C::NB];
  // operand r of step t, in the order of their first use: the first column block, the row blocks, the other columns
  auto read_one = [&](auto set, int slot, int t, auto which) {
    constexpr int k = decltype(set)::value, r = decltype(which)::value;
    const GG_LDS uint8_t* p = lds + slot * C::Slot;
    if constexpr (r >= 1 && r <= C::MB) {
      constexpr int i = r - 1;
      const int c = kA8 ? 2 * t + h : C::Blocks / 2 * h + t;   // e4m3: halves of two blocks, Blocks / 2 blocks apart
      xl[k][i] = *(const GG_LDS v4i*)(p + ra0 + 32 * C::RowA * i + 16 * (c ^ swa));
      if constexpr (kA8) xh[k][i] = *(const GG_LDS v4i*)(p + ra0 + 32 * C::RowA * i + 16 * ((c + C::Blocks) ^ swa));
    } else {
      constexpr int j = r == 0 ? 0 : r - C::MB;
      const int c = C::Blocks / 2 * h + t;
      wt[k][j] = *(const GG_LDS v4i*)(p + rb0 + 32 * C::RowB * j + 16 * (c ^ swb));
    }
  };
  // a lane's scales of stage st of its tile, in the buffer of chunk c
  auto read_scale = [&](int c, int st, auto which) {
    constexpr int r = decltype(which)::value;
    const GG_LDS uint8_t* p = lds + (c & 1) * C::ScaleBytes + C::Blocks * (st % C::Super);
    auto word = [&](const GG_LDS uint8_t* q) {
      return C::Blocks == 4 ? (int)*(const GG_LDS uint16_t*)q : *(const GG_LDS int*)q;
    };
    if constexpr (r < C::NB) nsw[r] = word(p + sb0 + 512 * r);
    else nsx[r - C::NB] = word(p + sa0 + 512 * (r - C::NB));
  };
  v16f acc[C::MB][C::NB];
  auto clear = [&] {
#pragma unroll
    for (int i = 0; i < C::MB; ++i)
#pragma unroll
      for (int j = 0; j < C::NB; ++j)
#pragma unroll
        for (int k = 0; k < 16; ++k) acc[i][j][k] = 0.f;
  };

  GG_LDS uint8_t* const lines = lds + C::LineOff + 32 * C::Line * wave;
  GG_LDS uint8_t* const bias_at = lds + C::BiasOff + C::BiasBytes * wave;
  auto fetch_bias = [&](const At& t) {                         // lands with the first stage that is waited for after it
    if constexpr (C::Line != 0) {
      if (e.bias == nullptr) return;
      const int n = t.n0 + 32 * C::NB * wn, size = e.bias_f32 ? 4 : 2;
      dma16(make_rsrc((const uint8_t*)e.bias + ((int64_t)t.g * a.N + n) * size, max(0, min(32 * C::NB, a.N - n)) * size),
            lds_u32(bias_at), 16 * lane);
    }
  };

  fetch_bias(tile);
  load_from(tile);
#pragma unroll
  for (int k = 0; k < C::S; ++k) {
    begin_stage();
#pragma unroll
    for (int j = 0; j < kPer; ++j) issue_one(k, j);
    end_stage();
  }
  wait_vmcnt<(C::S - 1) * kPer>();
  lds_barrier();
  constexpr int kMma = C::MB * C::NB, kReads = C::MB + C::NB;
  static_for<kReads>([&](auto r) {
    read_scale(0, 0, r);
    read_one(std::integral_constant<int, 0>{}, 0, 0, r);
  });
  clear();
  // Instructions go out in their order, and one that waits for its turn at LDS or the load path holds up the products
  // behind it: reads and loads are dealt out between the products, as many to each.
  int cur = 0, nxt = 1, st = 0, chunk = 0;
  for (;;) {
    // scales of blocks past K count as zero: what follows them in a row is not looked at
    const int left = all_blocks - C::Blocks * st - C::Blocks / 2 * h;
    const int mask = left >= 4 ? ~0 : left <= 0 ? 0 : (int)((1u << (8 * left)) - 1u);
#pragma unroll
    for (int j = 0; j < C::NB; ++j) sw[j] = nsw[j] & mask;
#pragma unroll
    for (int i = 0; i < C::MB; ++i) sx[i] = nsx[i] & mask;
    st = st + 1 == nst ? 0 : st + 1;
    chunk += st % C::Super == 0;                               // of the stage that comes, of this tile or the next
    static_for<C::T>([&](auto step) {
      constexpr int t = decltype(step)::value;
      constexpr bool kLast = t + 1 == C::T;
      static_for<kMma>([&](auto at) {
        constexpr int n = decltype(at)::value, j = n / C::MB, i = n % C::MB;
        acc[i][j] = mma<t, kA8>(wt[t & 1][j], xl[t & 1][i], xh[t & 1][i], acc[i][j], sw[j], sx[i]);
        if constexpr (kLast && n == 0) {
          // the stage that comes has landed for this wave (those after it may be in flight), then for all; every wave holds
          // its last operands of this one, whose slot is free
          keep_here(acc);
          wait_vmcnt<(C::S - 2) * kPer>();
          lds_barrier();
          begin_stage();
        }
        constexpr auto share = [](int all, int k) { return all * k / kMma; };
        static_for<share(kReads, n + 1) - share(kReads, n)>([&](auto d) {
          constexpr std::integral_constant<int, share(kReads, n) + decltype(d)::value> r;
          if constexpr (kLast) {
            read_scale(chunk, st, r);
            read_one(std::integral_constant<int, 0>{}, nxt, 0, r);
          } else {
            read_one(std::integral_constant<int, (t + 1) & 1>{}, cur, t + 1, r);
          }
        });
        if constexpr (kLast) {
#pragma unroll
          for (int d = share(kPer, n); d < share(kPer, n + 1); ++d) issue_one(cur, d);
        }
        __builtin_amdgcn_sched_barrier(0);
      });
    });
    keep_here(acc);
    end_stage();
    cur = nxt;
    nxt = nxt + 1 == C::S ? 0 : nxt + 1;
    if (st != 0) continue;
    store<kAct, C::MB, C::NB, C::Line>(acc, e, a.out, a.stride_out, tile.g, a.N, tile.row0 + 32 * C::MB * wm,
                                       tile.rows - 32 * C::MB * wm, tile.n0 + 32 * C::NB * wn, lane, lines, bias_at);
    if (next.rows == 0) break;                                 // nor are those that follow: tiles rise along a walk
    tile = next;
    fetch_bias(tile);
    block += grid;
    next = tile_at(block);
    clear();
  }
  wait_vmcnt<0>();                                             // loads of no tile write zeros to LDS
}

// Few rows (decoding): bound by reading the weights once and by how long the first loads take, so nothing but loads in
// flight counts: one row of one expert, 5760 x 2880, 6.3 us where a tile of 32 rows takes 10.2. A workgroup takes 16
// rows of one group and 16 NB columns; its four waves share K, wave w the pairs of steps w, w + 4, .. of 256 values:
// 128 bytes of a weight row, a whole line. No LDS stages; the waves' sums are added in their order at the end.
// v_mfma_scale_f32_16x16x128, weights as rows: lane 16 q + s feeds row s of either side, blocks 2 q and 2 q + 1 of
// the pair's eight, one to a step, its scales two neighbouring bytes.
namespace few {
constexpr int kWaves = 4, kNT = 256, kBatch = 3;    // pairs a wave has in flight: all of its share of up to 12

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
  const Tile at = find_tile<16>(load_groups<16>(a.group_offs, a.G, tile_rows_end(a), n_tn, lane), n_tn,
                                mid::tile_of_block(blockIdx.x));
  if (at.g < 0) return;                                        // more workgroups than tiles
  const int g = at.g;
  const int n_tm = (at.len + 15) / 16;                         // row tiles fastest: those of one group share its columns
  const int tn = at.in_g / n_tm, m0 = (at.in_g - tn * n_tm) * 16, n0 = tn * BN;
  const int rows = min(16, at.len - m0), cols = min(BN, a.N - n0);
  const int64_t row0 = (int64_t)at.start + m0;

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
