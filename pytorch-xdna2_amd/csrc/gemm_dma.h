// The 256 x 256 tile of the large bf16 products on gfx950, shared by gemm.hip and gated.hip: its
// XCD-aware order, the LDS DMA plans of its operands, and the k-loop of 16x16x32 MFMAs.  The
// kernels differ in how an operand's rows are found and in what becomes of the accumulators.
#pragma once

#include "common.h"
#include "mfma.h"

#include <type_traits>

namespace xdna {

enum StageMode { kAlongK = 0, kAlongRow = 1, kScalar = 2 };

constexpr int kT4 = 256;
typedef short g4i16x4 __attribute__((ext_vector_type(4)));
typedef unsigned int g2u2 __attribute__((ext_vector_type(2)));

// Workgroups go round-robin to the 8 XCDs (each with its own L2) in linear id order.  In
// launch order (x = column tile fastest) XCD x would take the column tiles x, x + 8, ...
// of every row, so each XCD would read all of A.  With xcd_group = G (the tile count a
// multiple of 8), XCD x takes tiles [x T/8, (x+1) T/8) of a grouped order (G tile rows at
// a time, rows fastest): a compact block of rows and columns per XCD, whose A and B tiles
// its L2 holds for the workgroups in flight.
constexpr int kGemmXcds = 8;

__device__ inline void xcd_tile_xy(int xcd_group, int& bx, int& by) {
  bx = blockIdx.x;
  by = blockIdx.y;
  if (xcd_group <= 0) return;
  const int nx = gridDim.x, my = gridDim.y;
  const int T = nx * my;
  const int L = by * nx + bx;
  const int t = (L % kGemmXcds) * (T / kGemmXcds) + L / kGemmXcds;
  const int gsz = xcd_group * nx;
  const int grp = t / gsz, r = t - grp * gsz;
  const int gm = min(xcd_group, my - grp * xcd_group);
  by = grp * xcd_group + r % gm;
  bx = r / gm;
}

constexpr int kK5 = 32, kNB5 = 4;
constexpr int kTile5 = kT4 * kK5;                          // elements of one operand's k-tile
constexpr size_t kGemm5Lds = size_t(kNB5) * 2 * kTile5 * 2;  // 4 buffers x (A, B): 128 KB

// One operand's DMA plan: per thread 4 loads of 16 bytes per k-tile (blocks 4 w + i of
// 1 KB, w the wave).  roff: the row part of the element offset (-1: rows past the
// operand), kq: the k offset within the k-tile.
struct G5Operand {
  i32x4_t rs;
  int roff[4];
  int kq[4];
  int s_k;
};

// kPerm16: the tile permutations of the 16x16x32 kernel (gemm6_kernel): k-contiguous,
// piece c of row r at c ^ 2 ((r >> 3) & 1), which the LDS serves without bank conflicts for
// reads of 16 rows x 4 pieces (the k-contiguous permutation above measured 2 conflict cycles
// per LDS-active cycle there); [k][row], for transposing reads that cover k rows R .. R+3
// and R+8 .. R+11 in one half-wave
template <int kMode, bool kPerm16 = false>
__device__ inline G5Operand g5_operand(const uint16_t* src, int64_t s_r, int64_t s_k, int r0, int rows, int K,
                                       int tid) {
  G5Operand o;
  const int64_t extent = ((int64_t(rows) - 1) * s_r + (int64_t(K) - 1) * s_k + 1) * 2;
  o.rs = lds_dma_rsrc(src, int(extent));
  o.s_k = int(s_k);
  const int lane = tid & 63, w = tid >> 6;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int j = 4 * w + i;
    if (kMode == kAlongK) {
      // block j: rows 16 j .. 16 j + 15, lane L at row 16 j + L / 4, position L % 4
      const int r = 16 * j + (lane >> 2);
      const int c = (lane & 3) ^ (kPerm16 ? 2 * ((r >> 3) & 1) : (r >> 2) & 3);
      o.roff[i] = r0 + r < rows ? int(int64_t(r0 + r) * s_r) : -1;
      o.kq[i] = c * 8;
    } else {
      // block j: k rows 2 j, 2 j + 1, lane L at k row 2 j + L / 32, position L % 32
      const int kr = 2 * j + (lane >> 5);
      const int q = (lane & 31) ^ (4 * (kr & 3) + (kPerm16 ? 2 * ((kr >> 3) & 1) : 0));
      o.roff[i] = r0 + 8 * q < rows ? (r0 + 8 * q) : -1;  // s_r == 1
      o.kq[i] = kr;
    }
  }
  return o;
}

// Byte offset of DMA load i of k-tile k0 .. k0 + 31 (masked past K: out of range).
__device__ inline int g5_off(const G5Operand& o, int i, int k0, int K) {
  const int k = k0 + o.kq[i];
  return o.roff[i] >= 0 && k < K ? (o.roff[i] + k * o.s_k) * 2 : 0x7FFFFFF0;
}

// The 4 DMA loads of k-tile k0 .. k0 + 31 (clamped, masked past K) into `tile`.
__device__ inline void g5_load(uint16_t* tile, const G5Operand& o, int k0, int K, int w) {
#pragma unroll
  for (int i = 0; i < 4; ++i) lds_dma16(o.rs, tile + (4 * w + i) * 512, g5_off(o, i, k0, K));
}

// 16 x 32 fragment of a k-contiguous [256][4 pieces] k-tile: rows rb + lane % 16, piece lane / 16;
// 16 x 32 fragment of a [k][row] k-tile (row-contiguous operand): two transposing reads.
// In 16-lane group g = lane / 16, lane j supplies (k row 8 g + 4 h + j / 4, rows rb + 4 (j % 4)
// .. +3) and receives row rb + j at k rows 8 g + 4 h .. +3 (h = 0, 1).  Piece q (8 rows) of
// k row kr sits at q ^ (4 (kr & 3) + 2 ((kr >> 3) & 1)): a half-wave's k rows R .. R+3 and
// R+8 .. R+11 fall on 16 distinct 16-byte positions of a 64-bank window.
template <int kMode>
__device__ inline u32x4_t g6_frag(const uint16_t* tile, int rb, int lane) {
  if (kMode == kAlongK) {
    const int r = rb + (lane & 15);
    const int c = (lane >> 4) ^ (2 * ((r >> 3) & 1));
    return *reinterpret_cast<const u32x4_t*>(tile + (r * 4 + c) * 8);
  }
  const int g = lane >> 4, j = lane & 15;
  const int kr = 8 * g + (j >> 2);
  const int rr = rb + 4 * (j & 3);
  const uint16_t* p = tile + (kr * 32 + ((rr >> 3) ^ (4 * (kr & 3) + 2 * ((kr >> 3) & 1)))) * 8 + (rr & 7);
  const g4i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) g4i16x4*)(p));
  const g4i16x4 hi =
      __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) g4i16x4*)(p + 4 * 32 * 8));
  const g2u2 a = __builtin_bit_cast(g2u2, lo), b = __builtin_bit_cast(g2u2, hi);
  return u32x4_t{a[0], a[1], b[0], b[1]};
}

// The k-loop over [kbeg, kend) of a workgroup of four waves (wave = 2 wn + wm owns rows 128 wm ..
// of A and 128 wn .. of B); kGemm5Lds bytes of LDS at smem.  An empty range still runs one
// k-tile: every load past kend is masked to zeros.  mfma16_fence before the accumulators are read.
template <int kModeA, int kModeB>
__device__ __forceinline__ void gemm6_loop(f32x4_t (&acc)[8][8], const G5Operand& oa, const G5Operand& ob, uint16_t* smem,
                                           int kbeg, int kend, int tid) {
  const int lane = tid & 63, wave = tid >> 6;
  const int wm = wave & 1, wn = wave >> 1;
  const int ntiles = kend > kbeg ? (kend - kbeg + kK5 - 1) / kK5 : 1;
  // one fragment set, each fragment read again for the next k-tile after its last MFMA
  // of this one: rows 0..3 of A and the B columns during the second half, rows 4..7 of A
  // during the next first half.  Both halves run column by column, so a fragment is read
  // at least 16 MFMAs before its first use.
  u32x4_t fa[8], fb[8];
  auto tbuf = [&](int t) { return smem + (t & (kNB5 - 1)) * 2 * kTile5; };
  auto load = [&](int t) {
    const int k_ = kbeg + min(t, ntiles - 1) * kK5;
    g5_load(tbuf(t), oa, k_, kend, wave);
    g5_load(tbuf(t) + kTile5, ob, k_, kend, wave);
  };
#pragma unroll
  for (int t = 0; t < kNB5; ++t) load(t);
  lds_dma_wait<8 * (kNB5 - 1)>();
  __builtin_amdgcn_s_barrier();
#pragma unroll
  for (int i = 0; i < 4; ++i) fa[i] = g6_frag<kModeA>(tbuf(0), wm * 128 + i * 16, lane);
#pragma unroll
  for (int j = 0; j < 8; ++j) fb[j] = g6_frag<kModeB>(tbuf(0) + kTile5, wn * 128 + j * 16, lane);
  // wave-uniform DMA state: resources and the LDS byte address of this wave's first
  // destination block (the loop adds buffer and block offsets as scalar arithmetic)
  const i32x4_t rsa = uniform_rsrc(oa.rs), rsb = uniform_rsrc(ob.rs);
  const int wave_u = __builtin_amdgcn_readfirstlane(wave);
  const uint32_t lds_w = lds_addr(smem) + uint32_t(4 * wave_u * 512 * 2);
  // k-tile t (kFirst: t == 0, whose MFMAs start the accumulators).  A 16x16x32 MFMA
  // occupies the matrix pipe for 16 cycles, so every LDS read and DMA is issued right
  // after one MFMA (never several after a group): the wave issues them while that MFMA
  // runs and the next MFMA is not held back.
  auto ktile = [&](int t, auto first) {
    constexpr bool kFirst = decltype(first)::value;
    // k of the DMA loads (k-tile t + kNB5): their offsets are formed in the second half
    const int kn = kbeg + min(t + kNB5, ntiles - 1) * kK5;
    const uint32_t m0n = lds_w + uint32_t(((t + kNB5) & (kNB5 - 1)) * 2 * kTile5 * 2);
    // first half (A rows 0..3) column by column; A rows 4..7 of this k-tile are read
    // after the second MFMA of columns 0..3
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mfma16_acc<kFirst>(acc[i][j], fa[i], fb[j]);
        if (i == 1 && j < 4) fa[4 + j] = g6_frag<kModeA>(tbuf(t), wm * 128 + (4 + j) * 16, lane);
        __builtin_amdgcn_sched_barrier(0);
      }
    // this wave's reads of buffer t are complete and its loads of k-tile t+1 have landed
    // (two k-tiles of loads may stay in flight): the barrier publishes k-tile t+1 and
    // frees buffer t
    lds_reads_wait();
    lds_dma_wait<8 * (kNB5 - 2)>();
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    // second half (A rows 4..7) column by column: DMA j of k-tile t+kNB5 after the
    // column's first MFMA, k-tile t+1's A row j (j < 4) after its second, its B column j
    // after the last (the last use of this k-tile's B column j)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      mfma16_acc<kFirst>(acc[4][j], fa[4], fb[j]);
      if (j < 4)
        lds_dma16_m0(rsa, m0n + uint32_t(j * 512 * 2), g5_off(oa, j, kn, kend));
      else
        lds_dma16_m0(rsb, m0n + uint32_t((kTile5 + (j - 4) * 512) * 2), g5_off(ob, j - 4, kn, kend));
      __builtin_amdgcn_sched_barrier(0);
      mfma16_acc<kFirst>(acc[5][j], fa[5], fb[j]);
      if (j < 4) fa[j] = g6_frag<kModeA>(tbuf(t + 1), wm * 128 + j * 16, lane);
      __builtin_amdgcn_sched_barrier(0);
      mfma16_acc<kFirst>(acc[6][j], fa[6], fb[j]);
      __builtin_amdgcn_sched_barrier(0);
      mfma16_acc<kFirst>(acc[7][j], fa[7], fb[j]);
      fb[j] = g6_frag<kModeB>(tbuf(t + 1) + kTile5, wn * 128 + j * 16, lane);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  ktile(0, std::true_type{});
  for (int t = 1; t < ntiles; ++t) ktile(t, std::false_type{});
  lds_dma_wait<0>();
}

}  // namespace xdna
