// Gated feed-forward on gfx950 MFMA: h = act(x Wg^T) * (x Wu^T), both projections, the
// activation and the product in one kernel, and its backward pass.  The reference would run
// these as separate mm / activation / mul ops (torch_xdna_device.cpp:4360-4417, 5124-5260).
//
// w holds [Wg; Wu], 2F rows of K.  The projections are summed in fp32 and stay there through
// the activation and the product; h is rounded once.  For training g and u are kept, in 20 bits
// each: a bf16 and 4 more bits of the mantissa, the two units' in one byte (M x 2F bf16, then
// M x F bytes).  The backward's products take [dg du] as bf16; with g and u in bf16 as well their
// rounding is the third of equal size in dx and dw (error of dx against 64 bits 1.75 times that of
// its own rounding, 1.4 times with the 4 bits), and the 4 bits cost a quarter of their traffic,
// where multiplying again would cost two more products.
//   dg = dh u act'(g), du = dh act(g), as [dg du] (M x 2F), so that dx = [dg du] w and
//   dw = [dg du]^T x are one product each.
//
// The linear layer y = act(x W^T + b) + r runs on the same tiles with an epilogue of its own.  For
// training it keeps the slope act'(v) as an fp16 times 2^15 (2 bytes a unit, 11 bits of mantissa
// down to 1.9e-9): what the backward multiplies dy by, without the activation again and within 2^-11,
// where a slope in bf16 would be a second rounding as large as that of dy act'(v) itself.  ReLU's slopes are bits, four
// units a byte, by which its gradient is selected (0 at a unit that is off, whatever comes in): the layer's traffic beside its
// products is a fifth less.  8192 x 1024 -> 4096 with bias, ReLU and residual: 96 us in a training pass (0.72 PFLOP/s: two
// rounds of tiles, each its k-loop and then its 128 KB of outputs, residual and slopes), 90 in a loop of its own and 84
// there without residual and slopes; dy and slopes to dp 25 (143 MB, 5.6 TB/s); 1 x 4096 -> 1024: 4.6.
#include "common.h"
#include "gemm_dma.h"
#include "mfma.h"

#include "../../include/xdna_hip.h"

namespace xdna {
namespace {

enum Act { kSilu = 0, kGelu = 1, kRelu = 2, kNone = 3 };

// The normal distribution function Phi(g) and e = exp(-g^2 / 2).  The lower tail keeps its relative
// accuracy (1 + erf(g / sqrt 2) loses it to the 1: 4 % off at -5, 0 from -5.5 on): Phi(-|g|) =
// e t P(t) with t = 1 / (1 + 0.3 |g|), which turns the half line into (0, 1].  P is the polynomial of
// degree 7 whose largest relative error on |g| <= 14 is least, 1.5e-7 (Lawson's weighted least squares
// on 4000 Chebyshev points; e underflows past 13.2).  The derivative shares e.  The block at 8192 x
// 1024 x 4096, forward and backward: 709 us; 767 with the library's erfc, 752 with its erf.
__device__ inline float2 normal_cdf(float g) {
  const float x = fabsf(g), e = __expf(-0.5f * g * g), t = __builtin_amdgcn_rcpf(fmaf(0.3f, x, 1.0f));
  float p = 0.035674773156642914f;
  p = fmaf(p, t, -0.1572030782699585f);
  p = fmaf(p, t, 0.20635350048542023f);
  p = fmaf(p, t, -0.05368364229798317f);
  p = fmaf(p, t, 0.12856163084506989f);
  p = fmaf(p, t, 0.09991349279880524f);
  p = fmaf(p, t, 0.12075395882129669f);
  p = fmaf(p, t, 0.11962930113077164f);
  const float tail = e * (t * p);
  return make_float2(g > 0.0f ? 1.0f - tail : tail, e);
}

template <int ACT>
__device__ inline float act_of(float g) {
  if constexpr (ACT == kSilu) return g * __builtin_amdgcn_rcpf(1.0f + __expf(-g));
  if constexpr (ACT == kGelu) return g * normal_cdf(g).x;
  return g > 0.0f ? g : (g != g ? g : 0.0f);
}

// act(g) and act'(g)
template <int ACT>
__device__ inline float2 act_pair(float g) {
  if constexpr (ACT == kSilu) {
    const float s = __builtin_amdgcn_rcpf(1.0f + __expf(-g));
    return make_float2(g * s, s * (1.0f + g * (1.0f - s)));
  }
  if constexpr (ACT == kGelu) {
    const float2 n = normal_cdf(g);
    return make_float2(g * n.x, n.x + g * 0.3989422804014327f * n.y);
  }
  return g > 0.0f ? make_float2(g, 1.0f) : make_float2(g != g ? g : 0.0f, 0.0f);
}

// ---- products in tiles, any sizes, alignments and row strides --------------------------------
// D[p][q] = sum over k of P[p][k] Q[q][k], written at out[q * ldc + p]: the p index is the one
// that is contiguous in memory, so that the 4 consecutive rows an MFMA accumulator quad holds
// are 4 consecutive elements of the output (and of [g u] beside it); the block's results go through
// LDS, so that 8 consecutive outputs are one access and consecutive threads continue the row
// (stored straight from the accumulators, each wave's store touched 32 rows: the epilogue of the
// projections of 3972 x 692 -> 998 units took most of its 64 us).  Each operand is contiguous
// along k, or along its rows (then staged [k][row] and transposed by the LDS reads).  Loads are
// 16 bytes at any element-aligned address (gfx950 takes them); out-of-range elements are zeros.
//
// Every wave multiplies a 64 x 64 block (2 x 2 MFMAs of 32x32x16: as many LDS reads as MFMAs):
//   wide tiles, 128 x 128: four waves side by side, k-tiles of 64;
//   narrow tiles, 64 x 64, where wide ones would leave CUs without work: eight waves on the
// same block, each with half its columns and two k-steps of a k-tile of 128 (few k-tiles: each
// costs a barrier), the four k parts added in wave order through LDS.  Where even they leave CUs
// without work (weight gradients: short outputs, k as long as the batch), plain products split k
// over the grid too, into fp32 partials that a second launch adds in order.
// What bounds small products is the latency of the k-tiles' loads: two k-tiles fly in registers
// while one is multiplied (one, with a k-step per wave and 64 more accumulators: 333 x 4096 -> 1367
// units 38 us, now 26; three do not fit the registers of two workgroups a CU).  Large ones are
// bounded by the LDS reads beside the MFMAs: 8192 x 512 x 2048 in wide tiles 27 us, 640 TFLOP/s.
// One barrier per k-tile.  Addresses are formed once, per vector and not per k-tile, and only the
// last k-tile is masked.  (Addresses and masks formed in every k-tile took more VALU time than the
// MFMAs: 445 us for the block at 4895 x 448 x 1506, forward and backward.)
enum TileEpi { kPlain = 0, kGated = 1, kGatedKeep = 2, kGatedGrad = 3, kLinear = 4 };

constexpr bool gated_epi(int epi) { return epi == kGated || epi == kGatedKeep; }
constexpr bool own_rows(int epi) { return epi == kPlain || epi == kLinear; }  // an output per row of P

struct TileOperand {
  const uint16_t* src;
  int64_t ld;  // between rows (k-contiguous), or between k (row-contiguous)
  int rows;
};

struct TileArgs {
  TileOperand p, q;
  int K;
  uint16_t* out;   // kPlain: D; kGated*: h; kGatedGrad: [dg du]
  int64_t ldc;
  uint16_t* gu;    // kGatedKeep: written; kGatedGrad: read.  The high parts, [q][2F] ...
  uint8_t* low;    // ... and the low ones, [q][F]: g's in bits 0-3, u's in bits 4-7
  int F;           // kGated*: p.src holds F gate rows, then F up rows (p.rows = F)
  int vec;         // 8-byte accesses of out and gu: their addresses and strides are multiples of 4
  float* part;     // kPlain with k split over blockIdx.z: [split][q][p] partials, else null
  int k_split;     // k per split (whole k-tiles)
  int nx, ny, group;  // the grid's tiles along p and along q, and the band of tile_at
  // kLinear
  int act;
  const uint16_t* bias;  // [p] or null
  const uint16_t* res;   // [q][p], row stride ldr, or null
  int64_t ldr;
  void* kept;            // the slopes, written where not null (xdna_linear_kept_bytes)
};

// A workgroup's tile.  Workgroups go to the XCDs (each with its own L2) in turn: XCD c takes the
// c-th eighth of the tiles in an order of splits, then bands of `group` tiles along q, within a
// band q fastest.  The tiles an XCD works on together so form a near-square block of one split,
// whose operands its L2 reads once; in launch order (p fastest) every XCD read all of both:
// 333 x 1000 -> 1367 units 15.0 us and so 12.3, 333 x 2048 -> 1367 23.9 and 18.5.
struct TileAt {
  int x, y, z;
};
__device__ inline TileAt tile_at(const TileArgs& a, int block, int n) {
  const int c = block % kGemmXcds;
  const int t = c * (n / kGemmXcds) + min(c, n % kGemmXcds) + block / kGemmXcds;
  const int plane = a.nx * a.ny, z = t / plane, r = t - z * plane;
  const int band = r / (a.group * a.nx), in = r - band * a.group * a.nx;
  const int high = min(a.group, a.ny - band * a.group);
  return {in / high, band * a.group + in % high, z};
}

// nx x ny tiles in `splits` splits as a grid of tile_at, `together` tiles at work on an XCD
int64_t plan_tiles(TileArgs& a, int64_t nx, int64_t ny, int64_t splits, int together) {
  a.nx = int(nx);
  a.ny = int(ny);
  const int64_t n = std::min({ceil_div(nx * ny * splits, int64_t(kGemmXcds)), nx * ny, int64_t(together)});
  int g = 1;
  while (g < ny && int64_t(g) * g < n) ++g;
  a.group = g;
  return nx * ny * splits;
}

typedef short i16x4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));

template <bool WIDE>
struct Tile {
  static constexpr int T = WIDE ? 128 : 64;        // rows of each operand
  static constexpr int KT = WIDE ? 64 : 128;       // k per k-tile
  static constexpr int NT = WIDE ? 256 : 512;      // threads
  static constexpr int V = T * KT / 8 / NT;        // 16-byte vectors per thread and operand
  static constexpr int NJ = WIDE ? 2 : 1;          // a wave's block: 64 x 32 NJ
  static constexpr int KS = WIDE ? 4 : 2;          // k-steps of a wave per k-tile
  static constexpr int PITCH = KT + 8;             // elements of a k-contiguous LDS row
  static constexpr int ELEMS = T * PITCH;          // (a [k][row] tile is smaller)
  static constexpr size_t LDS = size_t(2) * 2 * ELEMS * 2;
};

// Row of the operand that tile row r holds: itself, or (gated) 32 gate rows and the same 32
// units' up rows in turn, so that one wave has both.  Past the operand: its last row.
template <bool GATED>
__device__ inline int64_t tile_row(const TileArgs& a, const TileOperand& o, int r0, int r) {
  if constexpr (GATED) return min(r0 / 2 + (r >> 6) * 32 + (r & 31), a.F - 1) + int64_t((r >> 5) & 1) * a.F;
  return min(r0 + r, o.rows - 1);
}

// One operand's loads: per thread V vectors of 16 bytes of a k-tile, vector j at from[j] + t step,
// its k offset in the k-tile kq[j].  Every load is whole and none hangs on a branch, so that waiting
// for one k-tile leaves the younger ones in flight.  Results of rows past the operand are not
// stored, so what they multiply does not matter: a vector across a row-contiguous operand's end
// reads on into the next k row.  Only the last k-tile (LAST) needs care: vectors past the end of k
// read the last elements (the last k row) instead and are shifted (cleared) before they are stored,
// and so is a vector across the end of the last k row.
template <bool WIDE, bool ROWS, bool GATED>
struct TileLoads {
  using C = Tile<WIDE>;
  const uint16_t* from[C::V];
  int64_t ld;
  int kq[C::V];
  int over;  // row-contiguous: elements of the vectors past the operand's rows
  bool run;  // 8 elements along the contiguous direction exist

  __device__ inline void plan(const TileArgs& a, const TileOperand& o, int r0, int kbeg, int tid) {
    ld = o.ld;
    run = (ROWS ? o.rows : a.K) >= 8;
    over = 0;
#pragma unroll
    for (int j = 0; j < C::V; ++j) {
      const int i = tid + j * C::NT;
      if constexpr (!ROWS) {
        kq[j] = i % (C::KT / 8) * 8;
        from[j] = o.src + tile_row<GATED>(a, o, r0, i / (C::KT / 8)) * o.ld + kbeg + kq[j];
      } else {  // (NT is a multiple of the vectors along the rows: the same rows for every j)
        int r = r0 + i % (C::T / 8) * 8;
        kq[j] = i / (C::T / 8);
        over = max(r + 8 - o.rows, 0);
        if (r >= o.rows) r = run ? o.rows - 8 : 0, over = run ? 0 : 8;
        from[j] = o.src + int64_t(kbeg + kq[j]) * o.ld + r;
      }
    }
  }

  // The k-tile `t`: `left` is what k has from its start on.
  template <bool LAST>
  __device__ inline void load(Pix8 (&v)[C::V], int t, int left) const {
#pragma unroll
    for (int j = 0; j < C::V; ++j) {
      const uint16_t* p = from[j] + t * (ROWS ? C::KT * ld : int64_t(C::KT));
      if (LAST && left <= C::KT) {
        if (!ROWS) p -= max(kq[j] + 8 - left, 0);
        else if (kq[j] >= left - 1) p -= int64_t(kq[j] - left + 1) * ld + over;
      }
      v[j] = *reinterpret_cast<const Pix8*>(p);
    }
  }

  __device__ inline void align(Pix8 (&v)[C::V], int left) const {
    if (left > C::KT) return;
#pragma unroll
    for (int j = 0; j < C::V; ++j) {
      const int past = kq[j] + (ROWS ? 1 : 8) - left;
      if (past >= (ROWS ? 1 : 8)) v[j] = {{0u, 0u, 0u, 0u}};
      else if (past >= 0) v[j] = shifted(v[j], ROWS ? over : past);
    }
  }

  // load() and align() where an operand has fewer than 8 elements along its contiguous direction
  __device__ inline void load_short(Pix8 (&v)[C::V], int t, int left) const {
#pragma unroll
    for (int j = 0; j < C::V; ++j) {
      const bool in = kq[j] < left;  // (no address is formed for a vector that is not read)
      const uint16_t* p = in ? from[j] + t * (ROWS ? C::KT * ld : int64_t(C::KT)) : from[j];
      v[j] = row_vec(p, !in ? 0 : ROWS ? 8 - over : left - kq[j]);
    }
  }
};

// [k][row] tiles: 16-byte pieces of 8 rows, permuted by the k row so that the transposing reads'
// 4 k rows fall on distinct banks
template <bool WIDE>
__device__ inline int piece_at(int kr, int q) {
  return WIDE ? kr * 16 + (q ^ (4 * (kr & 3))) : kr * 8 + (q ^ (4 * ((kr >> 1) & 1)));
}

template <bool WIDE, bool ROWS>
__device__ inline void tile_store(uint16_t* lds, const Pix8 (&v)[Tile<WIDE>::V], int tid) {
  using C = Tile<WIDE>;
#pragma unroll
  for (int j = 0; j < C::V; ++j) {
    const int i = tid + j * C::NT;
    int at;
    if constexpr (!ROWS) at = i / (C::KT / 8) * C::PITCH + i % (C::KT / 8) * 8;
    else at = piece_at<WIDE>(i / (C::T / 8), i % (C::T / 8)) * 8;
    *reinterpret_cast<uint4*>(lds + at) = make_uint4(v[j].v[0], v[j].v[1], v[j].v[2], v[j].v[3]);
  }
}

// MFMA fragment: rows rb + lane % 32, k = 16 ks + 8 (lane / 32) .. +7
template <bool WIDE, bool ROWS>
__device__ inline bf16x8_t tile_frag(const uint16_t* lds, int rb, int ks, int lane) {
  if constexpr (!ROWS) {
    return as_bf16x8(*reinterpret_cast<const uint4*>(lds + (rb + (lane & 31)) * Tile<WIDE>::PITCH + ks * 16 + (lane >> 5) * 8));
  } else {
    const int g = lane >> 4, j = lane & 15;
    const int kr = 16 * ks + 8 * (g >> 1) + (j >> 2), r = rb + 16 * (g & 1) + 4 * (j & 3);
    const uint16_t* lo = lds + piece_at<WIDE>(kr, r >> 3) * 8 + (r & 7);
    const uint16_t* hi = lds + piece_at<WIDE>(kr + 4, r >> 3) * 8 + (r & 7);
    const u32x2_t a = __builtin_bit_cast(
        u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4_t*)(lo)));
    const u32x2_t b = __builtin_bit_cast(
        u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4_t*)(hi)));
    return as_bf16x8(u32x4_t{a[0], a[1], b[0], b[1]});
  }
}

// An fp32 value rounded to 20 bits (to nearest, ties away), in the high bits.  The sum cannot
// leave a NaN's or an infinity's class: a product of bf16 operands makes NaN with nothing in the
// low half.
__device__ inline uint32_t round20(float v) { return __float_as_uint(v) + 0x800u; }

// g's and u's low 4 bits of 4 units as 4 bytes
__device__ inline uint32_t low_bits(const uint32_t (&g)[4], const uint32_t (&u)[4]) {
  uint32_t b[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) b[e] = ((g[e] >> 12) & 15u) | ((u[e] >> 8) & 0xF0u);
  return (b[0] | b[1] << 8) | (b[2] | b[3] << 8) << 16;
}

// value e of 4 from its bf16 part (of a pair) and the units' low bytes; shift 0 for g, 4 for u
__device__ inline float kept(uint32_t pair, uint32_t low, int e, int shift) {
  const uint32_t hi = e & 1 ? pair & 0xFFFF0000u : pair << 16;
  return __uint_as_float(hi | (((low >> (8 * e + shift)) & 15u) << 12));
}

// n (up to 4) consecutive bf16 at p, as one 8-byte access where `vec`
__device__ inline void put4(uint16_t* p, const float (&v)[4], int n, int vec) {
  if (vec && n >= 4) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack2(v[0], v[1]), pack2(v[2], v[3]));
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < n) p[e] = f32_to_bf16(v[e]);
}

// g and u of 4 units (n of them in range) from the kept parts, and to them
__device__ inline void load_kept(const TileArgs& a, int q, int at, int n, float (&g)[4], float (&u)[4]) {
  const uint16_t* hi = a.gu + int64_t(q) * 2 * a.F + at;
  const uint8_t* lo = a.low + int64_t(q) * a.F + at;
  uint32_t gp[2] = {0, 0}, up[2] = {0, 0}, w = 0;
  if (a.vec && n >= 4) {
    const uint2 g2 = *reinterpret_cast<const uint2*>(hi), u2 = *reinterpret_cast<const uint2*>(hi + a.F);
    gp[0] = g2.x, gp[1] = g2.y, up[0] = u2.x, up[1] = u2.y;
    w = *reinterpret_cast<const uint32_t*>(lo);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n) {
        gp[e >> 1] |= uint32_t(hi[e]) << (16 * (e & 1));
        up[e >> 1] |= uint32_t(hi[a.F + e]) << (16 * (e & 1));
        w |= uint32_t(lo[e]) << (8 * e);
      }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) g[e] = kept(gp[e >> 1], w, e, 0), u[e] = kept(up[e >> 1], w, e, 4);
}

__device__ inline void store_kept(const TileArgs& a, int q, int at, int n, const float (&g)[4], const float (&u)[4]) {
  uint16_t* hi = a.gu + int64_t(q) * 2 * a.F + at;
  uint8_t* lo = a.low + int64_t(q) * a.F + at;
  uint32_t gb[4], ub[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) gb[e] = round20(g[e]), ub[e] = round20(u[e]);
  if (a.vec && n >= 4) {
    const auto pair = [](uint32_t x, uint32_t y) { return (x >> 16) | (y & 0xFFFF0000u); };
    *reinterpret_cast<uint2*>(hi) = make_uint2(pair(gb[0], gb[1]), pair(gb[2], gb[3]));
    *reinterpret_cast<uint2*>(hi + a.F) = make_uint2(pair(ub[0], ub[1]), pair(ub[2], ub[3]));
    *reinterpret_cast<uint32_t*>(lo) = low_bits(gb, ub);
    return;
  }
  const uint32_t w = low_bits(gb, ub);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < n) {
      hi[e] = uint16_t(gb[e] >> 16);
      hi[a.F + e] = uint16_t(ub[e] >> 16);
      lo[e] = uint8_t(w >> (8 * e));
    }
}

constexpr float kSlopeScale = 32768.0f;  // slopes are up to 1.13 in size: 37000 of fp16's 65504

// (The linear layer's activation is a value of the launch: an epilogue's few instructions are cheaper than four copies
// of every tile kernel.)

// N values v (the product's sums and the bias) to the layer's outputs, residual r added, and what is kept of their
// slopes: relu's as bits, the others' as fp16
template <int N>
struct LinearOut {
  float y[N];
  uint16_t slope[N];
  uint32_t bits;
};

template <int N>
__device__ inline LinearOut<N> linear_out(int act, const float (&v)[N], const float (&r)[N]) {
  LinearOut<N> o;
  o.bits = 0;
  if (act == kNone || act == kRelu) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const bool off = v[e] <= 0.0f;  // (a NaN is not: it passes value and gradient, as through the other fused ReLUs)
      o.bits |= off ? 0u : 1u << e;
      o.y[e] = (act == kRelu && off ? 0.0f : v[e]) + r[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float2 t = act == kSilu ? act_pair<kSilu>(v[e]) : act_pair<kGelu>(v[e]);
      o.y[e] = t.x + r[e];
      o.slope[e] = __builtin_bit_cast(uint16_t, static_cast<_Float16>(t.y * kSlopeScale));
    }
  }
  return o;
}

__host__ __device__ inline int64_t bit_bytes(int64_t units) { return (units + 3) / 4; }  // a row of relu's slopes

// 4 consecutive outputs: d0 (and for the gated forward the up projection d1) of row q, from
// column `at` on
template <int EPI, int ACT>
__device__ inline void put_quad(const TileArgs& a, int q, int at, const float (&d0)[4], const float (&d1)[4]) {
  if constexpr (EPI == kPlain) {
    put4(a.out + int64_t(q) * a.ldc + at, d0, a.p.rows - at, a.vec);
  } else if constexpr (EPI == kLinear) {
    const int n = min(a.p.rows - at, 4);
    float v[4], r[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = d0[e] + (a.bias && e < n ? bf16_to_f32(a.bias[at + e]) : 0.0f);
      r[e] = a.res && e < n ? bf16_to_f32(a.res[int64_t(q) * a.ldr + at + e]) : 0.0f;
    }
    const LinearOut<4> o = linear_out(a.act, v, r);
    put4(a.out + int64_t(q) * a.ldc + at, o.y, n, a.vec);
    if (a.kept && a.act == kRelu) {
      static_cast<uint8_t*>(a.kept)[q * bit_bytes(a.p.rows) + at / 4] = uint8_t(o.bits);
    } else if (a.kept) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < n) static_cast<uint16_t*>(a.kept)[int64_t(q) * a.p.rows + at + e] = o.slope[e];
    }
  } else if constexpr (EPI == kGatedGrad) {
    const int n = a.F - at;
    if (n <= 0) return;
    const int64_t row = int64_t(q) * 2 * a.F + at;
    float g[4], u[4], og[4], ou[4];
    load_kept(a, q, at, n, g, u);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 t = act_pair<ACT>(g[e]);
      og[e] = d0[e] * u[e] * t.y;
      ou[e] = d0[e] * t.x;
    }
    put4(a.out + row, og, n, a.vec);
    put4(a.out + row + a.F, ou, n, a.vec);
  } else {
    const int n = a.F - at;
    float h[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = act_of<ACT>(d0[e]) * d1[e];
    put4(a.out + int64_t(q) * a.F + at, h, n, a.vec);
    if constexpr (EPI == kGatedKeep) store_kept(a, q, at, n, d0, d1);
  }
}

struct __attribute__((packed, aligned(4))) Floats4 {  // 16 bytes at any fp32 element
  float v[4];
};

struct __attribute__((packed, aligned(1))) Bytes8 {
  uint32_t v[2];
};

__device__ inline Pix8 pack_vec(const float (&v)[8]) {
  return {{pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7])}};
}

// 8 units' kept projections (n in range), high parts and low bits
__device__ inline void load_kept8(const TileArgs& a, int q, int at, int n, Pix8& g, Pix8& u, Bytes8& low) {
  const uint16_t* hi = a.gu + int64_t(q) * 2 * a.F + at;
  const uint8_t* lo = a.low + int64_t(q) * a.F + at;
  g = row_vec(hi, n);
  u = row_vec(hi + a.F, n);
  if (n >= 8) {
    low = *reinterpret_cast<const Bytes8*>(lo);
    return;
  }
  low = {{0u, 0u}};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < n) low.v[e >> 2] |= uint32_t(lo[e]) << (8 * (e & 3));
}

__device__ inline void store_kept8(const TileArgs& a, int q, int at, int n, const float (&g)[8], const float (&u)[8]) {
  Pix8 gp, up;
  Bytes8 low;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    uint32_t gb[4], ub[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) gb[e] = round20(g[4 * x + e]), ub[e] = round20(u[4 * x + e]);
    low.v[x] = low_bits(gb, ub);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      gp.v[2 * x + e] = (gb[2 * e] >> 16) | (gb[2 * e + 1] & 0xFFFF0000u);
      up.v[2 * x + e] = (ub[2 * e] >> 16) | (ub[2 * e + 1] & 0xFFFF0000u);
    }
  }
  uint16_t* hi = a.gu + int64_t(q) * 2 * a.F + at;
  uint8_t* lo = a.low + int64_t(q) * a.F + at;
  put_vec(hi, gp, n);
  put_vec(hi + a.F, up, n);
  if (n >= 8) {
    *reinterpret_cast<Bytes8*>(lo) = low;
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < n) lo[e] = uint8_t(low.v[e >> 2] >> (8 * (e & 3)));
}

// [dg du] of 8 units from dh and the kept projections
template <int ACT>
__device__ inline void grad8(const float (&d)[8], const Pix8& g, const Pix8& u, const Bytes8& low, float (&dg)[8],
                             float (&du)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float2 t = act_pair<ACT>(kept(g.v[e >> 1], low.v[e >> 2], e & 3, 0));
    dg[e] = d[e] * kept(u.v[e >> 1], low.v[e >> 2], e & 3, 4) * t.y;
    du[e] = d[e] * t.x;
  }
}

__device__ inline void unpack8(const Pix8& p, float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(e & 1 ? p.v[e >> 1] & 0xFFFF0000u : p.v[e >> 1] << 16);
}

// the linear layer's bias at 8 columns (n in range), and a row's residual there
__device__ inline void load_bias8(const TileArgs& a, int at, int n, float (&bias)[8]) {
  const Pix8 none = {{0u, 0u, 0u, 0u}};
  unpack8(a.bias && n > 0 ? row_vec(a.bias + at, n) : none, bias);
}
__device__ inline Pix8 load_res8(const TileArgs& a, int q, int at, int n) {
  const Pix8 none = {{0u, 0u, 0u, 0u}};
  return a.res && n > 0 ? row_vec(a.res + int64_t(q) * a.ldr + at, n) : none;
}

// 8 outputs of the linear layer
__device__ inline void put_linear8(const TileArgs& a, int q, int at, int n, const float (&d)[8], const float (&bias)[8],
                                   const Pix8& res) {
  float v[8], r[8];
  unpack8(res, r);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = d[e] + bias[e];
  const LinearOut<8> o = linear_out(a.act, v, r);
  put_vec(a.out + int64_t(q) * a.ldc + at, pack_vec(o.y), n);
  if (a.kept && a.act == kRelu) {
    uint8_t* to = static_cast<uint8_t*>(a.kept) + q * bit_bytes(a.p.rows) + at / 4;
    to[0] = uint8_t(o.bits & 15u);
    if (n > 4) to[1] = uint8_t(o.bits >> 4);
  } else if (a.kept) {
    Pix8 s;
#pragma unroll
    for (int e = 0; e < 4; ++e) s.v[e] = uint32_t(o.slope[2 * e]) | uint32_t(o.slope[2 * e + 1]) << 16;
    put_vec(static_cast<uint16_t*>(a.kept) + int64_t(q) * a.p.rows + at, s, n);
  }
}

// 8 consecutive outputs of row q from column `at` on (n of them in range): d0, and for the gated
// forward the up projection d1
template <int EPI, int ACT>
__device__ inline void put_row8(const TileArgs& a, int q, int at, int n, const float (&d0)[8], const float (&d1)[8], int split) {
  if constexpr (own_rows(EPI)) {
    if (a.part) {
      float* to = a.part + (int64_t(split) * a.q.rows + q) * a.p.rows + at;
      if (n >= 8) {
        *reinterpret_cast<Floats4*>(to) = {{d0[0], d0[1], d0[2], d0[3]}};
        *reinterpret_cast<Floats4*>(to + 4) = {{d0[4], d0[5], d0[6], d0[7]}};
        return;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n) to[e] = d0[e];
      return;
    }
    put_vec(a.out + int64_t(q) * a.ldc + at, pack_vec(d0), n);
  } else if constexpr (EPI == kGatedGrad) {
    Pix8 g, u;
    Bytes8 low;
    load_kept8(a, q, at, n, g, u, low);
    float dg[8], du[8];
    grad8<ACT>(d0, g, u, low, dg, du);
    uint16_t* to = a.out + int64_t(q) * 2 * a.F + at;
    put_vec(to, pack_vec(dg), n);
    put_vec(to + a.F, pack_vec(du), n);
  } else {
    float h[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = act_of<ACT>(d0[e]) * d1[e];
    put_vec(a.out + int64_t(q) * a.F + at, pack_vec(h), n);
    if constexpr (EPI == kGatedKeep) store_kept8(a, q, at, n, d0, d1);
  }
}

// The linear layer's outputs of 8 columns from `at` on (n of them in range), rows r0, r0 + STEP, .. of ROWS: row(r) is
// row r's place in the output, sum(r, e) its product.  The bias is loaded once, the residual of four rows at a time from
// clamped places (row by row, each waited for its own: the epilogue of 8192 x 1024 -> 4096 took twice the k-loop).
template <int ROWS, int STEP, class Row, class Sum>
__device__ inline void put_linear_rows(const TileArgs& a, int r0, const Row& row, int at, int n, const Sum& sum) {
  constexpr int B = ROWS / STEP < 4 ? ROWS / STEP : 4;
  float bias[8];
  load_bias8(a, at, n, bias);
#pragma unroll 1
  for (int r = r0; r < ROWS; r += B * STEP) {
    Pix8 res[B];
#pragma unroll
    for (int u = 0; u < B; ++u) res[u] = load_res8(a, min(row(r + u * STEP), a.q.rows - 1), at, n);
#pragma unroll
    for (int u = 0; u < B; ++u) {
      const int q = row(r + u * STEP);
      float d[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = sum(r + u * STEP, e);
      if (q < a.q.rows) put_linear8(a, q, at, n, d, bias, res[u]);
    }
  }
}

// One tile, by a workgroup.
template <bool WIDE, bool PROWS, bool QROWS, int EPI, int ACT>
__device__ inline void tile_block(const TileArgs& a, const TileAt tile) {
  using C = Tile<WIDE>;
  constexpr bool GATED = gated_epi(EPI);
  extern __shared__ __attribute__((aligned(16))) uint16_t smem[];  // [2 buffers][P, Q]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wp = WIDE ? wave & 1 : 0, wq = WIDE ? wave >> 1 : wave & 1, wk = WIDE ? 0 : wave >> 1;
  const int p0 = tile.x * C::T, q0 = tile.y * C::T;
  f32x16_t acc[2][C::NJ];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < C::NJ; ++j) acc[i][j] = zero_acc();
  const int kbeg = own_rows(EPI) && a.part ? tile.z * a.k_split : 0;
  const int klen = (own_rows(EPI) && a.part ? min(a.K, kbeg + a.k_split) : a.K) - kbeg;
  TileLoads<WIDE, PROWS, GATED> lp;
  TileLoads<WIDE, QROWS, false> lq;
  lp.plan(a, a.p, p0, kbeg, tid);
  lq.plan(a, a.q, q0, kbeg, tid);
  const int tiles = (klen + C::KT - 1) / C::KT;
  const auto put = [&](const Pix8 (&rp)[C::V], const Pix8 (&rq)[C::V], int b) {
    uint16_t* to = smem + b * 2 * C::ELEMS;
    tile_store<WIDE, PROWS>(to, rp, tid);
    tile_store<WIDE, QROWS>(to + C::ELEMS, rq, tid);
  };
  const auto multiply = [&](int b) {
    const uint16_t* ps = smem + b * 2 * C::ELEMS;
    const uint16_t* qs = ps + C::ELEMS;
#pragma unroll
    for (int s = 0; s < C::KS; ++s) {
      const int ks = wk * C::KS + s;
      bf16x8_t fp[2], fq[C::NJ];
#pragma unroll
      for (int i = 0; i < 2; ++i) fp[i] = tile_frag<WIDE, PROWS>(ps, wp * 64 + i * 32, ks, lane);
#pragma unroll
      for (int j = 0; j < C::NJ; ++j) fq[j] = tile_frag<WIDE, QROWS>(qs, (wq * C::NJ + j) * 32, ks, lane);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < C::NJ; ++j) acc[i][j] = mfma_32x32x16(fp[i], fq[j], acc[i][j]);
    }
  };
  if (lp.run && lq.run) {
    Pix8 rp[2][C::V], rq[2][C::V];  // k-tile t's loads in set t % 2, its LDS buffer too
    const auto load = [&](int set, int t) {
      lp.template load<false>(rp[set], t, 0);
      lq.template load<false>(rq[set], t, 0);
    };
    const auto load_end = [&](int set, int t) {
      lp.template load<true>(rp[set], t, a.K - kbeg - t * C::KT);
      lq.template load<true>(rq[set], t, a.K - kbeg - t * C::KT);
    };
    const auto put_end = [&](int set, int t) {
      lp.align(rp[set], a.K - kbeg - t * C::KT);
      lq.align(rq[set], a.K - kbeg - t * C::KT);
      put(rp[set], rq[set], set);
    };
    load_end(0, 0);
    if (tiles > 1) load_end(1, 1);
    put_end(0, 0);
    __syncthreads();
    int t = 0;
    for (; t + 4 < tiles; t += 2) {  // (neither loads nor stores the last k-tile)
#pragma unroll
      for (int d = 0; d < 2; ++d) {
        load(d, t + d + 2);
        multiply(d);
        put(rp[d ^ 1], rq[d ^ 1], d ^ 1);  // that buffer's last reads ended before the previous barrier
        __syncthreads();
      }
    }
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      if (t + d < tiles) {
        if (d < 2 && t + d + 2 < tiles) load_end(d, t + d + 2);
        multiply(d & 1);
        if (t + d + 1 < tiles) put_end((d + 1) & 1, t + d + 1);
        __syncthreads();
      }
    }
  } else {
    for (int t = 0; t < tiles; ++t) {
      Pix8 rp[C::V], rq[C::V];
      lp.load_short(rp, t, a.K - kbeg - t * C::KT);
      lq.load_short(rq, t, a.K - kbeg - t * C::KT);
      put(rp, rq, t & 1);
      __syncthreads();
      multiply(t & 1);
    }
    __syncthreads();
  }
  // the block as [q][p] in fp32.  Accumulator quad (i, j, g): p 32 i + 8 g + 4 (lane / 32) .. +3,
  // q 32 j + lane % 32 of the wave's block.
  constexpr int EP = C::T + 4;  // (a quad's 16 rows on distinct banks)
  float* block = reinterpret_cast<float*>(smem);
  if constexpr (WIDE) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<float4*>(block + (wq * 64 + j * 32 + (lane & 31)) * EP + wp * 64 + i * 32 + 8 * g + 4 * (lane >> 5)) =
              make_float4(acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]);
  } else {
    // the eight waves' quads [wave][i][g][lane] in 64 KB, the four k parts of each summed by a
    // thread per (q half, g, lane) of both i
    float4* red = reinterpret_cast<float4*>(smem);
    const int g = wave & 3, half = wave >> 2;
    float4 sum[2];
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int y = 0; y < 4; ++y)
        red[((wave * 2 + x) * 4 + y) * 64 + lane] =
            make_float4(acc[x][0][4 * y], acc[x][0][4 * y + 1], acc[x][0][4 * y + 2], acc[x][0][4 * y + 3]);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      sum[i] = red[((half * 2 + i) * 4 + g) * 64 + lane];
#pragma unroll
      for (int w = 1; w < 4; ++w) {
        const float4 v = red[(((w * 2 + half) * 2 + i) * 4 + g) * 64 + lane];
        sum[i].x += v.x, sum[i].y += v.y, sum[i].z += v.z, sum[i].w += v.w;
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i)
      *reinterpret_cast<float4*>(block + (half * 32 + (lane & 31)) * EP + i * 32 + 8 * g + 4 * (lane >> 5)) = sum[i];
  }
  __syncthreads();
  // rows in windows of 8 outputs, consecutive threads along a row
  constexpr int kAcross = (GATED ? C::T / 2 : C::T) / 8;
  const int o = tid % kAcross;
  const int at = (GATED ? p0 / 2 : p0) + 8 * o, n = (own_rows(EPI) ? a.p.rows : a.F) - at;
  const float* from = block + (GATED ? (o >> 2) * 64 + (o & 3) * 8 : 8 * o);
  if (n <= 0) return;
  if constexpr (EPI == kLinear) {
    if (!a.part) {
      put_linear_rows<C::T, C::NT / kAcross>(a, tid / kAcross, [&](int r) { return q0 + r; }, at, n,
                                             [&](int r, int e) { return from[r * EP + e]; });
      return;
    }
  }
#pragma unroll 2
  for (int r = tid / kAcross; r < C::T; r += C::NT / kAcross) {
    if (q0 + r >= a.q.rows) break;
    float d0[8], d1[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) d0[e] = from[r * EP + e], d1[e] = GATED ? from[r * EP + 32 + e] : 0.0f;
    put_row8<EPI, ACT>(a, q0 + r, at, n, d0, d1, tile.z);
  }
}

template <bool WIDE, bool PROWS, bool QROWS, int EPI, int ACT>
__global__ __launch_bounds__(Tile<WIDE>::NT, WIDE ? 2 : 4) void tile_kernel(TileArgs a) {
  tile_block<WIDE, PROWS, QROWS, EPI, ACT>(a, tile_at(a, int(blockIdx.x), int(gridDim.x)));
}

// The block's gradients that follow dgu, dx = dgu w_in, dw_in = dgu^T x and dw_out = dy^T h, in one
// launch: at few hundred rows each alone has too few tiles or too few k-tiles to fill the chip, and
// its last round and its launch cost as much as its work.  The products with the longer k go first.
struct GradsArgs {
  TileArgs dx, dw_in, dw_out;
  int n_dx, n_in, n_out;  // tiles of each
  int dx_first;
};

template <bool WIDE>
__global__ __launch_bounds__(Tile<WIDE>::NT, WIDE ? 2 : 4) void grads_kernel(GradsArgs g) {
  const int i = int(blockIdx.x) - (g.dx_first ? g.n_dx : 0), n_w = g.n_in + g.n_out;
  if (i >= 0 && i < n_w) {
    const bool in = i < g.n_in;
    const TileArgs& a = in ? g.dw_in : g.dw_out;
    tile_block<WIDE, true, true, kPlain, kSilu>(a, tile_at(a, in ? i : i - g.n_in, in ? g.n_in : g.n_out));
  } else {
    tile_block<WIDE, true, false, kPlain, kSilu>(g.dx, tile_at(g.dx, i < 0 ? int(blockIdx.x) : i - n_w, g.n_dx));
  }
}

// out[q][p] = the partials of the k splits, added in order, four outputs a thread (Z splits'
// loads in flight)
template <int Z>
__global__ __launch_bounds__(256) void tile_join_kernel(TileArgs a, int splits) {
  const int64_t n = int64_t(a.q.rows) * a.p.rows;
  for (int64_t i = (int64_t(blockIdx.x) * 256 + threadIdx.x) * 4; i < n; i += int64_t(gridDim.x) * 1024) {
    float d[4] = {};
    const int m = int(n - i < 4 ? n - i : 4);
    for (int z = 0; z < splits; z += Z) {
      Floats4 v[Z];
#pragma unroll
      for (int u = 0; u < Z; ++u) {
        const float* p = a.part + int64_t(min(z + u, splits - 1)) * n + i;
        if (m == 4) {
          v[u] = *reinterpret_cast<const Floats4*>(p);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[u].v[e] = e < m ? p[e] : 0.0f;
        }
      }
#pragma unroll
      for (int u = 0; u < Z; ++u)
        if (z + u < splits) d[0] += v[u].v[0], d[1] += v[u].v[1], d[2] += v[u].v[2], d[3] += v[u].v[3];
    }
    if (a.ldc == a.p.rows && m == 4) {
      *reinterpret_cast<Pix4*>(a.out + i) = {pack2(d[0], d[1]), pack2(d[2], d[3])};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < m) {
          const int64_t q = (i + e) / a.p.rows;
          a.out[q * a.ldc + (i + e - q * a.p.rows)] = f32_to_bf16(d[e]);
        }
    }
  }
}

// The same for the linear layer: a thread per window of 8 outputs of a row.
__global__ __launch_bounds__(256) void linear_join_kernel(TileArgs a, int splits) {
  const int windows = (a.p.rows + 7) / 8;
  const int64_t total = int64_t(a.q.rows) * windows, plane = int64_t(a.q.rows) * a.p.rows;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < total; i += int64_t(gridDim.x) * 256) {
    const int q = int(i / windows), at = int(i - int64_t(q) * windows) * 8, n = min(a.p.rows - at, 8);
    const float* from = a.part + int64_t(q) * a.p.rows + at;
    float d[8] = {};
    for (int z = 0; z < splits; z += 4) {
      Floats4 v[4][2];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float* p = from + int64_t(min(z + u, splits - 1)) * plane;
        if (n == 8) {
          v[u][0] = *reinterpret_cast<const Floats4*>(p);
          v[u][1] = *reinterpret_cast<const Floats4*>(p + 4);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[u][e >> 2].v[e & 3] = e < n ? p[e] : 0.0f;
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (z + u < splits) {
#pragma unroll
          for (int e = 0; e < 8; ++e) d[e] += v[u][e >> 2].v[e & 3];
        }
    }
    float bias[8];
    load_bias8(a, at, n, bias);
    put_linear8(a, q, at, n, d, bias, load_res8(a, q, at, n));
  }
}

// dp = dy act'(v) from the kept slopes (null: 1), rounded once, and the column sums of the products
// before that rounding, for the bias: a workgroup takes 256 columns of every gridDim.y-th 8 rows, 32
// threads of 8 columns a row, and writes its sums as partials [gridDim.y][N].
struct LinearBwdArgs {
  const uint16_t* dy;     // [M][N], row stride ld
  int64_t ld;
  const void* kept;       // as the forward wrote them
  int bits;               // relu's
  uint16_t* dp;           // dense, or null
  float* part;            // or null
  int M, N;
};

__global__ __launch_bounds__(256) void linear_bwd_kernel(LinearBwdArgs a) {
  __shared__ float red[8][256];
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int at = blockIdx.x * 256 + lane * 8, n = min(a.N - at, 8);
  const int64_t bit_ld = bit_bytes(a.N);
  float sum[8] = {};
  if (n > 0) {
    const int step = gridDim.y * 8;
    for (int64_t q0 = int64_t(blockIdx.y) * 8 + row; q0 < a.M; q0 += 4 * int64_t(step)) {
      Pix8 d[4], k[4];
      uint32_t bits[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {  // (rows past the end: the last one again, unused)
        const int64_t q = min(q0 + int64_t(u) * step, int64_t(a.M - 1));
        d[u] = row_vec(a.dy + q * a.ld + at, n);
        if (a.bits) {
          const uint8_t* p = static_cast<const uint8_t*>(a.kept) + q * bit_ld + at / 4;
          bits[u] = p[0] | uint32_t(p[n > 4 ? 1 : 0]) << 4;
        } else if (a.kept) {
          k[u] = row_vec(static_cast<const uint16_t*>(a.kept) + q * a.N + at, n);
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t q = q0 + int64_t(u) * step;
        if (q >= a.M) break;
        float g[8];
        unpack8(d[u], g);
        if (a.bits) {  // (selected: a unit that is off has gradient 0, whatever dy is there)
#pragma unroll
          for (int e = 0; e < 8; ++e) g[e] = (bits[u] >> e) & 1u ? g[e] : 0.0f;
        } else if (a.kept) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            g[e] *= float(__builtin_bit_cast(_Float16, uint16_t(k[u].v[e >> 1] >> (16 * (e & 1))))) * (1.0f / kSlopeScale);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += g[e];
        if (a.dp) put_vec(a.dp + q * a.N + at, pack_vec(g), n);
      }
    }
  }
  if (!a.part) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) red[row][lane * 8 + e] = sum[e];
  __syncthreads();
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.N) return;
  float s = 0.0f;
#pragma unroll
  for (int r = 0; r < 8; ++r) s += red[r][threadIdx.x];
  a.part[int64_t(blockIdx.y) * a.N + c] = s;
}

// d_bias: the partials in order, 64 columns a workgroup, 16 waves
__global__ __launch_bounds__(1024) void linear_bias_kernel(const float* part, int parts, int N, uint16_t* d_bias) {
  __shared__ float red[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane;
  red[wave][lane] = c < N ? sum_strided8(0.0f, part + c, N, wave, 16, parts) : 0.0f;
  __syncthreads();
  if (wave != 0 || c >= N) return;
  float s = 0.0f;
#pragma unroll
  for (int w = 0; w < 16; ++w) s += red[w][lane];
  d_bias[c] = f32_to_bf16(s);
}

// ---- few rows -------------------------------------------------------------------------------------
// A step of decoding: bound by the weights' bytes, which pass once from memory to registers.  A
// workgroup takes 16 units (their gate and up rows) or `span` plain rows as the rows of 16x16x32
// MFMAs, its eight waves every eighth k-step, with the loads of up to 8 steps in flight; x's
// fragments come from L2.  The waves' sums are added in wave order through LDS.  (Sixteen waves
// were slower: 6.7 -> 7.3 us for 1 x 4096 -> 1024, 4.1 -> 4.6 for 1 x 1024 -> 4096.)  1 x 1024 ->
// 4096 units takes 5.9 us (16.8 MB, 2.8 TB/s with the launch), the product back 4.4; in narrow tiles
// 7.3 and 9.1.  32 rows 5.9 and 7.4; at 64 the two meet: 1024 -> 4096 8.2 and 7.4, 1000 -> 300 6.2
// and 7.5.
//   Fewer than 16 plain rows a workgroup (the MFMA's other rows repeat them) put every CU to work
// where there are few.  With up to 4 rows of x the repeats become useful: MFMA row (c, i) holds
// weight row i and column (c', m) row m of x, both at the c-th or c'-th of 4 chunks of 32 k, so
// that a load reads 1 KB of weights instead of 256 bytes; the products with c == c' are the sum's
// terms, the others are dropped.
constexpr int kFewGated = 64, kFewPlain = 16;  // most rows of x

template <int MT, int CH, int EPI, int ACT>
__global__ __launch_bounds__(512) void few_kernel(TileArgs a) {
  constexpr bool GATED = gated_epi(EPI);
  constexpr int PT = GATED ? 2 : 1, WAVES = 8, STEP = 32 * CH;
  extern __shared__ __attribute__((aligned(16))) float4 red[];  // [wave][PT][MT][lane]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int span = GATED ? 16 : CH > 1 ? 4 : a.F;  // units of the workgroup: 16, 8 or 4
  const int p0 = blockIdx.x * span, r = lane & 15;
  const int kq = (lane >> 4) * 8 + (CH > 1 ? (r >> 2) * 32 : 0);
  const uint16_t* wp[PT];
  const uint16_t* xp[MT];
  const int units = GATED ? a.F : a.p.rows;
#pragma unroll
  for (int p = 0; p < PT; ++p) wp[p] = a.p.src + (int64_t(min(p0 + (r & (span - 1)), units - 1)) + int64_t(p) * a.F) * a.p.ld + kq;
#pragma unroll
  for (int t = 0; t < MT; ++t) xp[t] = a.q.src + int64_t(min(t * 16 + (CH > 1 ? r & 3 : r), a.q.rows - 1)) * a.q.ld + kq;
  f32x4_t acc[PT][MT];
#pragma unroll
  for (int p = 0; p < PT; ++p)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[p][t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  const auto frag = [](const Pix8& v) { return as_bf16x8(u32x4_t{v.v[0], v.v[1], v.v[2], v.v[3]}); };
  const auto multiply = [&](const Pix8 (&w)[PT], const Pix8 (&x)[MT]) {
#pragma unroll
    for (int p = 0; p < PT; ++p)
#pragma unroll
      for (int t = 0; t < MT; ++t)
        acc[p][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(frag(w[p]), frag(x[t]), acc[p][t], 0, 0, 0);
  };
  const int whole = a.K / STEP;  // steps without a ragged end
  const auto batch = [&](int s0, auto steps) {
    constexpr int U = decltype(steps)::value;
    Pix8 w[U][PT], x[U][MT];
#pragma unroll
    for (int i = 0; i < U; ++i) {  // (steps past the end load the last one again, unused)
      const int k = min(s0 + i * WAVES, whole - 1) * STEP;
#pragma unroll
      for (int p = 0; p < PT; ++p) w[i][p] = *reinterpret_cast<const Pix8*>(wp[p] + k);
#pragma unroll
      for (int t = 0; t < MT; ++t) x[i][t] = *reinterpret_cast<const Pix8*>(xp[t] + k);
    }
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (s0 + i * WAVES < whole) multiply(w[i], x[i]);
  };
  int s0 = wave;
  if constexpr (MT == 1)
    for (; s0 + 7 * WAVES < whole; s0 += 8 * WAVES) batch(s0, std::integral_constant<int, 8>{});
  for (; s0 < whole; s0 += 4 * WAVES) batch(s0, std::integral_constant<int, 4>{});
  if (whole * STEP < a.K && whole % WAVES == wave) {
    const int n = a.K - whole * STEP - kq;
    Pix8 w[PT], x[MT];
#pragma unroll
    for (int p = 0; p < PT; ++p) w[p] = row_vec(wp[p] - kq + min(whole * STEP + kq, a.K), max(n, 0));
#pragma unroll
    for (int t = 0; t < MT; ++t) x[t] = row_vec(xp[t] - kq + min(whole * STEP + kq, a.K), max(n, 0));
    multiply(w, x);
  }
#pragma unroll
  for (int p = 0; p < PT; ++p)
#pragma unroll
    for (int t = 0; t < MT; ++t)
      red[((wave * PT + p) * MT + t) * 64 + lane] = make_float4(acc[p][t][0], acc[p][t][1], acc[p][t][2], acc[p][t][3]);
  __syncthreads();
  if constexpr (CH > 1) {
    // rows m of x by thread; chunk c's terms are with lanes 16 c + 4 c + m
    if (tid >= 4 || tid >= a.q.rows || p0 >= units) return;
    float d[4] = {}, none[4] = {};
#pragma unroll
    for (int w = 0; w < WAVES; ++w)
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const float4 v = red[w * 64 + 20 * c + tid];
        d[0] += v.x, d[1] += v.y, d[2] += v.z, d[3] += v.w;
      }
    put_quad<EPI, ACT>(a, tid, p0, d, none);
    return;
  }
  if (tid >= MT * 64) return;
  const int t = tid >> 6, q = t * 16 + r, at = p0 + 4 * (lane >> 4);
  if (q >= a.q.rows || at >= units || 4 * (lane >> 4) >= span) return;
  float d[2][4] = {};
#pragma unroll
  for (int p = 0; p < PT; ++p)
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float4 v = red[((w * PT + p) * MT + t) * 64 + lane];
      d[p][0] += v.x, d[p][1] += v.y, d[p][2] += v.z, d[p][3] += v.w;
    }
  put_quad<EPI, ACT>(a, q, at, d[0], d[1]);
}

// ---- large tiles --------------------------------------------------------------------------------
// The 256 x 256 tile of the library's large products (gemm_dma.h): operands that can be loaded as
// whole 16-byte vectors by the LDS DMA.  Rows of P (the hidden units) run along the MFMA's rows:
// a lane's accumulator quad is 4 consecutive units of one row of x.  For the projections P's tile
// rows hold 16 gate rows and the same 16 units' up rows in turn, so that one tile has both
// projections of 128 units.  One workgroup a CU (the accumulators take half the registers), so that
// nothing runs beside an epilogue: 8192 x 1024 -> 4096 with the kept projections takes 171 us (805
// TFLOP/s; its k-loop alone runs at about 1.1 PFLOP/s, the epilogue writes 235 MB), [dg du] from dy
// 139 us (the same bytes read, and 134 MB written).
template <bool ROWS>
constexpr int kDmaMode = ROWS ? kAlongRow : kAlongK;

// DMA plan of P = w for the projections: tile row r is unit f0 + 16 (r / 32) + r % 16, its gate
// row for even r / 16 and its up row for odd.
__device__ inline G5Operand gated_operand(const TileArgs& a, int f0, int tid) {
  G5Operand o = g5_operand<kAlongK, true>(a.p.src, a.p.ld, 1, 0, 2 * a.F, a.K, tid);
  const int lane = tid & 63, w = tid >> 6;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int j = 4 * w + i;  // tile rows 16 j .. 16 j + 15, lane L at row 16 j + L / 4
    const int f = f0 + 16 * (j >> 1) + (lane >> 2);
    o.roff[i] = f < a.F ? int((f + int64_t(j & 1) * a.F) * a.p.ld) : -1;
  }
  return o;
}

// The epilogue passes the accumulators through LDS, 128 rows of x at a time ([row][256 tile rows of
// P] in fp32, pitch 260: quads of 16 rows on distinct banks), so that every global access is 16
// bytes of a 256- or 512-byte run and the code is a short loop: stored straight from the
// accumulators (8-byte quads, straight-line code) the forward's epilogue took as long as the k-loop
// at K = 1024.
constexpr int kEpiRows = 128, kEpiPitch = kT4 + 4;
constexpr size_t kLargeLds = std::max(kGemm5Lds, size_t(kEpiRows) * kEpiPitch * 4);

template <bool PROWS, int EPI, int ACT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1)))
void gated_large_kernel(TileArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint16_t smem[];
  constexpr bool GATED = gated_epi(EPI);
  const int units = EPI == kLinear ? a.p.rows : a.F;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = wave & 1, wn = wave >> 1;
  const TileAt tile = tile_at(a, int(blockIdx.x), int(gridDim.x));
  const int f0 = tile.x * (GATED ? kT4 / 2 : kT4), q0 = tile.y * kT4;
  f32x4_t acc[8][8];
  {
    G5Operand op;
    if constexpr (GATED) op = gated_operand(a, f0, tid);
    else if constexpr (PROWS) op = g5_operand<kAlongRow, true>(a.p.src, 1, a.p.ld, f0, units, a.K, tid);
    else op = g5_operand<kAlongK, true>(a.p.src, a.p.ld, 1, f0, units, a.K, tid);
    const G5Operand oq = g5_operand<kAlongK, true>(a.q.src, a.q.ld, 1, q0, a.q.rows, a.K, tid);
    gemm6_loop<kDmaMode<PROWS>, kAlongK>(acc, op, oq, smem, 0, a.K, tid);
  }
  mfma16_fence(acc);
  float* epi = reinterpret_cast<float*>(smem);
  // threads of a row, 8 units each; rows per round
  constexpr int kAcross = (GATED ? kT4 / 2 : kT4) / 8, kRound = 256 / kAcross;
  const int o = tid % kAcross, rr = tid / kAcross;
  const int f = f0 + 8 * o;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    __syncthreads();  // the k-loop's (or the last half's) LDS reads are done
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        *reinterpret_cast<f32x4_t*>(epi + (wn * 64 + j * 16 + (lane & 15)) * kEpiPitch + wm * 128 + i * 16 + 4 * (lane >> 4)) =
            acc[i][half * 4 + j];
    __syncthreads();
    // LDS row r is row 128 (r / 64) + 64 half + r % 64 of the tile
    const auto row = [&](int r) { return q0 + 128 * (r >> 6) + 64 * half + (r & 63); };
    if constexpr (GATED) {
      const float* at = epi + (o >> 1) * 32 + (o & 1) * 8;
#pragma unroll 2
      for (int r = rr; r < kEpiRows; r += kRound) {
        float g[8], u[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = at[r * kEpiPitch + e], u[e] = at[r * kEpiPitch + 16 + e];
        if (row(r) < a.q.rows && f < a.F) put_row8<EPI, ACT>(a, row(r), f, 8, g, u, 0);
      }
    } else if constexpr (EPI == kLinear) {
      if (f < units)
        put_linear_rows<kEpiRows, kRound>(a, rr, row, f, min(units - f, 8),
                                          [&](int r, int e) { return epi[r * kEpiPitch + 8 * o + e]; });
    } else {
      // four rows' [g u] in flight: clamped addresses, no branch around the loads
#pragma unroll 1
      for (int r = rr; r < kEpiRows; r += 4 * kRound) {
        Pix8 kg[4], ku[4];
        Bytes8 kl[4];
#pragma unroll
        for (int n = 0; n < 4; ++n)
          load_kept8(a, min(row(r + n * kRound), a.q.rows - 1), min(f, a.F - 8), 8, kg[n], ku[n], kl[n]);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int q = row(r + n * kRound);
          float d[8], og[8], ou[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) d[e] = epi[(r + n * kRound) * kEpiPitch + 8 * o + e];
          grad8<ACT>(d, kg[n], ku[n], kl[n], og, ou);
          if (q < a.q.rows && f < a.F) {
            uint16_t* to = a.out + int64_t(q) * 2 * a.F + f;
            put_vec(to, pack_vec(og), 8);
            put_vec(to + a.F, pack_vec(ou), 8);
          }
        }
      }
    }
  }
}

// ---- dx and dw of a large linear layer in one launch -----------------------------------------
// The two products' 256 x 256 tiles, k split so that all of them are at work at once and end together: one by one, each
// is split to fill the CUs by itself, and both have their partials to write and add.
struct LargeGradsArgs {
  TileArgs dx, dw;
  int n_dx, n_dw;  // workgroups of each
};

template <bool QROWS>
__device__ __forceinline__ void large_plain(const TileArgs& a, const TileAt tile, uint16_t* smem) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = wave & 1, wn = wave >> 1;
  const int p0 = tile.x * kT4, q0 = tile.y * kT4, kbeg = tile.z * a.k_split;
  f32x4_t acc[8][8];
  {
    const G5Operand op = g5_operand<kAlongRow, true>(a.p.src, 1, a.p.ld, p0, a.p.rows, a.K, tid);
    G5Operand oq;
    if constexpr (QROWS) oq = g5_operand<kAlongRow, true>(a.q.src, 1, a.q.ld, q0, a.q.rows, a.K, tid);
    else oq = g5_operand<kAlongK, true>(a.q.src, a.q.ld, 1, q0, a.q.rows, a.K, tid);
    gemm6_loop<kAlongRow, kDmaMode<QROWS>>(acc, op, oq, smem, kbeg, min(a.K, kbeg + a.k_split), tid);
  }
  mfma16_fence(acc);
  float* epi = reinterpret_cast<float*>(smem);
  const int o = tid & 31, at = p0 + 8 * o;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        *reinterpret_cast<f32x4_t*>(epi + (wn * 64 + j * 16 + (lane & 15)) * kEpiPitch + wm * 128 + i * 16 + 4 * (lane >> 4)) =
            acc[i][half * 4 + j];
    __syncthreads();
#pragma unroll 4
    for (int r = tid >> 5; r < kEpiRows; r += 8) {
      const int q = q0 + 128 * (r >> 6) + 64 * half + (r & 63);
      float d[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = epi[r * kEpiPitch + 8 * o + e];
      if (q < a.q.rows && at < a.p.rows) put_row8<kPlain, kSilu>(a, q, at, a.p.rows - at, d, d, tile.z);
    }
  }
}

__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1)))
void linear_grads_large_kernel(LargeGradsArgs g) {
  extern __shared__ __attribute__((aligned(16))) uint16_t smem[];
  const int i = int(blockIdx.x);
  if (i < g.n_dx) large_plain<false>(g.dx, tile_at(g.dx, i, g.n_dx), smem);
  else large_plain<true>(g.dw, tile_at(g.dw, i - g.n_dx, g.n_dw), smem);
}

// ---- backward, elementwise: [dg du] from dh and the kept [g u] ------------------------------
// Bound by its bytes: 8192 x 4096 units, 370 MB, take 65 us (5.7 TB/s).
struct GatedBwdArgs {
  const uint16_t* dh;  // [M][F], row stride ld
  int64_t ld;
  TileArgs t;          // out: [dg du], gu, low, F, vec; q.rows: M
  int windows;         // windows of 4 per row
};

template <int ACT>
__global__ __launch_bounds__(256) void gated_bwd_kernel(GatedBwdArgs a) {
  const int64_t total = int64_t(a.t.q.rows) * a.windows;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < total; i += int64_t(gridDim.x) * 256) {
    const int q = int(i / a.windows);
    const int f = int(i - int64_t(q) * a.windows) * 4;
    const uint16_t* p = a.dh + q * a.ld + f;
    float d[4], none[4];
    const int n = min(4, a.t.F - f);
    if (n == 4) {
      const Pix4 v = *reinterpret_cast<const Pix4*>(p);
      d[0] = __uint_as_float(v.lo << 16), d[1] = __uint_as_float(v.lo & 0xFFFF0000u);
      d[2] = __uint_as_float(v.hi << 16), d[3] = __uint_as_float(v.hi & 0xFFFF0000u);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) d[e] = e < n ? bf16_to_f32(p[e]) : 0.0f;
    }
    put_quad<kGatedGrad, ACT>(a.t, q, f, d, none);
  }
}

int refuse(const char* what, const char* why) {
  set_error(std::string(what) + ": " + why);
  return -1;
}

constexpr int64_t kMaxSide = int64_t(1) << 30;
constexpr int64_t kMaxRows = int64_t(1) << 22;  // of x; of a plain product's second operand
constexpr int64_t kMaxOutputs = int64_t(1) << 42;  // (2^28 wide tiles: a grid has under 2^31)

const char* gated_fault(int64_t M, int64_t K, int64_t F, int act) {
  if (act < 0 || act > 2) return "activation must be 0 (silu), 1 (gelu) or 2 (relu)";
  if (M < 0 || M > kMaxSide || K < 1 || K > kMaxSide || F < 1 || F > kMaxSide / 2) return "sizes outside 1 .. 2^30";
  if (M > kMaxRows) return "too many rows";
  if (M * F > kMaxOutputs) return "too many outputs";
  return nullptr;
}

bool odd(const void* p) { return reinterpret_cast<uintptr_t>(p) & 1; }

template <bool WIDE, bool PROWS, bool QROWS, int EPI, int ACT>
bool launch_tile(TileArgs a, dim3 tiles, hipStream_t st) {
  using C = Tile<WIDE>;
  void (*f)(TileArgs) = tile_kernel<WIDE, PROWS, QROWS, EPI, ACT>;
  static const bool ok = hipFuncSetAttribute(reinterpret_cast<const void*>(f), hipFuncAttributeMaxDynamicSharedMemorySize,
                                             int(C::LDS)) == hipSuccess;
  if (!ok) return false;
  f<<<unsigned(plan_tiles(a, tiles.x, tiles.y, tiles.z, 64)), C::NT, C::LDS, st>>>(a);
  return true;
}

template <int MT, int CH, int EPI, int ACT>
bool launch_few(TileArgs a, hipStream_t st) {
  constexpr bool GATED = gated_epi(EPI);
  constexpr size_t lds = size_t(8) * (GATED ? 2 : 1) * MT * 1024;
  static_assert(lds <= 65536, "the waves' sums fit the LDS a launch has without asking");
  int span = CH > 1 ? 4 : 16;
  if (!GATED) {
    while (span > 4 && ceil_div(a.p.rows, span) < 256) span /= 2;
    a.F = span;
  }
  few_kernel<MT, CH, EPI, ACT><<<unsigned(ceil_div(GATED ? a.F : a.p.rows, span)), 512, lds, st>>>(a);
  return true;
}

void launch_join(const TileArgs& a, int splits, hipStream_t st) {
  const int64_t n = int64_t(a.q.rows) * a.p.rows;
  const unsigned grid = unsigned(std::min<int64_t>(ceil_div(n, int64_t(1024)), 4096));
  if (splits <= 2) tile_join_kernel<2><<<grid, 256, 0, st>>>(a, splits);
  else if (splits <= 4) tile_join_kernel<4><<<grid, 256, 0, st>>>(a, splits);
  else tile_join_kernel<8><<<grid, 256, 0, st>>>(a, splits);
}

// k split over the grid into `splits` parts, joined by a second launch
template <bool WIDE, bool PROWS, bool QROWS, int EPI>
bool launch_split(TileArgs a, dim3 tiles, int64_t splits, hipStream_t st) {
  constexpr int kt = Tile<WIDE>::KT;
  a.k_split = int(ceil_div(ceil_div(a.K, kt), splits)) * kt;
  tiles.z = unsigned(ceil_div(a.K, a.k_split));
  const int64_t n = int64_t(a.p.rows) * a.q.rows;
  a.part = static_cast<float*>(xdna_hip_cache_alloc(size_t(tiles.z) * size_t(n) * sizeof(float)));
  if (!a.part) return false;
  const bool ok = launch_tile<WIDE, PROWS, QROWS, EPI, kSilu>(a, tiles, st);
  if (ok && EPI == kLinear)
    linear_join_kernel<<<unsigned(std::min<int64_t>(ceil_div(int64_t(a.q.rows) * ceil_div(a.p.rows, 8), int64_t(256)), 4096)), 256, 0, st>>>(
        a, int(tiles.z));
  else if (ok) launch_join(a, int(tiles.z), st);
  xdna_hip_cache_free(a.part);  // stream-ordered reuse: the block's next user runs after the join
  return ok;
}

// What a product in tiles takes in us, `kt` k-tiles each: the grid in rounds of two tiles a CU,
// its last round alone on the CUs if it has no more tiles than they are.  Fitted to 100 products
// (64 .. 6000 x 64 .. 6000, k 100 .. 8000, all three layouts, either tile, k in 1 to 16 splits):
// 9 % off in the mean, and the choice by it 0.6 % off the best of each.
float tile_cost(bool wide, int64_t tiles, int64_t kt) {
  const float alone = wide ? 0.65f : 0.54f, paired = wide ? 1.2f : 1.1f;
  const int64_t full = (tiles - 1) / 512, rest = tiles - full * 512;
  return float(full) * (paired * float(kt) + (wide ? 1.1f : 2.75f)) + (rest <= 256 ? alone : paired) * float(kt) + (wide ? 6.5f : 4.6f);
}

// The same with k split: fp32 partials written and read, and the join's launch.
float split_cost(bool wide, int64_t tiles, int64_t kt, int64_t splits, int64_t outputs) {
  return tile_cost(wide, tiles * splits, ceil_div(kt, splits)) + 3.3f + float(outputs) * (float(splits) * 1.8e-6f + 0.4e-6f);
}

// Tiles and splits by the costs above, P x Q outputs (P in rows of the operand).  Measured, p x q x
// k, one of each outcome: 500 x 4001 x 700 narrow 10.0 us (wide 12.8, wide in two splits 25.0); 500
// x 6002 x 700 wide 16.3 (narrow 20.1); 1024 x 512 x 8192 narrow in four splits 26.1 (whole 36.6).
struct TileChoice {
  bool wide;
  int64_t splits;
  float cost;
};

int64_t tile_count(bool wide, int64_t P, int64_t Q) { return ceil_div(P, int64_t(wide ? 128 : 64)) * ceil_div(Q, int64_t(wide ? 128 : 64)); }
int64_t k_tiles(bool wide, int64_t K) { return ceil_div(K, int64_t(wide ? Tile<true>::KT : Tile<false>::KT)); }

TileChoice choose_tiles(int64_t P, int64_t Q, int64_t K, bool may_split) {
  TileChoice best = {false, 1, INFINITY};
  for (const bool wide : {false, true}) {
    const int64_t n = tile_count(wide, P, Q), kt = k_tiles(wide, K);
    const float whole = tile_cost(wide, n, kt);
    if (whole < best.cost) best = {wide, 1, whole};
    for (const int64_t s : {2, 3, 4, 6, 8, 12, 16}) {
      if (!may_split || 2 * s > kt || n * s > 1024) break;
      const float cost = split_cost(wide, n, kt, s, P * Q);
      if (cost < best.cost) best = {wide, s, cost};
    }
  }
  return best;
}

template <bool PROWS, bool QROWS, int EPI, int ACT>
bool launch_tiles(const TileArgs& a, hipStream_t st) {
  constexpr int side = EPI == kGated || EPI == kGatedKeep ? 2 : 1;  // tile rows per unit of p
  const auto tiles = [&](int t) { return dim3(unsigned(ceil_div(int64_t(a.p.rows) * side, t)), unsigned(ceil_div(a.q.rows, t))); };
  if constexpr (!PROWS && !QROWS) {
    if constexpr (own_rows(EPI)) {
      // chunks of k where k is long or the weight's rows are few: 4096 rows of 1024 take 4.1 us
      // without them and 6.0 with (a step per wave), 1024 rows of 4096 6.7 and 4.2
      if (a.q.rows <= 4 && (a.K >= 2048 || a.p.rows <= 2048)) return launch_few<1, 4, EPI, ACT>(a, st);
      if (a.q.rows <= kFewPlain) return launch_few<1, 1, EPI, ACT>(a, st);
    } else {
      if (a.q.rows <= 16) return launch_few<1, 1, EPI, ACT>(a, st);
      if (a.q.rows <= 32) return launch_few<2, 1, EPI, ACT>(a, st);
      if (a.q.rows <= kFewGated) return launch_few<4, 1, EPI, ACT>(a, st);
    }
  }
  const TileChoice c = choose_tiles(int64_t(a.p.rows) * side, a.q.rows, a.K, own_rows(EPI));
  const dim3 t = tiles(c.wide ? 128 : 64);
  if constexpr (own_rows(EPI)) {
    if (c.splits > 1)
      return c.wide ? launch_split<true, PROWS, QROWS, EPI>(a, t, c.splits, st) : launch_split<false, PROWS, QROWS, EPI>(a, t, c.splits, st);
  }
  return c.wide ? launch_tile<true, PROWS, QROWS, EPI, ACT>(a, t, st) : launch_tile<false, PROWS, QROWS, EPI, ACT>(a, t, st);
}

// What the gradients' three products take in one launch, in us: the tiles' work spread over the
// chip, or the longest tile.  Fitted as above to 50 blocks (16 .. 6000 rows, widths 64 .. 1024, 64 ..
// 4096 units; 10 % off in the mean): narrow tiles, wide tiles or apart by it, their geometric mean is
// 13.6 us, always apart 23.6.  333 x 1000 -> 1367: 23.2 narrow, 35.7 wide, 37.5 apart; 1628 x 723 ->
// 1767: 71.4, 61.0, 82.7; 143 x 308 -> 3370 (53 k-tiles for 15 tiles of dx): 33.0, 70.6, 27.1.
// `units`: rows of the input weight (2F, or the linear layer's).
float grads_cost(bool wide, int64_t M, int64_t K, int64_t units, int64_t F, int64_t N) {
  const int64_t n_dx = tile_count(wide, K, M), n_w = tile_count(wide, K, units) + (N ? tile_count(wide, F, N) : 0);
  const float k_dx = float(k_tiles(wide, units)), k_w = float(k_tiles(wide, M));
  const auto tile = [&](float k) { return wide ? 1.05f * k + 1.5f : 1.48f * k + 1.3f; };
  const float work = (float(n_dx) * tile(k_dx) + float(n_w) * tile(k_w)) / 512.0f, k = std::max(k_dx, k_w);
  return wide ? 4.0f + std::max(work, 0.73f * k + 1.1f) : 5.3f + std::max(work, 0.56f * k - 1.0f);
}

template <bool WIDE>
bool launch_grads(GradsArgs g, hipStream_t st) {
  using C = Tile<WIDE>;
  void (*f)(GradsArgs) = grads_kernel<WIDE>;
  static const bool ok = hipFuncSetAttribute(reinterpret_cast<const void*>(f), hipFuncAttributeMaxDynamicSharedMemorySize,
                                             int(C::LDS)) == hipSuccess;
  if (!ok) return false;
  const auto plan = [](TileArgs& a) {
    return a.p.rows ? int(plan_tiles(a, ceil_div(a.p.rows, C::T), ceil_div(a.q.rows, C::T), 1, 64)) : 0;
  };
  g.n_dx = plan(g.dx);
  g.n_in = plan(g.dw_in);
  g.n_out = plan(g.dw_out);
  g.dx_first = g.dx.K >= g.dw_in.K ? 1 : 0;
  f<<<unsigned(g.n_dx + g.n_in + g.n_out), C::NT, C::LDS, st>>>(g);
  return true;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7) == 0; }

// Operands the LDS DMA can load: 16-byte aligned rows, whole vectors of k (and of units where
// they are contiguous), 32-bit byte offsets.
bool dma_ok(const TileOperand& o, int64_t rows, int64_t K, bool along_rows) {
  const int64_t extent = along_rows ? (K - 1) * o.ld + rows : (rows - 1) * o.ld + K;
  return aligned16(o.src) && o.ld % 8 == 0 && extent * 2 < (int64_t(1) << 31);
}

template <bool PROWS, int EPI, int ACT>
bool launch_large(TileArgs a, dim3 tiles, hipStream_t st) {
  void (*f)(TileArgs) = gated_large_kernel<PROWS, EPI, ACT>;
  static const bool ok = hipFuncSetAttribute(reinterpret_cast<const void*>(f), hipFuncAttributeMaxDynamicSharedMemorySize,
                                             int(kLargeLds)) == hipSuccess;
  if (!ok) return false;
  f<<<unsigned(plan_tiles(a, tiles.x, tiles.y, 1, 32)), 256, kLargeLds, st>>>(a);
  return true;
}

// dx and dw on large tiles in one launch: their splits, such that all workgroups are at work at once, by the launch's cost
// in us.  Fitted to 8 sizes (3 % off at most): 0.87 a k-tile of the longest workgroup, and the split products' partials.
// Measured, this launch, the tiles' best and the GEMM for each product: 8192 x 1024 -> 4096 126, 166 and 168; 8192 x 1024 -> 1024
// 49, 64 and 174; 8192 x 512 -> 4096 85, 108 and 310; but 4096 x 1024 -> 4096 96, 83 and 107, 2048 x 1024 -> 2048 51, 31 and 131.
struct LargeGrads {
  int64_t s_dx, s_dw;
  float cost;  // infinite: the tiles alone are more than the CUs
};

float large_join(int64_t splits, int64_t outputs) { return splits > 1 ? 4.0f + float(outputs) * float(splits) * 1.6e-6f : 0.0f; }

LargeGrads plan_large_grads(int64_t M, int64_t K, int64_t N) {
  const int64_t t = kT4, n_dx = ceil_div(K, t) * ceil_div(M, t), n_dw = ceil_div(K, t) * ceil_div(N, t);
  const int64_t k_dx = ceil_div(N, int64_t(kK5)), k_dw = ceil_div(M, int64_t(kK5));
  LargeGrads best = {1, 1, INFINITY};
  for (int64_t a = 1; a <= 16; ++a)
    for (int64_t b = 1; b <= 16 && n_dx * a + n_dw * b <= 256; ++b) {
      const float cost = 4.0f + 0.87f * float(std::max(ceil_div(k_dx, a), ceil_div(k_dw, b))) + large_join(a, M * K) + large_join(b, N * K);
      if (cost < best.cost) best = {a, b, cost};
    }
  return best;
}

bool launch_grads_large(GradsArgs g, hipStream_t st) {
  static const bool ok = hipFuncSetAttribute(reinterpret_cast<const void*>(linear_grads_large_kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, int(kLargeLds)) == hipSuccess;
  if (!ok) return false;
  const LargeGrads p = plan_large_grads(g.dx.q.rows, g.dx.p.rows, g.dw_in.q.rows);
  const auto plan = [](TileArgs& a, int64_t splits) {
    a.k_split = int(ceil_div(ceil_div(a.K, kK5), splits)) * kK5;
    splits = ceil_div(a.K, a.k_split);
    if (splits > 1) {
      a.part = static_cast<float*>(xdna_hip_cache_alloc(size_t(splits) * size_t(a.p.rows) * size_t(a.q.rows) * sizeof(float)));
      if (!a.part) return int64_t(0);
    }
    return plan_tiles(a, ceil_div(a.p.rows, kT4), ceil_div(a.q.rows, kT4), splits, 32);
  };
  LargeGradsArgs l = {g.dx, g.dw_in, 0, 0};
  l.n_dx = int(plan(l.dx, p.s_dx));
  l.n_dw = l.n_dx ? int(plan(l.dw, p.s_dw)) : 0;
  const bool have = l.n_dx && l.n_dw;
  if (have) linear_grads_large_kernel<<<unsigned(l.n_dx + l.n_dw), 256, kLargeLds, st>>>(l);
  for (TileArgs* a : {&l.dx, &l.dw}) {
    if (!a->part) continue;
    if (have) launch_join(*a, int(ceil_div(a->K, a->k_split)), st);
    xdna_hip_cache_free(a->part);  // stream-ordered reuse: the block's next user runs after the join
  }
  return have;
}

// Large tiles where they give every CU one and fill the rounds that they take.  Measured, large
// and wide tiles in us: 8192 x 512 -> 1024 units (256 tiles) 27 and 34, 8192 x 1024 -> 4096 158 and
// 192; but 8192 x 512 -> 1024's gradient (128 tiles) 37 and 27, 4800 x 1024 -> 2048 (1.2 rounds) 64
// and 57.
template <int EPI, bool PROWS, int ACT>
bool launch_sized(const TileArgs& a, hipStream_t st) {
  constexpr bool GATED = gated_epi(EPI);
  const int64_t units = EPI == kLinear ? a.p.rows : a.F;
  const dim3 grid(unsigned(ceil_div(units, GATED ? kT4 / 2 : kT4)), unsigned(ceil_div(a.q.rows, kT4)));
  const int64_t n = int64_t(grid.x) * grid.y;
  const bool large = n >= 256 && 100 * n >= 65 * 256 * ceil_div(n, int64_t(256)) && a.K % 8 == 0 && (EPI == kLinear || (a.F % 8 == 0 && aligned16(a.out) && aligned16(a.gu))) &&
                     dma_ok(a.p, GATED ? 2 * units : units, a.K, PROWS) && dma_ok(a.q, a.q.rows, a.K, false);
  return large ? launch_large<PROWS, EPI, ACT>(a, grid, st) : launch_tiles<PROWS, false, EPI, ACT>(a, st);
}

template <int EPI, bool PROWS>
bool launch_gated(int act, const TileArgs& a, hipStream_t st) {
  if (act == kSilu) return launch_sized<EPI, PROWS, kSilu>(a, st);
  if (act == kGelu) return launch_sized<EPI, PROWS, kGelu>(a, st);
  return launch_sized<EPI, PROWS, kRelu>(a, st);
}

// out, the kept projections and the sizes the epilogues go by (gu: one block of xdna_gated_kept_bytes)
TileArgs kept_args(int64_t M, int64_t F, const void* gu, uint16_t* out) {
  TileArgs a = {};
  a.q.rows = int(M);
  a.F = int(F);
  a.out = out;
  a.gu = static_cast<uint16_t*>(const_cast<void*>(gu));
  a.low = reinterpret_cast<uint8_t*>(a.gu) + M * F * 4;
  a.vec = F % 4 == 0 && aligned8(out) && aligned8(gu) ? 1 : 0;
  return a;
}

// dx = d w and dw = d^T x of a product x w^T with `units` rows of w
GradsArgs input_grads(const uint16_t* d, int64_t ldd, const uint16_t* x, int64_t ldx, const uint16_t* w, int64_t ldw,
                      int64_t M, int64_t K, int64_t units, uint16_t* dx, uint16_t* dw) {
  GradsArgs g = {};
  g.dx.p = {w, ldw, int(K)};
  g.dx.q = {d, ldd, int(M)};
  g.dx.K = int(units);
  g.dx.out = dx;
  g.dx.ldc = K;
  g.dw_in.p = {x, M > 1 ? ldx : K, int(K)};
  g.dw_in.q = {d, ldd, int(units)};
  g.dw_in.K = int(M);
  g.dw_in.out = dw;
  g.dw_in.ldc = K;
  return g;
}

const char* linear_fault(int64_t M, int64_t K, int64_t N) {
  if (M < 0 || M > kMaxRows || K < 1 || K > kMaxSide || N < 1 || N > kMaxSide) return "sizes out of range";
  return M * N > kMaxOutputs ? "too many outputs" : nullptr;
}

// Row slices of the column sums: enough workgroups for the chip (four a CU), a row of each thread at least.
int64_t linear_parts(int64_t M, int64_t N) {
  if (M <= 0) return 0;
  return std::max<int64_t>(1, std::min(ceil_div(int64_t(1024), ceil_div(N, int64_t(256))), ceil_div(M, int64_t(8))));
}

// How dx and dw are best made: 0 apart, 1 together on small tiles, 2 together on large ones.
int grads_how(const GradsArgs& g) {
  const int64_t M = g.dx.q.rows, K = g.dx.p.rows, N = g.dx.K;
  const bool dma = K % 8 == 0 && N % 8 == 0 && dma_ok(g.dx.p, K, N, true) && dma_ok(g.dx.q, M, N, false) && dma_ok(g.dw_in.p, K, M, true) &&
                   dma_ok(g.dw_in.q, N, M, true);
  const float together = std::min(grads_cost(false, M, K, N, 0, 0), grads_cost(true, M, K, N, 0, 0));
  const float apart = choose_tiles(K, M, N, true).cost + choose_tiles(K, N, M, true).cost;
  if (dma && plan_large_grads(M, K, N).cost < std::min(together, apart)) return 2;
  return together < apart ? 1 : 0;
}

int launched(const char* what, bool ok) {
  return ok ? check_launch(what) : refuse(what, "no memory for partial sums, or a tile kernel's LDS size cannot be had");
}

}  // namespace
}  // namespace xdna

using namespace xdna;

extern "C" {

size_t xdna_gated_kept_bytes(int64_t M, int64_t F) {
  return M < 1 || F < 1 || M > kMaxSide || F > kMaxSide / 2 ? 0 : size_t(M) * size_t(F) * 5;
}

int xdna_gated_bf16(const uint16_t* x, int64_t ldx, const uint16_t* w, int64_t ldw, int64_t M, int64_t K, int64_t F,
                    int act, uint16_t* h, void* gu, void* stream) {
  const char* what = "xdna_gated_bf16";
  if (const char* why = gated_fault(M, K, F, act)) return refuse(what, why);
  if ((ldx < K && M > 1) || ldw < K) return refuse(what, "rows overlap");
  if (M == 0) return 0;
  if (!x || !w || !h) return refuse(what, "null operand");
  if (odd(x) || odd(w) || odd(h) || odd(gu)) return refuse(what, "misaligned operand");
  if (!admit_launch(what)) return -1;
  TileArgs a = kept_args(M, F, gu, h);
  a.p = {w, ldw, int(F)};
  a.q.src = x;
  a.q.ld = M > 1 ? ldx : K;
  a.K = int(K);
  hipStream_t st = as_stream(stream);
  return launched(what, gu ? launch_gated<kGatedKeep, false>(act, a, st) : launch_gated<kGated, false>(act, a, st));
}

int xdna_gated_mlp_bwd_bf16(const uint16_t* dy, int64_t lddy, const uint16_t* w_out, int64_t ldw, const void* gu,
                            int64_t M, int64_t N, int64_t F, int act, uint16_t* dgu, void* stream) {
  const char* what = "xdna_gated_mlp_bwd_bf16";
  if (const char* why = gated_fault(M, N, F, act)) return refuse(what, why);
  if ((lddy < N && M > 1) || (ldw < F && N > 1)) return refuse(what, "rows overlap");
  if (M == 0) return 0;
  if (!dy || !w_out || !gu || !dgu) return refuse(what, "null operand");
  if (odd(dy) || odd(w_out) || odd(gu) || odd(dgu)) return refuse(what, "misaligned operand");
  if (!admit_launch(what)) return -1;
  TileArgs a = kept_args(M, F, gu, dgu);
  a.p = {w_out, ldw, int(F)};
  a.q.src = dy;
  a.q.ld = M > 1 ? lddy : N;
  a.K = int(N);
  return launched(what, launch_gated<kGatedGrad, true>(act, a, as_stream(stream)));
}

int xdna_tile_mm_bf16(const uint16_t* p, int64_t ldp, int p_rows, const uint16_t* q, int64_t ldq, int q_rows, int64_t P,
                      int64_t Q, int64_t K, uint16_t* out, int64_t ldc, void* stream) {
  const char* what = "xdna_tile_mm_bf16";
  if (P < 0 || P > kMaxSide || Q < 0 || Q > kMaxRows || K < 1 || K > kMaxSide || P * Q > kMaxOutputs)
    return refuse(what, "sizes out of range");
  if ((p_rows != 0 && p_rows != 1) || (q_rows != 0 && q_rows != 1) || (q_rows && !p_rows))
    return refuse(what, "operands are k-contiguous (0) or row-contiguous (1), q only beside such a p");
  if (ldp < (p_rows ? P : K) || ldq < (q_rows ? Q : K) || ldc < P) return refuse(what, "rows overlap");
  if (P == 0 || Q == 0) return 0;
  if (!p || !q || !out) return refuse(what, "null operand");
  if (odd(p) || odd(q) || odd(out)) return refuse(what, "misaligned operand");
  if (!admit_launch(what)) return -1;
  TileArgs a = {};
  a.p = {p, ldp, int(P)};
  a.q = {q, ldq, int(Q)};
  a.K = int(K);
  a.out = out;
  a.ldc = ldc;
  a.vec = ldc % 4 == 0 && aligned8(out) ? 1 : 0;
  hipStream_t st = as_stream(stream);
  return launched(what, q_rows   ? launch_tiles<true, true, kPlain, kSilu>(a, st)
                        : p_rows ? launch_tiles<true, false, kPlain, kSilu>(a, st)
                                 : launch_tiles<false, false, kPlain, kSilu>(a, st));
}

int xdna_gated_grads_pick(int64_t M, int64_t K, int64_t F, int64_t N) {
  if (gated_fault(M, K, F, 0) || M == 0 || N < 0 || N > kMaxRows || F > kMaxRows / 2) return 0;
  const float apart = choose_tiles(K, M, 2 * F, true).cost + choose_tiles(K, 2 * F, M, true).cost +
                      (N ? choose_tiles(F, N, M, true).cost : 0.0f);
  return std::min(grads_cost(false, M, K, 2 * F, F, N), grads_cost(true, M, K, 2 * F, F, N)) < apart ? 1 : 0;
}

int xdna_gated_grads_bf16(const uint16_t* dgu, const uint16_t* x, int64_t ldx, const uint16_t* w_in, int64_t ldw,
                          const uint16_t* dy, int64_t lddy, const uint16_t* h, int64_t M, int64_t K, int64_t F, int64_t N,
                          uint16_t* dx, uint16_t* dw_in, uint16_t* dw_out, void* stream) {
  const char* what = "xdna_gated_grads_bf16";
  if (const char* why = gated_fault(M, K, F, 0)) return refuse(what, why);
  if (M == 0) return refuse(what, "no rows");
  if (N < 0 || N > kMaxRows || F > kMaxRows / 2 || 2 * F * K > kMaxOutputs || M * K > kMaxOutputs || N * F > kMaxOutputs)
    return refuse(what, "sizes out of range");
  if ((ldx < K && M > 1) || ldw < K || (N > 0 && lddy < N && M > 1)) return refuse(what, "rows overlap");
  if (!dgu || !x || !w_in || !dx || !dw_in || (N > 0 && (!dy || !h || !dw_out))) return refuse(what, "null operand");
  if (odd(dgu) || odd(x) || odd(w_in) || odd(dy) || odd(h) || odd(dx) || odd(dw_in) || odd(dw_out))
    return refuse(what, "misaligned operand");
  if (!admit_launch(what)) return -1;
  GradsArgs g = input_grads(dgu, 2 * F, x, ldx, w_in, ldw, M, K, 2 * F, dx, dw_in);
  if (N > 0) {
    g.dw_out.p = {h, F, int(F)};
    g.dw_out.q = {dy, M > 1 ? lddy : N, int(N)};
    g.dw_out.K = int(M);
    g.dw_out.out = dw_out;
    g.dw_out.ldc = F;
  }
  const bool wide = grads_cost(true, M, K, 2 * F, F, N) < grads_cost(false, M, K, 2 * F, F, N);
  hipStream_t st = as_stream(stream);
  return launched(what, wide ? launch_grads<true>(g, st) : launch_grads<false>(g, st));
}

int xdna_linear_bf16(const uint16_t* x, int64_t ldx, const uint16_t* w, int64_t ldw, int64_t M, int64_t K, int64_t N, int act,
                     const uint16_t* bias, const uint16_t* residual, int64_t ldr, uint16_t* y, void* kept, void* stream) {
  const char* what = "xdna_linear_bf16";
  if (const char* why = linear_fault(M, K, N)) return refuse(what, why);
  if (act < 0 || act > 3) return refuse(what, "activation must be 0 (silu), 1 (gelu), 2 (relu) or 3 (none)");
  if ((M > 1 && (ldx < K || (residual && ldr < N))) || (ldw < K && N > 1)) return refuse(what, "rows overlap");
  if (M == 0) return 0;
  if (!x || !w || !y) return refuse(what, "null operand");
  if (kept && act == kNone) return refuse(what, "no activation has no slopes");
  if (odd(x) || odd(w) || odd(bias) || odd(residual) || odd(y) || odd(kept)) return refuse(what, "misaligned operand");
  if (!admit_launch(what)) return -1;
  TileArgs a = {};
  a.p = {w, N > 1 ? ldw : K, int(N)};
  a.q = {x, M > 1 ? ldx : K, int(M)};
  a.K = int(K);
  a.out = y;
  a.ldc = N;
  a.vec = N % 4 == 0 && aligned8(y) ? 1 : 0;
  a.act = act;
  a.bias = bias;
  a.res = residual;
  a.ldr = M > 1 ? ldr : N;
  a.kept = kept;
  return launched(what, launch_sized<kLinear, false, kSilu>(a, as_stream(stream)));
}

size_t xdna_linear_kept_bytes(int64_t M, int64_t N, int act) {
  if (linear_fault(M, 1, N) || M == 0) return 0;
  return act == kSilu || act == kGelu ? size_t(M) * size_t(N) * 2 : act == kRelu ? size_t(M) * size_t(bit_bytes(N)) : 0;
}

size_t xdna_linear_bwd_workspace_bytes(int64_t M, int64_t N) {
  return linear_fault(M, 1, N) ? 0 : size_t(linear_parts(M, N)) * size_t(N) * sizeof(float);
}

int xdna_linear_bwd_bf16(const uint16_t* dy, int64_t ld, const void* kept, int act, int64_t M, int64_t N, uint16_t* dp,
                         uint16_t* d_bias, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "xdna_linear_bwd_bf16";
  if (const char* why = linear_fault(M, 1, N)) return refuse(what, why);
  if (ld < N && M > 1) return refuse(what, "rows overlap");
  if (act < 0 || act > 3) return refuse(what, "activation must be 0 (silu), 1 (gelu), 2 (relu) or 3 (none)");
  if (M > 0 && (!dy || (act != kNone && !kept))) return refuse(what, "null operand");
  if (odd(dy) || odd(kept) || odd(dp) || odd(d_bias)) return refuse(what, "misaligned operand");
  if (d_bias && M > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < xdna_linear_bwd_workspace_bytes(M, N)))
    return refuse(what, "workspace missing, misaligned or too small");
  if ((M == 0 || !dp) && !d_bias) return 0;
  if (!admit_launch(what)) return -1;
  hipStream_t st = as_stream(stream);
  LinearBwdArgs a = {dy, M > 1 ? ld : N, act == kNone ? nullptr : kept, act == kRelu, dp, d_bias ? static_cast<float*>(workspace) : nullptr, int(M), int(N)};
  const int64_t parts = linear_parts(M, N);
  if (M > 0) linear_bwd_kernel<<<dim3(unsigned(ceil_div(N, int64_t(256))), unsigned(parts)), 256, 0, st>>>(a);
  if (d_bias) linear_bias_kernel<<<unsigned(ceil_div(N, int64_t(64))), 1024, 0, st>>>(a.part, int(parts), int(N), d_bias);
  return check_launch(what);
}

int xdna_linear_grads_pick(const uint16_t* dp, int64_t lddp, const uint16_t* x, int64_t ldx, const uint16_t* w, int64_t ldw,
                           int64_t M, int64_t K, int64_t N) {
  if (linear_fault(M, K, N) || M == 0 || N > kMaxRows || N * K > kMaxOutputs || M * K > kMaxOutputs) return 0;
  return grads_how(input_grads(dp, M > 1 ? lddp : N, x, ldx, w, N > 1 ? ldw : K, M, K, N, nullptr, nullptr));
}

int xdna_linear_grads_bf16(const uint16_t* dp, int64_t lddp, const uint16_t* x, int64_t ldx, const uint16_t* w, int64_t ldw,
                           int64_t M, int64_t K, int64_t N, uint16_t* dx, uint16_t* dw, void* stream) {
  const char* what = "xdna_linear_grads_bf16";
  if (const char* why = linear_fault(M, K, N)) return refuse(what, why);
  if (M == 0) return refuse(what, "no rows");
  if (N > kMaxRows || N * K > kMaxOutputs || M * K > kMaxOutputs) return refuse(what, "sizes out of range");
  if ((M > 1 && (lddp < N || ldx < K)) || (ldw < K && N > 1)) return refuse(what, "rows overlap");
  if (!dp || !x || !w || !dx || !dw) return refuse(what, "null operand");
  if (odd(dp) || odd(x) || odd(w) || odd(dx) || odd(dw)) return refuse(what, "misaligned operand");
  if (!admit_launch(what)) return -1;
  const GradsArgs g = input_grads(dp, M > 1 ? lddp : N, x, ldx, w, N > 1 ? ldw : K, M, K, N, dx, dw);
  const bool wide = grads_cost(true, M, K, N, 0, 0) < grads_cost(false, M, K, N, 0, 0);
  hipStream_t st = as_stream(stream);
  if (grads_how(g) == 2) return launched(what, launch_grads_large(g, st));
  return launched(what, wide ? launch_grads<true>(g, st) : launch_grads<false>(g, st));
}

int xdna_gated_bwd_bf16(const uint16_t* dh, int64_t ld, const void* gu, int64_t M, int64_t F, int act, uint16_t* dgu,
                        void* stream) {
  const char* what = "xdna_gated_bwd_bf16";
  if (const char* why = gated_fault(M, 1, F, act)) return refuse(what, why);
  if (ld < F && M > 1) return refuse(what, "rows overlap");
  if (M == 0) return 0;
  if (!dh || !gu || !dgu) return refuse(what, "null operand");
  if (odd(dh) || odd(gu) || odd(dgu)) return refuse(what, "misaligned operand");
  if (!admit_launch(what)) return -1;
  GatedBwdArgs a = {};
  a.dh = dh;
  a.ld = M > 1 ? ld : F;
  a.t = kept_args(M, F, gu, dgu);
  a.windows = int(ceil_div(F, int64_t(4)));
  const unsigned grid = unsigned(std::min<int64_t>(ceil_div(M * a.windows, int64_t(256)), 16384));
  hipStream_t st = as_stream(stream);
  if (act == kSilu) gated_bwd_kernel<kSilu><<<grid, 256, 0, st>>>(a);
  else if (act == kGelu) gated_bwd_kernel<kGelu><<<grid, 256, 0, st>>>(a);
  else gated_bwd_kernel<kRelu><<<grid, 256, 0, st>>>(a);
  return check_launch(what);
}

}  // extern "C"
