// Layer norm of token rows on gfx950, alone or of a residual sum, and its backward pass.  The
// reference reaches layer norms only through its zero-copy CPU fallback
// (torch_xdna_device.cpp:5124-5260).
//
//   s = round(x + r) (the stored sum; s = x alone), m = mean(s), i = 1 / sqrt(mean((s - m)^2) + eps)
//   h = (s - m) i,  y = h w + b
//   a = dy w;  ds = i (a - mean(a) - h mean(a h)) (+ the sum's own gradient);  dw = sum of dy h,
//   db = sum of dy over the rows
//
// The norm is that of the sum as it is stored, so that the fused form gives the bits of an add
// followed by a norm, and the backward pass has the same h.  Everything is fp32 between one load
// and one rounding; the variance is summed from the differences to the mean (a row is in registers,
// so the second pass costs no memory).  In the same pass the differences' own mean c is summed: what the
// mean, a rounded sum and quotient, is off by (an ulp of a row far from zero is a large part of its
// deviation, and a constant row's is all of it: rows of 1000 gave -0.02 at width 1000, of 1e6 -1).  The
// differences are then s - m - c and the variance their squares' mean less c^2; what is kept for the
// gradient is m + c, rounded.  The gradients of w and b: a wave's rows add up in its
// lanes' registers, a workgroup's waves through LDS in wave order, the workgroups' partials by a
// second launch in order: no atomics, equal inputs give equal bits.
//
// Bound by HBM.  A row is held in registers: by one wave up to 2048 elements, by four waves up to
// 8192, by sixteen up to 16384; longer rows are read again for each pass.  65536 rows of 2048 in bf16: forward 106 us
// (537 MB, 5.1 TB/s), backward 165 (805 MB, 4.9) and 5 for the partials' sums; 8192 x 1024 with the residual sum: 15, 16
// and 4; one row of 1024: 3.1; 4099 x 515 in fp32: 7.8 (2.2 TB/s), 10.4 (2.4) and 3.9.
#include "common.h"

#include "../../include/xdna_hip.h"

namespace xdna {
namespace {

enum DType { kF32 = 1, kBf16 = 2 };

template <int DT>
struct Elem;
template <>
struct Elem<kF32> {
  typedef float T;
  struct __attribute__((packed, aligned(4))) Vec {
    float v[8];
  };
};
template <>
struct Elem<kBf16> {
  typedef uint16_t T;
  typedef Pix8 Vec;
};

__device__ inline float to_f32(float v) { return v; }
__device__ inline float to_f32(uint16_t v) { return bf16_to_f32(v); }
__device__ inline void put(float* p, float v) { *p = v; }
__device__ inline void put(uint16_t* p, float v) { *p = f32_to_bf16(v); }

__device__ inline void unpack(const Elem<kF32>::Vec& q, float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = q.v[e];
}
__device__ inline void unpack(const Pix8& q, float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(e & 1 ? q.v[e >> 1] & 0xFFFF0000u : q.v[e >> 1] << 16);
}
__device__ inline void pack(const float (&f)[8], Elem<kF32>::Vec& q) {
#pragma unroll
  for (int e = 0; e < 8; ++e) q.v[e] = f[e];
}
__device__ inline void pack(const float (&f)[8], Pix8& q) {
#pragma unroll
  for (int e = 0; e < 4; ++e) q.v[e] = uint32_t(f32_to_bf16(f[2 * e])) | uint32_t(f32_to_bf16(f[2 * e + 1])) << 16;
}

struct NormArgs {
  const void* x;       // rows of dim, row stride ldx
  const void* other;   // forward: the residual or null; backward: the sum's gradient or null
  const void* dy;      // backward
  int64_t ldx, ldo, lddy;
  int64_t rows;
  int dim;
  const void* weight;  // null: 1
  const void* bias;    // null: 0
  float eps;
  void* sum;           // forward with a residual: dense rows
  void* out;           // y, or dx (null: not asked for); dense rows
  float* stats;        // (mean, 1 / deviation) per row, or null
  float* part;         // backward: [workgroup][2][dim] partial sums, or null
};

// 8 elements of a row from column c on.  A vector across the row's end starts at dim - 8 instead
// (every load is whole and hangs on no branch); the elements it shares with its neighbour are left out
// of sums by the mask `from` (the first element that counts) and stored twice with the same value.
// Rows of fewer than 8 elements are read one by one.
struct Window {
  int c, from, n;  // start column, first element that counts, elements in range from c on
};

__device__ inline Window window(int c, int dim) {
  if (c + 8 <= dim) return {c, 0, 8};
  if (dim < 8) return {0, c == 0 ? 0 : 8, dim};
  return {dim - 8, c < dim ? c - (dim - 8) : 8, 8};  // (past the end: the last window, of which nothing counts)
}

// EVEN: dim is a multiple of 8, a window counts whole or not at all (one lane mask a window; a mask an
// element spills scalar registers)
template <int DT, bool EVEN = false>
__device__ inline typename Elem<DT>::Vec load8(const void* row, const Window& w) {
  typedef typename Elem<DT>::T T;
  typedef typename Elem<DT>::Vec Vec;
  const T* p = static_cast<const T*>(row) + w.c;
  if (EVEN || w.n >= 8) return *reinterpret_cast<const Vec*>(p);
  float f[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = e < w.n ? to_f32(p[e]) : 0.0f;
  Vec q;
  pack(f, q);
  return q;
}

template <int DT, bool EVEN = false>
__device__ inline void store8(void* row, const Window& w, const float (&f)[8]) {
  typedef typename Elem<DT>::T T;
  typedef typename Elem<DT>::Vec Vec;
  if (w.from >= 8) return;
  T* p = static_cast<T*>(row) + w.c;
  if (EVEN || w.n >= 8) {
    Vec q;
    pack(f, q);
    *reinterpret_cast<Vec*>(p) = q;
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < w.n) put(p + e, f[e]);
}

// an element counts in this thread's sums
template <bool EVEN>
__device__ inline bool counts(const Window& w, int e) {
  return EVEN ? w.from == 0 : e >= w.from && e < w.n;
}

// The sum over the wave, in every lane: quads, halves of 8 and rows of 16 by DPP, rows by gfx950's swaps: no LDS and
// no waits (six shuffles through LDS took 0.6 us of a row's 2).
template <int CTRL>
__device__ inline float dpp(float v) {
  return __uint_as_float(uint32_t(__builtin_amdgcn_update_dpp(0, int(__float_as_uint(v)), CTRL, 0xF, 0xF, true)));
}

__device__ inline float wave_sum(float v) {
  v += dpp<0xB1>(v);   // quad_perm 1 0 3 2
  v += dpp<0x4E>(v);   // quad_perm 2 3 0 1
  v += dpp<0x141>(v);  // row_half_mirror
  v += dpp<0x140>(v);  // row_mirror
  auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}

// The sums of N values over the WAVES waves that share a row, the same in every thread; `red` holds
// 2 x WAVES x N floats, used in turn by the calls (phase 0, 1, 0, ...), so that one barrier a call
// is enough.
template <int WAVES, int N>
__device__ inline void row_sums(float (&v)[N], float* red, int& phase) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
  if constexpr (WAVES > 1) {
    float* to = red + phase * WAVES * 2;
    phase ^= 1;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) to[(threadIdx.x >> 6) * N + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.0f;
    for (int w = 0; w < WAVES; ++w) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += to[w * N + i];
    }
  }
}

// 1 / sqrt(var + eps) from the mean square of differences that are all `off` too large
__device__ inline float inverse_deviation(float square, float off, float eps) {
  const float var = square - off * off;
  return 1.0f / sqrtf((var < 0.0f ? 0.0f : var) + eps);  // (NaN stays NaN)
}

constexpr int kRowWaves = 4;  // waves of a workgroup where each has rows of its own

// Forward.  WAVES waves share a row (1: each of a workgroup's four waves has its own rows), V
// vectors of 8 elements a thread.
template <int DT, int PT, int WAVES, int V, bool EVEN>
__global__ __launch_bounds__(64 * (WAVES == 1 ? kRowWaves : WAVES)) void fwd_kernel(NormArgs a) {
  typedef typename Elem<DT>::T T;
  __shared__ float red[2 * 2 * WAVES];
  const int lane = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x;
  const int64_t step = WAVES == 1 ? int64_t(gridDim.x) * kRowWaves : gridDim.x;
  int64_t r = WAVES == 1 ? int64_t(blockIdx.x) * kRowWaves + (threadIdx.x >> 6) : blockIdx.x;
  Window win[V];
#pragma unroll
  for (int j = 0; j < V; ++j) win[j] = window((lane + j * 64 * WAVES) * 8, a.dim);
  int phase = 0;
  const float scale = 1.0f / float(a.dim);
  for (; r < a.rows; r += step) {
    float v[V][8];
    float sums[1] = {0.0f};
    const T* x = static_cast<const T*>(a.x) + r * a.ldx;
    typename Elem<DT>::Vec q[V], o[V];
#pragma unroll
    for (int j = 0; j < V; ++j) q[j] = load8<DT, EVEN>(x, win[j]);
    if (a.other) {
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = load8<DT, EVEN>(static_cast<const T*>(a.other) + r * a.ldo, win[j]);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      unpack(q[j], v[j]);
      if (a.other) {
        float w[8];
        unpack(o[j], w);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] += w[e];
        typename Elem<DT>::Vec s;
        pack(v[j], s);
        unpack(s, v[j]);
        store8<DT, EVEN>(static_cast<T*>(a.sum) + r * a.dim, win[j], v[j]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) sums[0] += counts<EVEN>(win[j], e) ? v[j][e] : 0.0f;
    }
    row_sums<WAVES>(sums, red, phase);
    const float mean = sums[0] / float(a.dim);
    float dev[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[j][e] -= mean;
        dev[0] += counts<EVEN>(win[j], e) ? v[j][e] : 0.0f;
        dev[1] += counts<EVEN>(win[j], e) ? v[j][e] * v[j][e] : 0.0f;
      }
    row_sums<WAVES>(dev, red, phase);
    const float off = dev[0] * scale, inv = inverse_deviation(dev[1] * scale, off, a.eps);
    if (a.stats && lane == 0) {
      a.stats[2 * r] = mean + off;
      a.stats[2 * r + 1] = inv;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float w[8], b[8];
      if (a.weight) {
        unpack(load8<PT, EVEN>(a.weight, win[j]), w);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] = (v[j][e] - off) * (inv * w[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] = (v[j][e] - off) * inv;
      }
      if (a.bias) {
        unpack(load8<PT, EVEN>(a.bias, win[j]), b);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] += b[e];
      }
      store8<DT, EVEN>(static_cast<T*>(a.out) + r * a.dim, win[j], v[j]);
    }
  }
}

// Backward: dx and, with `part`, the workgroup's sums for dw and db.  GROUP rows are at work in a
// workgroup at once, each by WAVES waves.
template <int DT, int PT, int WAVES, int GROUP, int V, bool EVEN>
__global__ __launch_bounds__(64 * WAVES * GROUP) void bwd_kernel(NormArgs a) {
  typedef typename Elem<DT>::T T;
  static_assert(WAVES == 1 || GROUP == 1, "rows of several waves have the workgroup to themselves");
  extern __shared__ __attribute__((aligned(16))) float lds[];  // GROUP > 1: [GROUP][64 V 8]; else the row sums
  const int lane = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x, group = WAVES == 1 ? threadIdx.x >> 6 : 0;
  Window win[V];
  float dw[V][8], db[V][8];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    win[j] = window((lane + j * 64 * WAVES) * 8, a.dim);
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[j][e] = db[j][e] = 0.0f;
  }
  int phase = 0;
  const float scale = 1.0f / float(a.dim);
  // A row's loads fly beside the row before it where that costs no occupancy (at two waves a SIMD: 65536 x 2048 in bf16
  // 196 -> 187 us; with two vectors a thread it takes the fourth wave: 8192 x 1024 16.5 -> 20).
  constexpr bool kAhead = DT == kBf16 && WAVES < 16 && V == 4;
  typename Elem<DT>::Vec qx[V], qd[V];
  float2 stat;
  const auto load = [&](int64_t r) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      qx[j] = load8<DT, EVEN>(static_cast<const T*>(a.x) + r * a.ldx, win[j]);
      qd[j] = load8<DT, EVEN>(static_cast<const T*>(a.dy) + r * a.lddy, win[j]);
    }
    stat = make_float2(a.stats[2 * r], a.stats[2 * r + 1]);
  };
  const int64_t step = int64_t(gridDim.x) * GROUP;
  int64_t r = int64_t(blockIdx.x) * GROUP + group;
  if (kAhead && r < a.rows) load(r);
  for (; r < a.rows; r += step) {
    if (!kAhead) load(r);
    const float mean = stat.x, inv = stat.y;
    float sums[2] = {0.0f, 0.0f};
    float h[V][8], g[V][8];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      unpack(qx[j], h[j]);
      unpack(qd[j], g[j]);
      float w[8];
      if (a.weight) unpack(load8<PT, EVEN>(a.weight, win[j]), w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        h[j][e] = (h[j][e] - mean) * inv;
        const bool in = counts<EVEN>(win[j], e);
        dw[j][e] += in ? g[j][e] * h[j][e] : 0.0f;
        db[j][e] += in ? g[j][e] : 0.0f;
        if (a.weight) g[j][e] *= w[e];
        sums[0] += in ? g[j][e] : 0.0f;
        sums[1] += in ? g[j][e] * h[j][e] : 0.0f;
      }
    }
    if (kAhead && r + step < a.rows) load(r + step);
    if (!a.out) continue;
    row_sums<WAVES>(sums, lds, phase);
    const float ma = sums[0] * scale, mh = sums[1] * scale;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float d[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = inv * (g[j][e] - ma - h[j][e] * mh);
      if (a.other) {
        float o[8];
        unpack(load8<DT, EVEN>(static_cast<const T*>(a.other) + r * a.ldo, win[j]), o);
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] += o[e];
      }
      store8<DT, EVEN>(static_cast<T*>(a.out) + r * a.dim, win[j], d);
    }
  }
  if (!a.part) return;
  float* part = a.part + int64_t(blockIdx.x) * 2 * a.dim;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if constexpr (GROUP > 1) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < V; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) lds[(group * V + j) * 512 + e * 64 + lane] = which ? db[j][e] : dw[j][e];
      __syncthreads();
      // element (j, e, lane) is column 8 (lane + 64 j) + e of windows that count
      for (int i = threadIdx.x; i < V * 512; i += 64 * GROUP) {
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < GROUP; ++k) s += lds[k * V * 512 + i];
        const int j = i >> 9, e = (i >> 6) & 7;
        const Window w = window(((i & 63) + j * 64) * 8, a.dim);
        if (counts<EVEN>(w, e)) part[which * a.dim + w.c + e] = s;
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (counts<EVEN>(win[j], e)) part[which * a.dim + win[j].c + e] = which ? db[j][e] : dw[j][e];
    }
  }
}

// Rows past the register forms: a workgroup of 1024 threads a row, which it reads again for each pass.  A thread adds up to
// 16384 elements: compensated (Kahan), or squares that are alike put the variance 2e-4 off.
struct Compensated {
  float s = 0.0f, c = 0.0f;
  __device__ inline void add(float v) {
    const float y = v - c, t = s + y;
    c = (t - s) - y;
    s = t;
  }
};

template <int DT, int PT>
__global__ __launch_bounds__(1024) void long_fwd_kernel(NormArgs a) {
  typedef typename Elem<DT>::T T;
  typedef typename Elem<PT>::T P;
  __shared__ float red[2 * 2 * 16];
  int phase = 0;
  const float scale = 1.0f / float(a.dim);
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + r * a.ldx;
    T* s = static_cast<T*>(a.sum) + r * a.dim;
    Compensated sum, first, second;
    for (int c = threadIdx.x; c < a.dim; c += 1024) {
      float v = to_f32(x[c]);
      if (a.other) {
        put(s + c, v + to_f32(static_cast<const T*>(a.other)[r * a.ldo + c]));  // (read again by this thread alone)
        v = to_f32(s[c]);
      }
      sum.add(v);
    }
    if (a.other) x = s;
    float sums[1] = {sum.s};
    row_sums<16>(sums, red, phase);
    const float mean = sums[0] / float(a.dim);
    for (int c = threadIdx.x; c < a.dim; c += 1024) {
      const float v = to_f32(x[c]) - mean;
      first.add(v);
      second.add(v * v);
    }
    float dev[2] = {first.s, second.s};
    row_sums<16>(dev, red, phase);
    const float off = dev[0] * scale, inv = inverse_deviation(dev[1] * scale, off, a.eps);
    if (a.stats && threadIdx.x == 0) {
      a.stats[2 * r] = mean + off;
      a.stats[2 * r + 1] = inv;
    }
    for (int c = threadIdx.x; c < a.dim; c += 1024) {
      float v = (to_f32(x[c]) - mean - off) * inv;
      if (a.weight) v *= to_f32(static_cast<const P*>(a.weight)[c]);
      if (a.bias) v += to_f32(static_cast<const P*>(a.bias)[c]);
      put(static_cast<T*>(a.out) + r * a.dim + c, v);
    }
  }
}

template <int DT, int PT>
__global__ __launch_bounds__(1024) void long_dx_kernel(NormArgs a) {
  typedef typename Elem<DT>::T T;
  typedef typename Elem<PT>::T P;
  __shared__ float red[2 * 2 * 16];
  int phase = 0;
  const float scale = 1.0f / float(a.dim);
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + r * a.ldx;
    const T* dy = static_cast<const T*>(a.dy) + r * a.lddy;
    const float mean = a.stats[2 * r], inv = a.stats[2 * r + 1];
    const auto grad = [&](int c) { return to_f32(dy[c]) * (a.weight ? to_f32(static_cast<const P*>(a.weight)[c]) : 1.0f); };
    Compensated first, second;
    for (int c = threadIdx.x; c < a.dim; c += 1024) {
      const float g = grad(c);
      first.add(g);
      second.add(g * ((to_f32(x[c]) - mean) * inv));
    }
    float sums[2] = {first.s, second.s};
    row_sums<16>(sums, red, phase);
    const float ma = sums[0] * scale, mh = sums[1] * scale;
    for (int c = threadIdx.x; c < a.dim; c += 1024) {
      float d = inv * (grad(c) - ma - (to_f32(x[c]) - mean) * inv * mh);
      if (a.other) d += to_f32(static_cast<const T*>(a.other)[r * a.ldo + c]);
      put(static_cast<T*>(a.out) + r * a.dim + c, d);
    }
  }
}

// the sums of long rows: a thread per column, blockIdx.y every gridDim.y-th row
template <int DT>
__global__ __launch_bounds__(256) void long_part_kernel(NormArgs a) {
  typedef typename Elem<DT>::T T;
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.dim) return;
  float dw = 0.0f, db = 0.0f;
  for (int64_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
    const float g = to_f32(static_cast<const T*>(a.dy)[r * a.lddy + c]);
    dw += g * ((to_f32(static_cast<const T*>(a.x)[r * a.ldx + c]) - a.stats[2 * r]) * a.stats[2 * r + 1]);
    db += g;
  }
  a.part[int64_t(blockIdx.y) * 2 * a.dim + c] = dw;
  a.part[(int64_t(blockIdx.y) * 2 + 1) * a.dim + c] = db;
}

// dw and db from the workgroups' partials: 16 columns a workgroup, its 64 parts of 16 lanes every 64th partial, then the
// parts in order.
template <int PT>
__global__ __launch_bounds__(1024) void finish_kernel(const float* part, int parts, int dim, void* dweight, void* dbias) {
  typedef typename Elem<PT>::T P;
  __shared__ float red[64][17];
  const int column = threadIdx.x & 15, slice = threadIdx.x >> 4;
  const int64_t i = int64_t(blockIdx.x) * 16 + column, n = 2 * int64_t(dim);
  red[slice][column] = i < n ? sum_strided8(0.0f, part + i, n, slice, 64, parts) : 0.0f;
  __syncthreads();
  if (slice != 0 || i >= n) return;
  float s = 0.0f;
#pragma unroll
  for (int w = 0; w < 64; ++w) s += red[w][column];
  if (i < dim) {
    if (dweight) put(static_cast<P*>(dweight) + i, s);
  } else if (dbias) {
    put(static_cast<P*>(dbias) + (i - dim), s);
  }
}

int refuse(const char* what, const char* why) {
  set_error(std::string(what) + ": " + why);
  return -1;
}

bool misaligned(const void* p, int dt) { return reinterpret_cast<uintptr_t>(p) & (dt == kF32 ? 3 : 1); }

constexpr int64_t kMaxDim = int64_t(1) << 24, kMaxRows = int64_t(1) << 30;
constexpr int kWaveDim = 2048, kRegDim = 16384;  // widest row of one wave, of the register forms
constexpr int kBwdGroup = 8;                     // waves of a backward workgroup with rows of their own

// Workgroups of the backward pass: two a CU of rows by single waves (eight waves each), one a CU of
// longer rows; few rows, fewer.
int64_t bwd_groups(int64_t rows, int64_t dim) {
  if (rows <= 0) return 0;
  if (dim <= kWaveDim) {  // (as many rows for every wave)
    const int64_t each = ceil_div(rows, int64_t(512) * kBwdGroup);
    return ceil_div(rows, each * kBwdGroup);
  }
  if (dim <= kRegDim) return std::min<int64_t>(rows, dim <= 8192 ? 512 : 256);
  return std::min<int64_t>(rows, 64);
}

const char* norm_fault(int dt, int64_t rows, int64_t dim, int pt) {
  if (dt != kF32 && dt != kBf16) return "dtype must be 1 (fp32) or 2 (bf16)";
  if (pt != kF32 && pt != dt) return "parameters must be fp32 or of the rows' dtype";
  if (rows < 0 || rows > kMaxRows) return "row count outside 0 .. 2^30";
  if (dim < 1 || dim > kMaxDim) return "row length outside 1 .. 2^24";
  return nullptr;
}

template <int DT, int PT, int WAVES, int V>
void launch_fwd_rows(const NormArgs& a, hipStream_t st) {
  constexpr int per = WAVES == 1 ? kRowWaves : 1, threads = 64 * (WAVES == 1 ? kRowWaves : WAVES);
  const unsigned grid = unsigned(std::min<int64_t>(ceil_div(a.rows, int64_t(per)), 1 << 16));
  if (a.dim % 8 == 0) fwd_kernel<DT, PT, WAVES, V, true><<<grid, threads, 0, st>>>(a);
  else fwd_kernel<DT, PT, WAVES, V, false><<<grid, threads, 0, st>>>(a);
}

template <int DT, int PT>
void launch_fwd(const NormArgs& a, hipStream_t st) {
  if (a.dim <= 512) launch_fwd_rows<DT, PT, 1, 1>(a, st);
  else if (a.dim <= 1024) launch_fwd_rows<DT, PT, 1, 2>(a, st);
  else if (a.dim <= 2048) launch_fwd_rows<DT, PT, 1, 4>(a, st);
  else if (a.dim <= 4096) launch_fwd_rows<DT, PT, 4, 2>(a, st);
  else if (a.dim <= 8192) launch_fwd_rows<DT, PT, 4, 4>(a, st);
  else if (a.dim <= kRegDim) launch_fwd_rows<DT, PT, 16, 2>(a, st);
  else long_fwd_kernel<DT, PT><<<unsigned(std::min<int64_t>(a.rows, 1 << 16)), 1024, 0, st>>>(a);
}

template <int DT, int PT, int WAVES, int V, bool EVEN>
bool launch_bwd_form(const NormArgs& a, hipStream_t st) {
  constexpr int group = WAVES == 1 ? kBwdGroup : 1;
  constexpr size_t sums = size_t(2) * 2 * WAVES * sizeof(float), part = WAVES == 1 ? size_t(kBwdGroup) * V * 512 * sizeof(float) : 0;
  void (*f)(NormArgs) = bwd_kernel<DT, PT, WAVES, group, V, EVEN>;
  static const bool ok = hipFuncSetAttribute(reinterpret_cast<const void*>(f), hipFuncAttributeMaxDynamicSharedMemorySize,
                                             int(std::max(sums, part))) == hipSuccess;
  if (!ok) return false;
  f<<<unsigned(bwd_groups(a.rows, a.dim)), 64 * WAVES * group, a.part && part ? part : sums, st>>>(a);
  return true;
}

template <int DT, int PT, int WAVES, int V>
bool launch_bwd_rows(const NormArgs& a, hipStream_t st) {
  return a.dim % 8 == 0 ? launch_bwd_form<DT, PT, WAVES, V, true>(a, st) : launch_bwd_form<DT, PT, WAVES, V, false>(a, st);
}

template <int DT, int PT>
bool launch_bwd(const NormArgs& a, hipStream_t st) {
  if (a.dim <= 512) return launch_bwd_rows<DT, PT, 1, 1>(a, st);
  if (a.dim <= 1024) return launch_bwd_rows<DT, PT, 1, 2>(a, st);
  if (a.dim <= 2048) return launch_bwd_rows<DT, PT, 1, 4>(a, st);
  if (a.dim <= 4096) return launch_bwd_rows<DT, PT, 4, 2>(a, st);
  if (a.dim <= 8192) return launch_bwd_rows<DT, PT, 4, 4>(a, st);
  if (a.dim <= kRegDim) return launch_bwd_rows<DT, PT, 16, 2>(a, st);
  if (a.out) long_dx_kernel<DT, PT><<<unsigned(std::min<int64_t>(a.rows, 1 << 16)), 1024, 0, st>>>(a);
  if (a.part)
    long_part_kernel<DT><<<dim3(unsigned(ceil_div(a.dim, 256)), unsigned(bwd_groups(a.rows, a.dim))), 256, 0, st>>>(a);
  return true;
}

}  // namespace
}  // namespace xdna

using namespace xdna;

extern "C" {

int xdna_layer_norm(const void* x, int64_t ldx, const void* residual, int64_t ldr, int dtype, int64_t rows, int64_t dim,
                    const void* weight, const void* bias, int param_dtype, float eps, void* sum, void* y, float* stats,
                    void* stream) {
  const char* what = "xdna_layer_norm";
  if (const char* why = norm_fault(dtype, rows, dim, param_dtype)) return refuse(what, why);
  if (!(eps >= 0.0f) || eps > 3.0e38f) return refuse(what, "eps must be finite and not negative");
  if (rows > 1 && (ldx < dim || (residual && ldr < dim))) return refuse(what, "rows overlap");
  if (rows == 0) return 0;
  if (!x || !y || (residual && !sum)) return refuse(what, "null operand");
  if (misaligned(x, dtype) || misaligned(residual, dtype) || misaligned(sum, dtype) || misaligned(y, dtype) ||
      misaligned(weight, param_dtype) || misaligned(bias, param_dtype) || misaligned(stats, kF32))
    return refuse(what, "misaligned operand");
  if (!admit_launch(what)) return -1;
  NormArgs a = {};
  a.x = x;
  a.other = residual;
  a.ldx = rows > 1 ? ldx : dim;
  a.ldo = rows > 1 ? ldr : dim;
  a.rows = rows;
  a.dim = int(dim);
  a.weight = weight;
  a.bias = bias;
  a.eps = eps;
  a.sum = sum;
  a.out = y;
  a.stats = stats;
  hipStream_t st = as_stream(stream);
  if (dtype == kF32) launch_fwd<kF32, kF32>(a, st);
  else if (param_dtype == kF32) launch_fwd<kBf16, kF32>(a, st);
  else launch_fwd<kBf16, kBf16>(a, st);
  return check_launch(what);
}

size_t xdna_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t dim) {
  if (rows < 0 || rows > kMaxRows || dim < 1 || dim > kMaxDim) return 0;
  return size_t(bwd_groups(rows, dim)) * 2 * size_t(dim) * sizeof(float);
}

int xdna_layer_norm_bwd(const void* dy, int64_t lddy, const void* dsum, int64_t ldds, const void* x, int64_t ldx, int dtype,
                        int64_t rows, int64_t dim, const void* weight, int param_dtype, const float* stats, void* dx,
                        void* dweight, void* dbias, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "xdna_layer_norm_bwd";
  if (const char* why = norm_fault(dtype, rows, dim, param_dtype)) return refuse(what, why);
  if (rows > 1 && (lddy < dim || ldx < dim || (dsum && ldds < dim))) return refuse(what, "rows overlap");
  const bool params = dweight || dbias;
  if (rows > 0 && (!dy || !x || !stats)) return refuse(what, "null operand");
  if (misaligned(dy, dtype) || misaligned(dsum, dtype) || misaligned(x, dtype) || misaligned(dx, dtype) ||
      misaligned(weight, param_dtype) || misaligned(dweight, param_dtype) || misaligned(dbias, param_dtype) ||
      misaligned(stats, kF32))
    return refuse(what, "misaligned operand");
  if (params && rows > 0 &&
      (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < xdna_layer_norm_bwd_workspace_bytes(rows, dim)))
    return refuse(what, "workspace missing, misaligned or too small");
  if ((rows == 0 || !dx) && !params) return 0;
  if (!admit_launch(what)) return -1;
  NormArgs a = {};
  a.x = x;
  a.other = dsum;
  a.dy = dy;
  a.ldx = rows > 1 ? ldx : dim;
  a.ldo = rows > 1 ? ldds : dim;
  a.lddy = rows > 1 ? lddy : dim;
  a.rows = rows;
  a.dim = int(dim);
  a.weight = weight;
  a.out = dx;
  a.stats = const_cast<float*>(stats);
  a.part = params ? static_cast<float*>(workspace) : nullptr;
  hipStream_t st = as_stream(stream);
  if (rows > 0) {
    const bool ok = dtype == kF32            ? launch_bwd<kF32, kF32>(a, st)
                    : param_dtype == kF32 ? launch_bwd<kBf16, kF32>(a, st)
                                             : launch_bwd<kBf16, kBf16>(a, st);
    if (!ok) return refuse(what, "the kernel's LDS size cannot be had");
  }
  if (params) {
    const unsigned grid = unsigned(ceil_div(2 * dim, int64_t(16)));
    const int parts = int(bwd_groups(rows, dim));
    if (param_dtype == kF32) finish_kernel<kF32><<<grid, 1024, 0, st>>>(a.part, parts, a.dim, dweight, dbias);
    else finish_kernel<kBf16><<<grid, 1024, 0, st>>>(a.part, parts, a.dim, dweight, dbias);
  }
  return check_launch(what);
}

}  // extern "C"
