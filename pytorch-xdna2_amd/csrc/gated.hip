// Gated feed-forward on gfx950 MFMA: h = act(x Wg^T) * (x Wu^T), both projections, the
// activation and the product in one kernel, and its backward pass.  The reference would run
// these as separate mm / activation / mul ops (torch_xdna_device.cpp:4360-4417, 5124-5260).
//
// w holds [Wg; Wu], 2F rows of K.  The projections are summed in fp32 and stay there through
// the activation and the product; h is rounded once.  For training g and u are kept as bf16
// (the form the framework keeps every activation in): the backward reads them instead of
// multiplying again.
//   dg = dh u act'(g), du = dh act(g), as [dg du] (M x 2F), so that dx = [dg du] w and
//   dw = [dg du]^T x are one product each.
#include "common.h"
#include "mfma.h"

#include "../../include/xdna_hip.h"

namespace xdna {
namespace {

enum Act { kSilu = 0, kGelu = 1, kRelu = 2 };

template <int ACT>
__device__ inline float act_of(float g) {
  if constexpr (ACT == kSilu) return g / (1.0f + __expf(-g));
  if constexpr (ACT == kGelu) return g * 0.5f * (1.0f + erff(g * 0.70710678118654752f));
  return g > 0.0f ? g : (g != g ? g : 0.0f);
}

// act(g) and act'(g)
template <int ACT>
__device__ inline float2 act_pair(float g) {
  if constexpr (ACT == kSilu) {
    const float s = 1.0f / (1.0f + __expf(-g));
    return make_float2(g * s, s * (1.0f + g * (1.0f - s)));
  }
  if constexpr (ACT == kGelu) {
    const float cdf = 0.5f * (1.0f + erff(g * 0.70710678118654752f));
    return make_float2(g * cdf, cdf + g * 0.3989422804014327f * __expf(-0.5f * g * g));
  }
  return g > 0.0f ? make_float2(g, 1.0f) : make_float2(g != g ? g : 0.0f, 0.0f);
}

struct GatedArgs {
  const uint16_t* x;  // [M][K], row stride ldx
  const uint16_t* w;  // [2F][K], row stride ldw: gate rows, then up rows
  uint16_t* h;        // [M][F]
  uint16_t* gu;       // [M][2F] or null
  int M, K, F;
  int64_t ldx, ldw;
};

// ---- tiles of 64 rows x 64 hidden units ---------------------------------------------------
// Four waves of 32 x 32, each with a gate and an up accumulator; k-tiles of 64 in LDS ([row][k],
// pitch 72) with the next one's loads in registers meanwhile.  Loads are 16 bytes at any
// element-aligned address (gfx950 takes them), elements past K are zeros.
constexpr int kT = 64, kKT = 64, kP = 72;

__device__ inline Pix8 row_vec(const uint16_t* p, int n) {  // n elements, zeros after them
  if (n >= 8) return *reinterpret_cast<const Pix8*>(p);
  Pix8 q = {{0u, 0u, 0u, 0u}};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < n) q.v[e >> 1] |= uint32_t(p[e]) << ((e & 1) * 16);
  return q;
}

template <int ACT, bool KEEP>
__global__ __launch_bounds__(256) void gated_tile_kernel(GatedArgs a) {
  __shared__ __attribute__((aligned(16))) uint16_t xs[2][kT * kP];
  __shared__ __attribute__((aligned(16))) uint16_t ws[2][2 * kT * kP];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = wave & 1, wn = wave >> 1;
  const int m0 = blockIdx.y * kT, f0 = blockIdx.x * kT;
  const int lr = lane & 31, lk = (lane >> 5) * 8;
  f32x16_t g = zero_acc(), u = zero_acc();
  Pix8 rx[2], rw[4];
  const auto load = [&](int k0) {
    const int kv = k0 + (tid & 7) * 8;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int m = m0 + (tid >> 3) + j * 32;
      rx[j] = row_vec(a.x + int64_t(min(m, a.M - 1)) * a.ldx + min(kv, a.K), m < a.M ? a.K - kv : 0);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int f = f0 + (tid >> 3) + (j & 1) * 32;
      rw[j] = row_vec(a.w + (int64_t(min(f, a.F - 1)) + (j >> 1) * int64_t(a.F)) * a.ldw + min(kv, a.K), f < a.F ? a.K - kv : 0);
    }
  };
  const auto store = [&](int b) {
    const int at = (tid >> 3) * kP + (tid & 7) * 8;
#pragma unroll
    for (int j = 0; j < 2; ++j)
      *reinterpret_cast<uint4*>(xs[b] + at + j * 32 * kP) = make_uint4(rx[j].v[0], rx[j].v[1], rx[j].v[2], rx[j].v[3]);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<uint4*>(ws[b] + at + j * 32 * kP) = make_uint4(rw[j].v[0], rw[j].v[1], rw[j].v[2], rw[j].v[3]);
  };
  load(0);
  store(0);
  __syncthreads();
  int b = 0;
  for (int k0 = 0; k0 < a.K; k0 += kKT) {
    const bool more = k0 + kKT < a.K;
    if (more) load(k0 + kKT);
#pragma unroll
    for (int ks = 0; ks < kKT / 16; ++ks) {
      const bf16x8_t fx = as_bf16x8(*reinterpret_cast<const uint4*>(xs[b] + (wm * 32 + lr) * kP + ks * 16 + lk));
      const bf16x8_t fg = as_bf16x8(*reinterpret_cast<const uint4*>(ws[b] + (wn * 32 + lr) * kP + ks * 16 + lk));
      const bf16x8_t fu = as_bf16x8(*reinterpret_cast<const uint4*>(ws[b] + (kT + wn * 32 + lr) * kP + ks * 16 + lk));
      g = mfma_32x32x16(fx, fg, g);
      u = mfma_32x32x16(fx, fu, u);
    }
    if (more) store(b ^ 1);  // its last reads ended before the previous barrier
    __syncthreads();
    b ^= 1;
  }
  const int f = f0 + wn * 32 + lr;
  if (f >= a.F) return;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int m = m0 + wm * 32 + mfma_row(r, lane);
    if (m >= a.M) continue;
    a.h[int64_t(m) * a.F + f] = f32_to_bf16(act_of<ACT>(g[r]) * u[r]);
    if constexpr (KEEP) {
      a.gu[int64_t(m) * 2 * a.F + f] = f32_to_bf16(g[r]);
      a.gu[int64_t(m) * 2 * a.F + a.F + f] = f32_to_bf16(u[r]);
    }
  }
}

// ---- backward, elementwise: [dg du] from dh and the kept [g u] ------------------------------
struct GatedBwdArgs {
  const uint16_t* dh;  // [M][F], row stride ld
  const uint16_t* gu;  // [M][2F]
  uint16_t* dgu;       // [M][2F]
  int64_t M, ld;
  int F, windows;      // windows of 8 per row
};

template <int ACT>
__global__ __launch_bounds__(256) void gated_bwd_kernel(GatedBwdArgs a) {
  const int64_t total = a.M * a.windows;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < total; i += int64_t(gridDim.x) * 256) {
    const int64_t m = i / a.windows;
    const int f = int(i - m * a.windows) * 8, n = a.F - f;
    const uint16_t* gp = a.gu + m * 2 * a.F + f;
    uint16_t* dp = a.dgu + m * 2 * a.F + f;
    const Pix8 qd = row_vec(a.dh + m * a.ld + f, n), qg = row_vec(gp, n), qu = row_vec(gp + a.F, n);
    Pix8 og, ou;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t pg = 0, pu = 0;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const auto half = [&](uint32_t w) { return __uint_as_float(s ? w & 0xFFFF0000u : w << 16); };
        const float d = half(qd.v[e]), u = half(qu.v[e]);
        const float2 t = act_pair<ACT>(half(qg.v[e]));
        pg |= uint32_t(f32_to_bf16(d * u * t.y)) << (16 * s);
        pu |= uint32_t(f32_to_bf16(d * t.x)) << (16 * s);
      }
      og.v[e] = pg;
      ou.v[e] = pu;
    }
    if (n >= 8) {
      *reinterpret_cast<Pix8*>(dp) = og;
      *reinterpret_cast<Pix8*>(dp + a.F) = ou;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n) {
          dp[e] = uint16_t(og.v[e >> 1] >> (16 * (e & 1)));
          dp[a.F + e] = uint16_t(ou.v[e >> 1] >> (16 * (e & 1)));
        }
    }
  }
}

int refuse(const char* what, const char* why) {
  set_error(std::string(what) + ": " + why);
  return -1;
}

constexpr int64_t kMaxSide = int64_t(1) << 30;

const char* gated_fault(int64_t M, int64_t K, int64_t F, int act) {
  if (act < 0 || act > 2) return "activation must be 0 (silu), 1 (gelu) or 2 (relu)";
  if (M < 0 || M > kMaxSide || K < 1 || K > kMaxSide || F < 1 || F > kMaxSide / 2) return "sizes outside 1 .. 2^30";
  return nullptr;
}

bool odd(const void* p) { return reinterpret_cast<uintptr_t>(p) & 1; }

template <int ACT>
void launch_tile(const GatedArgs& a, hipStream_t st) {
  const dim3 grid(unsigned(ceil_div(a.F, kT)), unsigned(ceil_div(a.M, kT)));
  if (a.gu) gated_tile_kernel<ACT, true><<<grid, 256, 0, st>>>(a);
  else gated_tile_kernel<ACT, false><<<grid, 256, 0, st>>>(a);
}

}  // namespace
}  // namespace xdna

using namespace xdna;

extern "C" {

int xdna_gated_bf16(const uint16_t* x, int64_t ldx, const uint16_t* w, int64_t ldw, int64_t M, int64_t K, int64_t F,
                    int act, uint16_t* h, uint16_t* gu, void* stream) {
  const char* what = "xdna_gated_bf16";
  if (const char* why = gated_fault(M, K, F, act)) return refuse(what, why);
  if ((ldx < K && M > 1) || ldw < K) return refuse(what, "rows overlap");
  if (ceil_div(M, int64_t(kT)) > 65535) return refuse(what, "too many rows");
  if (M == 0) return 0;
  if (!x || !w || !h) return refuse(what, "null operand");
  if (odd(x) || odd(w) || odd(h) || odd(gu)) return refuse(what, "misaligned operand");
  if (!admit_launch(what)) return -1;
  const GatedArgs a = {x, w, h, gu, int(M), int(K), int(F), ldx, ldw};
  hipStream_t st = as_stream(stream);
  if (act == kSilu) launch_tile<kSilu>(a, st);
  else if (act == kGelu) launch_tile<kGelu>(a, st);
  else launch_tile<kRelu>(a, st);
  return check_launch(what);
}

int xdna_gated_bwd_bf16(const uint16_t* dh, int64_t ld, const uint16_t* gu, int64_t M, int64_t F, int act, uint16_t* dgu,
                        void* stream) {
  const char* what = "xdna_gated_bwd_bf16";
  if (const char* why = gated_fault(M, 1, F, act)) return refuse(what, why);
  if (M == 0) return 0;
  if (!dh || !gu || !dgu) return refuse(what, "null operand");
  if (odd(dh) || odd(gu) || odd(dgu)) return refuse(what, "misaligned operand");
  if (!admit_launch(what)) return -1;
  const GatedBwdArgs a = {dh, gu, dgu, M, ld, int(F), int(ceil_div(F, int64_t(8)))};
  const unsigned grid = unsigned(std::min<int64_t>(ceil_div(a.M * a.windows, int64_t(256)), 16384));
  hipStream_t st = as_stream(stream);
  if (act == kSilu) gated_bwd_kernel<kSilu><<<grid, 256, 0, st>>>(a);
  else if (act == kGelu) gated_bwd_kernel<kGelu><<<grid, 256, 0, st>>>(a);
  else gated_bwd_kernel<kRelu><<<grid, 256, 0, st>>>(a);
  return check_launch(what);
}

}  // extern "C"
