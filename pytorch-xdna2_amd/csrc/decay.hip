// Linear attention with a decay for each head, on gfx950 MFMA: the chunked form for training and
// prompts with its backward pass, and the recurrent form for single tokens.  The reference reaches
// such work only through its zero-copy CPU fallback (torch_xdna_device.cpp:5124-5260).
//
//   S_t = a S_{t-1} + k_t^T v_t,   o_t = scale q_t S_t,   a = exp(log_decay[head]),  S: Dk x Dv
//
// Chunks of C = 128 tokens: with S the state before a chunk and i, j places in it,
//   o_i = scale (sum over j <= i of a^(i-j) (q_i k_j) v_j + a^(i+1) q_i S),
//   S' = a^n S + sum over j of a^(n-1-j) k_j^T v_j         (n tokens in the chunk).
// The backward pass is three more walks of the same form.  With G_t the gradient of S_t, which
// obeys G_t = a G_{t+1} + scale q_t^T do_t,
//   dq_t = scale do_t S_t^T : the walk of (do, v, k), with S transposed,
//   dv_t = k_t G_t          : the walk of (k, q, do) from the last token to the first,
//   dk_t = v_t G_t^T        : the walk of (v, do, q), likewise, with G transposed,
// so one kernel does all four.  A backward walk starts from the final state's gradient R, which is
// not decayed before its first token, and ends at the first state's gradient: there the powers of a
// that q and k take are a^i and a^(n-j) in place of a^(i+1) and a^(n-1-j) (`lead` 0 for 1).
//
// A workgroup of four waves walks one sequence, head and 64 columns of v, the state in its registers
// in fp32.  Rounded to bf16 are the weighted scores and the state as an operand of q S (one rounding
// each beside the result's own, error against 64 bits 1.4 times that of the result's rounding);
// the weighted v of the state's own sum is carried in two bf16 (16 bits), since the state is fp32.
#include "common.h"
#include "mfma.h"

#include "../../include/xdna_hip.h"

namespace xdna {
namespace {

constexpr int kC = 128;       // tokens of a chunk: 32 for each wave
constexpr int kVB = 64;       // columns of v of a workgroup
constexpr int kMaxHead = 128;
constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

struct Heads {
  const uint16_t* p;
  int64_t sb, st, sh;
  int share;  // heads of the walk that read one head of this tensor
};

// One walk over all sequences: o = [scores by p_scale] v + q_scale [weights] q S, S from k and
// kv_scale v.
struct Walk {
  Heads q, k, v;
  int dk, dv;       // head sizes of k and q, and of v
  int vb;           // workgroups along dv
  int reverse;
  float p_scale, q_scale, kv_scale;
  void* out;        // dense [B][T][H][dv], bf16 or (wide) fp32
  int wide;
  const float* s0;  // state before the first token, [B][H] x (dk, dv by these strides), or null
  int64_t s0_k, s0_v;
  float* s1;        // the state behind the last token, dense, or null
  float* local;     // segments' own states [B][H][segments - 1] x (dk, dv by these strides)
  int64_t local_k, local_v;
};

struct DecayArgs {
  Walk walk[3];
  int64_t first[4];  // workgroups before each walk
  int n;             // walks
  int B, T, H;
  const float* log_decay;
  const void* lengths;  // null: T
  int index_bytes;
  int segments, chunks;  // of a sequence, and chunks of a segment
};

typedef short i16x4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));

__device__ inline float pow2(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ inline Pix8 vec_of(const uint16_t* p, int n) {  // n elements, zeros after them
  if (n >= 8) return *reinterpret_cast<const Pix8*>(p);
  Pix8 q = {{0u, 0u, 0u, 0u}};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < n) q.v[e >> 1] |= uint32_t(p[e]) << ((e & 1) * 16);
  return q;
}

__device__ inline uint32_t pack2(float a, float b) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}

// MFMA operand of a [k][row] tile in LDS: rows c0 + lane % 32, four k rows from k0 (of the lane's
// half) on and four from k1 on
__device__ inline bf16x8_t frag_tr(const uint16_t* tile, int pitch, int k0, int k1, int c0, int lane) {
  const int g = lane >> 4, j = lane & 15;
  const int c = c0 + 16 * (g & 1) + 4 * (j & 3);
  const uint16_t* lo = tile + (k0 + (j >> 2)) * pitch + c;
  const uint16_t* hi = tile + (k1 + (j >> 2)) * pitch + c;
  const u32x2_t a = __builtin_bit_cast(
      u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4_t*)(lo)));
  const u32x2_t b = __builtin_bit_cast(
      u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4_t*)(hi)));
  return as_bf16x8(u32x4_t{a[0], a[1], b[0], b[1]});
}

__device__ inline int64_t length_of(const DecayArgs& a, int b) {
  if (!a.lengths) return a.T;
  const int64_t n = a.index_bytes == 8 ? static_cast<const int64_t*>(a.lengths)[b] : static_cast<const int32_t*>(a.lengths)[b];
  return n < 0 ? 0 : n < a.T ? n : a.T;
}

template <int KT>
struct Lds {
  static constexpr int kPitch = KT + 16, vPitch = kVB + 16, sPitch = KT + 8;
  static constexpr int kElems = kC * kPitch, vElems = kC * vPitch, sElems = kVB * sPitch;
  static constexpr size_t bytes = size_t(kElems + vElems + sElems) * 2 + kC * sizeof(float);
};

// STATE: the state of a segment by itself, from zero, and no outputs.
template <int KT, bool STATE>
__global__ __launch_bounds__(kThreads, 2) void walk_kernel(DecayArgs a) {
  using L = Lds<KT>;
  constexpr int KV = KT / 16, VV = kVB / 16;  // 16-byte vectors a thread of a chunk of k and v
  constexpr int NS = KT / 64;                 // a wave's 32 x 32 tiles of the state
  extern __shared__ __attribute__((aligned(16))) uint16_t smem[];
  uint16_t* ks = smem;               // [token][dk]
  uint16_t* vs = ks + L::kElems;     // [token][dv]
  uint16_t* ss = vs + L::vElems;     // [dv][dk], the state before the chunk
  float* wt = reinterpret_cast<float*>(ss + L::sElems);  // [token] weight of v in the state's sum

  // workgroups of one sequence and head next to each other on one XCD (each has its own L2)
  const int n_all = int(gridDim.x), xcd = int(blockIdx.x) % 8;
  int64_t id = int64_t(xcd) * (n_all / 8) + min(xcd, n_all % 8) + int(blockIdx.x) / 8;
  const int wi = a.n > 2 && id >= a.first[2] ? 2 : a.n > 1 && id >= a.first[1] ? 1 : 0;
  const Walk& w = a.walk[wi];
  id -= a.first[wi];
  const int n_seg = STATE ? a.segments - 1 : a.segments;
  const int vb = int(id % w.vb);
  const int seg = int(id / w.vb % n_seg);
  const int head = int(id / (int64_t(w.vb) * n_seg) % a.H), batch = int(id / (int64_t(w.vb) * n_seg) / a.H);
  const int64_t bh = int64_t(batch) * a.H + head;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, half = lane >> 5;
  const int len = int(length_of(a, batch));
  const int seg_len = a.chunks * kC, begin = seg * seg_len;
  const int todo = max(0, min(len - begin, seg_len));  // tokens of this segment
  const int lead = w.reverse ? 0 : 1;
  float g2 = a.log_decay[head] * kLog2e;
  g2 = g2 < -1e4f ? -1e4f : g2;  // (exp(-inf) as exp(-1e4): 0, and 0 times it is 0)
  const int d0 = vb * kVB, dvn = min(w.dv - d0, kVB);  // columns of v

  const uint16_t* qp = w.q.p + batch * w.q.sb + int64_t(head / w.q.share) * w.q.sh;
  const uint16_t* kp = w.k.p + batch * w.k.sb + int64_t(head / w.k.share) * w.k.sh;
  const uint16_t* vp = w.v.p + batch * w.v.sb + int64_t(head / w.v.share) * w.v.sh + d0;
  // place i of the walk is this token
  const auto token = [&](int i) { return int64_t(w.reverse ? len - 1 - i : i); };

  // ---- tokens behind the sequence: zeros
  if constexpr (!STATE) {
    const int from = max(begin, len), to = min(begin + seg_len, a.T);
    for (int64_t i = tid; i < int64_t(to - from) * kVB; i += kThreads) {
      const int64_t t = from + i / kVB;
      const int c = int(i % kVB);
      if (c < dvn) {
        const int64_t at = ((int64_t(batch) * a.T + t) * a.H + head) * w.dv + d0 + c;
        if (w.wide) static_cast<float*>(w.out)[at] = 0.0f;
        else static_cast<uint16_t*>(w.out)[at] = 0;
      }
    }
  }
  const bool last = !STATE && w.s1 && seg == max(0, (len + seg_len - 1) / seg_len - 1);
  if (todo == 0 && !last && !STATE) return;

  // ---- the state: tile x of this wave is dk 32 kt(x) .., dv 32 (wave % 2) ..
  f32x16_t S[NS];
#pragma unroll
  for (int x = 0; x < NS; ++x) S[x] = zero_acc();
  const int vt = wave & 1;
  const auto dk_of = [&](int x, int i) { return 32 * ((wave >> 1) * NS + x) + mfma_row(i, lane); };
  const int dv_of = 32 * vt + l32;
  if constexpr (!STATE) {
    const auto add = [&](const float* s, int64_t sk, int64_t sv) {
#pragma unroll
      for (int x = 0; x < NS; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int dk = dk_of(x, i);
          if (dk < w.dk && dv_of < dvn) S[x][i] += s[dk * sk + (d0 + dv_of) * sv];
        }
    };
    const int64_t per = int64_t(w.dk) * w.dv;
    if (w.s0) add(w.s0 + bh * per, w.s0_k, w.s0_v);
    for (int j = 0; j < seg; ++j) {  // the segments before this one
      const float f = pow2(g2 * float(max(0, min(len - j * seg_len, seg_len))));
#pragma unroll
      for (int x = 0; x < NS; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i) S[x][i] *= f;
      add(w.local + (bh * (a.segments - 1) + j) * per, w.local_k, w.local_v);
    }
  }

  // ---- loads of a chunk
  Pix8 kr[KV], vr[VV];
  const auto load_kv = [&](int c0, int n) {
#pragma unroll
    for (int j = 0; j < KV; ++j) {
      const int i = tid + j * kThreads, r = i / (KT / 8), c = i % (KT / 8) * 8;
      kr[j] = {{0u, 0u, 0u, 0u}};
      if (r < n && c < w.dk) kr[j] = vec_of(kp + token(begin + c0 + r) * w.k.st + c, w.dk - c);
    }
#pragma unroll
    for (int j = 0; j < VV; ++j) {
      const int i = tid + j * kThreads, r = i / (kVB / 8), c = i % (kVB / 8) * 8;
      vr[j] = {{0u, 0u, 0u, 0u}};
      if (r < n && c < dvn) vr[j] = vec_of(vp + token(begin + c0 + r) * w.v.st + c, dvn - c);
    }
  };
  const auto store_kv = [&]() {
#pragma unroll
    for (int j = 0; j < KV; ++j) {
      const int i = tid + j * kThreads, r = i / (KT / 8), c = i % (KT / 8) * 8;
      *reinterpret_cast<uint4*>(ks + r * L::kPitch + c) = make_uint4(kr[j].v[0], kr[j].v[1], kr[j].v[2], kr[j].v[3]);
    }
#pragma unroll
    for (int j = 0; j < VV; ++j) {
      const int i = tid + j * kThreads, r = i / (kVB / 8), c = i % (kVB / 8) * 8;
      *reinterpret_cast<uint4*>(vs + r * L::vPitch + c) = make_uint4(vr[j].v[0], vr[j].v[1], vr[j].v[2], vr[j].v[3]);
    }
  };
  const auto store_weights = [&](int n) {
    if (tid < kC) wt[tid] = tid < n ? w.kv_scale * pow2(g2 * float(n - lead - tid)) : 0.0f;
  };
  const auto store_state = [&]() {
#pragma unroll
    for (int x = 0; x < NS; ++x)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<uint2*>(ss + dv_of * L::sPitch + dk_of(x, 4 * q)) =
            make_uint2(pack2(S[x][4 * q], S[x][4 * q + 1]), pack2(S[x][4 * q + 2], S[x][4 * q + 3]));
  };
  // q of the wave's 32 tokens: lane's token, k 16 kk + 8 half ..
  Pix8 qf[KT / 16];
  const auto load_q = [&](int c0, int n) {
    const int i = 32 * wave + l32;
#pragma unroll
    for (int kk = 0; kk < KT / 16; ++kk) {
      const int c = 16 * kk + 8 * half;
      qf[kk] = {{0u, 0u, 0u, 0u}};
      if (i < n && c < w.dk) qf[kk] = vec_of(qp + token(begin + c0 + i) * w.q.st + c, w.dk - c);
    }
  };
  const auto frag = [](const Pix8& v) { return as_bf16x8(u32x4_t{v.v[0], v.v[1], v.v[2], v.v[3]}); };

  // ---- weights of this lane's token (32 wave + l32) against the 16 tokens of its score registers:
  // inside the wave's own 32, and against the 32 before them
  float diag[16], off[16];
  float a32 = 0.0f, row_weight = 0.0f;
  if constexpr (!STATE) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int s = mfma_row(i, lane);
      diag[i] = l32 >= s ? w.p_scale * pow2(g2 * float(l32 - s)) : 0.0f;
      off[i] = w.p_scale * pow2(g2 * float(32 + l32 - s));
    }
    a32 = pow2(g2 * 32.0f);
    row_weight = w.q_scale * pow2(g2 * float(32 * wave + l32 + lead));
  }

  int n = min(todo, kC);
  if (todo > 0) {
    load_kv(0, n);
    if constexpr (!STATE) load_q(0, n);
    store_kv();
    store_weights(n);
    if constexpr (!STATE) store_state();
  }
  __syncthreads();
  for (int c0 = 0; c0 < todo; c0 += kC) {
    const int next = min(todo - c0 - kC, kC);  // tokens of the next chunk
    if (next > 0) load_kv(c0 + kC, next);
    if constexpr (!STATE) {
      const int i = 32 * wave + l32;
      f32x16_t o[2] = {zero_acc(), zero_acc()};  // [dv][token]
      if (32 * wave < n) {
#pragma unroll
        for (int kk = 0; kk < KT / 16; ++kk)
#pragma unroll
          for (int t = 0; t < 2; ++t)
            o[t] = mfma_32x32x16(as_bf16x8(*reinterpret_cast<const u32x4_t*>(ss + (32 * t + l32) * L::sPitch + 16 * kk + 8 * half)),
                                 frag(qf[kk]), o[t]);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int x = 0; x < 16; ++x) o[t][x] *= row_weight;
        float f = 1.0f;
        for (int j = wave; j >= 0; --j) {
          f32x16_t p = zero_acc();  // [key token][token]
#pragma unroll
          for (int kk = 0; kk < KT / 16; ++kk)
            p = mfma_32x32x16(as_bf16x8(*reinterpret_cast<const u32x4_t*>(ks + (32 * j + l32) * L::kPitch + 16 * kk + 8 * half)),
                              frag(qf[kk]), p);
          uint32_t pw[8];
          if (j == wave) {
#pragma unroll
            for (int x = 0; x < 8; ++x)
              pw[x] = pack2(diag[2 * x] != 0.0f ? p[2 * x] * diag[2 * x] : 0.0f,
                            diag[2 * x + 1] != 0.0f ? p[2 * x + 1] * diag[2 * x + 1] : 0.0f);
          } else {
#pragma unroll
            for (int x = 0; x < 8; ++x) pw[x] = pack2(p[2 * x] * (off[2 * x] * f), p[2 * x + 1] * (off[2 * x + 1] * f));
            f *= a32;
          }
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const bf16x8_t pf = as_bf16x8(u32x4_t{pw[4 * s], pw[4 * s + 1], pw[4 * s + 2], pw[4 * s + 3]});
            const int k0 = 32 * j + 16 * s + 4 * half;
#pragma unroll
            for (int t = 0; t < 2; ++t) o[t] = mfma_32x32x16(frag_tr(vs, L::vPitch, k0, k0 + 8, 32 * t, lane), pf, o[t]);
          }
        }
      }
      if (next > 0) load_q(c0 + kC, next);
      if (i < n) {
        const int64_t at = ((int64_t(batch) * a.T + token(begin + c0 + i)) * a.H + head) * w.dv + d0;
        if (w.wide) {
          float* to = static_cast<float*>(w.out) + at;
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int x = 0; x < 16; ++x) {
              const int c = 32 * t + mfma_row(x, lane);
              if (c < dvn) to[c] = o[t][x];
            }
        } else {
          uint16_t* to = static_cast<uint16_t*>(w.out) + at;
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int x = 0; x < 16; ++x) {
              const int c = 32 * t + mfma_row(x, lane);
              if (c < dvn) to[c] = f32_to_bf16(o[t][x]);
            }
        }
      }
    }
    // ---- the state behind the chunk
    const float f = pow2(g2 * float(n));
#pragma unroll
    for (int x = 0; x < NS; ++x)
#pragma unroll
      for (int i = 0; i < 16; ++i) S[x][i] *= f;
    for (int s = 0; 16 * s < n; ++s) {
      const int k0 = 16 * s + 8 * half;
      const bf16x8_t v = frag_tr(vs, L::vPitch, k0, k0 + 4, 32 * vt, lane);
      const u32x4_t vu = __builtin_bit_cast(u32x4_t, v);
      const float4 w0 = *reinterpret_cast<const float4*>(wt + k0), w1 = *reinterpret_cast<const float4*>(wt + k0 + 4);
      const float ww[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
      u32x4_t hi, lo;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x0 = __uint_as_float(vu[e] << 16) * ww[2 * e], x1 = __uint_as_float(vu[e] & 0xFFFF0000u) * ww[2 * e + 1];
        hi[e] = pack2(x0, x1);
        lo[e] = pack2(x0 - __uint_as_float(hi[e] << 16), x1 - __uint_as_float(hi[e] & 0xFFFF0000u));
      }
#pragma unroll
      for (int x = 0; x < NS; ++x) {
        const bf16x8_t k = frag_tr(ks, L::kPitch, k0, k0 + 4, 32 * ((wave >> 1) * NS + x), lane);
        S[x] = mfma_32x32x16(k, as_bf16x8(lo), S[x]);
        S[x] = mfma_32x32x16(k, as_bf16x8(hi), S[x]);
      }
    }
    if (next > 0) {
      __syncthreads();
      store_kv();
      if (next < kC) store_weights(next);
      if constexpr (!STATE) store_state();
      __syncthreads();
      n = next;
    }
  }
  if (STATE || last) {
    const int64_t per = int64_t(w.dk) * w.dv;
    float* to = STATE ? w.local + (bh * n_seg + seg) * per : w.s1 + bh * per;
#pragma unroll
    for (int x = 0; x < NS; ++x)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int dk = dk_of(x, i);
        if (dk < w.dk && dv_of < dvn) to[int64_t(dk) * w.dv + d0 + dv_of] = S[x][i];
      }
  }
}

// Gradients of shared heads: out[.., g, d] = the sum over the group's heads in order, rounded once.
__global__ __launch_bounds__(256) void group_kernel(const float* from, uint16_t* to, int64_t rows, int group, int d) {
  const int64_t n = rows * d;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) {
    const int64_t r = i / d;
    const float* p = from + r * group * d + (i - r * d);
    float s = 0.0f;
    for (int j = 0; j < group; ++j) s += p[int64_t(j) * d];
    to[i] = f32_to_bf16(s);
  }
}

// ---- single tokens --------------------------------------------------------------------------------
// S = a S + k^T v in place, o = scale q S.  Bound by the state's bytes, read and written once: a
// workgroup takes a head and 32 columns of v, a thread four columns of every 32nd row.
struct StepArgs {
  Heads q, k, v;
  int B, H, dk, dv;
  const float* log_decay;
  float* state;  // [slots][H][dk][dv]
  int64_t slots;
  const void* index;  // null: slot b
  int index_bytes;
  float scale;
  uint16_t* out;  // dense [B][H][dv]
  int tiles;      // of 32 columns
  int vec;        // rows of whole 16-byte vectors
};

__device__ inline int64_t slot_of(const StepArgs& a, int b) {
  if (!a.index) return b;
  return a.index_bytes == 8 ? static_cast<const int64_t*>(a.index)[b] : static_cast<const int32_t*>(a.index)[b];
}

__global__ __launch_bounds__(256) void step_kernel(StepArgs a) {
  __shared__ float red[4][32];
  const int tile = int(blockIdx.x) % a.tiles, head = int(blockIdx.x) / a.tiles % a.H, b = int(blockIdx.x) / a.tiles / a.H;
  const int tid = threadIdx.x, c = tile * 32 + (tid & 7) * 4, r0 = tid >> 3;
  const int64_t slot = slot_of(a, b);
  uint16_t* out = a.out + (int64_t(b) * a.H + head) * a.dv;
  // a slot past the pool, or one that an earlier sequence of the call has: no state is touched
  int bad = slot >= a.slots ? 1 : 0;
  if (a.index && slot >= 0)
    for (int i = tid; i < b; i += 256) bad |= slot_of(a, i) == slot ? 1 : 0;
  if (a.index) bad = __syncthreads_or(bad);
  if (slot < 0 || bad) {
    if (tid < 32 && tile * 32 + tid < a.dv) out[tile * 32 + tid] = slot < 0 ? 0 : 0x7FC0;
    return;
  }
  const uint16_t* q = a.q.p + b * a.q.sb + int64_t(head / a.q.share) * a.q.sh;
  const uint16_t* k = a.k.p + b * a.k.sb + int64_t(head / a.k.share) * a.k.sh;
  const uint16_t* v = a.v.p + b * a.v.sb + int64_t(head / a.v.share) * a.v.sh;
  float* S = a.state + (slot * a.H + head) * int64_t(a.dk) * a.dv + c;
  const float decay = pow2(a.log_decay[head] * kLog2e);
  const int n = min(4, a.dv - c);
  float o[4] = {}, vv[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) vv[e] = e < n ? bf16_to_f32(v[c + e]) : 0.0f;
  float s[kMaxHead / 32][4];
  if (n > 0) {
#pragma unroll
    for (int i = 0; i < kMaxHead / 32; ++i) {
      const int r = r0 + 32 * i;
      if (r < a.dk) {
        if (a.vec) {
          const float4 x = *reinterpret_cast<const float4*>(S + int64_t(r) * a.dv);
          s[i][0] = x.x, s[i][1] = x.y, s[i][2] = x.z, s[i][3] = x.w;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) s[i][e] = e < n ? S[int64_t(r) * a.dv + e] : 0.0f;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kMaxHead / 32; ++i) {
      const int r = r0 + 32 * i;
      if (r < a.dk) {
        const float kk = bf16_to_f32(k[r]), qq = bf16_to_f32(q[r]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[i][e] = fmaf(decay, s[i][e], kk * vv[e]);
          o[e] = fmaf(qq, s[i][e], o[e]);
        }
        if (a.vec) {
          *reinterpret_cast<float4*>(S + int64_t(r) * a.dv) = make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (e < n) S[int64_t(r) * a.dv + e] = s[i][e];
        }
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    o[e] += __shfl_xor(o[e], 8, 64);
    o[e] += __shfl_xor(o[e], 16, 64);
    o[e] += __shfl_xor(o[e], 32, 64);
    if ((tid & 63) < 8) red[tid >> 6][(tid & 7) * 4 + e] = o[e];
  }
  __syncthreads();
  if (tid < 32 && tile * 32 + tid < a.dv)
    out[tile * 32 + tid] = f32_to_bf16(a.scale * (red[0][tid] + red[1][tid] + red[2][tid] + red[3][tid]));
}

// ---- host -----------------------------------------------------------------------------------------
int refuse(const char* what, const char* why) {
  set_error(std::string(what) + ": " + why);
  return -1;
}

constexpr int64_t kMaxTokens = int64_t(1) << 30, kMaxGrid = (int64_t(1) << 31) - 1;

const char* sizes_fault(int64_t B, int64_t T, int64_t H, int64_t G, int64_t dk, int64_t dv) {
  if (B < 0 || B > (1 << 20) || T < 0 || T > kMaxTokens || H < 1 || H > (1 << 16)) return "batch, tokens or heads out of range";
  if (G < 1 || G > H || H % G) return "the heads of k and v must divide those of q";
  if (dk < 1 || dk > kMaxHead || dv < 1 || dv > kMaxHead) return "head sizes outside 1 .. 128";
  if (B * H * ceil_div(T, int64_t(kC)) * 6 > kMaxGrid) return "too many chunks";
  return nullptr;
}

bool odd(const void* p) { return reinterpret_cast<uintptr_t>(p) & 1; }
bool off4(const void* p) { return reinterpret_cast<uintptr_t>(p) & 3; }

const char* heads_fault(const xdna_heads_bf16* h) {
  if (!h || !h->data) return "null operand";
  if (odd(h->data)) return "misaligned operand";
  if (h->batch < 0 || h->token < 0 || h->head < 0) return "negative stride";
  return nullptr;
}

Heads heads_of(const xdna_heads_bf16* h, int64_t share) { return {h->data, h->batch, h->token, h->head, int(share)}; }

// Segments of a sequence: where the sequences and heads alone leave CUs without a workgroup.
struct Plan {
  int segments, chunks;
};

Plan plan_segments(int64_t workgroups, int64_t T) {
  const int64_t chunks = ceil_div(T, int64_t(kC));
  if (workgroups >= 256 || chunks < 2) return {1, int(std::max<int64_t>(chunks, 1))};
  const int64_t per = std::max<int64_t>(1, chunks / std::max<int64_t>(1, 512 / workgroups));
  return {int(ceil_div(chunks, per)), int(per)};
}

int blocks64(int64_t d) { return int(ceil_div(d, int64_t(kVB))); }

Plan fwd_plan(int64_t B, int64_t T, int64_t H, int64_t dv) { return plan_segments(B * H * blocks64(dv), T); }
Plan bwd_plan(int64_t B, int64_t T, int64_t H, int64_t dk, int64_t dv) {
  return plan_segments(B * H * (2 * blocks64(dk) + blocks64(dv)), T);
}

size_t local_floats(const Plan& p, int64_t B, int64_t H, int64_t dk, int64_t dv) {
  return size_t(p.segments - 1) * size_t(B * H) * size_t(dk * dv);
}

template <int KT, bool STATE>
bool launch_walks(DecayArgs& a, hipStream_t st) {
  void (*f)(DecayArgs) = walk_kernel<KT, STATE>;
  static const bool ok = hipFuncSetAttribute(reinterpret_cast<const void*>(f), hipFuncAttributeMaxDynamicSharedMemorySize,
                                             int(Lds<KT>::bytes)) == hipSuccess;
  if (!ok) return false;
  int64_t n = 0;
  for (int i = 0; i < a.n; ++i) {
    a.first[i] = n;
    a.walk[i].vb = blocks64(a.walk[i].dv);
    n += int64_t(a.B) * a.H * a.walk[i].vb * (STATE ? a.segments - 1 : a.segments);
  }
  f<<<unsigned(n), kThreads, Lds<KT>::bytes, st>>>(a);
  return true;
}

// The walks of one launch each where their keys' sizes are on the same side of 64.
template <bool STATE>
bool launch(const DecayArgs& a, const Walk* walks, int n, hipStream_t st) {
  for (const bool big : {true, false}) {
    DecayArgs b = a;
    b.n = 0;
    for (int i = 0; i < n; ++i)
      if ((walks[i].dk > 64) == big) b.walk[b.n++] = walks[i];
    if (b.n && !(big ? launch_walks<128, STATE>(b, st) : launch_walks<64, STATE>(b, st))) return false;
  }
  return true;
}

const char* common_fault(const float* log_decay, const void* lengths, int index_bytes, float scale) {
  if (!log_decay) return "null operand";
  if (off4(log_decay)) return "misaligned operand";
  if (lengths && index_bytes != 4 && index_bytes != 8) return "indices must be 4 or 8 bytes";
  if (lengths && (reinterpret_cast<uintptr_t>(lengths) & (index_bytes - 1))) return "misaligned operand";
  if (!(scale > -3.0e38f && scale < 3.0e38f)) return "scale must be finite";
  return nullptr;
}

bool workspace_bad(const void* ws, size_t have, size_t need) {
  return need && (!ws || (reinterpret_cast<uintptr_t>(ws) & 15) || have < need);
}

}  // namespace
}  // namespace xdna

using namespace xdna;

extern "C" {

size_t xdna_decay_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t dk, int64_t dv) {
  if (sizes_fault(B, T, H, H, dk, dv) || B == 0 || T == 0) return 0;
  return local_floats(fwd_plan(B, T, H, dv), B, H, dk, dv) * sizeof(float);
}

int xdna_decay_attention(const xdna_heads_bf16* q, const xdna_heads_bf16* k, const xdna_heads_bf16* v, int64_t B, int64_t T,
                         int64_t H, int64_t G, int64_t dk, int64_t dv, const float* log_decay, const void* lengths,
                         int index_bytes, float scale, const float* state, uint16_t* out, float* state_out, void* workspace,
                         size_t workspace_bytes, void* stream) {
  const char* what = "xdna_decay_attention";
  if (const char* why = sizes_fault(B, T, H, G, dk, dv)) return refuse(what, why);
  if (B == 0) return 0;
  if (T == 0) return refuse(what, "no tokens");
  for (const xdna_heads_bf16* h : {q, k, v})
    if (const char* why = heads_fault(h)) return refuse(what, why);
  if (const char* why = common_fault(log_decay, lengths, index_bytes, scale)) return refuse(what, why);
  if (!out) return refuse(what, "null operand");
  if (odd(out) || off4(state) || off4(state_out)) return refuse(what, "misaligned operand");
  if (workspace_bad(workspace, workspace_bytes, xdna_decay_workspace_bytes(B, T, H, dk, dv)))
    return refuse(what, "workspace missing, misaligned or too small");
  if (!admit_launch(what)) return -1;
  DecayArgs a = {};
  a.B = int(B), a.T = int(T), a.H = int(H);
  a.log_decay = log_decay;
  a.lengths = lengths;
  a.index_bytes = index_bytes;
  const Plan p = fwd_plan(B, T, H, dv);
  a.segments = p.segments, a.chunks = p.chunks;
  Walk w = {};
  w.q = heads_of(q, 1), w.k = heads_of(k, H / G), w.v = heads_of(v, H / G);
  w.dk = int(dk), w.dv = int(dv);
  w.p_scale = w.q_scale = scale;
  w.kv_scale = 1.0f;
  w.out = out;
  w.s0 = state;
  w.s0_k = dv, w.s0_v = 1;
  w.s1 = state_out;
  w.local = static_cast<float*>(workspace);
  w.local_k = dv, w.local_v = 1;
  hipStream_t st = as_stream(stream);
  const bool ok = (p.segments == 1 || launch<true>(a, &w, 1, st)) && launch<false>(a, &w, 1, st);
  return ok ? check_launch(what) : refuse(what, "the kernel's LDS size cannot be had");
}

size_t xdna_decay_bwd_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t G, int64_t dk, int64_t dv) {
  if (sizes_fault(B, T, H, G, dk, dv) || B == 0 || T == 0) return 0;
  // both states' segments, and with shared heads the fp32 gradients of each head's k and v
  return (2 * local_floats(bwd_plan(B, T, H, dk, dv), B, H, dk, dv) + (G < H ? size_t(B * T * H) * size_t(dk + dv) : 0)) *
         sizeof(float);
}

int xdna_decay_attention_bwd(const xdna_heads_bf16* dout, const float* d_state_out, const xdna_heads_bf16* q,
                             const xdna_heads_bf16* k, const xdna_heads_bf16* v, int64_t B, int64_t T, int64_t H, int64_t G,
                             int64_t dk, int64_t dv, const float* log_decay, const void* lengths, int index_bytes, float scale,
                             const float* state, uint16_t* d_q, uint16_t* d_k, uint16_t* d_v, float* d_state, void* workspace,
                             size_t workspace_bytes, void* stream) {
  const char* what = "xdna_decay_attention_bwd";
  if (const char* why = sizes_fault(B, T, H, G, dk, dv)) return refuse(what, why);
  if (B == 0) return 0;
  if (T == 0) return refuse(what, "no tokens");
  for (const xdna_heads_bf16* h : {dout, q, k, v})
    if (const char* why = heads_fault(h)) return refuse(what, why);
  if (const char* why = common_fault(log_decay, lengths, index_bytes, scale)) return refuse(what, why);
  if (!d_q || !d_k || !d_v) return refuse(what, "null operand");
  if (odd(d_q) || odd(d_k) || odd(d_v) || off4(d_state_out) || off4(state) || off4(d_state)) return refuse(what, "misaligned operand");
  if (workspace_bad(workspace, workspace_bytes, xdna_decay_bwd_workspace_bytes(B, T, H, G, dk, dv)))
    return refuse(what, "workspace missing, misaligned or too small");
  if (!admit_launch(what)) return -1;
  DecayArgs a = {};
  a.B = int(B), a.T = int(T), a.H = int(H);
  a.log_decay = log_decay;
  a.lengths = lengths;
  a.index_bytes = index_bytes;
  const Plan p = bwd_plan(B, T, H, dk, dv);
  a.segments = p.segments, a.chunks = p.chunks;
  const int64_t group = H / G;
  const Heads hd = heads_of(dout, 1), hq = heads_of(q, 1), hk = heads_of(k, group), hv = heads_of(v, group);
  float* local_s = static_cast<float*>(workspace);
  float* local_r = local_s + local_floats(p, B, H, dk, dv);
  float* wide_k = local_r + local_floats(p, B, H, dk, dv);
  float* wide_v = wide_k + B * T * H * dk;
  Walk w[3] = {};
  // dq: S transposed
  w[0].q = hd, w[0].k = hv, w[0].v = hk;
  w[0].dk = int(dv), w[0].dv = int(dk);
  w[0].p_scale = w[0].q_scale = scale;
  w[0].kv_scale = 1.0f;
  w[0].out = d_q;
  w[0].s0 = state;
  w[0].s0_k = 1, w[0].s0_v = dv;
  w[0].local = local_s;
  w[0].local_k = 1, w[0].local_v = dv;
  // dv
  w[1].q = hk, w[1].k = hq, w[1].v = hd;
  w[1].dk = int(dk), w[1].dv = int(dv);
  w[1].reverse = 1;
  w[1].p_scale = w[1].kv_scale = scale;
  w[1].q_scale = 1.0f;
  w[1].out = group > 1 ? static_cast<void*>(wide_v) : d_v;
  w[1].wide = group > 1;
  w[1].s0 = d_state_out;
  w[1].s0_k = dv, w[1].s0_v = 1;
  w[1].s1 = d_state;
  w[1].local = local_r;
  w[1].local_k = dv, w[1].local_v = 1;
  // dk: G transposed
  w[2] = w[1];
  w[2].q = hv, w[2].k = hd, w[2].v = hq;
  w[2].dk = int(dv), w[2].dv = int(dk);
  w[2].out = group > 1 ? static_cast<void*>(wide_k) : d_k;
  w[2].s0_k = 1, w[2].s0_v = dv;
  w[2].s1 = nullptr;
  w[2].local_k = 1, w[2].local_v = dv;
  hipStream_t st = as_stream(stream);
  bool ok = true;
  if (p.segments > 1) {
    // the segments' own states: S from (k, v) and G from (q, do), each [dk][dv]
    Walk s[2] = {w[0], w[1]};
    s[0].k = hk, s[0].v = hv;
    s[0].dk = int(dk), s[0].dv = int(dv);
    ok = launch<true>(a, s, 2, st);
  }
  ok = ok && launch<false>(a, w, 3, st);
  if (!ok) return refuse(what, "the kernel's LDS size cannot be had");
  if (group > 1) {
    const auto sum = [&](const float* from, uint16_t* to, int64_t d) {
      const unsigned grid = unsigned(std::min<int64_t>(ceil_div(B * T * G * d, int64_t(256)), 16384));
      group_kernel<<<grid, 256, 0, st>>>(from, to, B * T * G, int(group), int(d));
    };
    sum(wide_k, d_k, dk);
    sum(wide_v, d_v, dv);
  }
  return check_launch(what);
}

int xdna_decay_step(const xdna_heads_bf16* q, const xdna_heads_bf16* k, const xdna_heads_bf16* v, int64_t B, int64_t H,
                    int64_t G, int64_t dk, int64_t dv, const float* log_decay, float* state, int64_t slots, const void* index,
                    int index_bytes, float scale, uint16_t* out, void* stream) {
  const char* what = "xdna_decay_step";
  if (const char* why = sizes_fault(B, 1, H, G, dk, dv)) return refuse(what, why);
  if (slots < 0 || (!index && slots < B)) return refuse(what, "fewer states than sequences");
  if (B == 0) return 0;
  for (const xdna_heads_bf16* h : {q, k, v})
    if (const char* why = heads_fault(h)) return refuse(what, why);
  if (const char* why = common_fault(log_decay, index, index_bytes, scale)) return refuse(what, why);
  if (!out || (!state && slots)) return refuse(what, "null operand");
  if (odd(out) || off4(state)) return refuse(what, "misaligned operand");
  if (!admit_launch(what)) return -1;
  StepArgs a = {};
  a.q = heads_of(q, 1), a.k = heads_of(k, H / G), a.v = heads_of(v, H / G);
  a.B = int(B), a.H = int(H), a.dk = int(dk), a.dv = int(dv);
  a.log_decay = log_decay;
  a.state = state;
  a.slots = slots;
  a.index = index;
  a.index_bytes = index_bytes;
  a.scale = scale;
  a.out = out;
  a.tiles = int(ceil_div(dv, int64_t(32)));
  a.vec = dv % 4 == 0 && (reinterpret_cast<uintptr_t>(state) & 15) == 0 ? 1 : 0;
  step_kernel<<<unsigned(B * H * a.tiles), 256, 0, as_stream(stream)>>>(a);
  return check_launch(what);
}

}  // extern "C"
