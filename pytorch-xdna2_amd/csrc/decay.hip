// Linear attention with a decay for each head, on gfx950 MFMA: the chunked form for training and
// prompts with its backward pass, and the recurrent form for single tokens.  The reference reaches
// such work only through its zero-copy CPU fallback (torch_xdna_device.cpp:5124-5260).
//
//   S_t = a S_{t-1} + k_t^T v_t,   o_t = scale q_t S_t,   a = exp(log_decay[head]),  S: Dk x Dv
//
// Chunks of C = 64 tokens: with S the state before a chunk and i, j places in it,
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
// A workgroup walks one sequence, head and 64 columns of v, the state in its registers
// in fp32.  Rounded to bf16 is the state as an operand of q S (one rounding beside the result's own:
// error against 64 bits 1.25 times that of the result's rounding in training batches, 1.4 where nearly all
// comes from the state); the weighted scores go in two bf16 parts (one put sequences of a few tokens, whose rows share
// a few roundings, up to 1.8 times as far off; the second's products cost 1.5 % of a training batch), and the weighted v of
// the state's own sum in three (24 bits), since the state is fp32 (two leave it 2.8e-6 off).
#include "common.h"
#include "mfma.h"

#include "../../include/xdna_hip.h"

namespace xdna {
namespace {

constexpr int kC = 64;        // tokens of a chunk
constexpr int kVB = 64;       // columns of v of a workgroup
constexpr int kMaxHead = 128;
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
  int s0_k, s0_v;
  float* s1;        // the state behind the last token, dense, or null
  float* local;     // segments' own states [B][H][segments - 1] x (dk, dv by these strides)
  int local_k, local_v;
};

struct DecayArgs {
  Walk walk[3];
  int blocks;  // workgroups of all walks along their dv
  int B, T, H;
  const float* log_decay;
  const void* lengths;  // null: T
  int index_bytes;
  int segments, chunks;  // of a sequence, and chunks of a segment
  int scanned;           // Walk::local holds the states before segments 1, 2, .. (else the segments' own)
};

typedef short i16x4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));

__device__ inline float pow2(float x) { return __builtin_amdgcn_exp2f(x); }

// A value that the compiler takes for a new one: comparisons with it stay where they are written (hoisted
// out of the chunks' loop, the rare paths' lane masks took every scalar register and more).
template <class T>
__device__ inline T here(T v) {
  asm volatile("" : "+v"(v));
  return v;
}

struct __attribute__((packed, aligned(4))) Floats4 {
  float v[4];
};

__device__ inline void put4(float* row, int c, int d, bool vec, const f32x4_t& v) {  // columns c .. of d; vec: in whole fours
  if (vec) {
    if (c < d) *reinterpret_cast<Floats4*>(row + c) = {{v[0], v[1], v[2], v[3]}};
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (c + e < d) row[c + e] = v[e];
}

// Tiles in LDS: rows of W elements (64 or 128), in pieces of 8.  Piece p of row r is at p ^ swizzle(r): 16 lanes of a
// row read (16 rows x 4 pieces) and 32 of a transposing read (8 rows x 2 pieces) then fall on distinct banks.  (The writes
// of the state's operand form do meet on banks, 29 % of the LDS's cycles; in whole pieces or with rows 8 apart on other
// banks they meet less, and no call gets faster by more than the 2 % that others lose.)
template <int W>
__device__ inline int swizzle(int r) {
  return W == 128 ? 2 * (r & 7) : 2 * ((r >> 1) & 3);
}
template <int W>
__device__ inline int place(int r, int p) {
  return r * W + ((p ^ swizzle<W>(r)) * 8);
}

// A lane's byte offsets of the operands of 16x16x32 MFMAs in a tile, of which every other read differs by an XOR or
// an addition with constants (addresses formed one by one, hoisted out of the chunks' loop, spilled a hundred registers).
// With l = lane % 16, g = lane / 16:
//   row: row l, elements 8 g ..; elements 32 kk on: row ^ 64 kk; rows 16 on: + 16 rows.
//   tr: column l of rows 4 g .. +3, transposed; columns 16 x on: tr ^ 32 x; rows 16 on: + 16 rows.  An operand's eight k
//     are these four rows and those 16 further on (both operands of a product have the same order).
template <int W>
struct LaneAt {
  static constexpr uint32_t k16 = 16 * 2 * W;  // bytes of 16 rows
  uint32_t row, tr;
  __device__ inline explicit LaneAt(int lane) {
    const int l = lane & 15, g = lane >> 4;
    row = uint32_t(place<W>(l, g)) * 2u;
    tr = uint32_t(place<W>(4 * g + (l >> 2), (l & 3) >> 1) + 4 * (l & 1)) * 2u;
  }
};

template <class T>
__device__ inline T lds_at(uint32_t at) {
  return *reinterpret_cast<__attribute__((address_space(3))) const T*>(at);
}

__device__ inline bf16x8_t frag_row(uint32_t at) { return as_bf16x8(lds_at<u32x4_t>(at)); }

__device__ inline u32x4_t frag_tr(uint32_t lo, uint32_t hi) {
  const u32x2_t a = __builtin_bit_cast(
      u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<__attribute__((address_space(3))) i16x4_t*>(lo)));
  const u32x2_t b = __builtin_bit_cast(
      u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<__attribute__((address_space(3))) i16x4_t*>(hi)));
  return u32x4_t{a[0], a[1], b[0], b[1]};
}

__device__ inline f32x4_t mfma(const bf16x8_t& a, const bf16x8_t& b, const f32x4_t& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ inline f32x4_t zero4() { return f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}; }

// One of the two operands that go to LDS by chunks: rows of d elements, `step` from one token of the walk to
// the next (negative backwards).
struct Stream {
  const uint16_t* first;  // the segment's first token
  int64_t step;
  int d;
  bool narrow;  // no 8 elements up to the end of d in a row
};

// Rows sh .. 63 of a chunk (tokens c0 .. of the segment) into a tile, zeros in the rows before and behind d: by
// 16-byte LDS DMA, W / 32 instructions of each of four waves.  The caller waits.
//   A whole chunk takes one instruction each and little else: the lane's offset in a block of rows is one of two (lane_at[i
// % 2], out of range behind d), the blocks' and the chunks' are scalar.
template <int W>
struct Dma {
  static constexpr int P = W / 8, ROWS = 64 / P, N = W / 32;  // pieces of a row, rows of an instruction, instructions a wave
  uint32_t lane_at[2];
  uint32_t bytes;  // from row to row
  bool down;       // backwards: the chunk's last token has the lowest address

  __device__ inline Dma(const Stream& x, int lane) : bytes(uint32_t(x.step < 0 ? -x.step : x.step) * 2u), down(x.step < 0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = i * ROWS + lane / P, p = (lane % P) ^ swizzle<W>(r);
      lane_at[i] = p * 8 < x.d ? uint32_t(down ? ROWS - 1 - lane / P : lane / P) * bytes + uint32_t(p) * 16u : 0x7FFFFFF0u;
    }
  }

  __device__ inline i32x4_t rows(const Stream& x, int c0, int sh) const {
    return uniform_rsrc(lds_dma_rsrc(x.first + (c0 + (down ? kC - 1 - sh : 0)) * x.step, 0x7FFFFFE0));
  }

  __device__ inline void load_whole(const Stream& x, int c0, const uint16_t* tile, int wave) const {
    const i32x4_t rs = rows(x, c0, 0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int block = wave * N + i;
      const uint32_t at = uint32_t(down ? kC - (block + 1) * ROWS : block * ROWS) * bytes;
      lds_dma16_m0(rs, lds_addr(tile) + uint32_t(block) * 1024u, int(lane_at[i % 2]), at);
    }
  }

  __device__ inline void load_some(const Stream& x, int c0, int sh, const uint16_t* tile, int lane, int wave) const {
    const i32x4_t rs = rows(x, c0, sh);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = (wave * N + i) * ROWS + lane / P, p = (lane % P) ^ swizzle<W>(r);
      const uint32_t at = uint32_t(down ? kC - 1 - r : r - sh) * bytes + uint32_t(p) * 16u;
      lds_dma16_m0(rs, lds_addr(tile) + uint32_t(wave * N + i) * 1024u, r >= sh && p * 8 < x.d ? int(at) : 0x7FFFFFF0);
    }
  }
};

// 8 elements of a row of d (at least 8) from column c on: a row's last ones in a window that ends with it, so that every
// load is whole and hangs on no branch; `to_place` then puts them where they belong, zeros behind them.
__device__ inline Pix8 window8(const uint16_t* row, int c, int d) { return *reinterpret_cast<const Pix8*>(row + min(c, d - 8)); }
__device__ inline Pix8 to_place(const Pix8& v, int c, int d) { return c < d ? shifted(v, max(c + 8 - d, 0)) : Pix8{{0u, 0u, 0u, 0u}}; }

// The same as Dma for rows of any length, stride and alignment, through registers: loaded before a chunk's work, written to
// LDS behind it (one behind the other, the loads' way was in every chunk: heads of 127 took 271 us for 135).
template <int W>
struct Staged {
  static constexpr int P = W / 8, N = W / 32;
  Pix8 v[N];

  __device__ inline void load(const Stream& x, int c0, int sh, int t) {
    if (x.narrow) return;
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = window8(x.first + (c0 + max(t / P + i * (256 / P) - sh, 0)) * x.step, t % P * 8, x.d);
  }
  __device__ inline void store(const Stream& x, int c0, int sh, uint16_t* tile, int t) const {
    if (x.narrow) {  // (rows of under 8: element by element, here)
#pragma unroll 1
      for (int r = t / P; r < kC; r += 256 / P) put(tile, r, t % P, row_vec(x.first + (c0 + max(r - sh, 0)) * x.step, r >= sh && t % P == 0 ? x.d : 0));
      return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = t / P + i * (256 / P);
      put(tile, r, t % P, r >= sh ? to_place(v[i], t % P * 8, x.d) : Pix8{{0u, 0u, 0u, 0u}});
    }
  }
  __device__ static inline void put(uint16_t* tile, int r, int p, const Pix8& q) {
    *reinterpret_cast<uint4*>(tile + place<W>(r, p)) = make_uint4(q.v[0], q.v[1], q.v[2], q.v[3]);
  }
};

// This workgroup's place in an order whose neighbours are on one XCD (workgroups go to the 8 XCDs in turn).
__device__ inline int xcd_block() {
  const int n = int(gridDim.x), xcd = int(blockIdx.x) % 8;
  return xcd * (n / 8) + min(xcd, n % 8) + int(blockIdx.x) / 8;
}

__device__ inline int64_t length_of(const DecayArgs& a, int b) {
  if (!a.lengths) return a.T;
  const int64_t n = a.index_bytes == 8 ? static_cast<const int64_t*>(a.lengths)[b] : static_cast<const int32_t*>(a.lengths)[b];
  return n < 0 ? 0 : n < a.T ? n : a.T;
}

template <int KT>
struct Lds {  // two buffers each; of a segment's state by itself three, and none for the state's operand form
  static constexpr int k = kC * KT, v = kC * kVB, s = kVB * KT;
  static constexpr size_t bytes = size_t(2) * (k + v + s) * 2, state_bytes = size_t(3) * (k + v) * 2;
};

// STATE: the state of a segment by itself, from zero, and no outputs.
//
// Four waves have the outputs, 16 tokens of a chunk each, as [dv][token] so that a lane has one token.  Four more have
// the state, 16 columns of v each: while the outputs of a chunk are made they make the state behind it.  (All by four
// waves in turn, a chunk took 3.7 us with one workgroup a CU: a third of it the waits of one wave a SIMD, the rest
// scores, weights and the state's products one after the other.)  K and V of the next chunk are loaded while one is
// worked on, and the state before a chunk is in LDS twice, so that a chunk has one barrier.  A chunk of n < 64 tokens
// takes the tile's last n rows, its first ones are zeros: the weights inside a chunk, which go by differences and by the
// distance to its end, are those of every other.
//   A chunk takes 2.1 us with one workgroup a CU and 3.2 with two: MFMA a quarter to a third of it and VALU a third to two
// fifths, LDS reads about as much, a wave's products, scores and weights one after the other.  8 x 2048 tokens, 16 heads of
// 128: forward 73 us (256 workgroups, one a CU; 268 MB, 3.7 TB/s), backward 166 (three walks, 805 MB of rows, 480 MB read
// from memory and 197 written: 4.1 TB/s); 1 x 8192 tokens: the segments' states 20, their sums 7, the outputs 33.
//   DMA: rows of k and v are whole 16-byte pieces.
template <int KT, bool STATE, bool DMA>
__global__ __launch_bounds__(STATE ? 256 : 512, 4) void walk_kernel(DecayArgs a) {
  using L = Lds<KT>;
  constexpr int THREADS = STATE ? 256 : 512;
  constexpr int NS = KT / 16;  // a wave's 16 x 16 tiles of the state
  constexpr int KK = KT / 32;  // k-steps along a head
  extern __shared__ __attribute__((aligned(16))) uint16_t smem[];
  constexpr int BUFS = STATE ? 3 : 2;
  uint16_t* const ks = smem;              // [buffer][token][dk]
  uint16_t* const vs = ks + BUFS * L::k;  // [buffer][token][dv]
  static_assert(L::s == L::k, "a row's place in K and in the state's tile ([buffer][dv][dk]) differ by a constant");
  constexpr uint32_t kBuf = 2 * L::k, vBuf = 2 * L::v, kS = 2 * (2 * L::k + 2 * L::v);  // bytes

  // workgroups of one sequence and head, all walks', next to each other on one XCD: they read the same rows, and each XCD
  // has its own L2 (walk after walk, the backward of 8 x 2048 tokens, 16 heads of 128 took 177 us for 169, of 16 x 2048
  // with heads of 64 165 for 150)
  int id = xcd_block();
  int vb = id % a.blocks, wi = 0;
  id /= a.blocks;
  while (vb >= a.walk[wi].vb) vb -= a.walk[wi++].vb;
  const Walk& w = a.walk[wi];
  const int n_seg = STATE ? a.segments - 1 : a.segments;
  const int seg = id % n_seg, head = id / n_seg % a.H, batch = id / n_seg / a.H;
  const int64_t bh = int64_t(batch) * a.H + head;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int len = int(length_of(a, batch));
  const int seg_len = a.chunks * kC, begin = seg * seg_len;
  const int todo = max(0, min(len - begin, seg_len));  // tokens of this segment
  const int lead = w.reverse ? 0 : 1;
  float g2 = a.log_decay[head] * kLog2e;
  g2 = g2 < -1e4f ? -1e4f : g2;  // (exp(-inf) as exp(-1e4): 0, and 0 times it is 0)
  const int d0 = vb * kVB, dk = w.dk, dv = min(w.dv - d0, kVB);  // columns of k, and of v here

  // place i of the segment is token t0 + i or, backwards, t0 - i
  const int64_t t0 = w.reverse ? len - 1 - begin : begin;
  const auto step = [&](int64_t st) { return w.reverse ? -st : st; };
  const Stream kx = {w.k.p + batch * w.k.sb + int64_t(head / w.k.share) * w.k.sh + t0 * w.k.st, step(w.k.st), dk, dk < 8};
  const Stream vx = {w.v.p + batch * w.v.sb + int64_t(head / w.v.share) * w.v.sh + t0 * w.v.st + d0, step(w.v.st), dv, w.dv < 8};

  // ---- tokens behind the sequence: zeros
  if constexpr (!STATE) {
    const int from = max(begin, len), to = min(begin + seg_len, a.T);
    for (int64_t i = tid; i < int64_t(to - from) * kVB; i += THREADS) {
      const int64_t t = from + i / kVB;
      const int c = int(i % kVB);
      if (c < dv) {
        const int64_t at = ((int64_t(batch) * a.T + t) * a.H + head) * w.dv + d0 + c;
        if (w.wide) static_cast<float*>(w.out)[at] = 0.0f;
        else static_cast<uint16_t*>(w.out)[at] = 0;
      }
    }
  }
  const bool last = !STATE && w.s1 && seg == max(0, (len + seg_len - 1) / seg_len - 1);
  if (todo == 0 && !last && !STATE) return;

  const auto uniform = [](float v) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v))); };
  const uint32_t smem_at = lds_addr(smem);
  if (STATE || wave >= 4) {
    // ---- the state: register i of tile x of this wave is dk 16 x + 4 g + i, dv 16 vt + l16.  These waves load K and V too
    // (the others have the longer way through a chunk, and eight waves' loads at its start took a sixth of it).
    const int vt = STATE ? wave : wave - 4;
    const Dma<KT> k_dma(kx, lane);
    const Dma<kVB> v_dma(vx, lane);
    Staged<KT> k_staged;
    Staged<kVB> v_staged;
    const auto load = [&](int c0, int b) {  // chunk c0 .. into buffer b, or the registers that go there
      const int sh = max(0, kC - (todo - c0));
      if (DMA && sh == 0) {
        k_dma.load_whole(kx, c0, ks + b * L::k, vt);
        v_dma.load_whole(vx, c0, vs + b * L::v, vt);
      } else if constexpr (DMA) {
        const int l = here(lane);
        k_dma.load_some(kx, c0, sh, ks + b * L::k, l, vt);
        v_dma.load_some(vx, c0, sh, vs + b * L::v, l, vt);
      } else {
        const int t = here(64 * vt + lane);
        k_staged.load(kx, c0, sh, t);
        v_staged.load(vx, c0, sh, t);
      }
    };
    const auto write = [&](int c0, int b) {
      if constexpr (!DMA) {
        const int sh = max(0, kC - (todo - c0)), t = here(64 * vt + lane);
        k_staged.store(kx, c0, sh, ks + b * L::k, t);
        v_staged.store(vx, c0, sh, vs + b * L::v, t);
      }
    };
    if (todo > 0) load(0, 0), write(0, 0);
    if (STATE && todo > kC) load(kC, 1), write(kC, 1);
    f32x4_t S[NS];
#pragma unroll
    for (int x = 0; x < NS; ++x) S[x] = zero4();
    const int dv_of = 16 * vt + l16;
    const LaneAt<KT> k_at(lane);
    const LaneAt<kVB> v_at(lane);
    const uint32_t s_to = smem_at + kS + uint32_t(place<KT>(dv_of, g >> 1)) * 2u + uint32_t(g & 1) * 8u;
    const auto store_state = [&](int b) {
      const uint32_t to = here(s_to + uint32_t(b) * kBuf);
#pragma unroll
      for (int x = 0; x < NS; ++x)
        *reinterpret_cast<__attribute__((address_space(3))) u32x2_t*>(to ^ uint32_t(32 * x)) =
            u32x2_t{pack2(S[x][0], S[x][1]), pack2(S[x][2], S[x][3])};
    };
    if constexpr (!STATE) {
      const auto add = [&](const float* s, int sk, int sv) {  // (a state's places fit 32 bits: one base for all loads)
        const int rows = here(dk);
        const uint32_t column = uint32_t((d0 + min(dv_of, dv - 1)) * sv);
        f32x4_t v[NS];
#pragma unroll
        for (int x = 0; x < NS; ++x)
#pragma unroll
          for (int i = 0; i < 4; ++i) v[x][i] = s[column + uint32_t(min(16 * x + 4 * g + i, rows - 1) * sk)];
#pragma unroll
        for (int x = 0; x < NS; ++x)
#pragma unroll
          for (int i = 0; i < 4; ++i) S[x][i] += 16 * x + 4 * g + i < rows && dv_of < dv ? v[x][i] : 0.0f;
      };
      const int64_t per = int64_t(w.dk) * w.dv;
      if (w.s0 && !(seg > 0 && a.scanned)) add(w.s0 + bh * per, w.s0_k, w.s0_v);
      // the segments before this one: summed up by scan_kernel, or few
      if (seg > 0 && a.scanned) add(w.local + (bh * (a.segments - 1) + seg - 1) * per, w.local_k, w.local_v);
      for (int j = 0; j < seg && !a.scanned; ++j) {
        const float f = pow2(g2 * float(max(0, min(len - j * seg_len, seg_len))));
#pragma unroll
        for (int x = 0; x < NS; ++x) S[x] *= f;
        add(w.local + (bh * (a.segments - 1) + j) * per, w.local_k, w.local_v);
      }
      if (todo > 0) store_state(0);
    }
    // weights of v for the lane's tokens 32 s + 16 y + 4 g + e of a chunk (no exponent is negative)
    float weight[2][8];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) weight[s][e] = w.kv_scale * pow2(g2 * float(kC - lead - 32 * s - 16 * (e >> 2) - 4 * g - (e & 3)));
    int b = 0;
    for (int c0 = 0; c0 < todo; c0 += kC, b = STATE ? (b == 2 ? 0 : b + 1) : b ^ 1) {
      // this wave's loads and LDS writes of the chunk have landed; the barrier publishes everyone's, and everyone has left
      // the buffers that the next loads take.  A segment's state by itself has the loads of two chunks under way (one
      // ahead, it took 2.6 us a chunk, twice its work).
      lds_reads_wait();  // (its LDS writes; stated here, since the compiler leaves the barrier's own wait out beside the next line's)
      if constexpr (DMA) {
        if (STATE && c0 + kC < todo) lds_dma_wait<Dma<KT>::N + Dma<kVB>::N>();
        else lds_dma_wait<0>();
      }
      __syncthreads();
      const int coming = c0 + (STATE ? 2 : 1) * kC, to = STATE ? (b == 0 ? 2 : b - 1) : b ^ 1;
      // (at once: among the state's products they came later, and the forward of 8 x 2048 tokens, 16 heads of 128, took 76 us
      // for 69, the backward 169 for 165)
      if (coming < todo) load(coming, to);
      const uint32_t k_tr = here(k_at.tr + smem_at + uint32_t(b) * kBuf);
      const uint32_t v_tr = (v_at.tr ^ uint32_t(32 * vt)) + smem_at + BUFS * kBuf + uint32_t(b) * vBuf;
      constexpr uint32_t k16 = LaneAt<KT>::k16, v16 = LaneAt<kVB>::k16;
      const float f = pow2(g2 * float(min(todo - c0, kC)));
#pragma unroll
      for (int x = 0; x < NS; ++x) S[x] *= f;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const u32x4_t vu = frag_tr(v_tr + 2 * s * v16, v_tr + (2 * s + 1) * v16);
        u32x4_t part[3];  // v weighted, in three bf16
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x0 = __uint_as_float(vu[e] << 16) * weight[s][2 * e];
          float x1 = __uint_as_float(vu[e] & 0xFFFF0000u) * weight[s][2 * e + 1];
#pragma unroll
          for (int y = 0; y < 3; ++y) {
            part[y][e] = pack2(x0, x1);
            x0 -= __uint_as_float(part[y][e] << 16);
            x1 -= __uint_as_float(part[y][e] & 0xFFFF0000u);
          }
        }
#pragma unroll
        for (int x0 = 0; x0 < NS; x0 += 4) {
          bf16x8_t k[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const uint32_t at = k_tr ^ uint32_t(32 * (x0 + x));
            k[x] = as_bf16x8(frag_tr(at + 2 * s * k16, at + (2 * s + 1) * k16));
          }
#pragma unroll
          for (int y = 2; y >= 0; --y)
#pragma unroll
            for (int x = 0; x < 4; ++x) S[x0 + x] = mfma(k[x], as_bf16x8(part[y]), S[x0 + x]);
        }
      }
      if (coming < todo) write(coming, to);
      if (!STATE && c0 + kC < todo) store_state(b ^ 1);
    }
    if (STATE || last) {
      const int64_t per = int64_t(w.dk) * w.dv;
      float* to = STATE ? w.local + (bh * n_seg + seg) * per : w.s1 + bh * per;
      const int rows = here(dk);
      if (dv_of < dv) {
#pragma unroll
        for (int x = 0; x < NS; ++x)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (16 * x + 4 * g + i < rows) to[uint32_t((16 * x + 4 * g + i) * w.dv + d0 + dv_of)] = S[x][i];
      }
    }
  } else if constexpr (!STATE) {
    // ---- the outputs of tokens 16 wave .. of a chunk
    const uint16_t* const qp = w.q.p + batch * w.q.sb + int64_t(head / w.q.share) * w.q.sh + t0 * w.q.st;
    const int64_t q_step = step(w.q.st), o_step = step(int64_t(a.H) * w.dv);
    const int64_t o_at = (int64_t(batch) * a.T + t0) * a.H * w.dv + int64_t(head) * w.dv + d0;
    const int row = 16 * wave + l16;
    // q: the lane's token, k 32 kk + 8 g .. (those of no token are not stored; columns past the head meet zeros of k and of
    // the state)
    Pix8 qf[KK];
    const auto load_q = [&](int c0) {
      const int sh = max(0, kC - (todo - c0));
      const uint16_t* from = qp + (c0 + max(row - sh, 0)) * q_step;
      const int d = here(dk);
      if (DMA && dk == KT) {
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) qf[kk] = *reinterpret_cast<const Pix8*>(from + 32 * kk + 8 * g);
      } else if (DMA || d >= 8) {
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) qf[kk] = window8(from, 32 * kk + 8 * g, d);
      } else {
        qf[0] = row_vec(from, d);
      }
    };
    const auto place_q = [&] {  // (with DMA a row is whole pieces: they are in place, and those past it meet zeros)
      if constexpr (!DMA) {
        const int d = here(dk);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
          const int c = 32 * kk + 8 * g;
          qf[kk] = d >= 8 ? to_place(qf[kk], c, d) : c == 0 ? qf[0] : Pix8{{0u, 0u, 0u, 0u}};
        }
      }
    };
    const auto frag = [](const Pix8& v) { return as_bf16x8(u32x4_t{v.v[0], v.v[1], v.v[2], v.v[3]}); };
    if (todo > 0) load_q(0);
    // weights of this lane's token against the 4 keys of its score registers: of its own 16 tokens, and of the 16
    // before them (d tiles before: times a^(16 (d - 1)); no exponent is negative)
    float diag[4], off[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int apart = l16 - 4 * g - i;
      diag[i] = apart >= 0 ? w.p_scale * pow2(g2 * float(apart)) : 0.0f;
      off[i] = w.p_scale * pow2(g2 * float(16 + apart));
    }
    const float a16 = uniform(pow2(g2 * 16.0f)), a32 = uniform(pow2(g2 * 32.0f));
    const LaneAt<KT> k_at(lane);
    const LaneAt<kVB> v_at(lane);
    constexpr uint32_t k16 = LaneAt<KT>::k16, v16 = LaneAt<kVB>::k16;
    int b = 0;
    for (int c0 = 0; c0 < todo; c0 += kC, b ^= 1) {
      lds_reads_wait();
      __syncthreads();
      const int sh = max(0, kC - (todo - c0));
      f32x4_t o[4];  // [dv][token], four tiles of 16 columns
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = zero4();
      if (16 * wave + 16 > sh) {
        place_q();
        const uint32_t k_row = here(k_at.row + smem_at + uint32_t(b) * kBuf), s_row = k_row + kS;
        const uint32_t v_tr = here(v_at.tr + smem_at + 2 * kBuf + uint32_t(b) * vBuf);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[j] = mfma(frag_row((s_row ^ uint32_t(64 * kk)) + j * k16), frag(qf[kk]), o[j]);
        const float row_weight = w.q_scale * pow2(g2 * float(max(row - sh, 0) + lead));
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] *= row_weight;
        for (int s = 0; 2 * s <= wave; ++s) {  // keys 32 s .. +31
          const bool two = 2 * s < wave;       // (their second 16 are not all behind)
          f32x4_t p[2] = {zero4(), zero4()};   // [key][token]
          const uint32_t k_s = k_row + uint32_t(s) * (2 * k16);
#pragma unroll
          for (int kk = 0; kk < KK; ++kk) p[0] = mfma(frag_row(k_s ^ uint32_t(64 * kk)), frag(qf[kk]), p[0]);
          if (two) {
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) p[1] = mfma(frag_row((k_s ^ uint32_t(64 * kk)) + k16), frag(qf[kk]), p[1]);
          }
          uint32_t pw[2][4] = {};  // the weighted scores and what their rounding to bf16 left
          const auto scores = [&](int y, int apart) {  // `apart` tiles before the wave's own
            const float f = apart == 3 ? a32 : apart == 2 ? a16 : 1.0f;
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = p[y][i] * (apart == 0 ? diag[i] : off[i] * f);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t hi = pack2(x[2 * i], x[2 * i + 1]);
              pw[0][2 * y + i] = hi;
              pw[1][2 * y + i] = pack2(x[2 * i] - __uint_as_float(hi << 16), x[2 * i + 1] - __uint_as_float(hi & 0xFFFF0000u));
            }
          };
          scores(0, wave - 2 * s);
          if (two) scores(1, wave - 2 * s - 1);
          if (2 * s + 2 > wave && c0 + kC < todo) load_q(c0 + kC);  // (after q's last use: the next chunk's into its registers)
          const uint32_t v_s = v_tr + uint32_t(s) * (2 * v16);
          bf16x8_t vf[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) vf[j] = as_bf16x8(frag_tr(v_s ^ uint32_t(32 * j), (v_s ^ uint32_t(32 * j)) + v16));
#pragma unroll
          for (int y = 1; y >= 0; --y) {
            const bf16x8_t pf = as_bf16x8(u32x4_t{pw[y][0], pw[y][1], pw[y][2], pw[y][3]});
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = mfma(vf[j], pf, o[j]);
          }
        }
      }
      if (row >= sh) {
        const int64_t at = o_at + (c0 + row - sh) * o_step;
        const int d = here(dv);
        if (w.wide) {
#pragma unroll
          for (int j = 0; j < 4; ++j) put4(static_cast<float*>(w.out) + at, 16 * j + 4 * g, d, w.dv % 4 == 0, o[j]);
        } else {
          // a lane's quads of columns 4 g .. of two tiles to columns 8 g .. of 32: a 64-byte run of a token's row a store
          uint16_t* to = static_cast<uint16_t*>(w.out) + at;
#pragma unroll
          for (int j = 0; j < 4; j += 2) {
            uint32_t q[2][2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const auto m = __builtin_amdgcn_permlane32_swap(pack2(o[j][2 * x], o[j][2 * x + 1]),
                                                              pack2(o[j + 1][2 * x], o[j + 1][2 * x + 1]), false, false);
              const auto n = __builtin_amdgcn_permlane16_swap(m[0], m[1], false, false);
              q[0][x] = n[0], q[1][x] = n[1];
            }
            put_vec(to + 16 * j + 8 * g, {{q[0][0], q[0][1], q[1][0], q[1][1]}}, d - 16 * j - 8 * g);
          }
        }
      }
    }
  }
}

// The segments' own states to the states before segments 1, 2, ..: in place, a thread an element, the segments' loads
// eight ahead.  s0: the state before the first (dense [B][H][dk][dv], or null).  Latency-bound (four elements a thread
// took 6.2 us for 4.5 at 18 heads of 64 x 64 and 12 segments, 7.2 for 6.4 at 16 of 128 x 128 and 7).
struct ScanArgs {
  float* local;
  const float* s0;
  int per, count;  // elements of a state, segments - 1
};

__global__ __launch_bounds__(256) void scan_kernel(ScanArgs x, ScanArgs y, DecayArgs a) {
  const ScanArgs& s = blockIdx.z ? y : x;
  const int i = int(blockIdx.x) * 256 + int(threadIdx.x), bh = blockIdx.y;
  if (i >= s.per) return;
  float* p = s.local + int64_t(bh) * s.count * s.per + i;
  constexpr int A = 8;
  float v[A];
  const auto load = [&](int j0) {
#pragma unroll
    for (int u = 0; u < A; ++u) v[u] = p[int64_t(min(j0 + u, s.count - 1)) * s.per];
  };
  load(0);  // (before the length and the decay are known)
  const int len = int(length_of(a, bh / a.H)), seg_len = a.chunks * kC;
  float g2 = a.log_decay[bh % a.H] * kLog2e;
  g2 = g2 < -1e4f ? -1e4f : g2;
  float S = s.s0 ? s.s0[int64_t(bh) * s.per + i] : 0.0f;
  for (int j0 = 0; j0 < s.count; j0 += A) {
    if (j0 > 0) load(j0);
#pragma unroll
    for (int u = 0; u < A; ++u) {
      const int j = j0 + u;
      if (j >= s.count) break;
      S = S * pow2(g2 * float(max(0, min(len - j * seg_len, seg_len)))) + v[u];
      p[int64_t(j) * s.per] = S;
    }
  }
}

// Gradients of shared heads: out[.., g, d] = the sum over the group's heads in order, rounded once.  2^lanes threads a row
// of an output head, four columns each.  Bound by the fp32 gradients' bytes: 53 us for 537 MB of them (8 x 2048 tokens, 16
// heads of 128 by fours; a column a thread 92).
struct GroupArgs {
  const float* from[2];  // of k and v
  uint16_t* to[2];
  int d[2], lanes[2];
  int64_t rows;
  int group;
};

__global__ __launch_bounds__(256) void group_kernel(GroupArgs a) {
  const int which = blockIdx.y, d = a.d[which], lanes = a.lanes[which];
  const int c = (threadIdx.x & ((1 << lanes) - 1)) * 4, n = d - c, per = 256 >> lanes;
  if (n <= 0) return;
  for (int64_t r = int64_t(blockIdx.x) * per + (threadIdx.x >> lanes); r < a.rows; r += int64_t(gridDim.x) * per) {
    const float* p = a.from[which] + r * a.group * d + c;
    float s[4] = {};
    for (int j0 = 0; j0 < a.group; j0 += 4) {
      float v[4][4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float* q = p + int64_t(min(j0 + u, a.group - 1)) * d;
        if (n >= 4) {
          const Floats4 f = *reinterpret_cast<const Floats4*>(q);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[u][e] = f.v[e];
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[u][e] = e < n ? q[e] : 0.0f;
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (j0 + u < a.group) {
#pragma unroll
          for (int e = 0; e < 4; ++e) s[e] += v[u][e];
        }
    }
    put_vec(a.to[which] + r * d + c, {{pack2(s[0], s[1]), pack2(s[2], s[3]), 0u, 0u}}, min(n, 4));
  }
}

// ---- single tokens --------------------------------------------------------------------------------
// S = a S + k^T v in place, o = scale q S.  Bound by the state's bytes, read and written once: a
// workgroup takes a head and 32 columns of v, a thread four columns of every 32nd row.  64 x 16 heads of 128: 26 us, 5.1
// TB/s.  Where tiles share lines of memory, those of a head are on one XCD, whose L2 puts the lines together (heads of 127
// 49 -> 34 us, of 100 32 -> 21; heads of 128 are 1 us faster spread out).
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
  int lines;      // and a tile's rows whole lines of memory
};

__device__ inline int64_t slot_of(const StepArgs& a, int b) {
  if (!a.index) return b;
  return a.index_bytes == 8 ? static_cast<const int64_t*>(a.index)[b] : static_cast<const int32_t*>(a.index)[b];
}

__global__ __launch_bounds__(256) void step_kernel(StepArgs a) {
  __shared__ float red[4][32];
  const int id = a.lines ? int(blockIdx.x) : xcd_block(), tile = id % a.tiles, head = id / a.tiles % a.H, b = id / a.tiles / a.H;
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
        } else if (n == 4) {
          const Floats4 x = *reinterpret_cast<const Floats4*>(S + int64_t(r) * a.dv);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[i][e] = x.v[e];
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
        } else if (n == 4) {
          *reinterpret_cast<Floats4*>(S + int64_t(r) * a.dv) = {{s[i][0], s[i][1], s[i][2], s[i][3]}};
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

constexpr int64_t kMaxTokens = int64_t(1) << 30;
constexpr int64_t kMaxWalks = (int64_t(1) << 23) - 1;  // workgroups of a launch (512 threads: under 2^32 of them)
constexpr int64_t kSplitWalks = 256;                   // most workgroups whose sequences are cut into segments

const char* sizes_fault(int64_t B, int64_t T, int64_t H, int64_t G, int64_t dk, int64_t dv) {
  if (B < 0 || B > (1 << 20) || T < 0 || T > kMaxTokens || H < 1 || H > (1 << 16)) return "batch, tokens or heads out of range";
  if (G < 1 || G > H || H % G) return "the heads of k and v must divide those of q";
  if (dk < 1 || dk > kMaxHead || dv < 1 || dv > kMaxHead) return "head sizes outside 1 .. 128";
  if (B * H * 6 > kMaxWalks) return "too many sequences and heads";  // (three walks of two blocks of columns)
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

constexpr int kScanFrom = 5;  // segments from which on their states are summed up by a launch

// Segments of a sequence, where its call has no workgroup for every CU, by what it takes in us.  Fitted to 21 shapes (1 to
// 8 sequences of 300 to 32768 tokens, 2 to 32 heads of 32, 64 or 128, both directions, whole and in 2 to 64 segments; 8 % off
// in the mean, the choice under 2 % slower than the best in the mean and 15 % at most): a chunk takes 1.4 with few
// workgroups, 1.7 with one on each CU, and with two 2.8 forward and 3.2 backward (three walks' rows from memory); of the
// segments' own states 0.43 a workgroup on a CU, at least 1.1; heads up to 64 three quarters of that; the states' sums 0.94 a
// MB.  1 x 8192 tokens, 16 heads of 128, forward: 193 us whole, 60 in 8 segments, 56 in 16, 97 in 64; 4 x 5000, 4 heads of
// 64: 99, 32, 24 and 32; backward of 1 x 8192 199 whole, 113 in 8, 129 in 16.
struct Plan {
  int segments, chunks;
};

// `chunk`: a chunk's time against that of heads of 128, `two`: that with two workgroups on each CU
float walk_cost(int64_t workgroups, int64_t chunks, float chunk, float two) {
  const auto round = [&](float n) { return n <= 256.0f ? 1.4f + 0.3f * n / 256.0f : 1.7f + (two - 1.7f) * (n - 256.0f) / 256.0f; };
  const int64_t rest = workgroups % 512;
  return 5.4f + float(chunks) * chunk * (two * float(workgroups / 512) + (rest ? round(float(rest)) : 0.0f));
}

// `walks`, `states`: workgroups of a segment's walks and of its states; `state_mb`: bytes of all heads' states
Plan plan_segments(int64_t walks, int64_t states, float state_mb, int64_t T, bool big, float two) {
  const int64_t chunks = ceil_div(T, int64_t(kC));
  const float size = big ? 1.0f : 0.75f;
  Plan best = {1, int(std::max<int64_t>(chunks, 1))};
  // (every CU has one: backward of 6 x 2048 tokens, 16 heads of 128, 130 us whole, 149 in 2 segments, 182 in 4; of 3 x
  // 4096, 157, 169 and 170)
  if (walks > kSplitWalks) return best;
  float least = 0.95f * walk_cost(walks, chunks, size, two);  // (cut for a gain beyond the fit's errors)
  for (int64_t n = 2; n <= std::min<int64_t>(chunks, 256); n += n < 64 ? 1 : 32) {
    const int64_t per = ceil_div(chunks, n), segments = ceil_div(chunks, per);
    const float own = 3.4f + float(per) * size * std::max(1.1f, 0.43f * float(states * (segments - 1)) / 256.0f);
    const float join = segments >= kScanFrom ? 2.9f + (0.94f * state_mb + 0.08f) * float(segments - 1) : 1.25f * float(segments - 1);
    const float cost = walk_cost(walks * segments, per, size, two) + own + join;
    if (cost < least) least = cost, best = {int(segments), int(per)};
  }
  return best;
}

int blocks64(int64_t d) { return int(ceil_div(d, int64_t(kVB))); }

Plan fwd_plan(int64_t B, int64_t T, int64_t H, int64_t dk, int64_t dv) {
  const int64_t n = B * H * blocks64(dv);
  return plan_segments(n, n, float(B * H * dk * dv) * 4e-6f, T, dk > 64, 2.8f);
}
Plan bwd_plan(int64_t B, int64_t T, int64_t H, int64_t dk, int64_t dv) {
  return plan_segments(B * H * (2 * blocks64(dk) + blocks64(dv)), 2 * B * H * blocks64(dv), float(B * H * dk * dv) * 8e-6f, T,
                       dk > 64 || dv > 64, 3.2f);
}

size_t local_floats(const Plan& p, int64_t B, int64_t H, int64_t dk, int64_t dv) {
  return size_t(p.segments - 1) * size_t(B * H) * size_t(dk * dv);
}

// 16-byte aligned rows, and offsets inside a chunk that 31 bits hold
bool dma_rows(const Heads& h) {
  return (reinterpret_cast<uintptr_t>(h.p) & 15) == 0 && h.sb % 8 == 0 && h.st % 8 == 0 && h.sh % 8 == 0 && h.st < (int64_t(1) << 23);
}

template <int KT, bool STATE, bool DMA>
bool launch_walks(const DecayArgs& a, hipStream_t st) {
  constexpr size_t bytes = STATE ? Lds<KT>::state_bytes : Lds<KT>::bytes;
  void (*f)(DecayArgs) = walk_kernel<KT, STATE, DMA>;
  static const bool ok = hipFuncSetAttribute(reinterpret_cast<const void*>(f), hipFuncAttributeMaxDynamicSharedMemorySize,
                                             int(bytes)) == hipSuccess;
  if (!ok) return false;
  const int64_t n = int64_t(a.B) * a.H * a.blocks * (STATE ? a.segments - 1 : a.segments);
  f<<<unsigned(n), STATE ? 256 : 512, bytes, st>>>(a);
  return true;
}

// All walks in one launch, on tiles for the largest of their keys' heads (walks of sizes on both sides of 64 in a launch
// each took 26 us where one takes 16: 3 x 777 tokens, 6 heads of 48 and 80).
template <bool STATE>
bool launch(DecayArgs a, const Walk* walks, int n, hipStream_t st) {
  bool big = false, dma = true;
  a.blocks = 0;
  for (int i = 0; i < n; ++i) {
    Walk& w = a.walk[i] = walks[i];
    w.vb = blocks64(w.dv);
    a.blocks += w.vb;
    big |= w.dk > 64;
    dma = dma && w.dk % 8 == 0 && w.dv % 8 == 0 && dma_rows(w.k) && dma_rows(w.v);
  }
  if (dma) return big ? launch_walks<128, STATE, true>(a, st) : launch_walks<64, STATE, true>(a, st);
  return big ? launch_walks<128, STATE, false>(a, st) : launch_walks<64, STATE, false>(a, st);
}

// the segments' own states, and where they are many the states before them
template <int N>
bool launch_segments(DecayArgs& a, const Walk (&walks)[N], const float* const (&s0)[N], hipStream_t st) {
  if (a.segments == 1) return true;
  if (!launch<true>(a, walks, N, st)) return false;
  a.scanned = a.segments >= kScanFrom ? 1 : 0;
  if (!a.scanned) return true;
  const int per = walks[0].dk * walks[0].dv;
  ScanArgs s[2] = {};
  for (int i = 0; i < N; ++i) s[i] = {walks[i].local, s0[i], per, a.segments - 1};
  scan_kernel<<<dim3(unsigned(ceil_div(per, 256)), unsigned(a.B * a.H), N), 256, 0, st>>>(s[0], s[1], a);
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
  return local_floats(fwd_plan(B, T, H, dk, dv), B, H, dk, dv) * sizeof(float);
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
  const Plan p = fwd_plan(B, T, H, dk, dv);
  a.segments = p.segments, a.chunks = p.chunks;
  Walk w = {};
  w.q = heads_of(q, 1), w.k = heads_of(k, H / G), w.v = heads_of(v, H / G);
  w.dk = int(dk), w.dv = int(dv);
  w.p_scale = w.q_scale = scale;
  w.kv_scale = 1.0f;
  w.out = out;
  w.s0 = state;
  w.s0_k = int(dv), w.s0_v = 1;
  w.s1 = state_out;
  w.local = static_cast<float*>(workspace);
  w.local_k = int(dv), w.local_v = 1;
  hipStream_t st = as_stream(stream);
  const bool ok = launch_segments<1>(a, {w}, {state}, st) && launch<false>(a, &w, 1, st);
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
  w[0].s0_k = 1, w[0].s0_v = int(dv);
  w[0].local = local_s;
  w[0].local_k = 1, w[0].local_v = int(dv);
  // dv
  w[1].q = hk, w[1].k = hq, w[1].v = hd;
  w[1].dk = int(dk), w[1].dv = int(dv);
  w[1].reverse = 1;
  w[1].p_scale = w[1].kv_scale = scale;
  w[1].q_scale = 1.0f;
  w[1].out = group > 1 ? static_cast<void*>(wide_v) : d_v;
  w[1].wide = group > 1;
  w[1].s0 = d_state_out;
  w[1].s0_k = int(dv), w[1].s0_v = 1;
  w[1].s1 = d_state;
  w[1].local = local_r;
  w[1].local_k = int(dv), w[1].local_v = 1;
  // dk: G transposed
  w[2] = w[1];
  w[2].q = hv, w[2].k = hd, w[2].v = hq;
  w[2].dk = int(dv), w[2].dv = int(dk);
  w[2].out = group > 1 ? static_cast<void*>(wide_k) : d_k;
  w[2].s0_k = 1, w[2].s0_v = int(dv);
  w[2].s1 = nullptr;
  w[2].local_k = 1, w[2].local_v = int(dv);
  hipStream_t st = as_stream(stream);
  // the segments' own states: S from (k, v) and G from (q, do), each [dk][dv]
  Walk s[2] = {w[0], w[1]};
  s[0].k = hk, s[0].v = hv;
  s[0].dk = int(dk), s[0].dv = int(dv);
  if (!launch_segments<2>(a, s, {state, d_state_out}, st) || !launch<false>(a, w, 3, st)) return refuse(what, "the kernel's LDS size cannot be had");
  if (group > 1) {
    GroupArgs g = {{wide_k, wide_v}, {d_k, d_v}, {int(dk), int(dv)}, {}, B * T * G, int(group)};
    for (int i = 0; i < 2; ++i)
      while (4 << g.lanes[i] < g.d[i]) ++g.lanes[i];
    const int64_t rows = 256 >> std::max(g.lanes[0], g.lanes[1]);
    group_kernel<<<dim3(unsigned(std::min<int64_t>(ceil_div(g.rows, rows), 16384)), 2), 256, 0, st>>>(g);
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
  a.lines = dv % 32 == 0 && (reinterpret_cast<uintptr_t>(state) & 127) == 0 ? 1 : 0;
  step_kernel<<<unsigned(B * H * a.tiles), 256, 0, as_stream(stream)>>>(a);
  return check_launch(what);
}

}  // extern "C"
