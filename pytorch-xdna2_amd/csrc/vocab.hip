// Rows over a vocabulary on gfx950: log probabilities of given tokens with entropy and top
// alternatives, distillation from a teacher's top logits, and the gradients of both.  The
// reference reaches such rows only through its zero-copy CPU fallback
// (torch_xdna_device.cpp:5124-5260).
//
// Mathematics, per row of logits z with temperature tau, x = z / tau:
//   m = max z, s = sum exp((z - m) / tau), q = exp((z - m) / tau) / s;
//   log probability of token y: (z_y - m) / tau - ln s;
//   entropy: ln s - u / (tau s), u = sum exp((z - m) / tau) (z - m);
//   pieces of a row join by m = max m_i, w_i = exp((m_i - m) / tau), s = sum w_i s_i,
//   u = sum w_i (u_i + (m_i - m) s_i).
// The gradients take m and 1 / s from the forward: both hold q to a few fp32 roundings,
// where m / tau + ln s in one number would lose its last bits to the size of m.
// A row of -inf only has s = 0: log probabilities -inf, entropy 0, gradient 0; an element of
// -inf adds nothing anywhere (its e (z - m) would be 0 * inf).  NaN and +inf make the row's
// results NaN.
//
// Layout: a workgroup streams a row (or, where there are few rows, a piece of one: a second
// launch joins the pieces in order), each thread with a running maximum and sums of its own
// that are rescaled once per 4 loaded windows; the workgroup joins its threads once at the end.
// Every sum has a fixed order, so equal inputs give equal bits.  The largest entries need no
// second read of the row either: the threads' own maxima bound the top-th largest element, and
// only the threads whose maximum reaches the bound look at their elements again.  The gradient
// kernels stream: read z, write dz.
#include "common.h"

#include "../../include/xdna_hip.h"

namespace xdna {
namespace {

constexpr int kWin = 4;               // 16-byte windows of a thread per step
constexpr int kMaxTop = 64;           // alternatives: one group maximum per lane bounds them
constexpr int kMaxPieces = 64;        // pieces of a row: their lists fit the join's LDS
constexpr int kMaxTeacher = 1024;     // teacher entries per row (held in LDS by the gradient)
constexpr int64_t kMaxVocab = int64_t(1) << 22;
constexpr int kCandidates = 1024;     // LDS list of elements that may be among the largest
constexpr int kScan = 8;              // windows that the selection reads at once
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.402823466e38f;  // z - m of a term of weight 0: 0 times it is 0, where 0 * -inf is NaN

// VW elements of a 16-byte window (any element-aligned address: global accesses of gfx950
// take one), as fp32
template <typename T>
struct Win;
template <>
struct Win<float> {
  static constexpr int VW = 4;
};
template <>
struct Win<uint16_t> {
  static constexpr int VW = 8;
};

struct Raw {
  uint32_t w[4];
};

template <typename T>
__device__ inline float raw_get(const Raw& r, int e) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(r.w[e]);
  return __uint_as_float((e & 1) ? (r.w[e >> 1] & 0xFFFF0000u) : (r.w[e >> 1] << 16));
}

template <typename T>
__device__ inline void raw_set(Raw& r, int e, float v) {
  if constexpr (sizeof(T) == 4) {
    r.w[e] = __float_as_uint(v);
  } else {
    const uint32_t h = f32_to_bf16(v);
    if (e & 1) r.w[e >> 1] = (r.w[e >> 1] & 0xFFFFu) | (h << 16);
    else r.w[e >> 1] = (r.w[e >> 1] & 0xFFFF0000u) | h;
  }
}

template <typename T>
__device__ inline float load_one(const T* p) {
  if constexpr (sizeof(T) == 4) return *p;
  else return bf16_to_f32(*p);
}

template <typename T>
__device__ inline void store_one(T* p, float v) {
  if constexpr (sizeof(T) == 4) *p = v;
  else *p = f32_to_bf16(v);
}

// The window of p: whole, or its first n elements and -inf after them.
template <typename T>
__device__ inline Raw load_win(const T* p, int n) {
  Raw r;
  if (n >= Win<T>::VW) {
    const Pix8 q = *reinterpret_cast<const Pix8*>(p);
#pragma unroll
    for (int k = 0; k < 4; ++k) r.w[k] = q.v[k];
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) r.w[k] = sizeof(T) == 4 ? 0xFF800000u : 0xFF80FF80u;
#pragma unroll
    for (int e = 0; e < Win<T>::VW; ++e)
      if (e < n) raw_set<T>(r, e, load_one<T>(p + e));
  }
  return r;
}

template <typename T>
__device__ inline void store_win(T* p, const Raw& r, int n) {
  if (n >= Win<T>::VW) {
    Pix8 q;
#pragma unroll
    for (int k = 0; k < 4; ++k) q.v[k] = r.w[k];
    *reinterpret_cast<Pix8*>(p) = q;
  } else {
#pragma unroll
    for (int e = 0; e < Win<T>::VW; ++e)
      if (e < n) store_one<T>(p + e, raw_get<T>(r, e));
  }
}

// 1 where p starts inside a word: windows of whole words start one element before it or after it.
template <typename T>
__device__ inline int word_skip(const T* p) {
  return sizeof(T) == 2 ? int(reinterpret_cast<uintptr_t>(p) >> 1) & 1 : 0;
}

__device__ inline float exp2_hw(float v) { return __builtin_amdgcn_exp2f(v); }

// ---- order of the alternatives: value descending, index ascending ------------------------
// An unsigned key that grows with the value (-0 as +0, NaN above all, as sorting puts it)
// over the inverted index: unique per element, and never 0.
__device__ inline uint32_t order_key(float v) {
  v = v != v ? __uint_as_float(0x7FC00000u) : v + 0.0f;
  const uint32_t b = __float_as_uint(v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ inline float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }
__device__ inline uint64_t entry_of(uint32_t key, int idx) { return (uint64_t(key) << 32) | uint32_t(~idx); }
__device__ inline int entry_index(uint64_t e) { return int(~uint32_t(e)); }

__device__ inline uint64_t lane64(uint64_t v, int lane) {
  return (uint64_t(uint32_t(__builtin_amdgcn_readlane(int(v >> 32), lane))) << 32) |
         uint32_t(__builtin_amdgcn_readlane(int(uint32_t(v)), lane));
}

__device__ inline float wave_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}

__device__ inline float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

struct RowStat {
  float m, s, u;
};

struct LogprobOut {
  const void* targets;  // [rows] token indices, negative: not scored
  int index_bytes;
  float* log_probs;
  float* entropy;
  float2* stats;  // [rows] m and 1 / s (0 for a row of -inf)
  float* top_log_probs;  // [rows][top]
  int64_t* top_ids;
  int top;
};

struct DistillOut {
  const void* ids;  // [rows][k] token indices, negative: absent
  int index_bytes;
  const void* teacher;  // [rows][k] logits, -inf: absent
  int teacher_dtype;
  const float* weight;  // [rows] or null: all 1
  int k;
  float tau;
  float2* stats;  // [rows] m and 1 / s
  float* p;       // [rows][k]
  float* loss;    // [rows] the row's weighted loss
  float* share;   // [rows] the row's weight, 0 where it has no valid entry or one past the vocabulary
};

struct RowArgs {
  const void* z;
  int64_t ld;
  int64_t rows;
  int V;
  int piece, pieces;  // elements per piece (a multiple of 8), pieces per row
  float inv_tau;
  RowStat* stat;   // [rows][pieces] where pieces > 1
  uint64_t* list;  // [rows][pieces][top] where pieces > 1
  LogprobOut lp;
  DistillOut ds;
};

enum RowMode { kLogprob = 0, kDistill = 1 };

__device__ inline int64_t index_at(const void* p, int bytes, int64_t i) {
  return bytes == 8 ? static_cast<const int64_t*>(p)[i] : int64_t(static_cast<const int32_t*>(p)[i]);
}

// ln q of a logit: (z - m) / tau - ln s, -inf throughout a row of -inf (log_s = ln 0)
__device__ inline float log_q(const RowStat& st, float log_s, float z, float inv_tau) {
  return st.s == 0.0f ? -INFINITY : (z - st.m) * inv_tau - log_s;
}

__device__ inline float2 kept_stats(const RowStat& st) {
  return st.s == 0.0f ? make_float2(0.0f, 0.0f) : make_float2(st.m, 1.0f / st.s);
}

__device__ inline float teacher_at(const DistillOut& d, int64_t i) {
  return d.teacher_dtype == 1 ? static_cast<const float*>(d.teacher)[i]
                              : bf16_to_f32(static_cast<const uint16_t*>(d.teacher)[i]);
}

// What the end of a row needs from memory, loaded before the row's logits are (a chain of two
// or three loads there would wait a memory latency each).  One entry per thread: the target, or
// the lane's first teacher entry.
struct Early {
  int64_t id = -1;
  float z = 0.0f, t = 0.0f, weight = 1.0f;
};

template <typename T, int MODE>
__device__ inline Early early_loads(const RowArgs& a, int64_t row) {
  Early r;
  if (MODE == kLogprob) {
    if (threadIdx.x == 0) r.id = index_at(a.lp.targets, a.lp.index_bytes, row);
  } else if (threadIdx.x < 64) {
    if (int(threadIdx.x) < a.ds.k) {
      r.id = index_at(a.ds.ids, a.ds.index_bytes, row * a.ds.k + threadIdx.x);
      r.t = teacher_at(a.ds, row * a.ds.k + threadIdx.x);
    }
    if (a.ds.weight) r.weight = a.ds.weight[row];
  }
  if (r.id >= 0 && r.id < a.V) r.z = load_one<T>(static_cast<const T*>(a.z) + row * a.ld + r.id);
  return r;
}

// A row's log probability, entropy and kept statistics (one thread).
__device__ inline void logprob_row(const RowArgs& a, int64_t row, const RowStat& st, const Early& early) {
  const float log_s = logf(st.s);
  a.lp.stats[row] = kept_stats(st);
  a.lp.entropy[row] = st.s == 0.0f ? 0.0f : log_s - st.u * a.inv_tau / st.s;
  a.lp.log_probs[row] = early.id >= a.V ? NAN : early.id >= 0 ? log_q(st, log_s, early.z, a.inv_tau) : 0.0f;
}

__device__ inline void top_store(const RowArgs& a, int64_t row, int rank, uint64_t e, const RowStat& st, float log_s) {
  a.lp.top_log_probs[row * a.lp.top + rank] = log_q(st, log_s, key_value(uint32_t(e >> 32)), a.inv_tau);
  a.lp.top_ids[row * a.lp.top + rank] = entry_index(e);
}

// A row's distillation loss from its statistics (one wave): its first 64 entries are in `early`.  A
// sum over the entries: two of one token are two terms (joining them would change the loss by a
// constant and take a search per entry).
template <typename T>
__device__ inline void distill_row(const RowArgs& a, int64_t row, const RowStat& st, const Early& early) {
  const DistillOut& d = a.ds;
  const int lane = threadIdx.x & 63;
  const float log_s = logf(st.s);
  const int64_t at = row * d.k;
  bool bad = false;  // an entry that is present names no token of the vocabulary
  const auto entry = [&](int j) {
    Early r = early;
    if (j >= 64) {
      r.id = index_at(d.ids, d.index_bytes, at + j);
      r.t = teacher_at(d, at + j);
    }
    bad |= r.id >= a.V && r.t != -INFINITY;
    if (r.id < 0 || r.id >= a.V) r.t = -INFINITY;  // absent
    return r;
  };
  float tm = -INFINITY;
  for (int j = lane; j < d.k; j += 64) tm = fmaxf(tm, entry(j).t);
  tm = wave_max(tm);
  const float c = a.inv_tau * kLog2e;
  float ts = 0.0f;
  bool some = false;
  for (int j = lane; j < d.k; j += 64) {
    const float t = entry(j).t;
    if (t != -INFINITY) ts += exp2_hw((t - tm) * c), some = true;
  }
  ts = wave_sum(ts);
  const float inv = 1.0f / ts, log_ts = logf(ts);
  float sum = 0.0f;
  for (int j = lane; j < d.k; j += 64) {
    const Early r = entry(j);
    float p = 0.0f;
    if (r.t != -INFINITY) {
      p = exp2_hw((r.t - tm) * c) * inv;
      const float z = j < 64 ? r.z : load_one<T>(static_cast<const T*>(a.z) + row * a.ld + r.id);
      // p ln(p / q) is 0 where p underflows, also against q = 0
      if (p != 0.0f) sum += p * (((r.t - tm) * a.inv_tau - log_ts) - log_q(st, log_s, z, a.inv_tau));
    }
    d.p[at + j] = p;
  }
  sum = wave_sum(sum);
  const bool any_bad = __any(bad), any_some = __any(some);
  if (lane == 0) {
    const float w = any_some && !any_bad ? early.weight : 0.0f;  // 0: out of the gradient too
    d.stats[row] = kept_stats(st);
    d.share[row] = w;
    d.loss[row] = early.weight == 0.0f ? 0.0f : any_bad ? NAN : w == 0.0f ? 0.0f : w * (d.tau * (d.tau * sum));  // (tau^2 alone may leave fp32)
  }
}

// ---- selection of the largest entries ----------------------------------------------------------

template <int NT>
struct TopShared {
  uint64_t best[NT > 64 ? NT : 1];  // the threads' largest, by group
  uint64_t cand[kCandidates + kMaxTop];
  uint64_t bound;
  int count, ties, total[NT / 64];
};

// The top-th largest of 64 groups' largest entries (a group: threads of one lane, skewed by
// wave), 0 where fewer groups hold one: at least `top` entries reach it, and in rows without
// special order hardly more.  For nearly as many entries as groups the threads themselves are the
// groups: the least of 64 maxima lets 4 to 5 times as many entries through as are asked for (64 of
// 1 x 131072 took 37 us before their join, so 13; 40 of them 18 either way).
template <int NT>
__device__ inline uint64_t group_bound(uint64_t best, int top, TopShared<NT>& sh) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if constexpr (NT > 64) {
    if (top > 48) {
      sh.best[tid] = best;
      if (tid == 0) sh.bound = 0, sh.count = 0;
      __syncthreads();
      int rank = 0;
#pragma unroll 8
      for (int t = 0; t < NT; ++t) rank += sh.best[t] > best ? 1 : 0;
      if (rank == top - 1 && best != 0) sh.bound = best;  // (entries are unique: one thread at most)
      __syncthreads();
      return sh.bound;
    }
  }
  if constexpr (NT > 64) {
    sh.best[wave * 64 + ((lane + 17 * wave) & 63)] = best;
    __syncthreads();
  }
  if (wave == 0) {
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) best = sh.best[w * 64 + lane] > best ? sh.best[w * 64 + lane] : best;
    int rank = 0;
#pragma unroll 16
    for (int l = 0; l < 64; ++l) rank += lane64(best, l) > best ? 1 : 0;
    const uint64_t hit = __ballot(rank == top - 1 && best != 0);
    const uint64_t bound = hit ? lane64(best, __builtin_amdgcn_readfirstlane(__ffsll(static_cast<unsigned long long>(hit)) - 1)) : 0;
    if (lane == 0) sh.bound = bound, sh.count = 0;
  }
  __syncthreads();
  return sh.bound;
}

// Ranks the n candidates (entries are unique: their order of arrival does not matter) and
// hands the first `top` to put(rank, entry); `fill`: entry 0 for ranks past them.
template <int NT, typename Put>
__device__ inline void rank_candidates(const TopShared<NT>& sh, int n, int top, bool fill, Put put) {
  for (int c = threadIdx.x; c < n; c += NT) {
    const uint64_t en = sh.cand[c];
    int rank = 0;
#pragma unroll 4
    for (int o = 0; o < n; ++o) rank += sh.cand[o] > en ? 1 : 0;
    if (rank < top) put(rank, en);
  }
  if (fill)
    for (int c = n + int(threadIdx.x); c < top; c += NT) put(c, uint64_t(0));
}

template <int NT>
__device__ inline int block_count(int n, TopShared<NT>& sh) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
  if constexpr (NT > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.total[threadIdx.x >> 6] = n;
    __syncthreads();
    n = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) n += sh.total[w];
  }
  return n;
}

// The `top` largest of the piece z[skip, len) (element 0 has index lo in its row), through
// put(rank, entry).  m: the thread's maximum over its windows tid, tid + NT, ...
//   Usual rows: the elements of value at least the bound go to an LDS list, found by the threads
// whose maximum reaches it.
//   Rows where that list overflows, or where the bound is -inf (fewer allowed tokens than asked
// for): the elements above the bound only, and as many equal ones as are still wanted in index
// order, by a scan that ends when it has them.
//   Rows where even those overflow (the largest elements sit in few groups) or that hold NaN:
// the exact top-th largest key by bisection, then the same.
template <typename T, int NT, typename Put>
__device__ inline void select_top(const T* z, int skip, int lo, int len, int top, bool fill, float m, bool nan,
                                  TopShared<NT>& sh, Put put) {
  constexpr int VW = Win<T>::VW;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const bool mine = tid * VW < len;
  uint32_t bound = uint32_t(group_bound<NT>(mine ? uint64_t(order_key(m)) << 32 | uint32_t(~tid) : 0, top, sh) >> 32);
  const uint32_t lowest = order_key(-INFINITY);
  if (bound == 0) bound = lowest;
  const auto scan = [&](uint32_t from, bool all) {  // entries of key >= from to the list
    const float fb = key_value(from);
    const auto take = [&](const Raw& r, int at) {
      float wm = raw_get<T>(r, 0);
#pragma unroll
      for (int e = 1; e < VW; ++e) wm = fmaxf(wm, raw_get<T>(r, e));
      if (!all && !(wm >= fb)) return;
#pragma unroll
      for (int e = 0; e < VW; ++e) {
        const uint32_t key = order_key(raw_get<T>(r, e));
        if (at + e >= skip && at + e < len && key >= from) {
          const int c = atomicAdd(&sh.count, 1);
          if (c < kCandidates) sh.cand[c] = entry_of(key, lo + at + e);
        }
      }
    };
    if (all || m >= fb) {
      // the few threads that are here wait for a round of kScan windows at once (4096 x 50001: 140
      // us with two, 122 with eight)
      const int whole = len / VW;
      for (int w = tid; w < whole; w += kScan * NT) {
        Raw r[kScan];
#pragma unroll
        for (int i = 0; i < kScan; ++i) {
          const Pix8 q = *reinterpret_cast<const Pix8*>(z + min(w + i * NT, whole - 1) * VW);
#pragma unroll
          for (int k = 0; k < 4; ++k) r[i].w[k] = q.v[k];
        }
#pragma unroll
        for (int i = 0; i < kScan; ++i)
          if (w + i * NT < whole) take(r[i], (w + i * NT) * VW);
      }
      if (whole * VW < len && whole % NT == tid) take(load_win<T>(z + whole * VW, len - whole * VW), whole * VW);
    }
    __syncthreads();
    return sh.count;
  };
  if (!nan && bound > lowest) {
    const int n = scan(bound, false);
    if (n <= kCandidates) {
      rank_candidates<NT>(sh, n, top, fill, put);
      return;
    }
  }
  int n = kCandidates + 1;
  if (!nan) {
    __syncthreads();
    if (tid == 0) sh.count = 0;
    __syncthreads();
    n = scan(bound + 1, false);
  }
  if (n > kCandidates) {
    bound = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t trial = bound | (1u << bit);
      int c = 0;
      for (int at = tid * VW; at < len; at += NT * VW) {
        const Raw r = load_win<T>(z + at, len - at);
#pragma unroll
        for (int e = 0; e < VW; ++e) c += at + e >= skip && at + e < len && order_key(raw_get<T>(r, e)) >= trial ? 1 : 0;
      }
      if (block_count<NT>(c, sh) >= top) bound = trial;
    }
    __syncthreads();
    if (tid == 0) sh.count = 0;
    __syncthreads();
    n = scan(bound + 1, true);  // fewer than top
  }
  // elements equal to the bound, in index order
  int want = top - n;
  for (int base = 0; base < len && want > 0; base += NT * VW) {
    const int at = base + tid * VW;
    int hits = 0;
    if (at < len) {
      const Raw r = load_win<T>(z + at, len - at);
#pragma unroll
      for (int e = 0; e < VW; ++e) hits |= (at + e >= skip && at + e < len && order_key(raw_get<T>(r, e)) == bound ? 1 : 0) << e;
    }
    int before = __popc(hits);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int t = __shfl_up(before, o, 64);
      if (lane >= o) before += t;
    }
    int all = __shfl(before, 63, 64);
    before -= __popc(hits);
    if constexpr (NT > 64) {
      __syncthreads();
      if (lane == 0) sh.total[wave] = all;
      __syncthreads();
      all = 0;
#pragma unroll
      for (int w = 0; w < NT / 64; ++w) {
        before += w < wave ? sh.total[w] : 0;
        all += sh.total[w];
      }
    }
    for (; hits && before < want; hits &= hits - 1, ++before)
      sh.cand[n + before] = entry_of(bound, lo + at + __ffs(hits) - 1);
    n += min(want, all);
    want -= min(want, all);
  }
  __syncthreads();
  rank_candidates<NT>(sh, n, top, fill, put);
}

// ---- forward ----------------------------------------------------------------------------------

template <typename T>
struct Steps {  // kWin windows of a thread
  Raw r[kWin];
};

// One thread's running statistics over another kWin windows: the new maximum first, then the
// old sums rescaled to it (by 0 while there were none) and the windows' terms.
template <typename T, bool ENT>
__device__ inline void accumulate(const Steps<T>& w, float c, float& m, float& s, float& u) {
  constexpr int VW = Win<T>::VW;
  float top = m;
#pragma unroll
  for (int i = 0; i < kWin; ++i)
#pragma unroll
    for (int e = 0; e < VW; ++e) top = fmaxf(top, raw_get<T>(w.r[i], e));
  const float m0 = top == -INFINITY ? 0.0f : top;
  if (top > m) {
    const float d = m == -INFINITY ? -INFINITY : m - m0;
    const float k = exp2_hw(d * c);
    s *= k;
    if (ENT) u = fmaf(fmaxf(d, kLowest), s, k * u);
    m = top;
  }
#pragma unroll
  for (int i = 0; i < kWin; ++i)
#pragma unroll
    for (int e = 0; e < VW; ++e) {
      const float d = raw_get<T>(w.r[i], e) - m0;
      const float x = exp2_hw(d * c);
      s += x;
      if (ENT) u = fmaf(x, fmaxf(d, kLowest), u);
    }
}

// (m, s, u) of several threads or pieces, joined at the overall maximum M
template <bool ENT>
__device__ inline void rescale(float M, float c, float m, float& s, float& u) {
  const float d = m == M ? 0.0f : m - M;
  const float k = s == 0.0f ? 0.0f : exp2_hw(d * c);  // s == 0: nothing but -inf (or nothing at all)
  if (ENT) u = s == 0.0f ? 0.0f : fmaf(fmaxf(d, kLowest), s * k, k * u);
  s *= k;
}

// A row (or a piece of one): statistics, and for log probabilities its largest entries.  Bound by
// the bytes of z where the rows are long: 4096 x 131072 in bf16 229 us (4.7 TB/s) for distillation;
// 1024 x 32768 in fp32 41 us (3.3 TB/s: four workgroups a CU, whose starts and joins show); 4096 x
// 50001 with 5 alternatives 100 to 109 us (4 TB/s), 79 without (5.2 TB/s): five waves a SIMD, so
// that others stream while one workgroup selects (with four a tenth more).  Few
// rows are bound by latency: 4 x 131072 with 20 alternatives, in 128 pieces, 9.6 us and the join 6.3.
template <typename T, int NT, int MODE, bool TOP>
__global__ __launch_bounds__(NT, 5) void row_kernel(RowArgs a) {
  constexpr int VW = Win<T>::VW, kStep = NT * VW * kWin;
  constexpr bool ENT = MODE == kLogprob;
  __shared__ float red[3][NT / 64];
  __shared__ TopShared<TOP ? NT : 64> sh;
  const int tid = threadIdx.x;
  const int64_t items = a.rows * a.pieces;
  const float c = a.inv_tau * kLog2e;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t row = a.pieces == 1 ? item : item / a.pieces;
    int lo = a.pieces == 1 ? 0 : int(item - row * a.pieces) * a.piece;
    int len = min(a.piece, a.V - lo);
    const T* z = static_cast<const T*>(a.z) + row * a.ld + lo;
    // windows start at whole words: where z does not, one element earlier, which is left out (its
    // word holds z's first element too).  4096 x 50001 takes 79 us so, with 5 alternatives 109; 91 and 123 with
    // windows across the words.
    const int skip = word_skip(z);
    z -= skip, lo -= skip, len += skip;
    const auto leave_out = [&](Steps<T>& w) {
      if (sizeof(T) == 2 && skip && tid == 0) w.r[0].w[0] = (w.r[0].w[0] & 0xFFFF0000u) | 0xFF80u;  // -inf
    };
    Early early;
    if (a.pieces == 1) early = early_loads<T, MODE>(a, row);
    float m = -INFINITY, s = 0.0f, u = 0.0f;
    const int whole = len / kStep * kStep;  // elements in whole steps of the workgroup
    const auto load = [&](int at) {
      Steps<T> w;
#pragma unroll
      for (int i = 0; i < kWin; ++i) {
        const Pix8 q = *reinterpret_cast<const Pix8*>(z + at + (tid + i * NT) * VW);
#pragma unroll
        for (int k = 0; k < 4; ++k) w.r[i].w[k] = q.v[k];
      }
      return w;
    };
    if (whole > 0) {
      Steps<T> next = load(0);
      for (int at = kStep; at < whole; at += kStep) {
        Steps<T> w = next;
        next = load(at);
        if (at == kStep) leave_out(w);
        accumulate<T, ENT>(w, c, m, s, u);
      }
      if (whole == kStep) leave_out(next);
      accumulate<T, ENT>(next, c, m, s, u);
    }
    if (whole < len) {
      Steps<T> w;
#pragma unroll
      for (int i = 0; i < kWin; ++i) {
        const int at = whole + (tid + i * NT) * VW;
        w.r[i] = load_win<T>(z + min(at, len), len - at);
      }
      if (whole == 0) leave_out(w);
      accumulate<T, ENT>(w, c, m, s, u);
    }
    float M = wave_max(m);
    if constexpr (NT > 64) {
      __syncthreads();
      if ((tid & 63) == 0) red[0][tid >> 6] = M;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < NT / 64; ++w) M = fmaxf(M, red[0][w]);
    }
    rescale<ENT>(M, c, m, s, u);
    s = wave_sum(s);
    if (ENT) u = wave_sum(u);
    if constexpr (NT > 64) {
      if ((tid & 63) == 0) red[1][tid >> 6] = s, red[2][tid >> 6] = u;
      __syncthreads();
      s = red[1][0], u = red[2][0];
#pragma unroll
      for (int w = 1; w < NT / 64; ++w) s += red[1][w], u += red[2][w];
    }
    const RowStat st = {M, s, u};
    if (a.pieces > 1) {
      if (tid == 0) a.stat[item] = st;
      if constexpr (TOP) {
        uint64_t* list = a.list + item * a.lp.top;
        select_top<T, NT>(z, skip, lo, len, a.lp.top, true, m, s != s, sh, [&](int rank, uint64_t e) { list[rank] = e; });
      }
    } else if constexpr (MODE == kLogprob) {
      if (tid == 0) logprob_row(a, row, st, early);
      if constexpr (TOP) {
        const float log_s = logf(st.s);
        select_top<T, NT>(z, skip, lo, len, a.lp.top, false, m, s != s, sh,
                          [&](int rank, uint64_t e) { top_store(a, row, rank, e, st, log_s); });
      }
    } else {
      if (tid < 64) distill_row<T>(a, row, st, early);
    }
    if (TOP) __syncthreads();  // the next item reuses the LDS lists
  }
}

// Joins the pieces of a row, in piece order: one workgroup per row.
constexpr int kJoinThreads = 256;

template <typename T, int MODE, bool TOP>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(RowArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint64_t lists[];
  __shared__ TopShared<TOP ? kJoinThreads : 64> sh;
  constexpr bool ENT = MODE == kLogprob;
  const int tid = threadIdx.x, lane = tid & 63;
  const float c = a.inv_tau * kLog2e;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    if (MODE == kDistill && tid >= 64) continue;
    const Early early = early_loads<T, MODE>(a, row);
    const int n = a.pieces * a.lp.top;
    uint64_t best = 0;
    if constexpr (TOP) {
      // by rank and then piece, so that the largest (the lists are in order) are spread over the
      // threads: one thread's bound lets few others through
      for (int i = tid; i < n; i += kJoinThreads) {
        const int rank = i / a.pieces, piece = i - rank * a.pieces;
        const uint64_t e = a.list[row * n + piece * a.lp.top + rank];
        lists[i] = e;
        best = e > best ? e : best;
      }
    }
    RowStat q = {-INFINITY, 0.0f, 0.0f};  // (a row has at most 64 pieces)
    if (lane < a.pieces) q = a.stat[row * a.pieces + lane];
    const float m = wave_max(q.m);
    rescale<ENT>(m, c, q.m, q.s, q.u);
    const RowStat st = {m, wave_sum(q.s), wave_sum(q.u)};
    if constexpr (MODE == kDistill) {
      distill_row<T>(a, row, st, early);
    } else {
      if (tid == 0) logprob_row(a, row, st, early);
      if constexpr (TOP) {
        const float log_s = logf(st.s);
        uint64_t bound = group_bound<kJoinThreads>(best, a.lp.top, sh);
        bound = bound ? bound : 1;
        const auto collect = [&] {
          for (int i = tid; i < n; i += kJoinThreads)
            if (lists[i] >= bound) {
              const int at = atomicAdd(&sh.count, 1);
              if (at < kCandidates) sh.cand[at] = lists[i];
            }
          __syncthreads();
          return sh.count;
        };
        int count = collect();
        if (count > kCandidates) {  // the exact top-th largest entry, by bisection
          bound = 0;
          for (int bit = 63; bit >= 0; --bit) {
            const uint64_t trial = bound | (uint64_t(1) << bit);
            int k = 0;
            for (int i = tid; i < n; i += kJoinThreads) k += lists[i] >= trial ? 1 : 0;
            if (block_count<kJoinThreads>(k, sh) >= a.lp.top) bound = trial;
          }
          __syncthreads();
          if (tid == 0) sh.count = 0;
          __syncthreads();
          count = collect();
        }
        rank_candidates<kJoinThreads>(sh, count, a.lp.top, false,
                                      [&](int rank, uint64_t e) { top_store(a, row, rank, e, st, log_s); });
        __syncthreads();
      }
    }
  }
}

// ---- gradients: one pass, read z, write dz ---------------------------------------------------

struct LogprobBwdArgs {
  const void* z;
  int64_t ld;
  void* dz;  // [rows][V]
  int64_t rows;
  int V, piece, pieces;
  float inv_tau;
  const void* targets;
  int index_bytes;
  const float2* stats;
  const float* entropy;
  const float* d_log_probs;  // [rows] or null
  const float* d_entropy;    // [rows] or null
};

constexpr int kBwdThreads = 256;

// dz_v = (g (1[v = y] - q_v) - h q_v (ln q_v + H)) / tau, g and h the row's incoming
// gradients.  Rows without either are written as zeros and not read.  Bound by its bytes: 1024 x
// 32768 in fp32, 268 MB, take 43 us (6.2 TB/s).
template <typename T>
__global__ __launch_bounds__(kBwdThreads) void logprob_bwd_kernel(LogprobBwdArgs a) {
  constexpr int VW = Win<T>::VW;
  const int64_t items = a.rows * a.pieces;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t row = a.pieces == 1 ? item : item / a.pieces;
    const int lo = a.pieces == 1 ? 0 : int(item - row * a.pieces) * a.piece;
    const int len = min(a.piece, a.V - lo);
    const T* z = static_cast<const T*>(a.z) + row * a.ld + lo;
    T* dz = static_cast<T*>(a.dz) + row * a.V + lo;
    const float2 ms = a.stats[row];
    const int64_t y64 = index_at(a.targets, a.index_bytes, row);
    const bool scored = y64 >= 0 && y64 < a.V;
    const int y = scored ? int(y64) - lo : -1;
    float g = a.d_log_probs && scored ? a.d_log_probs[row] * a.inv_tau : 0.0f;
    const float h = a.d_entropy ? a.d_entropy[row] * a.inv_tau : 0.0f;
    const bool none = (g == 0.0f && h == 0.0f) || ms.y == 0.0f;
    const float c = a.inv_tau * kLog2e;
    const float H = a.entropy[row] + logf(ms.y);
    const auto window = [&](int at, int n) {
      Raw o = {{0u, 0u, 0u, 0u}};
      if (!none) {
        const Raw r = load_win<T>(z + at, n);
#pragma unroll
        for (int e = 0; e < VW; ++e) {
          const float d = raw_get<T>(r, e) - ms.x;
          const float q = exp2_hw(d * c) * ms.y;
          // selected by q: ln q is -inf at a masked token, or h times it is (q NaN stays NaN)
          float v = q == 0.0f ? 0.0f : -q * (g + h * (d * a.inv_tau + H));
          if (at + e == y) v += g;
          raw_set<T>(o, e, v);
        }
      }
      store_win<T>(dz + at, o, n);
    };
    // (4096 x 50001 in bf16: 162 us; 170 with stores across the words, 195 with the last
    // window's elements one by one too)
    const int skip = word_skip(dz);
    if (len >= VW) {  // the first and the last window overlap their neighbours: the same values twice
#pragma unroll 4
      for (int at = skip + int(threadIdx.x) * VW; at < len; at += kBwdThreads * VW) window(min(at, len - VW), VW);
      if (skip && threadIdx.x == kBwdThreads - 1) window(0, VW);
    } else if (threadIdx.x == 0) {
      window(0, len);
    }
  }
}

struct DistillBwdArgs {
  const void* z;
  int64_t ld;
  void* dz;
  int64_t rows;
  int V, piece, pieces;
  float inv_tau, tau;
  const void* ids;
  int index_bytes;
  int k;
  const float* p;
  const float2* stats;
  const float* share;
  const float* inv_weight;  // [1]: 1 / sum of the rows' weights, or null: 1
  const void* go;           // a scalar, or [rows]
  int go_dtype, go_rows;
};

// dz_v = coef (q_v - sum over the entries of token v of p), coef = go * share * tau [/ sum of
// weights].  The piece is written without its teacher entries first; behind the barrier the
// (few) entries' tokens are written again, each with the sum of all its entries' p, which
// every one of them computes alike (a row may name a token twice).  Bound by its bytes: 4096 x
// 131072 in bf16, 2.1 GB, take 363 us (5.9 TB/s).
template <typename T>
__global__ __launch_bounds__(kBwdThreads) void distill_bwd_kernel(DistillBwdArgs a) {
  constexpr int VW = Win<T>::VW;
  __shared__ int ids[kMaxTeacher];
  __shared__ float ps[kMaxTeacher];
  const int64_t items = a.rows * a.pieces;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t row = a.pieces == 1 ? item : item / a.pieces;
    const int lo = a.pieces == 1 ? 0 : int(item - row * a.pieces) * a.piece;
    const int len = min(a.piece, a.V - lo);
    const T* z = static_cast<const T*>(a.z) + row * a.ld + lo;
    T* dz = static_cast<T*>(a.dz) + row * a.V + lo;
    const int64_t gi = a.go_rows ? row : 0;
    const float go = a.go_dtype == 1 ? static_cast<const float*>(a.go)[gi]
                                     : bf16_to_f32(static_cast<const uint16_t*>(a.go)[gi]);
    const float share = a.share[row];
    const float2 ms = a.stats[row];
    const bool none = share == 0.0f || ms.y == 0.0f;
    const float coef = none ? 0.0f : go * (a.inv_weight ? share * *a.inv_weight : share) * a.tau;
    for (int j = threadIdx.x; j < a.k; j += kBwdThreads) {
      const int64_t id = index_at(a.ids, a.index_bytes, row * a.k + j) - lo;
      ids[j] = id >= 0 && id < len ? int(id) : -1;
      ps[j] = a.p[row * a.k + j];
    }
    const float c = a.inv_tau * kLog2e, cq = coef * ms.y;
    const auto window = [&](int at, int n) {
      Raw o = {{0u, 0u, 0u, 0u}};
      if (!none) {
        const Raw r = load_win<T>(z + at, n);
#pragma unroll
        for (int e = 0; e < VW; ++e) raw_set<T>(o, e, cq * exp2_hw((raw_get<T>(r, e) - ms.x) * c));
      }
      store_win<T>(dz + at, o, n);
    };
    const int skip = word_skip(dz);
    if (len >= VW) {  // the first and the last window overlap their neighbours: the same values twice
#pragma unroll 4
      for (int at = skip + int(threadIdx.x) * VW; at < len; at += kBwdThreads * VW) window(min(at, len - VW), VW);
      if (skip && threadIdx.x == kBwdThreads - 1) window(0, VW);
    } else if (threadIdx.x == 0) {
      window(0, len);
    }
    __syncthreads();
    if (!none)
      for (int j = threadIdx.x; j < a.k; j += kBwdThreads) {
        const int id = ids[j];
        if (id < 0) continue;
        float p = 0.0f;
        for (int i = 0; i < a.k; ++i) p += ids[i] == id ? ps[i] : 0.0f;
        store_one<T>(dz + id, cq * exp2_hw((load_one<T>(z + id) - ms.x) * c) - coef * p);
      }
    __syncthreads();
  }
}

// loss = sum of the rows' losses [/ sum of their weights], in fixed order (fp64): 4096 rows 4.9 us
template <bool MEAN>
__global__ __launch_bounds__(1024) void distill_total_kernel(const float* __restrict__ loss,
                                                             const float* __restrict__ share, int64_t rows,
                                                             float* __restrict__ out, float* __restrict__ inv_weight) {
  __shared__ double red[2][16];
  double l = 0.0, w = 0.0;
  for (int64_t i = threadIdx.x; i < rows; i += 1024) l += double(loss[i]), w += double(share[i]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o, 64), w += __shfl_xor(w, o, 64);
  if ((threadIdx.x & 63) == 0) red[0][threadIdx.x >> 6] = l, red[1][threadIdx.x >> 6] = w;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) l += red[0][i], w += red[1][i];
    const double inv = !MEAN ? 1.0 : w != 0.0 ? 1.0 / w : 0.0;
    out[0] = float(MEAN && w == 0.0 && l == l ? 0.0 : l * inv);
    inv_weight[0] = float(inv);
  }
}

// ---- launch plans --------------------------------------------------------------------------------

struct Plan {
  int threads, piece, pieces;
};

// Whole rows where they are short or come near filling the chip, else pieces of equal length, of at
// least half a step of the workgroup, and their join.  Measured, pieces and whole rows in us (bf16):
// 400 x 131072 26.7 and 20.8, 300 x 131072 with 5 alternatives 38 and 45; 300 x 50001 12.8 and 12.0;
// 1 x 32000 7.1 and 5.4, with 20 alternatives 15.0 and 16.2, 200 x 32000 with 20 23 and 19.
// One wave a row where that is short and there are enough of them (no barriers): 3000 x 6000 9.4 and
// 12.0 with four waves, 3000 x 4000 with 5 alternatives 17 and 27, but 200 x 4000 10.3 and 8.6.
Plan row_plan(int64_t rows, int64_t V) {
  Plan p;
  p.threads = V <= 2048 || (V <= 6144 && rows >= 1024) ? 64 : 256;
  const bool whole = V <= 32768 || rows >= 384 || (rows >= 256 && V <= 65536);
  p.pieces = whole ? 1 : int(std::min<int64_t>({ceil_div(V, int64_t(4096)), ceil_div(int64_t(1024), rows), kMaxPieces}));
  p.piece = int(ceil_div(ceil_div(V, int64_t(p.pieces)), int64_t(8)) * 8);
  p.pieces = int(ceil_div(V, int64_t(p.piece)));
  return p;
}

Plan bwd_plan(int64_t V) {
  Plan p;
  p.threads = kBwdThreads;
  p.pieces = int(ceil_div(V, int64_t(16384)));
  p.piece = int(ceil_div(ceil_div(V, int64_t(p.pieces)), int64_t(8)) * 8);
  p.pieces = int(ceil_div(V, int64_t(p.piece)));
  return p;
}

// A grid's workgroups: its threads stay under 2^32, the kernels stride over the rest.
unsigned grid_of(int64_t items, int threads) {
  return unsigned(std::min<int64_t>(items, (int64_t(1) << 31) / threads));
}

size_t list_offset(int64_t rows, const Plan& p) {
  return size_t(ceil_div(rows * p.pieces * int64_t(sizeof(RowStat)), int64_t(16))) * 16;
}

size_t row_workspace(int64_t rows, int64_t V, int top) {
  const Plan p = row_plan(rows, V);
  if (p.pieces == 1) return 0;
  return list_offset(rows, p) + size_t(rows) * p.pieces * top * sizeof(uint64_t);
}

template <typename T, int MODE, bool TOP>
void launch_row(const Plan& p, const RowArgs& a, hipStream_t st) {
  const int64_t items = a.rows * a.pieces;
  if (p.threads == 64) row_kernel<T, 64, MODE, TOP><<<grid_of(items, 64), 64, 0, st>>>(a);
  else row_kernel<T, 256, MODE, TOP><<<grid_of(items, 256), 256, 0, st>>>(a);
  if (a.pieces > 1) {
    const size_t lds = TOP ? size_t(a.pieces) * a.lp.top * sizeof(uint64_t) : 0;
    join_kernel<T, MODE, TOP><<<grid_of(a.rows, kJoinThreads), kJoinThreads, lds, st>>>(a);
  }
}

bool rows_ok(const char* what, const void* z, int dtype, int64_t rows, int64_t V, int64_t ld, float tau) {
  std::string why;
  if (dtype != 1 && dtype != 2) why = "dtype must be 1 (fp32) or 2 (bf16)";
  else if (rows < 0) why = "negative row count";
  else if (V < 1 || V > kMaxVocab) why = "vocabulary outside 1 .. 2^22";
  else if (ld < V) why = "rows overlap";
  else if (!(tau > 0.0f) || !(tau < INFINITY)) why = "temperature must be positive and finite";
  else if (!(1.0f / tau * kLog2e < INFINITY)) why = "temperature too small: log2(e) / temperature is infinite";
  else if (rows > (int64_t(1) << 40) / V) why = "too many logits";
  else if (rows > 0 && !z) why = "null logits";
  else if (reinterpret_cast<uintptr_t>(z) % (dtype == 1 ? 4 : 2)) why = "misaligned logits";
  if (why.empty()) return true;
  set_error(std::string(what) + ": " + why);
  return false;
}

int refuse(const char* what, const char* why) {
  set_error(std::string(what) + ": " + why);
  return -1;
}

bool off(const void* p, unsigned bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }

bool workspace_ok(const char* what, const void* ws, size_t have, size_t need) {
  if (!need || (ws && have >= need && (reinterpret_cast<uintptr_t>(ws) & 15) == 0)) return true;
  refuse(what, "workspace missing, misaligned or too small");
  return false;
}

}  // namespace
}  // namespace xdna

using namespace xdna;

extern "C" {

size_t xdna_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int top) {
  if (rows < 1 || vocab < 1 || vocab > kMaxVocab || top < 0 || top > kMaxTop || rows > (int64_t(1) << 40) / vocab) return 0;
  return row_workspace(rows, vocab, top);
}

int xdna_token_logprobs(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t ld, const void* targets,
                        int index_bytes, float tau, int top, float* log_probs, float* entropy, float* stats,
                        float* top_log_probs, int64_t* top_ids, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "xdna_token_logprobs";
  if (!rows_ok(what, logits, dtype, rows, vocab, ld, tau)) return -1;
  if (top < 0 || top > kMaxTop || top > vocab) return refuse(what, "top outside 0 .. min(64, vocabulary)");
  if (index_bytes != 4 && index_bytes != 8) return refuse(what, "indices of 4 or 8 bytes");
  if (rows == 0) return 0;
  if (!targets || !log_probs || !entropy || !stats || (top && (!top_log_probs || !top_ids)))
    return refuse(what, "null operand");
  if (off(stats, 8)) return refuse(what, "misaligned stats");
  if (!workspace_ok(what, workspace, workspace_bytes, row_workspace(rows, vocab, top))) return -1;
  if (!admit_launch(what)) return -1;
  const Plan p = row_plan(rows, vocab);
  RowArgs a = {};
  a.z = logits;
  a.ld = ld;
  a.rows = rows;
  a.V = int(vocab);
  a.piece = p.piece;
  a.pieces = p.pieces;
  a.inv_tau = 1.0f / tau;
  a.stat = static_cast<RowStat*>(workspace);
  a.list = reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + (p.pieces > 1 ? list_offset(rows, p) : 0));
  a.lp = {targets, index_bytes, log_probs, entropy, reinterpret_cast<float2*>(stats), top_log_probs, top_ids, top};
  hipStream_t st = as_stream(stream);
  if (dtype == 1) top ? launch_row<float, kLogprob, true>(p, a, st) : launch_row<float, kLogprob, false>(p, a, st);
  else top ? launch_row<uint16_t, kLogprob, true>(p, a, st) : launch_row<uint16_t, kLogprob, false>(p, a, st);
  return check_launch(what);
}

int xdna_token_logprobs_bwd(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t ld, const void* targets,
                            int index_bytes, float tau, const float* stats, const float* entropy,
                            const float* d_log_probs, const float* d_entropy, void* d_logits, void* stream) {
  const char* what = "xdna_token_logprobs_bwd";
  if (!rows_ok(what, logits, dtype, rows, vocab, ld, tau)) return -1;
  if (index_bytes != 4 && index_bytes != 8) return refuse(what, "indices of 4 or 8 bytes");
  if (rows == 0) return 0;
  if (!targets || !stats || !entropy || !d_logits) return refuse(what, "null operand");
  if (off(stats, 8) || off(d_logits, dtype == 1 ? 4 : 2)) return refuse(what, "misaligned operand");
  if (!admit_launch(what)) return -1;
  const Plan p = bwd_plan(vocab);
  const LogprobBwdArgs a = {logits, ld, d_logits, rows, int(vocab), p.piece, p.pieces, 1.0f / tau, targets, index_bytes,
                            reinterpret_cast<const float2*>(stats), entropy, d_log_probs, d_entropy};
  hipStream_t st = as_stream(stream);
  const unsigned grid = grid_of(rows * p.pieces, kBwdThreads);
  if (dtype == 1) logprob_bwd_kernel<float><<<grid, kBwdThreads, 0, st>>>(a);
  else logprob_bwd_kernel<uint16_t><<<grid, kBwdThreads, 0, st>>>(a);
  return check_launch(what);
}

size_t xdna_distill_workspace_bytes(int64_t rows, int64_t vocab) {
  if (rows < 1 || vocab < 1 || vocab > kMaxVocab || rows > (int64_t(1) << 40) / vocab) return 0;
  return row_workspace(rows, vocab, 0);
}

int xdna_distill(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t ld, const void* ids,
                 int index_bytes, const void* teacher, int teacher_dtype, int k, float tau, const float* weight,
                 int reduction, float* row_loss, float* row_share, float* stats, float* p, float* loss, float* inv_weight,
                 void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "xdna_distill";
  if (!rows_ok(what, logits, dtype, rows, vocab, ld, tau)) return -1;
  if (k < 1 || k > kMaxTeacher) return refuse(what, "teacher entries outside 1 .. 1024");
  if (index_bytes != 4 && index_bytes != 8) return refuse(what, "indices of 4 or 8 bytes");
  if (teacher_dtype != 1 && teacher_dtype != 2) return refuse(what, "teacher logits are fp32 or bf16");
  if (reduction < 0 || reduction > 2) return refuse(what, "reduction must be 0 (none), 1 (mean) or 2 (sum)");
  if (reduction != 0 && (!loss || !inv_weight)) return refuse(what, "null operand");
  if (rows > 0 && (!ids || !teacher || !row_loss || !row_share || !stats || !p)) return refuse(what, "null operand");
  if (off(stats, 8)) return refuse(what, "misaligned stats");
  if (!workspace_ok(what, workspace, workspace_bytes, rows > 0 ? row_workspace(rows, vocab, 0) : 0)) return -1;
  if (!admit_launch(what)) return -1;
  hipStream_t st = as_stream(stream);
  if (rows > 0) {
    const Plan pl = row_plan(rows, vocab);
    RowArgs a = {};
    a.z = logits;
    a.ld = ld;
    a.rows = rows;
    a.V = int(vocab);
    a.piece = pl.piece;
    a.pieces = pl.pieces;
    a.inv_tau = 1.0f / tau;
    a.stat = static_cast<RowStat*>(workspace);
    a.ds = {ids, index_bytes, teacher, teacher_dtype, weight, k, tau, reinterpret_cast<float2*>(stats), p, row_loss, row_share};
    if (dtype == 1) launch_row<float, kDistill, false>(pl, a, st);
    else launch_row<uint16_t, kDistill, false>(pl, a, st);
  }
  if (reduction == 1) distill_total_kernel<true><<<1, 1024, 0, st>>>(row_loss, row_share, rows, loss, inv_weight);
  else if (reduction == 2) distill_total_kernel<false><<<1, 1024, 0, st>>>(row_loss, row_share, rows, loss, inv_weight);
  return check_launch(what);
}

int xdna_distill_bwd(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t ld, const void* ids,
                     int index_bytes, int k, float tau, const float* row_share, const float* stats, const float* p,
                     const float* inv_weight, const void* go, int go_dtype, int go_rows, void* d_logits, void* stream) {
  const char* what = "xdna_distill_bwd";
  if (!rows_ok(what, logits, dtype, rows, vocab, ld, tau)) return -1;
  if (k < 1 || k > kMaxTeacher) return refuse(what, "teacher entries outside 1 .. 1024");
  if (index_bytes != 4 && index_bytes != 8) return refuse(what, "indices of 4 or 8 bytes");
  if (go_dtype != 1 && go_dtype != 2) return refuse(what, "the incoming gradient is fp32 or bf16");
  if (rows == 0) return 0;
  if (!ids || !row_share || !stats || !p || !go || !d_logits) return refuse(what, "null operand");
  if (off(stats, 8) || off(d_logits, dtype == 1 ? 4 : 2)) return refuse(what, "misaligned operand");
  if (!admit_launch(what)) return -1;
  const Plan pl = bwd_plan(vocab);
  const DistillBwdArgs a = {logits, ld, d_logits, rows, int(vocab), pl.piece, pl.pieces, 1.0f / tau, tau, ids,
                            index_bytes, k, p, reinterpret_cast<const float2*>(stats), row_share, inv_weight, go, go_dtype, go_rows ? 1 : 0};
  hipStream_t st = as_stream(stream);
  const unsigned grid = grid_of(rows * pl.pieces, kBwdThreads);
  if (dtype == 1) distill_bwd_kernel<float><<<grid, kBwdThreads, 0, st>>>(a);
  else distill_bwd_kernel<uint16_t><<<grid, kBwdThreads, 0, st>>>(a);
  return check_launch(what);
}

}  // extern "C"
