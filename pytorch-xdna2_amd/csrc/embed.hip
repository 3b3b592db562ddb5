// Embedding rows on gfx950: lookup with scaling, and its gradient by sorted tokens.  The
// reference reaches both through its zero-copy CPU fallback (torch_xdna_device.cpp:5124-5260).
//
//   y[t] = scale W[id_t];   dW[v] = scale sum over {t: id_t = v} of dy[t], 0 for other rows.
//
// The gradient sorts the token positions by id (stable) and sums each id's rows in that order
// in fp32, rounded once: the same inputs give the same bits, and no token, however common,
// makes others wait for its row.
//   Order of up to kRankItems positions: by counting.  A workgroup holds all ids in LDS and
// counts, for 64 positions, the ids that come before: one launch and no passes.  The count
// grows with the square of the positions; above, a radix sort in blocks, a histogram and a
// scatter launch per digit of up to 9 bits (two digits serve every vocabulary below 2^18).
//   The rows of dW that no token names have to be written too: the ordering launches, which are
// bound by latency, share the writing of zeros to all of dW among their other workgroups.
//   Sum: a wave takes a chunk of sorted positions and 64 windows of 16 bytes of the columns.  A
// run of one id inside the chunk is written straight to dW; the parts of a run that crosses
// chunks go to fp32 partials (one slot for the run that came in, one for the run that goes
// on), which a last launch joins in chunk order.
//   Ids outside the table: their lookup gives NaN rows, their gradient is dropped (an id is
// data on the device: there is nothing to raise without waiting for it).
#include "common.h"

#include "../../include/xdna_hip.h"

namespace xdna {
namespace {

constexpr int kMinChunk = 8, kMaxChunk = 64;  // sorted positions per wave (a group of loads; its lanes)
constexpr int kSortPer = 8;          // positions per thread of a sorting workgroup
constexpr int kSortThreads = 1024;
constexpr int kSortItems = kSortPer * kSortThreads;
constexpr int kSortWaves = kSortThreads / 64;
// Ids in LDS (64 KB).  The whole gradient in 15000 rows of 64 by counting and by the radix sort, in
// us: 1000 positions 16 and 28, 4096 19 and 36, 16384 35 and 48, 20000 66 and 49.
constexpr int kRankItems = 16384;
constexpr int kDigitBits = 9, kDigits = 1 << kDigitBits;

template <typename T>
struct EW {
  static constexpr int n = 16 / int(sizeof(T));
};

template <typename T>
__device__ inline void unpack(const Pix8& q, float (&v)[EW<T>::n]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(q.v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[2 * e] = __uint_as_float(q.v[e] << 16);
      v[2 * e + 1] = __uint_as_float(q.v[e] & 0xFFFF0000u);
    }
  }
}

template <typename T>
__device__ inline Pix8 pack(const float (&v)[EW<T>::n]) {
  Pix8 q;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e) q.v[e] = __float_as_uint(v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      q.v[e] = uint32_t(f32_to_bf16(v[2 * e])) | (uint32_t(f32_to_bf16(v[2 * e + 1])) << 16);
  }
  return q;
}

template <typename T>
__device__ inline float one(const T* p) {
  if constexpr (sizeof(T) == 4) return *p;
  else return bf16_to_f32(*p);
}

template <typename T>
__device__ inline void put_one(T* p, float v) {
  if constexpr (sizeof(T) == 4) *p = v;
  else *p = f32_to_bf16(v);
}

// The n (at most a window's) elements at p, zeros after them.
template <typename T>
__device__ inline Pix8 window(const T* p, int n) {
  if (n >= EW<T>::n) return *reinterpret_cast<const Pix8*>(p);
  float v[EW<T>::n];
#pragma unroll
  for (int e = 0; e < EW<T>::n; ++e) v[e] = e < n ? one<T>(p + e) : 0.0f;
  return pack<T>(v);
}

template <typename T>
__device__ inline void put_window(T* p, const float (&v)[EW<T>::n], int n) {
  if (n >= EW<T>::n) {
    *reinterpret_cast<Pix8*>(p) = pack<T>(v);
    return;
  }
#pragma unroll
  for (int e = 0; e < EW<T>::n; ++e)
    if (e < n) put_one<T>(p + e, v[e]);
}

__device__ inline int64_t id_at(const void* ids, int index_bytes, int64_t i) {
  return index_bytes == 8 ? static_cast<const int64_t*>(ids)[i] : int64_t(static_cast<const int32_t*>(ids)[i]);
}

struct LookupArgs {
  const void* ids;
  int index_bytes;
  int64_t tokens;
  const void* w;
  int64_t ld;
  void* y;
  int vocab, dim;
  float scale;
  int tx;  // threads along a row: a power of two up to 64
};

// Bound by its writes (and the rows it reads): 64 / tx rows per wave, 16 bytes per lane.  65536 rows
// of 2048 in bf16 take 76 us (537 MB, 7.0 TB/s; rows named again come from the caches), one row 2.3.
template <typename T>
__global__ __launch_bounds__(256) void lookup_kernel(LookupArgs a) {
  constexpr int W = EW<T>::n;
  const int ty = threadIdx.x / a.tx, tx = threadIdx.x & (a.tx - 1);
  const int rows = 256 / a.tx;
  for (int64_t t = int64_t(blockIdx.x) * rows + ty; t < a.tokens; t += int64_t(gridDim.x) * rows) {
    const int64_t id = id_at(a.ids, a.index_bytes, t);
    const bool ok = id >= 0 && id < a.vocab;
    const T* src = static_cast<const T*>(a.w) + (ok ? id : 0) * a.ld;
    T* dst = static_cast<T*>(a.y) + t * a.dim;
#pragma unroll 4
    for (int at = tx * W; at < a.dim; at += a.tx * W) {
      const int n = a.dim - at;
      float v[W];
      unpack<T>(window<T>(src + at, n), v);
#pragma unroll
      for (int e = 0; e < W; ++e) v[e] = ok ? v[e] * a.scale : NAN;
      put_window<T>(dst + at, v, n);
    }
  }
}

// ---- stable sort of the positions by id ------------------------------------------------------

struct SortArgs {
  const void* ids;
  int index_bytes;
  int n, vocab;
  int64_t padding;
  int shift, bits;         // this pass's digit
  const uint32_t* key_in;  // null: from ids
  const uint32_t* pos_in;
  uint32_t* key;
  uint32_t* pos;
  uint32_t* hist;          // [blocks][kDigits]
  int blocks;
  char* fill;              // zeros for fill_bytes bytes, by the workgroups past the sorting ones
  int64_t fill_bytes;
};

// Ids without a gradient (padding, outside the table) sort behind all others.
__device__ inline uint32_t sort_key(const SortArgs& a, int64_t i) {
  const int64_t id = id_at(a.ids, a.index_bytes, i);
  return id < 0 || id >= a.vocab || id == a.padding ? uint32_t(a.vocab) : uint32_t(id);
}

// fill_bytes are whole 16-byte vectors but for the last launch's end
__device__ inline void zero_fill(const SortArgs& a, int block, int blocks, int threads) {
  const int64_t whole = a.fill_bytes >> 4;
  const int64_t step = int64_t(blocks) * threads;
  uint4* to = reinterpret_cast<uint4*>(a.fill);
  for (int64_t i = int64_t(block) * threads + threadIdx.x; i < whole; i += step) to[i] = make_uint4(0, 0, 0, 0);
  if (block == 0 && threadIdx.x < ((a.fill_bytes & 15) >> 1))
    reinterpret_cast<uint16_t*>(to + whole)[threadIdx.x] = 0;
}

// Order by counting: workgroup b finds the places of positions 64 b .. 64 b + 63 (lane l: 64 b +
// l), each of its 16 waves against a sixteenth of all keys, read from LDS four at a time.  A key
// comes before an equal one at a later position.  4099 positions take 11 us (a third of it LDS reads
// and compares), 8192 beside 102 MB of zeros 17.5 (5.9 TB/s).  With the radix sort and a fill of its
// own, lookup and gradient of 8192 rows of 1024 took 72 us, so 44.
__global__ __launch_bounds__(kSortThreads) void rank_kernel(SortArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint32_t keys[];  // [n rounded up to 64]
  __shared__ uint32_t part[kSortThreads];
  if (int(blockIdx.x) >= a.blocks) {
    zero_fill(a, int(blockIdx.x) - a.blocks, int(gridDim.x) - a.blocks, kSortThreads);
    return;
  }
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int groups = a.blocks;
  // (clamped positions: the loads of a round are issued together)
  for (int base = 0; base < groups * 64; base += 8 * kSortThreads) {
    uint32_t k[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) k[j] = sort_key(a, min(base + j * kSortThreads + tid, a.n - 1));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = base + j * kSortThreads + tid;
      if (i < groups * 64) keys[i] = i < a.n ? k[j] : 0xFFFFFFFFu;
    }
  }
  __syncthreads();
  const int own = blockIdx.x;
  const uint32_t mine = keys[own * 64 + lane];
  uint32_t count = 0;
  for (int g = wave; g < groups; g += kSortWaves) {
    const uint4* q = reinterpret_cast<const uint4*>(keys + g * 64);
    if (g == own) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint4 v = q[i];
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) count += w[e] < mine || (w[e] == mine && 4 * i + e < lane) ? 1u : 0u;
      }
    } else {
      // keys below `least` come before: mine itself, or one more where equal ones do (keys of
      // real positions are below 2^31)
      const uint32_t least = mine + (g < own ? 1u : 0u);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint4 v = q[i];
        count += (v.x < least ? 1u : 0u) + (v.y < least ? 1u : 0u) + (v.z < least ? 1u : 0u) + (v.w < least ? 1u : 0u);
      }
    }
  }
  part[tid] = count;
  __syncthreads();
  if (wave == 0) {
#pragma unroll
    for (int w = 1; w < kSortWaves; ++w) count += part[w * 64 + lane];
    const int i = own * 64 + lane;
    if (i < a.n) a.key[count] = mine, a.pos[count] = uint32_t(i);
  }
}

// Ranks of this thread's items within the workgroup's items of equal digit, in item order
// (wave w holds items [512 w, +512), lane l item 64 j + l of them): lanes of equal digit by
// ballots over the digit's bits, counts per wave in LDS.
__device__ inline void wave_rank(const uint32_t (&digit)[kSortPer], int bits, uint32_t* count, int lane,
                                 uint32_t (&rank)[kSortPer]) {
  const uint64_t below = (uint64_t(1) << lane) - 1;
#pragma unroll
  for (int j = 0; j < kSortPer; ++j) {
    uint64_t same = ~uint64_t(0);
    for (int b = 0; b < bits; ++b) {
      const uint64_t set = __ballot((digit[j] >> b) & 1);
      same &= (digit[j] >> b) & 1 ? set : ~set;
    }
    const uint32_t before = count[digit[j]];
    rank[j] = before + uint32_t(__popcll(same & below));
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if ((same & below) == 0) count[digit[j]] = before + uint32_t(__popcll(same));
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// Exclusive prefix sum over the first kDigits threads of the workgroup.
__device__ inline uint32_t digit_prefix(uint32_t v, uint32_t* red) {
  const int tid = threadIdx.x, lane = tid & 63;
  uint32_t s = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t t = __shfl_up(s, o, 64);
    if (lane >= o) s += t;
  }
  if (tid < kDigits && lane == 63) red[tid >> 6] = s;
  __syncthreads();
  uint32_t base = 0;
  if (tid < kDigits)
    for (int w = 0; w < (tid >> 6); ++w) base += red[w];
  __syncthreads();
  return base + s - v;
}

// One pass in blocks of kSortItems: digit counts of each block (bound by latency and by the zeros
// written beside it: 65536 positions, two passes and 537 MB of zeros take 107 us, 5.0 TB/s) ...
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(SortArgs a) {
  __shared__ uint32_t count[kDigits];
  if (int(blockIdx.x) >= a.blocks) {
    zero_fill(a, int(blockIdx.x) - a.blocks, int(gridDim.x) - a.blocks, kSortThreads);
    return;
  }
  const int tid = threadIdx.x;
  if (tid < kDigits) count[tid] = 0;
  __syncthreads();
  const uint32_t mask = (1u << a.bits) - 1;
#pragma unroll
  for (int j = 0; j < kSortPer; ++j) {
    const int64_t i = int64_t(blockIdx.x) * kSortItems + j * kSortThreads + tid;
    if (i < a.n) atomicAdd(&count[((a.key_in ? a.key_in[i] : sort_key(a, i)) >> a.shift) & mask], 1u);
  }
  __syncthreads();
  if (tid < kDigits) a.hist[int64_t(blockIdx.x) * kDigits + tid] = count[tid];
}

// ... and the scatter to their places: smaller digits of all blocks, the digit in earlier
// blocks, then the rank in this one.
__global__ __launch_bounds__(kSortThreads) void sort_scatter_kernel(SortArgs a) {
  __shared__ uint32_t count[kSortWaves * kDigits];
  __shared__ uint32_t red[kDigits / 64];
  if (int(blockIdx.x) >= a.blocks) {
    zero_fill(a, int(blockIdx.x) - a.blocks, int(gridDim.x) - a.blocks, kSortThreads);
    return;
  }
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t first = int64_t(blockIdx.x) * kSortItems + wave * (64 * kSortPer) + lane;
  const uint32_t mask = (1u << a.bits) - 1;
  uint32_t key[kSortPer], pos[kSortPer], rank[kSortPer], digit[kSortPer];
#pragma unroll
  for (int j = 0; j < kSortPer; ++j) {
    const int64_t i = first + j * 64;
    const bool ok = i < a.n;
    key[j] = !ok ? 0xFFFFFFFFu : a.key_in ? a.key_in[i] : sort_key(a, i);
    pos[j] = !ok ? 0u : a.pos_in ? a.pos_in[i] : uint32_t(i);
    digit[j] = (key[j] >> a.shift) & mask;
  }
  uint32_t* mine = count + wave * kDigits;
#pragma unroll
  for (int d = 0; d < kDigits / 64; ++d) mine[d * 64 + lane] = 0;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  wave_rank(digit, a.bits, mine, lane, rank);
  uint32_t all = 0, before = 0;
  if (tid < kDigits) {
#pragma unroll 8
    for (int b = 0; b < a.blocks; ++b) {
      const uint32_t h = a.hist[int64_t(b) * kDigits + tid];
      all += h;
      before += b < int(blockIdx.x) ? h : 0;
    }
  }
  uint32_t place = digit_prefix(all, red) + before;  // (its barriers also publish the counts)
  if (tid < kDigits)
    for (int w = 0; w < kSortWaves; ++w) {
      const uint32_t c = count[w * kDigits + tid];
      count[w * kDigits + tid] = place;
      place += c;
    }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kSortPer; ++j)
    if (first + j * 64 < a.n) {
      const uint32_t at = mine[digit[j]] + rank[j];
      a.key[at] = key[j];
      a.pos[at] = pos[j];
    }
}

// ---- sums over the sorted positions --------------------------------------------------------

struct SumArgs {
  const uint32_t* key;
  const uint32_t* pos;
  int n, vocab, dim, slices;  // slices of 64 windows along dim
  int chunk, chunks;
  const void* dy;
  int64_t ld;
  void* dw;      // [vocab][dim]
  float* part;   // [chunks][2][pitch]
  int pitch;     // dim rounded up to windows
  float scale;
};

template <int W>
__device__ inline void put_part(float* p, const float (&v)[W]) {
#pragma unroll
  for (int e = 0; e < W; e += 4) *reinterpret_cast<float4*>(p + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
}

template <int W>
__device__ inline void add_part(float (&v)[W], const float* p) {
#pragma unroll
  for (int e = 0; e < W; e += 4) {
    const float4 q = *reinterpret_cast<const float4*>(p + e);
    v[e] += q.x, v[e + 1] += q.y, v[e + 2] += q.z, v[e + 3] += q.w;
  }
}

// Bound by the bytes of scattered rows: 65536 rows of 2048 in bf16 into 131072 take 116 us (268 MB
// read, 212 MB written: 4.1 TB/s).  Chunks of 8 to 64 positions: as long as they leave every CU 16
// waves, since each edge may cost a partial.
template <typename T>
__global__ __launch_bounds__(256) void sum_kernel(SumArgs a) {
  constexpr int W = EW<T>::n, G = 8;  // rows in flight
  const int lane = threadIdx.x & 63;
  const int64_t item = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (item >= int64_t(a.chunks) * a.slices) return;
  const int chunk = __builtin_amdgcn_readfirstlane(int(item / a.slices));
  const int slice = __builtin_amdgcn_readfirstlane(int(item - int64_t(chunk) * a.slices));
  const int first = chunk * a.chunk;
  const int count = min(a.chunk, a.n - first);
  const int col = (slice * 64 + lane) * W;
  const int width = a.dim - col;  // below 1: this lane has no column
  // the chunk's keys and positions by lane; the neighbours' keys
  uint32_t k = 0xFFFFFFFFu, ps = 0;
  if (lane < count) k = a.key[first + lane], ps = a.pos[first + lane];
  const uint32_t prev = first > 0 ? a.key[first - 1] : 0xFFFFFFFFu;
  const uint32_t next = first + count >= a.n ? 0xFFFFFFFFu : a.key[first + count];
  const T* dy = static_cast<const T*>(a.dy);
  const auto load = [&](int base, Pix8 (&q)[G]) {
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const int at = min(base + i, count - 1);
      q[i] = {{0u, 0u, 0u, 0u}};
      if (uint32_t(__builtin_amdgcn_readlane(k, at)) < uint32_t(a.vocab) && width > 0)
        q[i] = window<T>(dy + int64_t(uint32_t(__builtin_amdgcn_readlane(ps, at))) * a.ld + col, width);
    }
  };
  float acc[W];
#pragma unroll
  for (int e = 0; e < W; ++e) acc[e] = 0.0f;
  bool came_in = uint32_t(__builtin_amdgcn_readlane(k, 0)) == prev;
  Pix8 nq[G];
  load(0, nq);
  for (int base = 0; base < count; base += G) {
    Pix8 q[G];
#pragma unroll
    for (int i = 0; i < G; ++i) q[i] = nq[i];
    if (base + G < count) load(base + G, nq);
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const int at = base + i;
      if (at >= count) break;
      const uint32_t id = __builtin_amdgcn_readlane(k, at);
      if (id >= uint32_t(a.vocab)) return;  // the rest of the order has no gradient
      float v[W];
      unpack<T>(q[i], v);
#pragma unroll
      for (int e = 0; e < W; ++e) acc[e] += v[e];
      const bool edge = at + 1 == count;
      const bool ends = (edge ? next : uint32_t(__builtin_amdgcn_readlane(k, min(at + 1, 63)))) != id;
      if (!ends && !edge) continue;
      if (width > 0) {
        if (ends && !came_in) {
#pragma unroll
          for (int e = 0; e < W; ++e) v[e] = acc[e] * a.scale;
          put_window<T>(static_cast<T*>(a.dw) + int64_t(id) * a.dim + col, v, width);
        } else {
          put_part<W>(a.part + (int64_t(chunk) * 2 + (came_in ? 0 : 1)) * a.pitch + col, acc);
        }
      }
#pragma unroll
      for (int e = 0; e < W; ++e) acc[e] = 0.0f;
      came_in = false;
    }
  }
}

// Joins the runs that cross chunks: a workgroup for the chunk where a run begins and a slice of
// the columns; of a long run each of its four waves adds a quarter, in order.  Most workgroups find
// no run to join: 65536 rows 7.7 us.
template <typename T>
__global__ __launch_bounds__(256) void sum_join_kernel(SumArgs a) {
  constexpr int W = EW<T>::n;
  __shared__ __attribute__((aligned(16))) float quarter[3][64 * W];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int chunk = int(blockIdx.x) / a.slices, slice = int(blockIdx.x) - chunk * a.slices;
  const int first = chunk * a.chunk;
  const int64_t after = int64_t(first) + a.chunk;  // chunk + 1 exists: position `after` does
  const uint32_t id = a.key[after - 1];
  if (id >= uint32_t(a.vocab) || a.key[after] != id) return;
  if (a.key[first] == id && first > 0 && a.key[first - 1] == id) return;  // it began earlier
  // chunks after this one that the run reaches: chunk + 1, and further while the first position
  // of a next one still holds id
  int reach = 1;
  for (;;) {
    const int64_t at = (int64_t(chunk) + reach + lane + 1) * a.chunk;
    const bool on = at < a.n && a.key[at] == id;
    const uint64_t stop = ~__ballot(on);
    if (stop) {
      reach += __ffsll(static_cast<unsigned long long>(stop)) - 1;
      break;
    }
    reach += 64;
  }
  const bool shared = reach > 16;
  if (!shared && wave > 0) return;
  const int col = (slice * 64 + lane) * W;
  const int width = a.dim - col;
  float acc[W];
#pragma unroll
  for (int e = 0; e < W; ++e) acc[e] = 0.0f;
  if (width > 0) {
    const int64_t step = 2 * int64_t(a.pitch);
    const float* from = a.part + int64_t(chunk) * step + col;
    if (wave == 0) add_part<W>(acc, from + a.pitch);
    const int share = (reach + 3) / 4;
    const int lo = shared ? 1 + wave * share : 1, hi = shared ? min(reach, lo + share - 1) : reach;
#pragma unroll 8
    for (int j = lo; j <= hi; ++j) add_part<W>(acc, from + j * step);
  }
  if (shared) {
    if (wave > 0) put_part<W>(&quarter[wave - 1][lane * W], acc);
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 0; w < 3; ++w) add_part<W>(acc, &quarter[w][lane * W]);
  }
  if (width <= 0) return;
#pragma unroll
  for (int e = 0; e < W; ++e) acc[e] *= a.scale;
  put_window<T>(static_cast<T*>(a.dw) + int64_t(id) * a.dim + col, acc, width);
}

// ---- workspace: sorted keys and positions (twice where passes go between buffers), block
// counts, partials -----------------------------------------------------------------------------

int64_t up16(int64_t b) { return (b + 15) & ~int64_t(15); }

struct GradPlan {
  int bits, passes, pass_bits, blocks, chunk, chunks, pitch;
  bool rank;
  int64_t keys, hist, part, total;  // byte sizes and the total
};

GradPlan grad_plan(int64_t tokens, int64_t vocab, int64_t dim) {
  GradPlan p;
  p.bits = 1;
  while ((int64_t(1) << p.bits) <= vocab) ++p.bits;  // keys 0 .. vocab
  p.passes = int(ceil_div(p.bits, kDigitBits));
  p.pass_bits = int(ceil_div(p.bits, p.passes));
  p.rank = tokens <= kRankItems;
  p.blocks = int(ceil_div(tokens, int64_t(p.rank ? 64 : kSortItems)));
  p.pitch = int(ceil_div(dim, int64_t(8)) * 8);
  // chunks that give 4096 waves (four a SIMD)
  p.chunk = kMinChunk;
  while (p.chunk < kMaxChunk && ceil_div(tokens, int64_t(2 * p.chunk)) * ceil_div(dim, int64_t(512)) >= 4096) p.chunk *= 2;
  p.chunks = int(ceil_div(tokens, int64_t(p.chunk)));
  p.keys = up16(tokens * 4);
  p.hist = p.rank ? 0 : up16(int64_t(p.blocks) * kDigits * 4);
  p.part = int64_t(p.chunks) * 2 * p.pitch * 4;
  p.total = p.keys * (p.rank ? 2 : 4) + p.hist + p.part;
  return p;
}

constexpr int64_t kMaxTokens = int64_t(1) << 30, kMaxRows = int64_t(1) << 30, kMaxDim = int64_t(1) << 20;

int refuse(const char* what, const char* why) {
  set_error(std::string(what) + ": " + why);
  return -1;
}

const char* embed_fault(int index_bytes, int64_t tokens, int dtype, int64_t vocab, int64_t dim) {
  if (index_bytes != 4 && index_bytes != 8) return "indices of 4 or 8 bytes";
  if (dtype != 1 && dtype != 2) return "dtype must be 1 (fp32) or 2 (bf16)";
  if (tokens < 0 || tokens > kMaxTokens) return "token count outside 0 .. 2^30";
  if (vocab < 1 || vocab > kMaxRows) return "table rows outside 1 .. 2^30";
  if (dim < 1 || dim > kMaxDim) return "row length outside 1 .. 2^20";
  return nullptr;
}

bool off_element(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % (dtype == 1 ? 4 : 2) != 0; }

template <typename T>
void launch_sums(const SumArgs& s, hipStream_t st) {
  const int64_t items = int64_t(s.chunks) * s.slices;
  sum_kernel<T><<<unsigned(ceil_div(items, int64_t(4))), 256, 0, st>>>(s);
  if (s.chunks > 1) sum_join_kernel<T><<<unsigned(int64_t(s.chunks - 1) * s.slices), 256, 0, st>>>(s);
}

// Workgroups for a share of the zeros: 64 KB each, up to four a CU.
unsigned fillers(int64_t bytes) {
  return unsigned(std::max<int64_t>(bytes > 0 ? 1 : 0, std::min<int64_t>(ceil_div(bytes, int64_t(65536)), 1024)));
}

}  // namespace
}  // namespace xdna

using namespace xdna;

extern "C" {

int xdna_embed(const void* ids, int index_bytes, int64_t tokens, const void* weight, int dtype, int64_t vocab,
               int64_t dim, int64_t ld, float scale, void* out, void* stream) {
  const char* what = "xdna_embed";
  if (const char* why = embed_fault(index_bytes, tokens, dtype, vocab, dim)) return refuse(what, why);
  if (ld < dim && vocab > 1) return refuse(what, "table rows overlap");
  if (tokens == 0) return 0;
  if (!ids || !weight || !out) return refuse(what, "null operand");
  if (off_element(weight, dtype) || off_element(out, dtype)) return refuse(what, "misaligned operand");
  if (!admit_launch(what)) return -1;
  LookupArgs a = {ids, index_bytes, tokens, weight, ld, out, int(vocab), int(dim), scale, 1};
  const int64_t windows = ceil_div(dim, int64_t(dtype == 1 ? 4 : 8));
  while (a.tx < 64 && a.tx < windows) a.tx *= 2;
  const unsigned grid = unsigned(std::min<int64_t>(ceil_div(tokens, int64_t(256 / a.tx)), 16384));
  hipStream_t st = as_stream(stream);
  if (dtype == 1) lookup_kernel<float><<<grid, 256, 0, st>>>(a);
  else lookup_kernel<uint16_t><<<grid, 256, 0, st>>>(a);
  return check_launch(what);
}

size_t xdna_embed_bwd_workspace_bytes(int64_t tokens, int64_t vocab, int64_t dim) {
  if (tokens < 1 || tokens > kMaxTokens || vocab < 1 || vocab > kMaxRows || dim < 1 || dim > kMaxDim) return 0;
  return size_t(grad_plan(tokens, vocab, dim).total);
}

int xdna_embed_bwd(const void* ids, int index_bytes, int64_t tokens, const void* grad, int dtype, int64_t ld,
                   int64_t vocab, int64_t dim, int64_t padding, float scale, void* d_weight, void* workspace,
                   size_t workspace_bytes, void* stream) {
  const char* what = "xdna_embed_bwd";
  if (const char* why = embed_fault(index_bytes, tokens, dtype, vocab, dim)) return refuse(what, why);
  if (ld < dim && tokens > 1) return refuse(what, "gradient rows overlap");
  if (!d_weight || (tokens > 0 && (!ids || !grad))) return refuse(what, "null operand");
  if ((reinterpret_cast<uintptr_t>(d_weight) & 15) || off_element(grad, dtype)) return refuse(what, "misaligned operand");
  const GradPlan p = grad_plan(std::max<int64_t>(tokens, 1), vocab, dim);
  if (tokens > 0 && (!workspace || workspace_bytes < size_t(p.total) || (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return refuse(what, "workspace missing, misaligned or too small");
  if (int64_t(p.chunks) * ceil_div(dim, int64_t(64) * (dtype == 1 ? 4 : 8)) > kMaxGridX256)
    return refuse(what, "too many rows and columns");
  if (!admit_launch(what)) return -1;
  hipStream_t st = as_stream(stream);
  SortArgs s = {};
  s.ids = ids;
  s.index_bytes = index_bytes;
  s.n = int(tokens);
  s.vocab = int(vocab);
  s.padding = padding;
  s.fill = static_cast<char*>(d_weight);
  s.fill_bytes = vocab * dim * (dtype == 1 ? 4 : 2);
  if (tokens == 0) {  // nothing to order
    sort_count_kernel<<<fillers(s.fill_bytes), kSortThreads, 0, st>>>(s);
    return check_launch(what);
  }
  char* ws = static_cast<char*>(workspace);
  uint32_t* buf[4];  // key, position, and the other side of the passes
  for (int i = 0; i < (p.rank ? 2 : 4); ++i, ws += p.keys) buf[i] = reinterpret_cast<uint32_t*>(ws);
  s.hist = reinterpret_cast<uint32_t*>(ws);
  ws += p.hist;
  int side = 0;
  s.blocks = p.blocks;
  if (p.rank) {
    static const bool lds_ok = hipFuncSetAttribute(reinterpret_cast<const void*>(&rank_kernel),
                                                   hipFuncAttributeMaxDynamicSharedMemorySize, kRankItems * 4) == hipSuccess;
    if (!lds_ok) return refuse(what, "cannot enable the ordering kernel's LDS size");
    s.key = buf[0];
    s.pos = buf[1];
    rank_kernel<<<unsigned(p.blocks) + fillers(s.fill_bytes), kSortThreads, size_t(p.blocks) * 256, st>>>(s);
  } else {
    const int64_t all = s.fill_bytes, share = ceil_div(all, int64_t(2 * p.passes) * 16) * 16;
    const auto next_share = [&](int i) {  // of the i-th launch
      const int64_t lo = std::min(all, i * share), hi = std::min(all, lo + share);
      s.fill = static_cast<char*>(d_weight) + lo;
      s.fill_bytes = hi - lo;
      return unsigned(p.blocks) + fillers(s.fill_bytes);
    };
    for (int i = 0; i < p.passes; ++i) {
      s.shift = i * p.pass_bits;
      s.bits = p.pass_bits;
      s.key_in = i ? buf[side] : nullptr;
      s.pos_in = i ? buf[side + 1] : nullptr;
      side = i ? 2 - side : 0;
      s.key = buf[side];
      s.pos = buf[side + 1];
      const unsigned count_grid = next_share(2 * i);
      sort_count_kernel<<<count_grid, kSortThreads, 0, st>>>(s);
      const unsigned scatter_grid = next_share(2 * i + 1);
      sort_scatter_kernel<<<scatter_grid, kSortThreads, 0, st>>>(s);
    }
  }
  SumArgs m = {};
  m.key = buf[side];
  m.pos = buf[side + 1];
  m.n = int(tokens);
  m.vocab = int(vocab);
  m.dim = int(dim);
  m.slices = int(ceil_div(dim, int64_t(64) * (dtype == 1 ? 4 : 8)));
  m.chunk = p.chunk;
  m.chunks = p.chunks;
  m.pitch = p.pitch;
  m.dy = grad;
  m.ld = ld;
  m.dw = d_weight;
  m.part = reinterpret_cast<float*>(ws);
  m.scale = scale;
  if (dtype == 1) launch_sums<float>(m, st);
  else launch_sums<uint16_t>(m, st);
  return check_launch(what);
}

}  // extern "C"
