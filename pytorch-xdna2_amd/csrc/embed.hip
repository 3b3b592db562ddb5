// Embedding rows on gfx950: lookup with scaling, and its gradient by sorted tokens.  The
// reference reaches both through its zero-copy CPU fallback (torch_xdna_device.cpp:5124-5260).
//
//   y[t] = scale W[id_t];   dW[v] = scale sum over {t: id_t = v} of dy[t], 0 for other rows.
//
// The gradient sorts the token positions by id (stable, least significant digit first) and
// sums each id's rows in that order in fp32, rounded once: the same inputs give the same
// bits, and no token, however common, makes others wait for its row.
//   Sort: up to kSortItems positions in one workgroup's LDS, all digits in one launch; more
// in blocks, a histogram and a scatter launch per digit.  Digits have up to 9 bits: two
// passes serve every vocabulary below 2^18.
//   The rows of dW that no token names have to be written too: the sort's first launch,
// which fills a few CUs only, writes all of dW with zeros in its other workgroups.
//   Sum: a wave takes kChunk sorted positions and 64 windows of 16 bytes of the columns.  A
// run of one id inside the chunk is written straight to dW; the parts of a run that crosses
// chunks go to fp32 partials (one slot for the run that came in, one for the run that goes
// on), which a last launch joins in chunk order.
//   Ids outside the table: their lookup gives NaN rows, their gradient is dropped (an id is
// data on the device: there is nothing to raise without waiting for it).
#include "common.h"

#include "../../include/xdna_hip.h"

namespace xdna {
namespace {

constexpr int kChunk = 32;           // sorted positions per wave
constexpr int kSortPer = 8;          // positions per thread of a sorting workgroup
constexpr int kSortThreads = 1024;
constexpr int kSortItems = kSortPer * kSortThreads;
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

// Bound by its writes (and the rows it reads): 64 / tx rows per wave, 16 bytes per lane.
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
  int shift, bits;         // this pass's digit (block form)
  int passes, pass_bits;   // all passes (one-workgroup form)
  const uint32_t* key_in;  // null: from ids
  const uint32_t* pos_in;
  uint32_t* key;
  uint32_t* pos;
  uint32_t* hist;          // [blocks][kDigits]
  int blocks;
  uint4* fill;             // zeros for fill_bytes bytes, by the workgroups past the sorting ones
  int64_t fill_bytes;
};

// Ids without a gradient (padding, outside the table) sort behind all others.
__device__ inline uint32_t sort_key(const SortArgs& a, int64_t i) {
  const int64_t id = id_at(a.ids, a.index_bytes, i);
  return id < 0 || id >= a.vocab || id == a.padding ? uint32_t(a.vocab) : uint32_t(id);
}

__device__ inline void zero_fill(const SortArgs& a, int block, int blocks, int threads) {
  const int64_t whole = a.fill_bytes >> 4;
  const int64_t step = int64_t(blocks) * threads;
  for (int64_t i = int64_t(block) * threads + threadIdx.x; i < whole; i += step) a.fill[i] = make_uint4(0, 0, 0, 0);
  if (block == 0 && threadIdx.x < ((a.fill_bytes & 15) >> 1))
    reinterpret_cast<uint16_t*>(a.fill + whole)[threadIdx.x] = 0;
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

constexpr int kSortWaves = kSortThreads / 64;
constexpr size_t kSortLds = size_t(2) * kSortItems * 4 + size_t(kSortWaves) * kDigits * 4;

// All passes over up to kSortItems positions in LDS (workgroup 0; the others fill dW).
__global__ __launch_bounds__(kSortThreads) void sort_small_kernel(SortArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
  if (blockIdx.x > 0) {
    zero_fill(a, int(blockIdx.x) - 1, int(gridDim.x) - 1, kSortThreads);
    return;
  }
  __shared__ uint32_t red[kDigits / 64];
  uint32_t* keys = lds;
  uint32_t* poss = lds + kSortItems;
  uint32_t* count = lds + 2 * kSortItems;  // [waves][kDigits]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int first = wave * (64 * kSortPer) + lane;
  uint32_t key[kSortPer], pos[kSortPer], rank[kSortPer], digit[kSortPer];
#pragma unroll
  for (int j = 0; j < kSortPer; ++j) {
    const int i = first + j * 64;
    // places past the end hold the greatest key and the last positions: they stay last
    key[j] = i < a.n ? sort_key(a, i) : 0xFFFFFFFFu;
    pos[j] = uint32_t(i);
  }
  for (int p = 0; p < a.passes; ++p) {
    const int shift = p * a.pass_bits;
    const uint32_t mask = (1u << a.pass_bits) - 1;
    uint32_t* mine = count + wave * kDigits;
#pragma unroll
    for (int d = 0; d < kDigits / 64; ++d) mine[d * 64 + lane] = 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < kSortPer; ++j) digit[j] = (key[j] >> shift) & mask;
    wave_rank(digit, a.pass_bits, mine, lane, rank);
    __syncthreads();
    // counts -> first places: digits in order, waves in order within a digit
    uint32_t total = 0;
    if (tid < kDigits)
      for (int w = 0; w < kSortWaves; ++w) total += count[w * kDigits + tid];
    uint32_t place = digit_prefix(total, red);
    if (tid < kDigits)
      for (int w = 0; w < kSortWaves; ++w) {
        const uint32_t c = count[w * kDigits + tid];
        count[w * kDigits + tid] = place;
        place += c;
      }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kSortPer; ++j) {
      const uint32_t at = mine[digit[j]] + rank[j];
      keys[at] = key[j];
      poss[at] = pos[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kSortPer; ++j) key[j] = keys[first + j * 64], pos[j] = poss[first + j * 64];
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < kSortPer; ++j) {
    const int i = first + j * 64;
    if (i < a.n) a.key[i] = key[j], a.pos[i] = pos[j];
  }
}

// One pass in blocks of kSortItems: digit counts of each block ...
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
  int chunks;
  const void* dy;
  int64_t ld;
  void* dw;      // [vocab][dim]
  float* part;   // [chunks][2][dim]
  float scale;
};

template <typename T>
__global__ __launch_bounds__(256) void sum_kernel(SumArgs a) {
  constexpr int W = EW<T>::n;
  const int lane = threadIdx.x & 63;
  const int64_t item = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (item >= int64_t(a.chunks) * a.slices) return;
  const int chunk = __builtin_amdgcn_readfirstlane(int(item / a.slices));
  const int slice = __builtin_amdgcn_readfirstlane(int(item - int64_t(chunk) * a.slices));
  const int first = chunk * kChunk;
  const int count = min(kChunk, a.n - first);
  const int col = (slice * 64 + lane) * W;
  const int width = a.dim - col;  // below 1: this lane has no column
  // the chunk's keys in lanes 0 .. 31, the neighbours' in lanes 32 and 33
  uint32_t k = 0xFFFFFFFFu, ps = 0;
  if (lane < count) k = a.key[first + lane], ps = a.pos[first + lane];
  if (lane == 32 && first > 0) k = a.key[first - 1];
  if (lane == 33 && first + count < a.n) k = a.key[first + count];
  const uint32_t prev = __builtin_amdgcn_readlane(k, 32), next = __builtin_amdgcn_readlane(k, 33);
  const T* dy = static_cast<const T*>(a.dy);
  float acc[W];
#pragma unroll
  for (int e = 0; e < W; ++e) acc[e] = 0.0f;
  bool came_in = __builtin_amdgcn_readlane(k, 0) == prev;
  for (int base = 0; base < count; base += 8) {
    Pix8 q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = base + i;
      const uint32_t id = at < count ? __builtin_amdgcn_readlane(k, at) : 0xFFFFFFFFu;
      q[i] = {{0u, 0u, 0u, 0u}};
      if (id < uint32_t(a.vocab) && width > 0)
        q[i] = window<T>(dy + int64_t(__builtin_amdgcn_readlane(ps, at)) * a.ld + col, width);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = base + i;
      if (at >= count) break;
      const uint32_t id = __builtin_amdgcn_readlane(k, at);
      if (id >= uint32_t(a.vocab)) return;  // the rest of the order has no gradient
      float v[W];
      unpack<T>(q[i], v);
#pragma unroll
      for (int e = 0; e < W; ++e) acc[e] += v[e];
      const uint32_t after = at + 1 < count ? __builtin_amdgcn_readlane(k, at + 1) : next;
      const bool ends = at + 1 < count || first + count < a.n ? after != id : true;
      if (!ends && at + 1 < count) continue;
      if (width > 0) {
        if (ends && !came_in) {
#pragma unroll
          for (int e = 0; e < W; ++e) v[e] = acc[e] * a.scale;
          put_window<T>(static_cast<T*>(a.dw) + int64_t(id) * a.dim + col, v, width);
        } else {
          float* to = a.part + (int64_t(chunk) * 2 + (came_in ? 0 : 1)) * a.dim + col;
#pragma unroll
          for (int e = 0; e < W; ++e)
            if (e < width) to[e] = acc[e];
        }
      }
#pragma unroll
      for (int e = 0; e < W; ++e) acc[e] = 0.0f;
      came_in = false;
    }
  }
}

// Joins the runs that cross chunks: the wave of the chunk where a run begins.
template <typename T>
__global__ __launch_bounds__(256) void sum_join_kernel(SumArgs a) {
  constexpr int W = EW<T>::n;
  const int lane = threadIdx.x & 63;
  const int64_t item = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (item >= int64_t(a.chunks - 1) * a.slices) return;
  const int chunk = __builtin_amdgcn_readfirstlane(int(item / a.slices));
  const int slice = __builtin_amdgcn_readfirstlane(int(item - int64_t(chunk) * a.slices));
  const int last = (chunk + 1) * kChunk - 1;  // chunk + 1 exists: position last + 1 does
  const uint32_t id = a.key[last];
  if (id >= uint32_t(a.vocab) || a.key[last + 1] != id) return;
  const int first = chunk * kChunk;
  if (a.key[first] == id && first > 0 && a.key[first - 1] == id) return;  // it began earlier
  // chunks after this one that the run reaches: chunk + 1, and further while the last position
  // of a chunk and the first of the next still hold id
  int reach = 1;
  for (;;) {
    const int64_t c = int64_t(chunk) + reach + lane;  // does the run go on past chunk c?
    const int64_t at = (c + 1) * kChunk;
    const bool on = at < a.n && a.key[at] == id;
    const uint64_t stop = ~__ballot(on);
    if (stop) {
      reach += __ffsll(static_cast<unsigned long long>(stop)) - 1;
      break;
    }
    reach += 64;
  }
  const int col = (slice * 64 + lane) * W;
  const int width = a.dim - col;
  if (width <= 0) return;
  float acc[W];
  const float* from = a.part + (int64_t(chunk) * 2 + 1) * a.dim + col;
#pragma unroll
  for (int e = 0; e < W; ++e) acc[e] = e < width ? from[e] : 0.0f;
#pragma unroll 8
  for (int j = 1; j <= reach; ++j) {
    const float* p = a.part + int64_t(chunk + j) * 2 * a.dim + col;
#pragma unroll
    for (int e = 0; e < W; ++e) acc[e] += e < width ? p[e] : 0.0f;
  }
#pragma unroll
  for (int e = 0; e < W; ++e) acc[e] *= a.scale;
  put_window<T>(static_cast<T*>(a.dw) + int64_t(id) * a.dim + col, acc, width);
}

// ---- workspace: sorted keys and positions (twice where passes go between buffers), block
// counts, partials -----------------------------------------------------------------------------

int64_t up16(int64_t b) { return (b + 15) & ~int64_t(15); }

struct GradPlan {
  int bits, passes, pass_bits, blocks, chunks;
  int64_t keys, hist, part, total;  // byte sizes and the total
};

GradPlan grad_plan(int64_t tokens, int64_t vocab, int64_t dim) {
  GradPlan p;
  p.bits = 1;
  while ((int64_t(1) << p.bits) <= vocab) ++p.bits;  // keys 0 .. vocab
  p.passes = int(ceil_div(p.bits, kDigitBits));
  p.pass_bits = int(ceil_div(p.bits, p.passes));
  p.blocks = int(ceil_div(tokens, int64_t(kSortItems)));
  p.chunks = int(ceil_div(tokens, int64_t(kChunk)));
  p.keys = up16(tokens * 4);
  p.hist = p.blocks > 1 ? up16(int64_t(p.blocks) * kDigits * 4) : 0;
  p.part = up16(int64_t(p.chunks) * 2 * dim * 4);
  p.total = p.keys * (p.blocks > 1 ? 4 : 2) + p.hist + p.part;
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
  if (s.chunks > 1)
    sum_join_kernel<T><<<unsigned(ceil_div(int64_t(s.chunks - 1) * s.slices, int64_t(4))), 256, 0, st>>>(s);
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
  if (!d_weight || (tokens > 0 && (!ids || !grad))) return refuse(what, "null operand");
  if ((reinterpret_cast<uintptr_t>(d_weight) & 15) || off_element(grad, dtype)) return refuse(what, "misaligned operand");
  const GradPlan p = grad_plan(std::max<int64_t>(tokens, 1), vocab, dim);
  if (tokens > 0 && (!workspace || workspace_bytes < size_t(p.total) || (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return refuse(what, "workspace missing, misaligned or too small");
  static const bool lds_ok = hipFuncSetAttribute(reinterpret_cast<const void*>(&sort_small_kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, int(kSortLds)) == hipSuccess;
  if (!lds_ok) return refuse(what, "cannot enable the sort's LDS size");
  if (!admit_launch(what)) return -1;
  hipStream_t st = as_stream(stream);
  SortArgs s = {};
  s.ids = ids;
  s.index_bytes = index_bytes;
  s.n = int(tokens);
  s.vocab = int(vocab);
  s.padding = padding;
  s.fill = static_cast<uint4*>(d_weight);
  s.fill_bytes = vocab * dim * (dtype == 1 ? 4 : 2);
  // 32 KB of zeros per filling workgroup and round
  const unsigned fillers = unsigned(std::max<int64_t>(1, std::min<int64_t>(ceil_div(s.fill_bytes, int64_t(32768)), 1024)));
  if (tokens == 0) {  // nothing to sort: workgroup 0 of the counting kernel fills as well
    sort_count_kernel<<<fillers, kSortThreads, 0, st>>>(s);
    return check_launch(what);
  }
  char* ws = static_cast<char*>(workspace);
  uint32_t* buf[4];  // key, position, and the other side of the passes
  for (int i = 0; i < (p.blocks > 1 ? 4 : 2); ++i, ws += p.keys) buf[i] = reinterpret_cast<uint32_t*>(ws);
  s.hist = reinterpret_cast<uint32_t*>(ws);
  ws += p.hist;
  int side = 0;
  if (p.blocks == 1) {
    s.passes = p.passes;
    s.pass_bits = p.pass_bits;
    s.key = buf[0];
    s.pos = buf[1];
    sort_small_kernel<<<1 + fillers, kSortThreads, kSortLds, st>>>(s);
  } else {
    s.blocks = p.blocks;
    for (int i = 0; i < p.passes; ++i) {
      s.shift = i * p.pass_bits;
      s.bits = p.pass_bits;
      s.key_in = i ? buf[side] : nullptr;
      s.pos_in = i ? buf[side + 1] : nullptr;
      side = i ? 2 - side : 0;
      s.key = buf[side];
      s.pos = buf[side + 1];
      sort_count_kernel<<<unsigned(p.blocks) + (i ? 0 : fillers), kSortThreads, 0, st>>>(s);
      sort_scatter_kernel<<<unsigned(p.blocks), kSortThreads, 0, st>>>(s);
    }
  }
  SumArgs m = {};
  m.key = buf[side];
  m.pos = buf[side + 1];
  m.n = int(tokens);
  m.vocab = int(vocab);
  m.dim = int(dim);
  m.slices = int(ceil_div(dim, int64_t(64) * (dtype == 1 ? 4 : 8)));
  m.chunks = p.chunks;
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
