// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   fwd: y[n] = scale * W[id[n]]                       (rows of D values)
//   bwd: dW[v] = scale * sum_{n: id[n] = v} dy[n]      (zeros where no n)
//
// Both are bound by memory: N*D values read and written forward, N*D read
// and V*D written backward. The backward pass never adds with atomics, so it
// gives the same bits each time: the tokens are sorted by (id, position) and
// each id's rows are then summed in the order of their positions.
#include <algorithm>

#include "kernels.h"
#include "lm_util.h"

namespace axon {

namespace {

using namespace lm;

constexpr int kThreads = 256;

// ------------------------------------------------------------------ forward
//
// A group of `lanes` lanes copies up to kFwdVecs 16-byte vectors of one row;
// wide rows are spread over gridDim.y. 32768 rows of 4096 bf16 from a table
// of 128256, 12549 of them different as in a text: 79 us, 4.7 TB/s (91 us right
// behind a gradient, whose last zeros still go to memory then); 8 rows of 2048: 2.3 us, the latency of two
// dependent loads and a store. An id outside [0, V) gives a row of
// NaN: the kernel reads nothing for it, and the caller sees it in the loss.

constexpr int kFwdVecs = 4;

template <typename T, typename I>
__global__ __launch_bounds__(kThreads) void embed_fwd_kernel(
    const I* __restrict__ ids, const T* __restrict__ w, T* __restrict__ y,
    int64_t n, int64_t vocab, int64_t dim, int64_t wstride, float scale,
    int lanes) {
  constexpr int V = kVec<T>;
  const int64_t row =
      static_cast<int64_t>(blockIdx.x) * (kThreads / lanes) +
      threadIdx.x / lanes;
  if (row >= n) return;
  const int64_t c0 =
      (static_cast<int64_t>(blockIdx.y) * kFwdVecs * lanes +
       threadIdx.x % lanes) * V;
  const int64_t id = static_cast<int64_t>(ids[row]);
  const bool known = id >= 0 && id < vocab;
  const T* src = w + (known ? id * wstride : 0);
  T* dst = y + row * dim;
  const float s = known ? scale : __builtin_nanf("");
  u32x4 r[kFwdVecs];
#pragma unroll
  for (int k = 0; k < kFwdVecs; ++k) {
    const int64_t c = c0 + static_cast<int64_t>(k) * lanes * V;
    if (c + V <= dim) r[k] = known ? load16(src + c) : u32x4{0, 0, 0, 0};
  }
#pragma unroll
  for (int k = 0; k < kFwdVecs; ++k) {
    const int64_t c = c0 + static_cast<int64_t>(k) * lanes * V;
    if (c + V <= dim) {
      float f[V];
      unpack<T>(r[k], f);
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] *= s;
      store16(dst + c, pack<T>(f));
    } else {
      for (int64_t i = c; i < dim; ++i)
        dst[i] = static_cast<T>((known ? static_cast<float>(src[i]) : 0.f) * s);
    }
  }
}

// ----------------------------------------------------------- sorting tokens
//
// A key is id << 32 | position: keys differ from each other, so any way of
// sorting them gives one order. Ids that take no part (padding, or outside
// [0, V)) get the id V and end up behind all others.
//
// Within tiles a key's place is counted: the smaller ids in the tile, and the
// equal ones before it. All pairs are compared, a tile's length for each
// token, but over the whole chip and without a barrier in between: a bitonic
// sort of 2048 keys by one block took 15 us, the count takes 5. (A tile of
// 8192 would save their merge, but took 22 us instead of 9 and 7.)
//
// Then runs are merged, up to kMergeRuns at a time: a key's place in the
// merged run is its place in its own run plus the number of smaller keys in
// each of the others. One merge does for up to 32768 tokens, two for up to
// 524288.

constexpr int kTile = 2048;
constexpr int kRankThreads = 1024;
constexpr int kRankKeys = 64;  // keys that a block places, one for each lane
constexpr int kMergeRuns = 16;

// dW is filled with zeros by further blocks of the sorting launches, which
// leave memory idle; each writes kFillUnits units of 16 bytes. (1.05 GB of
// zeros and the keys of 32768 tokens: 82 + 96 us, 5.9 TB/s; the keys alone take
// 11 + 7.)
constexpr int kFillUnits = 4096;

struct Fill {
  u32x4* at;
  int64_t units;
  __host__ __device__ int64_t blocks() const {
    return (units + kFillUnits - 1) / kFillUnits;
  }
};

// Of the launch's blocks, every second one fills until the others (or the
// fill) run out: blocks start in order, and either kind alone would take all
// CUs first. Returns this block's number among its kind; *fills says which.
__device__ __forceinline__ int64_t kind_of(int64_t block, int64_t others,
                                           int64_t fills_in_all,
                                           bool* fills) {
  const int64_t pairs = min(others, fills_in_all);
  if (block < 2 * pairs) {
    *fills = block & 1;
    return block >> 1;
  }
  *fills = fills_in_all > others;
  return block - pairs;
}

template <int kBlock>
__device__ __forceinline__ void fill(const Fill& f, int64_t block) {
  const int64_t begin = block * kFillUnits + threadIdx.x;
#pragma unroll
  for (int k = 0; k < kFillUnits / kBlock; ++k)
    if (begin + k * kBlock < f.units)
      f.at[begin + k * kBlock] = u32x4{0, 0, 0, 0};
}

template <typename I>
__global__ __launch_bounds__(kRankThreads) void embed_rank_kernel(
    const I* __restrict__ ids, uint64_t* __restrict__ keys, int64_t n,
    int64_t vocab, int64_t padding, int64_t blocks, Fill f) {
  bool fills;
  const int64_t block = kind_of(blockIdx.x, blocks, f.blocks(), &fills);
  if (fills) {
    fill<kRankThreads>(f, block);
    return;
  }
  constexpr int kWaves = kRankThreads / 64;
  constexpr int kPart = kTile / kWaves;  // keys that a wave compares with
  __shared__ alignas(16) uint32_t s[kTile];
  __shared__ int counts[kWaves][kRankKeys];
  const int64_t first = block * kRankKeys;
  const int64_t base = first / kTile * kTile;
  const int len = static_cast<int>(min<int64_t>(kTile, n - base));
  for (int i = threadIdx.x; i < kTile; i += kRankThreads) {
    uint32_t key = ~0u;  // never smaller than another
    if (i < len) {
      const int64_t id = static_cast<int64_t>(ids[base + i]);
      key = static_cast<uint32_t>(
          id >= 0 && id < vocab && id != padding ? id : vocab);
    }
    s[i] = key;
  }
  __syncthreads();
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int mine = static_cast<int>(first - base) + lane;
  const uint32_t key = s[mine];
  int count = 0;
  const int from = wave * kPart, to = min(from + kPart, len);
  const int own = static_cast<int>(first - base);
  // An equal id counts if it stands before: k <= key is k < key + 1. Waves
  // whose keys all stand on one side of the block's own need no comparison
  // of positions.
  const bool mixed = from < own + kRankKeys && from + kPart > own;
  const uint32_t bound = key + (from < own ? 1 : 0);
  if (!mixed) {
#pragma unroll 4
    for (int j = from; j < to; j += 4) {
      const u32x4 k = *reinterpret_cast<const u32x4*>(&s[j]);
#pragma unroll
      for (int e = 0; e < 4; ++e) count += k[e] < bound;
    }
  } else {
#pragma unroll 4
    for (int j = from; j < to; j += 4) {
      const u32x4 k = *reinterpret_cast<const u32x4*>(&s[j]);
#pragma unroll
      for (int e = 0; e < 4; ++e) count += k[e] < key + (j + e < mine ? 1 : 0);
    }
  }
  counts[wave][lane] = count;
  __syncthreads();
  if (wave == 0 && mine < len) {
    int place = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) place += counts[w][lane];
    keys[base + place] = static_cast<uint64_t>(key) << 32 |
                         static_cast<uint32_t>(base + mine);
  }
}

// Keys below `key` in the sorted run p[0..n).
__device__ __forceinline__ int64_t count_below(const uint64_t* p, int64_t n,
                                               uint64_t key) {
  int64_t lo = 0, hi = n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (p[mid] < key)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo;
}

// A block places 64 keys, which stand next to each other in one run: wave r
// bisects run r for all of them, along nearly the same path, so that its loads
// touch few lines (32768 tokens 7 us; with a lane for each run 12).
__global__ __launch_bounds__(kMergeRuns * 64) void embed_merge_kernel(
    const uint64_t* __restrict__ in, uint64_t* __restrict__ out, int64_t n,
    int64_t run, int64_t blocks, Fill f) {
  bool fills;
  const int64_t block = kind_of(blockIdx.x, blocks, f.blocks(), &fills);
  if (fills) {
    fill<kMergeRuns * 64>(f, block);
    return;
  }
  __shared__ int64_t places[kMergeRuns][64];
  const int r = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t i = block * 64 + lane;
  const int64_t at = min(i, n - 1);
  const uint64_t key = in[at];
  const int64_t group = at / (run * kMergeRuns) * (run * kMergeRuns);
  const int64_t mine = at / run * run;
  const int64_t start = group + r * run;
  places[r][lane] =
      start == mine ? group + (at - mine)
      : start < n   ? count_below(in + start, min(run, n - start), key)
                    : 0;
  __syncthreads();
  if (r == 0 && i < n) {
    int64_t place = 0;
#pragma unroll
    for (int w = 0; w < kMergeRuns; ++w) place += places[w][lane];
    out[place] = key;
  }
}

// ------------------------------------------------------------ summing rows
//
// The sorted positions are cut into chunks of equal length, whatever the
// tokens' frequencies: a wave sums one chunk over one slice of columns and
// writes each id's row when the id changes. Rows of an id that crosses a
// chunk's border go to fp32 partial sums (slot 0: the id came from the chunk
// before; slot 1: it starts here and goes on), which a second kernel joins
// in order.
//
// A chunk has 64 tokens at most: each lane loads one key, and reading them
// from the lanes makes ids and row addresses uniform, so that changes of the
// id are scalar branches and kRowsAhead rows are in flight. The rows of dy are
// read once, past the caches, which are full of dW's zeros: 32768 rows of 4096
// bf16 take 78 us (5.0 TB/s, with the rows of dW) and took 119 through them.

constexpr int kRowsAhead = 8;
constexpr int kMaxChunk = 64;

// kRows: rows are whole 16-byte vectors (kWhole); or their last vector is not
// (kTail), and its lane reads a whole one that ends with the row, of whose
// columns the first kept ones are the lane's before; or they are shorter than
// a vector (kNarrow).
enum { kWhole, kTail, kNarrow };

template <typename T, int kRows>
__global__ __launch_bounds__(kThreads) void embed_sum_kernel(
    const uint64_t* __restrict__ keys, const T* __restrict__ dy,
    T* __restrict__ dw, float* __restrict__ part, int64_t n, int64_t vocab,
    int64_t dim, int chunk, int64_t nchunks, int slices, float scale) {
  constexpr int V = kVec<T>;
  const int lane = threadIdx.x & 63;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * (kThreads / 64) +
                       __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t ci = unit / slices;
  if (ci >= nchunks) return;
  const int64_t column = (unit % slices) * 64 * V + lane * V;
  const bool active = column < dim;
  const int64_t c0 = kRows == kTail ? min(column, dim - V) : column;
  const int kept = kRows == kTail ? static_cast<int>(column - c0) : 0;
  const int width = kRows == kNarrow ? static_cast<int>(dim) : V;
  const int64_t begin = ci * chunk;
  const int len = static_cast<int>(min<int64_t>(chunk, n - begin));

  const uint64_t mine = lane < len ? keys[begin + lane] : ~0ull;
  const uint32_t none = static_cast<uint32_t>(vocab);
  const uint32_t before =
      begin > 0 ? static_cast<uint32_t>(keys[begin - 1] >> 32) : none;
  const uint32_t after = begin + len < n
                             ? static_cast<uint32_t>(keys[begin + len] >> 32)
                             : none;
  auto id_at = [&](int k) {
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(
        static_cast<int>(mine >> 32), k));
  };
  auto row_at = [&](int k) {
    return static_cast<uint32_t>(
        __builtin_amdgcn_readlane(static_cast<int>(mine), k));
  };

  float acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
  uint32_t cur = id_at(0);
  bool first = before == cur;

  auto flush = [&](bool goes_on) {
    if (cur == none || !active) return;
    if (first || goes_on) {
      float* p = part + (ci * 2 + (first ? 0 : 1)) * dim + c0;
      if (kRows == kWhole || (kRows == kTail && kept == 0)) {
#pragma unroll
        for (int i = 0; i < V; i += 4) store16(p + i, pack<float>(acc + i));
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (i >= kept && i < width) p[i] = acc[i];
      }
    } else {
      T* p = dw + static_cast<int64_t>(cur) * dim + c0;
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] *= scale;
      if (kRows == kWhole || (kRows == kTail && kept == 0)) {
        store16(p, pack<T>(acc));
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (i >= kept && i < width) p[i] = static_cast<T>(acc[i]);
      }
    }
  };

  for (int p0 = 0; p0 < len; p0 += kRowsAhead) {
    u32x4 r[kRowsAhead];
#pragma unroll
    for (int k = 0; k < kRowsAhead; ++k) {
      r[k] = u32x4{0, 0, 0, 0};
      if (p0 + k < len && id_at(p0 + k) != none) {
        const T* src = dy + static_cast<int64_t>(row_at(p0 + k)) * dim + c0;
        if (kRows != kNarrow) {
          if (active) r[k] = load16_once(src);
        } else if (active) {
          T t[V] = {};
#pragma unroll
          for (int i = 0; i < V; ++i)
            if (i < width) t[i] = src[i];
          __builtin_memcpy(&r[k], t, 16);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kRowsAhead; ++k) {
      if (p0 + k < len) {
        const uint32_t id = id_at(p0 + k);
        if (id != cur) {
          flush(false);
          first = false;
          cur = id;
#pragma unroll
          for (int i = 0; i < V; ++i) acc[i] = 0.f;
        }
        float f[V];
        unpack<T>(r[k], f);
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] += f[i];
      }
    }
  }
  flush(after == cur);
}

// One block joins one chunk's slot 1 with the slots 0 behind it, if an id
// starts in that chunk and goes on: wave w of kJoinWaves takes chunks w,
// w + kJoinWaves, ..., kJoinAhead of them at a time, and the waves' sums are
// added in order. Where the id ends is seen from the first keys of the next 64
// chunks, one for each lane, and found by bisection only behind those. (8192
// tokens of one id, 512 chunks, 1024 columns: 142 us with 4 waves that wait
// for each chunk.)
constexpr int kJoinCols = 4;  // columns of a lane
constexpr int kJoinWaves = 8;
constexpr int kJoinAhead = 8;

template <typename T>
__global__ __launch_bounds__(kJoinWaves * 64) void embed_join_kernel(
    const uint64_t* __restrict__ keys, const float* __restrict__ part,
    T* __restrict__ dw, int64_t n, int64_t vocab, int64_t dim, int chunk,
    float scale) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t ci = blockIdx.x;
  const int64_t begin = ci * chunk, end = begin + chunk;
  if (end >= n) return;
  const int64_t at = min(end + static_cast<int64_t>(lane) * chunk, n - 1);
  const uint32_t next = static_cast<uint32_t>(keys[at] >> 32);
  const uint32_t id = __builtin_amdgcn_readfirstlane(next);
  const uint32_t before = static_cast<uint32_t>(keys[end - 1] >> 32);
  const uint32_t earlier =
      static_cast<uint32_t>(keys[begin > 0 ? begin - 1 : 0] >> 32);
  // Does it start here? Else an earlier chunk joins it.
  if (id >= vocab || before != id || (begin > 0 && earlier == id)) return;
  // Chunk ci + l is reached if its first key has the id.
  const uint64_t on =
      __ballot(next == id && end + static_cast<int64_t>(lane) * chunk < n);
  int64_t last = ci + __builtin_ctzll(~on | (1ull << 63));
  if (on == ~0ull) {
    const uint64_t after = (static_cast<uint64_t>(id) + 1) << 32;
    last = (end + count_below(keys + end, n - end, after) - 1) / chunk;
  }
  __shared__ float s[kJoinWaves][kJoinCols][64];
  const int64_t c0 = static_cast<int64_t>(blockIdx.y) * 64 * kJoinCols + lane;
  float acc[kJoinCols] = {};
  for (int64_t k = ci + wave; k <= last; k += kJoinWaves * kJoinAhead) {
    float v[kJoinAhead][kJoinCols];
#pragma unroll
    for (int a = 0; a < kJoinAhead; ++a) {
      const int64_t from = k + a * kJoinWaves;
      const float* p = part + (from * 2 + (from == ci ? 1 : 0)) * dim;
#pragma unroll
      for (int i = 0; i < kJoinCols; ++i) {
        v[a][i] = 0.f;
        if (from <= last && c0 + i * 64 < dim) v[a][i] = p[c0 + i * 64];
      }
    }
#pragma unroll
    for (int a = 0; a < kJoinAhead; ++a)
#pragma unroll
      for (int i = 0; i < kJoinCols; ++i) acc[i] += v[a][i];
  }
#pragma unroll
  for (int i = 0; i < kJoinCols; ++i) s[wave][i][lane] = acc[i];
  __syncthreads();
  // Wave w finishes column w of each lane.
  const int64_t c = c0 + wave * 64;
  if (wave < kJoinCols && c < dim) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) sum += s[w][wave][lane];
    dw[id * dim + c] = static_cast<T>(sum * scale);
  }
}
static_assert(kJoinCols <= kJoinWaves, "a wave for each column");

struct SumPlan {
  int chunk;
  int64_t nchunks;
  int slices;
};

// Chunks are as long as still leaves about 1024 waves (one for each SIMD), and
// 8 to 64 tokens. Shorter ones leave the sums' time as it is and make more
// rows to join: for 8192 tokens of 1024 bf16 values, chunks of 8, 16 and 32
// took 7.6 + 14.3, 8.4 + 8.1 and 11.8 + 5.7 us (sums + join).
SumPlan sum_plan(int64_t n, int64_t dim, int vec) {
  SumPlan p;
  p.slices = static_cast<int>((dim + 64 * vec - 1) / (64 * vec));
  p.chunk = 8;
  while (p.chunk < kMaxChunk && n / p.chunk * p.slices > 1024) p.chunk *= 2;
  p.nchunks = (n + p.chunk - 1) / p.chunk;
  return p;
}

template <typename T, typename I>
void bwd(const I* ids, const T* dy, T* dw, uint64_t* keys, float* part,
         int64_t n, int64_t vocab, int64_t dim, int64_t padding, float scale,
         hipStream_t stream) {
  // The allocation of dw is rounded up to 16 bytes for the fill.
  int64_t left = (vocab * dim * static_cast<int64_t>(sizeof(T)) + 15) / 16;
  int passes = 1;
  for (int64_t run = kTile; run < n; run *= kMergeRuns) ++passes;
  u32x4* at = reinterpret_cast<u32x4*>(dw);
  auto next_fill = [&] {  // an equal share for each launch that is left
    const int64_t blocks =
        (left + kFillUnits * passes - 1) / (kFillUnits * passes);
    const Fill f = {at, std::min(left, blocks * kFillUnits)};
    at += f.units;
    left -= f.units;
    --passes;
    return f;
  };
  const int64_t ranks = (n + kRankKeys - 1) / kRankKeys;
  Fill f = next_fill();
  hipLaunchKernelGGL(embed_rank_kernel<I>,
                     dim3(static_cast<unsigned>(ranks + f.blocks())),
                     dim3(kRankThreads), 0, stream, ids, keys, n, vocab,
                     padding, ranks, f);
  if (n == 0) return;
  uint64_t* other = keys + n;
  for (int64_t run = kTile; run < n; run *= kMergeRuns) {
    f = next_fill();
    const int64_t blocks = (n + 63) / 64;
    hipLaunchKernelGGL(embed_merge_kernel,
                       dim3(static_cast<unsigned>(blocks + f.blocks())),
                       dim3(kMergeRuns * 64), 0, stream, keys, other, n, run, blocks,
                       f);
    std::swap(keys, other);
  }
  const SumPlan p = sum_plan(n, dim, kVec<T>);
  const int64_t units = p.nchunks * p.slices;
  auto* sum = dim % kVec<T> == 0 ? &embed_sum_kernel<T, kWhole>
              : dim > kVec<T>   ? &embed_sum_kernel<T, kTail>
                                : &embed_sum_kernel<T, kNarrow>;
  hipLaunchKernelGGL(sum, dim3(static_cast<unsigned>((units + 3) / 4)),
                     dim3(kThreads), 0, stream, keys, dy, dw, part, n, vocab,
                     dim, p.chunk, p.nchunks, p.slices, scale);
  if (p.nchunks > 1)
    hipLaunchKernelGGL(embed_join_kernel<T>,
                       dim3(static_cast<unsigned>(p.nchunks - 1),
                            static_cast<unsigned>((dim + 64 * kJoinCols - 1) /
                                                 (64 * kJoinCols))),
                       dim3(kJoinWaves * 64), 0, stream, keys, part, dw, n,
                       vocab, dim, p.chunk, scale);
}

template <typename T, typename I>
void fwd(const I* ids, const T* w, T* y, int64_t n, int64_t vocab, int64_t dim,
         int64_t wstride, float scale, hipStream_t stream) {
  int lanes = 1;
  while (lanes < 64 && lanes * kVec<T> < dim) lanes *= 2;
  const int rows = kThreads / lanes;
  const int64_t cols = static_cast<int64_t>(lanes) * kVec<T> * kFwdVecs;
  hipLaunchKernelGGL((embed_fwd_kernel<T, I>),
                     dim3(static_cast<unsigned>((n + rows - 1) / rows),
                          static_cast<unsigned>((dim + cols - 1) / cols)),
                     dim3(kThreads), 0, stream, ids, w, y, n, vocab, dim,
                     wstride, scale, lanes);
}

}  // namespace

int64_t embed_part_floats(int64_t n, int64_t dim, int elem_size) {
  const SumPlan p = sum_plan(n, dim, 16 / elem_size);
  return p.nchunks * 2 * dim;
}

void launch_embed_fwd(int dtype, bool ids64, const void* ids, const void* w,
                      void* y, int64_t n, int64_t vocab, int64_t dim,
                      int64_t wstride, float scale, hipStream_t stream) {
  auto go = [&](auto t) {
    using T = decltype(t);
    if (ids64)
      fwd(static_cast<const int64_t*>(ids), static_cast<const T*>(w),
          static_cast<T*>(y), n, vocab, dim, wstride, scale, stream);
    else
      fwd(static_cast<const int32_t*>(ids), static_cast<const T*>(w),
          static_cast<T*>(y), n, vocab, dim, wstride, scale, stream);
  };
  if (dtype == kFloat) go(float{});
  if (dtype == kHalf) go(_Float16{});
  if (dtype == kBF16) go(__bf16{});
}

void launch_embed_bwd(int dtype, bool ids64, const void* ids, const void* dy,
                      void* dw, uint64_t* keys, float* part, int64_t n,
                      int64_t vocab, int64_t dim, int64_t padding, float scale,
                      hipStream_t stream) {
  auto go = [&](auto t) {
    using T = decltype(t);
    if (ids64)
      bwd(static_cast<const int64_t*>(ids), static_cast<const T*>(dy),
          static_cast<T*>(dw), keys, part, n, vocab, dim, padding, scale,
          stream);
    else
      bwd(static_cast<const int32_t*>(ids), static_cast<const T*>(dy),
          static_cast<T*>(dw), keys, part, n, vocab, dim, padding, scale,
          stream);
  };
  if (dtype == kFloat) go(float{});
  if (dtype == kHalf) go(_Float16{});
  if (dtype == kBF16) go(__bf16{});
}

}  // namespace axon
