// Cross entropy over the last dimension, with the logits' gradient.
//
//   m = max_j x_j,  S = sum_j exp(x_j - m)
//   loss = (1 - e) (ln S + m - x_t) + e (ln S + m - mean_j x_j)
//   dx_j = g (exp(x_j - m) / S - (1 - e) [j = t] - e / V)
//
// for a row of V logits with label t and label smoothing e. Bound by memory:
// the forward pass reads the logits once (running maximum and sum, in fp32),
// the backward pass reads them again and writes the gradient; nothing of the
// logits' size is kept between. Rows whose label is ignored are not read, and
// their gradient is zeros.
#include <algorithm>
#include <type_traits>

#include "kernels.h"
#include "lm_util.h"

namespace axon {

namespace {

using namespace lm;

constexpr int kThreads = 256;
// Below every finite value's exponent range that matters: exp(x - kLowest) is
// 0 for x = -inf, and no (-inf) - (-inf) occurs in the running sums.
constexpr float kLowest = -3.402823466e+38f;
constexpr float kLog2e = 1.44269504088896340736f;

// exp by the hardware's exp2 (1 ulp; 0 below 2^-126), on a difference that is
// exact for the values that matter in a sum.
__device__ __forceinline__ float exp_of(float d) {
  return __builtin_amdgcn_exp2f(d * kLog2e);
}

// Running maximum, sum of exp(x - max), and (for smoothing) sum of x times
// down(V): a few classes masked by fp32's lowest value would take their plain
// sum past its range.
struct Stat {
  float m, s, x;
};

// The power of two in [1 / 4V, 1 / 2V]: exact as a factor.
__host__ __device__ __forceinline__ float down(int64_t vocab) {
  float d = 0.5f;
  for (; vocab > 1; vocab = (vocab + 1) / 2) d *= 0.5f;
  return d;
}

__device__ __forceinline__ Stat join(Stat a, Stat b) {
  const float m = fmaxf(a.m, b.m);
  return {m, a.s * exp_of(a.m - m) + b.s * exp_of(b.m - m), a.x + b.x};
}

// Values before the next border of a 128-byte line, which a group handles one
// by one, so that its vectors lie on such borders: rows of an odd length
// start anywhere. (32768 rows of 30522 bf16, both passes past the caches: 1241
// us with vectors from each row's start, 1021 with this.)
template <typename T>
__device__ __forceinline__ int head_of(const T* p, int len) {
  const uintptr_t past = reinterpret_cast<uintptr_t>(p) & 127;
  return min(len, static_cast<int>(((128 - past) & 127) / sizeof(T)));
}

template <bool kOnce, typename T>
__device__ __forceinline__ u32x4 load(const T* p) {
  return kOnce ? load16_once(p) : load16(p);
}
template <bool kOnce, typename T>
__device__ __forceinline__ void store(T* p, u32x4 r) {
  if (kOnce)
    store16_once(p, r);
  else
    store16(p, r);
}

// Row r of logits [outer, inner, V] with strides; labels are dense.
struct Rows {
  int64_t inner, stride_outer, stride_inner;
  __device__ __forceinline__ int64_t at(int64_t r) const {
    return r / inner * stride_outer + r % inner * stride_inner;
  }
};

// What a row's statistics and its label's logit make of it: (m, 1/S) for the
// backward pass, and the loss.
__device__ __forceinline__ float row_loss(Stat st, float xt, bool known,
                                          int64_t vocab, float eps) {
  if (!known) return __builtin_nanf("");
  const float ln_s = logf(st.s);
  float loss = (ln_s + (st.m - xt)) * (1.f - eps);
  if (eps > 0.f) {
    // In 64 bits: the mean may be a rounding past fp32's range.
    const double mean = st.x / (static_cast<double>(down(vocab)) * vocab);
    loss = static_cast<float>(loss + (ln_s + (st.m - mean)) * eps);
  }
  return loss;
}

// A group of G threads reads one segment of one row; where rows are not cut
// (kWhole) it finishes the row as well. 8192 rows of 128256 bf16 in 311 us,
// 6.8 TB/s: memory, and nearly arithmetic as well (an exp2 at a quarter of the
// rate and 5 other instructions for a value, 240 us). So the running maximum
// is moved once for each vector, which costs an exp2 more for 4 or 8 values.
template <typename T, int G, bool kSmooth, bool kWhole>
__global__ __launch_bounds__(kThreads) void ce_stat_kernel(
    const T* __restrict__ x, Rows rows, const int64_t* __restrict__ target,
    int64_t ignore, int64_t n, int64_t vocab, int64_t seg_len, int segs,
    int64_t once_rows, float small, float eps, float unlabelled,
    Stat* __restrict__ stat, float2* __restrict__ kept,
    float* __restrict__ losses) {
  constexpr int V = kVec<T>;
  constexpr int kAhead = 4;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * (kThreads / G) +
                       threadIdx.x / G;
  const int64_t row = kWhole ? unit : unit / segs;
  const int64_t label = row < n ? target[row] : ignore;
  const bool reads = label != ignore;
  const int t = threadIdx.x % G;
  if (kWhole && !reads && t == 0 && row < n) losses[row] = unlabelled;
  if (G == kThreads && !reads) return;
  const bool known = label >= 0 && label < vocab;
  Stat st = {kLowest, 0.f, 0.f};
  float xt = 0.f;
  if (reads) {
    const int64_t begin = kWhole ? 0 : unit % segs * seg_len;
    const int len = static_cast<int>(kWhole ? vocab
                                            : min(seg_len, vocab - begin));
    const T* p = x + rows.at(row) + begin;
    if (kWhole && known) xt = static_cast<float>(p[label]);
    auto take_one = [&](float f) {
      const float m = fmaxf(st.m, f);
      st.s = st.s * exp_of(st.m - m) + exp_of(f - m);
      if (kSmooth) st.x = fmaf(f, small, st.x);
      st.m = m;
    };
    auto take = [&](u32x4 r) {
      float f[V];
      unpack<T>(r, f);
      float m = st.m;
#pragma unroll
      for (int q = 0; q < V; ++q) m = fmaxf(m, f[q]);
      float s = st.s * exp_of(st.m - m);
#pragma unroll
      for (int q = 0; q < V; ++q) {
        s += exp_of(f[q] - m);
        if (kSmooth) st.x = fmaf(f[q], small, st.x);
      }
      st.m = m;
      st.s = s;
    };
    const int head = head_of(p, len);
    for (int j = t; j < head; j += G) take_one(static_cast<float>(p[j]));
    const T* body = p + head;
    const int full = (len - head) / V;
    auto vectors = [&](auto once) {
      constexpr bool kOnce = decltype(once)::value;
      int i = t;
      for (; i + (kAhead - 1) * G < full; i += kAhead * G) {
        u32x4 r[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
          r[k] = load<kOnce>(body + (i + k * G) * V);
#pragma unroll
        for (int k = 0; k < kAhead; ++k) take(r[k]);
      }
      // Up to three are left: loaded together as well.
      u32x4 r[kAhead - 1];
#pragma unroll
      for (int k = 0; k < kAhead - 1; ++k)
        if (i + k * G < full) r[k] = load<kOnce>(body + (i + k * G) * V);
#pragma unroll
      for (int k = 0; k < kAhead - 1; ++k)
        if (i + k * G < full) take(r[k]);
    };
    if (row < once_rows)
      vectors(std::true_type{});
    else
      vectors(std::false_type{});
    for (int j = head + full * V + t; j < len; j += G)
      take_one(static_cast<float>(p[j]));
  }
#pragma unroll
  for (int off = (G < 64 ? G : 64) / 2; off > 0; off >>= 1) {
    Stat o;
    o.m = __shfl_xor(st.m, off, 64);
    o.s = __shfl_xor(st.s, off, 64);
    o.x = kSmooth ? __shfl_xor(st.x, off, 64) : 0.f;
    st = join(st, o);
  }
  if (G > 64) {
    __shared__ Stat lds[kThreads / 64];
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = st;
    __syncthreads();
    if (threadIdx.x == 0)
      for (int w = 1; w < kThreads / 64; ++w) st = join(st, lds[w]);
  }
  if (t != 0 || !reads) return;
  if (kWhole) {
    kept[row] = make_float2(st.m, 1.f / st.s);
    losses[row] = row_loss(st, xt, known, vocab, eps);
  } else {
    stat[unit] = st;
  }
}

// Joins the segments of rows that were cut.
__global__ __launch_bounds__(kThreads) void ce_join_kernel(
    const void* __restrict__ x, int dtype, Rows rows,
    const int64_t* __restrict__ target, int64_t ignore, int64_t n,
    int64_t vocab, int segs, float eps, float unlabelled,
    const Stat* __restrict__ stat, float2* __restrict__ kept,
    float* __restrict__ losses) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (row >= n) return;
  const int64_t t = target[row];
  if (t == ignore) {
    losses[row] = unlabelled;
    return;
  }
  const bool known = t >= 0 && t < vocab;
  const int64_t at = rows.at(row) + (known ? t : 0);
  const float xt =
      dtype == kFloat  ? static_cast<const float*>(x)[at]
      : dtype == kHalf ? static_cast<float>(static_cast<const _Float16*>(x)[at])
                       : static_cast<float>(static_cast<const __bf16*>(x)[at]);
  Stat st = stat[row * segs];
#pragma unroll 4
  for (int k = 1; k < segs; ++k) st = join(st, stat[row * segs + k]);
  kept[row] = make_float2(st.m, 1.f / st.s);
  losses[row] = row_loss(st, xt, known, vocab, eps);
}

// Sums the rows' losses and counts the labels, in 64 bits: one block for up
// to kSumRows rows, else partial sums of that many each and a second launch
// over those (`in`). A row without a label holds kUnlabelled: no loss is
// -inf, since S >= 1 and m >= x_t wherever the loss is a number.
constexpr int kSumThreads = 1024;
constexpr int64_t kSumRows = 16384;
constexpr float kUnlabelled = -__builtin_inff();

__global__ __launch_bounds__(kSumThreads) void ce_sum_kernel(
    const float* __restrict__ losses, int64_t n, const double* __restrict__ in,
    double* __restrict__ out, bool mean, float* __restrict__ loss,
    float* __restrict__ factor) {
  double sum = 0.0, count = 0.0;
  const int64_t begin = static_cast<int64_t>(blockIdx.x) * kSumRows;
  const int64_t end = min(n, begin + kSumRows);
  if (in) {
    for (int64_t i = begin + threadIdx.x; i < end; i += kSumThreads) {
      sum += in[2 * i];
      count += in[2 * i + 1];
    }
  } else {
#pragma unroll 8
    for (int64_t i = begin + threadIdx.x; i < end; i += kSumThreads) {
      const float l = losses[i];
      sum += l == kUnlabelled ? 0.0 : static_cast<double>(l);
      count += l == kUnlabelled ? 0.0 : 1.0;
    }
  }
  __shared__ double lds[2][kSumThreads / 64];
  sum = wave_sum(sum);
  count = wave_sum(count);
  if ((threadIdx.x & 63) == 0) {
    lds[0][threadIdx.x >> 6] = sum;
    lds[1][threadIdx.x >> 6] = count;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  sum = count = 0.0;
  for (int w = 0; w < kSumThreads / 64; ++w) {
    sum += lds[0][w];
    count += lds[1][w];
  }
  if (out) {
    out[2 * blockIdx.x] = sum;
    out[2 * blockIdx.x + 1] = count;
  } else {
    *loss = static_cast<float>(mean ? sum / count : sum);
    *factor = static_cast<float>(mean ? 1.0 / count : 1.0);
  }
}

// The gradient of one segment of one row by a group of G threads: the logits
// again and 1/S, no division. 8192 rows of 128256 bf16 in 773 us, 5.4 TB/s of
// reading and writing (a copy reaches 4.9); 8192 rows of 30522 of which 15 of
// 100 have a label in 114 us, 5.0 TB/s.
template <typename T, int G, bool kOnce>
__global__ __launch_bounds__(kThreads) void ce_grad_kernel(
    const T* __restrict__ x, Rows rows, const int64_t* __restrict__ target,
    int64_t ignore, int64_t n, int64_t vocab, int64_t seg_len, int segs,
    int64_t once_rows, float eps, const float2* __restrict__ kept, const float* __restrict__ gout,
    int gstride, const float* __restrict__ factor, T* __restrict__ dx) {
  constexpr int V = kVec<T>;
  constexpr int kAhead = 4;
  // Last rows first: they are in the cache.
  const int64_t unit =
      static_cast<int64_t>(gridDim.x - 1 - blockIdx.x) * (kThreads / G) +
      threadIdx.x / G;
  const int64_t row = unit / segs;
  if (row >= n) return;
  const int t = threadIdx.x % G;
  const int64_t begin = unit % segs * seg_len;
  const int len = static_cast<int>(min(seg_len, vocab - begin));
  T* q = dx + row * vocab + begin;
  const int head = head_of(q, len);
  const int full = (len - head) / V;
  const int tail = head + full * V;
  T* qbody = q + head;
  const int64_t label = target[row];
  if (label == ignore) {
    const u32x4 zero = {0, 0, 0, 0};
    for (int j = t; j < head; j += G) q[j] = static_cast<T>(0.f);
    for (int i = t; i < full; i += G) store<kOnce>(qbody + i * V, zero);
    for (int j = tail + t; j < len; j += G) q[j] = static_cast<T>(0.f);
    return;
  }
  const T* p = x + rows.at(row) + begin;
  const T* body = p + head;
  float g = gout[row * gstride];
  if (factor) g *= *factor;
  const bool known = label >= 0 && label < vocab;
  if (!known) g = __builtin_nanf("");
  const float2 st = kept[row];
  const float scale = st.y * g;
  const float off = eps > 0.f ? g * eps / static_cast<float>(vocab) : 0.f;
  const float hit = g * (1.f - eps);
  // The label's place in this segment, if it is here.
  const int at = known && label >= begin && label - begin < len
                     ? static_cast<int>(label - begin)
                     : -1;
  auto one = [&](int j) {
    const float v = exp_of(static_cast<float>(p[j]) - st.x) * scale - off;
    q[j] = static_cast<T>(j == at ? v - hit : v);
  };
  auto put = [&](u32x4 r, int i) {
    float f[V];
    unpack<T>(r, f);
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = exp_of(f[e] - st.x) * scale - off;
    const int in = at - head - i * V;
    if (in >= 0 && in < V) {
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = e == in ? f[e] - hit : f[e];
    }
    store<kOnce>(qbody + i * V, pack<T>(f));
  };
  auto vectors = [&](auto once) {
    constexpr bool kReadOnce = decltype(once)::value;
    int i = t;
    for (; i + (kAhead - 1) * G < full; i += kAhead * G) {
      u32x4 r[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        r[k] = load<kReadOnce>(body + (i + k * G) * V);
#pragma unroll
      for (int k = 0; k < kAhead; ++k) put(r[k], i + k * G);
    }
    u32x4 r[kAhead - 1];
#pragma unroll
    for (int k = 0; k < kAhead - 1; ++k)
      if (i + k * G < full) r[k] = load<kReadOnce>(body + (i + k * G) * V);
#pragma unroll
    for (int k = 0; k < kAhead - 1; ++k)
      if (i + k * G < full) put(r[k], i + k * G);
  };
  for (int j = t; j < head; j += G) one(j);
  if (kOnce && row < once_rows)
    vectors(std::true_type{});
  else
    vectors(std::false_type{});
  for (int j = tail + t; j < len; j += G) one(j);
}

// 16 lanes for a row of up to 160 vectors of 16 bytes, a wave for one of up to
// 1024 where there are rows enough for it, a block for a longer one. 65536
// rows of bf16, loss and gradient: of 1100 logits 27 + 51 us by 16 lanes, 40 +
// 63 by waves, 100 + 118 by blocks; of 8000 162 + 369 by waves, 208 + 394 by
// blocks; of 12000 (half as many) 120 + 279 and 125 + 263.
//
// Up to 256 long rows are cut into 512 / n segments, whole numbers of them, of
// 4096 logits or more, and joined by a launch of its own; more rows stay whole.
// 511 rows of 32003 fp16 took 8.4 us whole, 11.3 and 12.7 in 2 and 4 segments;
// 64 rows of 128256 8.1 us in 8 segments, 11.3 in 31. As it is, a call for 64,
// 96, 160 and 256 rows of 128256 bf16 takes 8.9, 9.6, 12.5 and 16.2 us in 8, 5, 3
// and 2 segments, one for 257, 300, 400 and 511 whole rows 18.0, 19.5, 19.4 and
// 21.6.
struct Plan {
  int group;
  int segs;
  int64_t seg_len;
};

constexpr int kFew = 160, kSome = 1024;  // vectors of a row

Plan plan_of(int64_t n, int64_t vocab, int64_t size) {
  const int64_t vectors = vocab * size / 16;
  if (vectors <= kFew) return {16, 1, vocab};
  if (vectors <= kSome && (n >= 2048 || vectors <= 128)) return {64, 1, vocab};
  const int64_t want = std::max<int64_t>(1, 512 / std::max<int64_t>(n, 1));
  const int64_t most = std::max<int64_t>(1, vocab / 4096);
  const int64_t segs = std::min(want, most);
  const int64_t len = ((vocab + segs - 1) / segs + 15) / 16 * 16;
  return {kThreads, static_cast<int>((vocab + len - 1) / len), len};
}

int64_t size_of(int dtype) { return dtype == kFloat ? 4 : 2; }

unsigned blocks_of(const Plan& p, int64_t n) {
  const int per = kThreads / p.group;
  return static_cast<unsigned>((n * p.segs + per - 1) / per);
}

// Rows that go past the caches, in both passes, as all of the gradient does
// then: the chip's last cache (256 MB) keeps the last kKeep bytes of the
// logits from the forward to the backward pass, which takes the rows from the
// last to the first; streaming the others through it would displace them.
// Forward and backward of 4096 x 30528 bf16 (250 MB): all through the caches
// 154 us, all past them 136, kKeep of 64, 128, 192 MB 135, 128, 122; of
// 8192 x 128256 (2.1 GB): 1207, 1140, and 1131, 1125, 1116, 1096 in that order
// of rows. Smaller logits are cached whole.
constexpr int64_t kKeep = int64_t{192} << 20;

int64_t once_rows_of(int64_t n, int64_t vocab, size_t size) {
  return std::max<int64_t>(
      0, n - kKeep / (vocab * static_cast<int64_t>(size)));
}

template <typename T, bool kSmooth>
auto* stat_kernel(const Plan& p) {
  if (p.segs > 1) return &ce_stat_kernel<T, kThreads, kSmooth, false>;
  return p.group == 16   ? &ce_stat_kernel<T, 16, kSmooth, true>
         : p.group == 64 ? &ce_stat_kernel<T, 64, kSmooth, true>
                         : &ce_stat_kernel<T, kThreads, kSmooth, true>;
}

template <typename T>
void stat_pass(const Plan& p, const void* x, Rows rows, const int64_t* target,
               int64_t ignore, int64_t n, int64_t vocab, float eps,
               float unlabelled, Stat* stat, float2* kept, float* losses,
               hipStream_t stream) {
  auto* k = eps > 0.f ? stat_kernel<T, true>(p) : stat_kernel<T, false>(p);
  hipLaunchKernelGGL(k, dim3(blocks_of(p, n)), dim3(kThreads), 0, stream,
                     static_cast<const T*>(x), rows, target, ignore, n, vocab,
                     p.seg_len, p.segs, once_rows_of(n, vocab, sizeof(T)),
                     down(vocab), eps, unlabelled, stat, kept, losses);
}

template <typename T, bool kOnce>
auto* grad_kernel(const Plan& p) {
  return p.group == 16   ? &ce_grad_kernel<T, 16, kOnce>
         : p.group == 64 ? &ce_grad_kernel<T, 64, kOnce>
                         : &ce_grad_kernel<T, kThreads, kOnce>;
}

template <typename T>
void grad_pass(const Plan& p, const void* x, Rows rows, const int64_t* target,
               int64_t ignore, int64_t n, int64_t vocab, float eps,
               const float2* kept, const float* gout, int gstride,
               const float* factor, void* dx, hipStream_t stream) {
  const int64_t once = once_rows_of(n, vocab, sizeof(T));
  auto* k = once ? grad_kernel<T, true>(p) : grad_kernel<T, false>(p);
  hipLaunchKernelGGL(k, dim3(blocks_of(p, n)), dim3(kThreads), 0, stream,
                     static_cast<const T*>(x), rows, target, ignore, n, vocab,
                     p.seg_len, p.segs, once, eps, kept, gout, gstride, factor,
                     static_cast<T*>(dx));
}

int64_t sum_blocks(int64_t n) { return (n + kSumRows - 1) / kSumRows; }

}  // namespace

// A launch takes fewer than 2^32 threads; the second one of ce_sum_kernel
// has one block.
int64_t ce_max_rows(int dtype, int64_t vocab) {
  const int group = plan_of(1 << 20, vocab, size_of(dtype)).group;
  return std::min<int64_t>((int64_t{1} << 32) / group - kThreads,
                           kSumRows * kSumRows);
}

// Partial sums, the rows' losses, and statistics of segments.
int64_t ce_scratch_bytes(int dtype, int64_t n, int64_t vocab) {
  const int segs = plan_of(n, vocab, size_of(dtype)).segs;
  return sum_blocks(n) * 2 * static_cast<int64_t>(sizeof(double)) +
         n * static_cast<int64_t>(sizeof(float)) +
         (segs > 1 ? n * segs * static_cast<int64_t>(sizeof(Stat)) : 0);
}

void launch_ce_fwd(int dtype, const void* x, int64_t inner,
                   int64_t stride_outer, int64_t stride_inner,
                   const int64_t* target, int64_t ignore, int64_t n,
                   int64_t vocab, float eps, int reduction, void* scratch,
                   float* kept_, float* loss, float* factor,
                   hipStream_t stream) {
  const Plan p = plan_of(n, vocab, size_of(dtype));
  const Rows rows = {inner, stride_outer, stride_inner};
  const int64_t blocks = sum_blocks(n);
  double* sums = static_cast<double*>(scratch);
  float* own = reinterpret_cast<float*>(sums + 2 * blocks);
  float* losses = reduction ? own : loss;
  Stat* stat = reinterpret_cast<Stat*>(own + n);
  float2* kept = reinterpret_cast<float2*>(kept_);
  const float unlabelled = reduction ? kUnlabelled : 0.f;
  if (n > 0) {
    auto* pass = dtype == kFloat  ? stat_pass<float>
                 : dtype == kHalf ? stat_pass<_Float16>
                                  : stat_pass<__bf16>;
    pass(p, x, rows, target, ignore, n, vocab, eps, unlabelled, stat, kept,
         losses, stream);
    if (p.segs > 1)
      hipLaunchKernelGGL(ce_join_kernel,
                         dim3(static_cast<unsigned>((n + kThreads - 1) / kThreads)),
                         dim3(kThreads), 0, stream, x, dtype, rows, target,
                         ignore, n, vocab, p.segs, eps, unlabelled, stat, kept,
                         losses);
  }
  if (!reduction) return;
  const bool mean = reduction == 1;
  hipLaunchKernelGGL(ce_sum_kernel, dim3(static_cast<unsigned>(
                         std::max<int64_t>(1, blocks))),
                     dim3(kSumThreads), 0, stream, losses, n, nullptr,
                     blocks > 1 ? sums : nullptr, mean, loss, factor);
  if (blocks > 1)
    hipLaunchKernelGGL(ce_sum_kernel, dim3(1), dim3(kSumThreads), 0, stream,
                       nullptr, blocks, sums, nullptr, mean, loss, factor);
}

void launch_ce_bwd(int dtype, const void* x, int64_t inner,
                   int64_t stride_outer, int64_t stride_inner,
                   const int64_t* target, int64_t ignore, int64_t n,
                   int64_t vocab, float eps, const float* kept,
                   const float* gout, int gstride, const float* factor,
                   void* dx, hipStream_t stream) {
  const Plan p = plan_of(n, vocab, size_of(dtype));
  const Rows rows = {inner, stride_outer, stride_inner};
  auto* pass = dtype == kFloat  ? grad_pass<float>
               : dtype == kHalf ? grad_pass<_Float16>
                                : grad_pass<__bf16>;
  pass(p, x, rows, target, ignore, n, vocab, eps,
       reinterpret_cast<const float2*>(kept), gout, gstride, factor, dx,
       stream);
}

}  // namespace axon
