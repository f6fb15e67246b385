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

// exp by the hardware's exp2 (1 ulp), on a difference that is exact for the
// values that matter in a sum.
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
// (kWhole) it finishes the row as well.
template <typename T, int G, bool kSmooth, bool kWhole>
__global__ __launch_bounds__(kThreads) void ce_stat_kernel(
    const T* __restrict__ x, Rows rows, const int64_t* __restrict__ target,
    int64_t ignore, int64_t n, int64_t vocab, int64_t seg_len, int segs,
    float small, float eps, Stat* __restrict__ stat, float2* __restrict__ kept,
    float* __restrict__ losses) {
  constexpr int V = kVec<T>;
  constexpr int kAhead = 4;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * (kThreads / G) +
                       threadIdx.x / G;
  const int64_t row = kWhole ? unit : unit / segs;
  const int64_t label = row < n ? target[row] : ignore;
  const bool reads = label != ignore;
  const int t = threadIdx.x % G;
  if (kWhole && !reads && t == 0 && row < n) losses[row] = 0.f;
  if (G == kThreads && !reads) return;
  const bool known = label >= 0 && label < vocab;
  Stat st = {kLowest, 0.f, 0.f};
  float xt = 0.f;
  if (reads) {
    const int64_t begin = kWhole ? 0 : unit % segs * seg_len;
    const int64_t len = kWhole ? vocab : min(seg_len, vocab - begin);
    const T* p = x + rows.at(row) + begin;
    if (kWhole && known) xt = static_cast<float>(p[label]);
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
    const int64_t full = len / V;
    int64_t i = t;
    for (; i + (kAhead - 1) * G < full; i += kAhead * G) {
      u32x4 r[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) r[k] = load16(p + (i + k * G) * V);
#pragma unroll
      for (int k = 0; k < kAhead; ++k) take(r[k]);
    }
    for (; i < full; i += G) take(load16(p + i * V));
    for (int64_t j = full * V + t; j < len; j += G) {
      const float f = static_cast<float>(p[j]);
      const float m = fmaxf(st.m, f);
      st.s = st.s * exp_of(st.m - m) + exp_of(f - m);
      if (kSmooth) st.x = fmaf(f, small, st.x);
      st.m = m;
    }
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
    int64_t vocab, int segs, float eps, const Stat* __restrict__ stat,
    float2* __restrict__ kept, float* __restrict__ losses) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (row >= n) return;
  const int64_t t = target[row];
  if (t == ignore) {
    losses[row] = 0.f;
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
// over those (`sums` in, `losses` null).
constexpr int kSumThreads = 1024;
constexpr int64_t kSumRows = 16384;

__global__ __launch_bounds__(kSumThreads) void ce_sum_kernel(
    const float* __restrict__ losses, const int64_t* __restrict__ target,
    int64_t ignore, int64_t n, const double* __restrict__ in,
    double* __restrict__ out, bool mean, float* __restrict__ loss,
    float* __restrict__ factor) {
  double sum = 0.0, count = 0.0;
  const int64_t begin = static_cast<int64_t>(blockIdx.x) * kSumRows;
  const int64_t end = min(n, begin + kSumRows);
#pragma unroll 4
  for (int64_t i = begin + threadIdx.x; i < end; i += kSumThreads) {
    sum += in ? in[2 * i] : static_cast<double>(losses[i]);
    count += in ? in[2 * i + 1] : (target[i] != ignore ? 1.0 : 0.0);
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

template <typename T, int G>
__global__ __launch_bounds__(kThreads) void ce_grad_kernel(
    const T* __restrict__ x, Rows rows, const int64_t* __restrict__ target,
    int64_t ignore, int64_t n, int64_t vocab, int64_t seg_len, int segs,
    float eps, const float2* __restrict__ kept, const float* __restrict__ gout,
    int gstride, const float* __restrict__ factor, T* __restrict__ dx) {
  constexpr int V = kVec<T>;
  constexpr int kAhead = 4;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * (kThreads / G) +
                       threadIdx.x / G;
  const int64_t row = unit / segs;
  if (row >= n) return;
  const int t = threadIdx.x % G;
  const int64_t begin = unit % segs * seg_len;
  const int64_t len = min(seg_len, vocab - begin);
  const int64_t full = len / V;
  T* q = dx + row * vocab + begin;
  const int64_t label = target[row];
  if (label == ignore) {
    for (int64_t i = t; i < full; i += G) store16(q + i * V, u32x4{0, 0, 0, 0});
    for (int64_t j = full * V + t; j < len; j += G) q[j] = static_cast<T>(0.f);
    return;
  }
  const T* p = x + rows.at(row) + begin;
  float g = gout[row * gstride];
  if (factor) g *= *factor;
  if (label < 0 || label >= vocab) g = __builtin_nanf("");
  const float2 st = kept[row];
  const float scale = st.y * g;
  const float off = eps > 0.f ? g * eps / static_cast<float>(vocab) : 0.f;
  const float hit = g * (1.f - eps);
  const int64_t at = label - begin;  // the label's place in this segment
  auto value = [&](float f, int64_t j) {
    float v = exp_of(f - st.x) * scale - off;
    return j == at ? v - hit : v;
  };
  int64_t i = t;
  for (; i + (kAhead - 1) * G < full; i += kAhead * G) {
    u32x4 r[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) r[k] = load16(p + (i + k * G) * V);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      float f[V];
      unpack<T>(r[k], f);
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = value(f[e], (i + k * G) * V + e);
      store16(q + (i + k * G) * V, pack<T>(f));
    }
  }
  for (; i < full; i += G) {
    float f[V];
    unpack<T>(load16(p + i * V), f);
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = value(f[e], i * V + e);
    store16(q + i * V, pack<T>(f));
  }
  for (int64_t j = full * V + t; j < len; j += G)
    q[j] = static_cast<T>(value(static_cast<float>(p[j]), j));
}

// 16 lanes for a row of up to 128 logits, a wave for one of up to 1024, a
// block for a longer one. Where the rows are too few to fill the chip (2048
// blocks), long ones are cut into segments of 4096 logits or more.
struct Plan {
  int group;
  int segs;
  int64_t seg_len;
};

Plan plan_of(int64_t n, int64_t vocab) {
  if (vocab <= 128) return {16, 1, vocab};
  if (vocab <= 1024) return {64, 1, vocab};
  const int64_t want = std::max<int64_t>(1, 2048 / std::max<int64_t>(n, 1));
  const int64_t most = std::max<int64_t>(1, vocab / 4096);
  const int64_t segs = std::min(want, most);
  const int64_t len = ((vocab + segs - 1) / segs + 15) / 16 * 16;
  return {kThreads, static_cast<int>((vocab + len - 1) / len), len};
}

unsigned blocks_of(const Plan& p, int64_t n) {
  const int per = kThreads / p.group;
  return static_cast<unsigned>((n * p.segs + per - 1) / per);
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
               int64_t ignore, int64_t n, int64_t vocab, float eps, Stat* stat,
               float2* kept, float* losses, hipStream_t stream) {
  auto* k = eps > 0.f ? stat_kernel<T, true>(p) : stat_kernel<T, false>(p);
  hipLaunchKernelGGL(k, dim3(blocks_of(p, n)), dim3(kThreads), 0, stream,
                     static_cast<const T*>(x), rows, target, ignore, n, vocab,
                     p.seg_len, p.segs, down(vocab), eps, stat, kept, losses);
}

template <typename T>
void grad_pass(const Plan& p, const void* x, Rows rows, const int64_t* target,
               int64_t ignore, int64_t n, int64_t vocab, float eps,
               const float2* kept, const float* gout, int gstride,
               const float* factor, void* dx, hipStream_t stream) {
  auto* k = p.group == 16   ? &ce_grad_kernel<T, 16>
            : p.group == 64 ? &ce_grad_kernel<T, 64>
                            : &ce_grad_kernel<T, kThreads>;
  hipLaunchKernelGGL(k, dim3(blocks_of(p, n)), dim3(kThreads), 0, stream,
                     static_cast<const T*>(x), rows, target, ignore, n, vocab,
                     p.seg_len, p.segs, eps, kept, gout, gstride, factor,
                     static_cast<T*>(dx));
}

int64_t sum_blocks(int64_t n) { return (n + kSumRows - 1) / kSumRows; }

}  // namespace

// Partial sums, the rows' losses, and statistics of segments.
int64_t ce_scratch_bytes(int64_t n, int64_t vocab) {
  const int segs = plan_of(n, vocab).segs;
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
  const Plan p = plan_of(n, vocab);
  const Rows rows = {inner, stride_outer, stride_inner};
  const int64_t blocks = sum_blocks(n);
  double* sums = static_cast<double*>(scratch);
  float* own = reinterpret_cast<float*>(sums + 2 * blocks);
  float* losses = reduction ? own : loss;
  Stat* stat = reinterpret_cast<Stat*>(own + n);
  float2* kept = reinterpret_cast<float2*>(kept_);
  if (n > 0) {
    auto* pass = dtype == kFloat  ? stat_pass<float>
                 : dtype == kHalf ? stat_pass<_Float16>
                                  : stat_pass<__bf16>;
    pass(p, x, rows, target, ignore, n, vocab, eps, stat, kept, losses,
         stream);
    if (p.segs > 1)
      hipLaunchKernelGGL(ce_join_kernel,
                         dim3(static_cast<unsigned>((n + kThreads - 1) / kThreads)),
                         dim3(kThreads), 0, stream, x, dtype, rows, target,
                         ignore, n, vocab, p.segs, eps, stat, kept, losses);
  }
  if (!reduction) return;
  const bool mean = reduction == 1;
  hipLaunchKernelGGL(ce_sum_kernel, dim3(static_cast<unsigned>(
                         std::max<int64_t>(1, blocks))),
                     dim3(kSumThreads), 0, stream, losses, target, ignore, n,
                     nullptr, blocks > 1 ? sums : nullptr, mean, loss, factor);
  if (blocks > 1)
    hipLaunchKernelGGL(ce_sum_kernel, dim3(1), dim3(kSumThreads), 0, stream,
                       nullptr, nullptr, ignore, blocks, sums, nullptr, mean,
                       loss, factor);
}

void launch_ce_bwd(int dtype, const void* x, int64_t inner,
                   int64_t stride_outer, int64_t stride_inner,
                   const int64_t* target, int64_t ignore, int64_t n,
                   int64_t vocab, float eps, const float* kept,
                   const float* gout, int gstride, const float* factor,
                   void* dx, hipStream_t stream) {
  const Plan p = plan_of(n, vocab);
  const Rows rows = {inner, stride_outer, stride_inner};
  auto* pass = dtype == kFloat  ? grad_pass<float>
               : dtype == kHalf ? grad_pass<_Float16>
                                : grad_pass<__bf16>;
  pass(p, x, rows, target, ignore, n, vocab, eps,
       reinterpret_cast<const float2*>(kept), gout, gstride, factor, dx,
       stream);
}

}  // namespace axon
