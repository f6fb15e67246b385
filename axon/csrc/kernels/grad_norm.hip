// Norm over all gradients, and the gradients scaled by it:
//
//   r = (sum g^2)^(1/2), sum |g| or max |g| over all tensors
//   c = min(1, max_norm / (r + 1e-6));  g <- c g
//
// Bound by memory: the gradients are read once for the norm, and read and
// written once more where c < 1 (a norm within the bound leaves them alone).
// Sums are in 64 bits: a norm up to the largest fp32 value comes out finite,
// small gradients do not vanish when squared. No atomics: block b takes
// chunks b, b + grid, ... and its partial sum has a place of its own, so the
// same gradients give the same bits.
//
// Measured: the norm of 1.5G bf16 values 529 us (5.7 TB/s), of 25.6M fp32
// values 16.0 us (6.4 TB/s); the squares in 64 bits hide behind the loads. 335M
// bf16 values in two tables: norm 141 us (4.7 TB/s), scaling 217 us (6.2 TB/s
// of reading and writing).
#include <algorithm>

#include "grad_norm.h"
#include "lm_util.h"

namespace axon {

namespace {

using namespace lm;

constexpr int kThreads = 256;
constexpr int kMaxBlocks = 2048;  // 8 blocks of 4 waves on each CU

struct Sum {  // type 1 and 2
  static __device__ double join(double a, double b) { return a + b; }
};
struct Most {  // type 0: NaN wins
  static __device__ double join(double a, double b) {
    return (b > a || b != b) ? b : a;
  }
};

template <int kType>
__device__ __forceinline__ double add(double acc, float f) {
  const double d = static_cast<double>(f);
  if (kType == 2) return fma(d, d, acc);
  if (kType == 1) return acc + fabs(d);
  return Most::join(acc, fabs(d));
}

template <typename J, int kBlock = kThreads>
__device__ double block_join(double v) {
  __shared__ double lds[kBlock / 64];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = J::join(v, __shfl_xor(v, off, 64));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = lds[0];
  for (int w = 1; w < kBlock / 64; ++w) v = J::join(v, lds[w]);
  return v;
}

// Finds the tensor that a chunk belongs to, the last one with first[i] <= c:
// each lane holds three of the table's borders, so that it takes a comparison
// of all at once. (With a bisection of the arguments, a chain of loads for
// each chunk: norm of 335M bf16 values 150 us instead of 139, scaling 219
// instead of 213.)
struct Finder {
  int32_t border[kGradTensors / 64];

  __device__ __forceinline__ explicit Finder(const GradTable& t) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int k = 0; k < kGradTensors / 64; ++k)
      border[k] =
          lane + k * 64 < t.count ? t.first[lane + k * 64] : 0x7fffffff;
  }
  // The tensor's number; *first is the chunk that it starts with.
  __device__ __forceinline__ int find(int c, int* first) const {
    int i = -1;
#pragma unroll
    for (int k = 0; k < kGradTensors / 64; ++k)
      i += __popcll(__ballot(border[k] <= c));
    const int held = i < 64 ? border[0] : i < 128 ? border[1] : border[2];
    *first = __builtin_amdgcn_readlane(held, i & 63);
    return i;
  }
};
static_assert(kGradTensors == 192, "three borders for each lane");

template <typename T, int kType>
__global__ __launch_bounds__(kThreads) void grad_partial_kernel(
    const GradTable t, double* __restrict__ partial) {
  constexpr int V = kVec<T>;
  constexpr int kAhead = 4;
  double acc = 0.0;
  const int chunks = t.first[t.count];
  const Finder finder(t);
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    int first;
    const int i = finder.find(c, &first);
    const int64_t begin = static_cast<int64_t>(c - first) * kGradChunk;
    const T* p = static_cast<const T*>(t.ptr[i]) + begin;
    const int len = static_cast<int>(min(kGradChunk, t.n[i] - begin));
    const int full = len / V;
    int k = threadIdx.x;
    for (; k + (kAhead - 1) * kThreads < full; k += kAhead * kThreads) {
      u32x4 r[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) r[a] = load16(p + (k + a * kThreads) * V);
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        float f[V];
        unpack<T>(r[a], f);
#pragma unroll
        for (int e = 0; e < V; ++e) acc = add<kType>(acc, f[e]);
      }
    }
    for (; k < full; k += kThreads) {
      float f[V];
      unpack<T>(load16(p + k * V), f);
#pragma unroll
      for (int e = 0; e < V; ++e) acc = add<kType>(acc, f[e]);
    }
    for (int j = full * V + threadIdx.x; j < len; j += kThreads)
      acc = add<kType>(acc, static_cast<float>(p[j]));
  }
  using J = std::conditional_t<kType == 0, Most, Sum>;
  acc = block_join<J>(acc);
  if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

// (norm, factor) of the partial sums, in every thread of the block, and the
// same bits in every block.
template <int kType, int kBlock = kThreads>
__device__ __forceinline__ float2 finish(const double* __restrict__ partial,
                                         int blocks, float max_norm) {
  using J = std::conditional_t<kType == 0, Most, Sum>;
  double acc = 0.0;
  for (int i = threadIdx.x; i < blocks; i += kBlock)
    acc = J::join(acc, partial[i]);
  acc = block_join<J, kBlock>(acc);
  const float norm = static_cast<float>(kType == 2 ? sqrt(acc) : acc);
  const float c = max_norm / (norm + 1e-6f);
  return make_float2(norm, c > 1.f ? 1.f : c);  // NaN stays
}

constexpr int kFinishThreads = 1024;

template <int kType>
__global__ __launch_bounds__(kFinishThreads) void grad_finish_kernel(
    const double* __restrict__ partial, int blocks, float max_norm,
    float2* __restrict__ out) {
  const float2 r = finish<kType, kFinishThreads>(partial, blocks, max_norm);
  if (threadIdx.x == 0) *out = r;
}

// kType >= 0: every block joins the (few) partial sums itself, and the first
// one writes the result; kType < 0: the factor is there.
template <typename T, int kType>
__global__ __launch_bounds__(kThreads) void grad_scale_kernel(
    const GradTable t, const float* __restrict__ factor,
    const double* __restrict__ partial, int blocks, float max_norm,
    float2* __restrict__ out) {
  constexpr int V = kVec<T>;
  constexpr int kAhead = 4;
  float c;
  if constexpr (kType < 0) {
    c = *factor;
  } else {
    const float2 r = finish<kType>(partial, blocks, max_norm);
    c = r.y;
    if (blockIdx.x == 0 && threadIdx.x == 0) *out = r;
  }
  if (c == 1.f) return;
  const int chunks = t.first[t.count];
  const Finder finder(t);
  // From the last chunk to the first: the norm has just read the last ones,
  // and the chip's last cache holds 256 MB of them.
  for (int b = chunks - 1 - static_cast<int>(blockIdx.x); b >= 0;
       b -= gridDim.x) {
    int first;
    const int i = finder.find(b, &first);
    const int64_t begin = static_cast<int64_t>(b - first) * kGradChunk;
    T* p = static_cast<T*>(t.ptr[i]) + begin;
    const int len = static_cast<int>(min(kGradChunk, t.n[i] - begin));
    const int full = len / V;
    int k = threadIdx.x;
    for (; k + (kAhead - 1) * kThreads < full; k += kAhead * kThreads) {
      u32x4 r[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) r[a] = load16(p + (k + a * kThreads) * V);
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        float f[V];
        unpack<T>(r[a], f);
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] *= c;
        store16(p + (k + a * kThreads) * V, pack<T>(f));
      }
    }
    for (; k < full; k += kThreads) {
      float f[V];
      unpack<T>(load16(p + k * V), f);
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] *= c;
      store16(p + k * V, pack<T>(f));
    }
    for (int j = full * V + threadIdx.x; j < len; j += kThreads)
      p[j] = static_cast<T>(static_cast<float>(p[j]) * c);
  }
}

template <int kType>
void partial_of(const GradTable& t, int dtype, double* partial,
                hipStream_t stream) {
  auto* k = dtype == kFloat  ? grad_partial_kernel<float, kType>
            : dtype == kHalf ? grad_partial_kernel<_Float16, kType>
                             : grad_partial_kernel<__bf16, kType>;
  hipLaunchKernelGGL(k, dim3(grad_norm_blocks(t)), dim3(kThreads), 0, stream, t,
                     partial);
}

}  // namespace

int grad_norm_blocks(const GradTable& t) {
  return std::min(kMaxBlocks, t.first[t.count]);
}

void launch_grad_partial(const GradTable& t, int dtype, int type,
                         double* partial, hipStream_t stream) {
  if (type == 2) partial_of<2>(t, dtype, partial, stream);
  if (type == 1) partial_of<1>(t, dtype, partial, stream);
  if (type == 0) partial_of<0>(t, dtype, partial, stream);
}

void launch_grad_finish(const double* partial, int blocks, int type,
                        float max_norm, float* out, hipStream_t stream) {
  auto* k = type == 2   ? grad_finish_kernel<2>
            : type == 1 ? grad_finish_kernel<1>
                        : grad_finish_kernel<0>;
  hipLaunchKernelGGL(k, dim3(1), dim3(kFinishThreads), 0, stream, partial, blocks,
                     max_norm, reinterpret_cast<float2*>(out));
}

namespace {

template <int kType>
void scale(const GradTable& t, int dtype, const float* factor,
           const double* partial, int blocks, float max_norm, float* out,
           hipStream_t stream) {
  auto* k = dtype == kFloat  ? grad_scale_kernel<float, kType>
            : dtype == kHalf ? grad_scale_kernel<_Float16, kType>
                             : grad_scale_kernel<__bf16, kType>;
  hipLaunchKernelGGL(k, dim3(grad_norm_blocks(t)), dim3(kThreads), 0, stream, t,
                     factor, partial, blocks, max_norm,
                     reinterpret_cast<float2*>(out));
}

}  // namespace

void launch_grad_scale(const GradTable& t, int dtype, const float* factor,
                       hipStream_t stream) {
  scale<-1>(t, dtype, factor, nullptr, 0, 0.f, nullptr, stream);
}

bool grad_clip_folds(int blocks) { return blocks <= 2 * kThreads; }

void launch_grad_clip(const GradTable& t, int dtype, int type,
                      const double* partial, int blocks, float max_norm,
                      float* out, hipStream_t stream) {
  if (type == 2)
    scale<2>(t, dtype, nullptr, partial, blocks, max_norm, out, stream);
  if (type == 1)
    scale<1>(t, dtype, nullptr, partial, blocks, max_norm, out, stream);
  if (type == 0)
    scale<0>(t, dtype, nullptr, partial, blocks, max_norm, out, stream);
}

}  // namespace axon
