// Shared device helpers of the language-model kernels (embedding.hip,
// cross_entropy.hip, grad_norm.hip): 16-byte vectors of float / fp16 / bf16
// at any element alignment, and wave64 reductions.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <cstring>

namespace axon {
namespace lm {

// at::ScalarType codes.
constexpr int kHalf = 5, kFloat = 6, kBF16 = 15;

using u32x4 = uint32_t __attribute__((ext_vector_type(4)));
using f32x2 = float __attribute__((ext_vector_type(2)));
using bf16x2 = __bf16 __attribute__((ext_vector_type(2)));
using f16x2 = _Float16 __attribute__((ext_vector_type(2)));

// Values of T in 16 bytes.
template <typename T>
constexpr int kVec = 16 / static_cast<int>(sizeof(T));

// 16 bytes from any address that T may have. Rows of an odd length start
// anywhere; gfx950 loads and stores 16 bytes at any alignment, so there is
// no separate path for the first values of a row.
template <typename T>
__device__ __forceinline__ u32x4 load16(const T* p) {
  u32x4 r;
  __builtin_memcpy(&r, p, 16);
  return r;
}
template <typename T>
__device__ __forceinline__ void store16(T* p, u32x4 r) {
  __builtin_memcpy(p, &r, 16);
}

// The same for data that is read or written once: it goes past the caches
// without displacing what is in them.
template <typename T>
__device__ __forceinline__ u32x4 load16_once(const T* p) {
  using Any = u32x4 __attribute__((aligned(sizeof(T))));
  return __builtin_nontemporal_load(reinterpret_cast<const Any*>(p));
}
template <typename T>
__device__ __forceinline__ void store16_once(T* p, u32x4 r) {
  using Any = u32x4 __attribute__((aligned(sizeof(T))));
  __builtin_nontemporal_store(r, reinterpret_cast<Any*>(p));
}

template <typename T>
__device__ __forceinline__ void unpack(u32x4 r, float* f);
template <>
__device__ __forceinline__ void unpack<float>(u32x4 r, float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // (bit_cast of a vector's element itself takes the first one's bits.)
    const uint32_t u = r[i];
    f[i] = __builtin_bit_cast(float, u);
  }
}
template <>
__device__ __forceinline__ void unpack<__bf16>(u32x4 r, float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __builtin_bit_cast(float, r[i] << 16);
    f[2 * i + 1] = __builtin_bit_cast(float, r[i] & 0xffff0000u);
  }
}
template <>
__device__ __forceinline__ void unpack<_Float16>(u32x4 r, float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t u = r[i];
    const f16x2 h = __builtin_bit_cast(f16x2, u);
    f[2 * i] = static_cast<float>(h[0]);
    f[2 * i + 1] = static_cast<float>(h[1]);
  }
}

// Rounds to nearest even, once.
template <typename T>
__device__ __forceinline__ u32x4 pack(const float* f);
template <>
__device__ __forceinline__ u32x4 pack<float>(const float* f) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(uint32_t, f[i]);
  return r;
}
template <>
__device__ __forceinline__ u32x4 pack<__bf16>(const float* f) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x2 v = {f[2 * i], f[2 * i + 1]};
    r[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
  }
  return r;
}
template <>
__device__ __forceinline__ u32x4 pack<_Float16>(const float* f) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x2 v = {f[2 * i], f[2 * i + 1]};
    r[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
  }
  return r;
}

template <typename V>
__device__ __forceinline__ V wave_sum(V v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

}  // namespace lm
}  // namespace axon
