// Element types and small vectors of the token-path kernels (layer norm,
// rotary positions): every value is computed in fp32 and rounded once to the
// tensor's type when it is stored.
#pragma once

#include <cuda_fp16.h>

#include "pkv_common.cuh"

namespace pkv {

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) {
  return __half2float(v);
}
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// N consecutive elements, loaded and stored as one access of N * sizeof(T)
// bytes (<= 16) when the address is a multiple of that.
template <typename T, int N>
struct alignas(N * sizeof(T)) Vec {
  T v[N];
};

template <typename T, int N>
__device__ __forceinline__ Vec<T, N> ld_vec(const T* p) {
  return *reinterpret_cast<const Vec<T, N>*>(p);
}
template <typename T, int N>
__device__ __forceinline__ void st_vec(T* p, const Vec<T, N>& v) {
  *reinterpret_cast<Vec<T, N>*>(p) = v;
}

// Asynchronous copy of N elements (4, 8 or 16 bytes) into shared memory.  A
// thread that copies only what it reads itself needs no barrier: its own
// wait_group orders the copy before its loads.
template <typename T, int N>
__device__ __forceinline__ void cp_async(void* dst, const T* src) {
  const uint32_t d = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
  constexpr int kBytes = N * int(sizeof(T));
  static_assert(kBytes == 4 || kBytes == 8 || kBytes == 16, "cp.async copies 4, 8 or 16 bytes");
  if constexpr (kBytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(d), "l"(src), "n"(kBytes)
                 : "memory");
}
__device__ __forceinline__ void cp_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Two 16-bit elements of a word: one instruction a value to widen them (bf16
// is the upper half of fp32), one to round a pair.
template <typename T>
__device__ __forceinline__ void unpack2(uint32_t w, float& lo, float& hi);
template <>
__device__ __forceinline__ void unpack2<__nv_bfloat16>(uint32_t w, float& lo, float& hi) {
  lo = __uint_as_float(w << 16);
  hi = __uint_as_float(w & 0xffff0000u);
}
template <>
__device__ __forceinline__ void unpack2<__half>(uint32_t w, float& lo, float& hi) {
  const __half2 h = *reinterpret_cast<const __half2*>(&w);
  const float2 f = __half22float2(h);
  lo = f.x;
  hi = f.y;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// A vector's elements as fp32, and fp32 rounded into a vector.
template <typename T, int N>
__device__ __forceinline__ void widen(const Vec<T, N>& v, float* f) {
  if constexpr (sizeof(T) == 2 && N >= 2) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) unpack2<T>(w[i], f[2 * i], f[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = to_f32(v.v[i]);
  }
}
template <typename T, int N>
__device__ __forceinline__ Vec<T, N> narrow(const float* f) {
  Vec<T, N> v;
  if constexpr (sizeof(T) == 2 && N >= 2) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) w[i] = pack2<T>(f[2 * i], f[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v.v[i] = from_f32<T>(f[i]);
  }
  return v;
}

// N consecutive elements as fp32, in accesses of up to 16 bytes (aligned to
// that where N > 1).
template <typename T, int N>
__device__ __forceinline__ void ld_f32(const T* p, float (&f)[N]) {
  constexpr int M = N * sizeof(T) > 16 ? int(16 / sizeof(T)) : N;
#pragma unroll
  for (int i = 0; i < N; i += M) {
    widen<T, M>(ld_vec<T, M>(p + i), f + i);
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Whether `p` and a row stride (elements) keep every row on a boundary of n
// elements of `size` bytes.
inline bool vec_ok(const void* p, int64_t row_stride, int n, int size) {
  return p == nullptr ||
         (reinterpret_cast<uintptr_t>(p) % (uintptr_t(n) * size) == 0 && row_stride % n == 0);
}

}  // namespace pkv
