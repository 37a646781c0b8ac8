// Device helpers shared by the mixture-of-experts and distillation kernels:
// element types, 16-byte vectors, wave and workgroup reductions.
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace bcjr {

// Element types by the ids of the C ABI (BCJR_F32, BCJR_BF16, BCJR_F16).  The
// 16-bit types are held as their bits; all arithmetic is float32.
struct F32 {
  using raw = float;
  static __device__ __forceinline__ float get(raw x) { return x; }
  static __device__ __forceinline__ raw put(float x) { return x; }
};
struct BF16 {
  using raw = uint16_t;
  static __device__ __forceinline__ float get(raw x) { return __uint_as_float((uint32_t)x << 16); }
  static __device__ __forceinline__ raw put(float x) {  // to nearest, ties to even
    return __builtin_bit_cast(uint16_t, (__bf16)x);
  }
};
struct F16 {
  using raw = uint16_t;
  static __device__ __forceinline__ float get(raw x) { return (float)__builtin_bit_cast(_Float16, x); }
  static __device__ __forceinline__ raw put(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
};

// 16 bytes of elements: 4 of float32, 8 of the 16-bit types.
template <class E>
struct alignas(16) Vec16 {
  static constexpr int N = 16 / sizeof(typename E::raw);
  typename E::raw v[N];
};

// The same 16 bytes as four registers, and their elements.  (Arrays of 16-bit
// elements that live long are kept one to a register.)
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <class E>
__device__ __forceinline__ void unpack16(u32x4 v, float* z) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(typename E::raw) == 4) {
      z[i] = __uint_as_float(v[i]);
    } else {
      z[2 * i] = E::get((typename E::raw)(v[i] & 0xffffu));
      z[2 * i + 1] = E::get((typename E::raw)(v[i] >> 16));
    }
  }
}
template <class E>
__device__ __forceinline__ u32x4 pack16(const float* z) {
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(typename E::raw) == 4)
      v[i] = __float_as_uint(z[i]);
    else
      v[i] = (uint32_t)E::put(z[2 * i]) | (uint32_t)E::put(z[2 * i + 1]) << 16;
  }
  return v;
}

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int o = 32; o; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
  return x;
}

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

// Sum and maximum over a workgroup of NW waves; every thread gets the result.
// `part` holds NW floats and may be reused after the next barrier.
template <int NW>
__device__ __forceinline__ float group_sum(float x, float* part) {
  x = wave_sum(x);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NW; ++i) s += part[i];
  return s;
}

template <int NW>
__device__ __forceinline__ float group_max(float x, float* part) {
  x = wave_max(x);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
  __syncthreads();
  float s = part[0];
#pragma unroll
  for (int i = 1; i < NW; ++i) s = fmaxf(s, part[i]);
  return s;
}

// Stores v past the caches.  (Between the two, the compiler would join it with a
// plain store of the same in another branch.)
template <class V>
__device__ __forceinline__ void store_past(V* to, V v) {
  asm volatile("" ::: "memory");
  __builtin_nontemporal_store(v, to);
  asm volatile("" ::: "memory");
}

}  // namespace bcjr
