// Eight consecutive elements of a flat tensor as floats: 16-byte accesses for
// 16-bit types, two of them for fp32.  `chunk` counts eights from the base,
// which is 16-byte aligned.
#pragma once

#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace lsrm {

// The eight elements as loaded (a load in flight costs 4 or 8 registers).
template <typename T>
struct Raw8 {
  uint4 u[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ Raw8<T> load8_raw(const T* base, long long chunk) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i)
    r.u[i] = reinterpret_cast<const uint4*>(base)[chunk * (sizeof(T) / 2) + i];
  return r;
}

template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, float* f) {
  const T* e = reinterpret_cast<const T*>(r.u);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (float)e[i];
}

template <typename T>
__device__ __forceinline__ void load8(const T* base, long long chunk, float* f) {
  unpack8(load8_raw(base, chunk), f);
}

template <typename T>
__device__ __forceinline__ void store8(T* base, long long chunk, const float* f) {
  if constexpr (sizeof(T) == 2) {
    uint4 u;
    T* e = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = (T)f[i];
    reinterpret_cast<uint4*>(base)[chunk] = u;
  } else {
    reinterpret_cast<float4*>(base)[2 * chunk] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(base)[2 * chunk + 1] = make_float4(f[4], f[5], f[6], f[7]);
  }
}

// The elements [lo, hi) of a chunk only (element 8 * chunk + i for i in the range).
template <typename T>
__device__ __forceinline__ void load8_part(const T* base, long long chunk, int lo, int hi, float* f) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (i >= lo && i < hi) ? (float)base[8 * chunk + i] : 0.f;
}

template <typename T>
__device__ __forceinline__ void store8_part(T* base, long long chunk, int lo, int hi, const float* f) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i >= lo && i < hi) base[8 * chunk + i] = (T)f[i];
}

}  // namespace lsrm
