// Eight consecutive elements of a flat tensor as floats: 16-byte accesses for
// 16-bit types, two of them for fp32.  `chunk` counts eights from the base,
// which is 16-byte aligned.
#pragma once

#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace lsrm {

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  return (float)v;
}

template <typename T>
__device__ __forceinline__ void load8(const T* base, long long chunk, float* f) {
  if constexpr (sizeof(T) == 2) {
    const uint4 u = reinterpret_cast<const uint4*>(base)[chunk];
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)e[i];
  } else {
    const float4 a = reinterpret_cast<const float4*>(base)[2 * chunk];
    const float4 b = reinterpret_cast<const float4*>(base)[2 * chunk + 1];
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  }
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
