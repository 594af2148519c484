// Dropout whose mask is never stored: y = x / (1 - p) where the element's
// Philox word (philox.cuh) is kept, else 0.  The backward pass is the same
// call on the gradient.  A thread takes eight elements (two counter blocks).
//
// Bound by the generator's arithmetic, not by HBM.  537 million elements: bf16
// 486 us (4.4 TB/s), fp16 471, fp32 (half as many) 415; a plain copy 329.  The
// 36 products of eight elements, four cycles a warp, are 260 us of that, and the
// logical operations beside them fill the other pipe: ALU 58 % of the cycles,
// FMA 43 %, issue slots 62 %, DRAM 41 % (67 million elements); the warps wait
// for a math pipe first.  Of 475 us before the scaling went to 32 bits: 340
// without the generator's last seven rounds, 437 without the memory.  Loading an
// iteration ahead does not help: the warps that are resident hide the loads.
#include <algorithm>

#include "host_util.h"
#include "philox.cuh"
#include "vec8.cuh"

namespace lsrm {
namespace {

// Two packed 16-bit values times 1 / (1 - p): the 32-bit product rounded once,
// right for infinities and at both ends of the type's range.  (The scale as
// the sum of two 16-bit values would save two conversions and 2 % of the time,
// and turns infinities into NaN.)
__device__ __forceinline__ uint32_t scale2(uint32_t x, float s, __nv_bfloat16) {
  const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x));
  const __nv_bfloat162 r = __floats2bfloat162_rn(f.x * s, f.y * s);
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t scale2(uint32_t x, float s, __half) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x));
  const __half2 r = __floats2half2_rn(f.x * s, f.y * s);
  return *reinterpret_cast<const uint32_t*>(&r);
}

template <typename T>
__global__ void __launch_bounds__(256) dropout_kernel(const T* __restrict__ x, T* __restrict__ y, long long n,
                                                      const DropoutParams d) {
  const long long full = n >> 3;
  const long long stride = (long long)gridDim.x * blockDim.x;
  long long c = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  PhiloxHigh ph;
  for (; c < full; c += stride) {
    Raw8<T> r = load8_raw(x, c);  // in flight over the generator's rounds
    if constexpr (sizeof(T) == 2) {
      uint32_t w[8], *v = reinterpret_cast<uint32_t*>(r.u);
      dropout_words(d, ph, c, w);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t s = scale2(v[i], d.scale, T());
        if (w[2 * i] < d.threshold) s &= 0xffff0000u;
        if (w[2 * i + 1] < d.threshold) s &= 0xffffu;
        v[i] = s;
      }
      reinterpret_cast<uint4*>(y)[c] = r.u[0];
    } else {
      float f[8];
      unpack8(r, f);
      dropout8(d, ph, c, f);
      store8(y, c, f);
    }
  }
  if (c == full && (n & 7)) {
    float f[8];
    load8_part(x, c, 0, (int)(n & 7), f);
    dropout8(d, ph, c, f);
    store8_part(y, c, 0, (int)(n & 7), f);
  }
}

template <typename T>
int launch_dropout(const void* x, void* y, long long n, const DropoutParams& d, cudaStream_t s) {
  const int grid = (int)std::min<long long>((n / 8 + 256) / 256,
                                            (long long)num_sms() * resident_blocks<dropout_kernel<T>>(256));
  dropout_kernel<<<grid, 256, 0, s>>>(static_cast<const T*>(x), static_cast<T*>(y), n, d);
  LSRM_LAUNCH_CHECK();
  return LSRM_OK;
}

}  // namespace
}  // namespace lsrm

using namespace lsrm;

extern "C" int lsrm_dropout(int64_t n, int32_t dtype, double p, uint64_t seed, uint64_t offset, const void* x, void* y,
                            void* stream) {
  LSRM_CHECK_ARG(n >= 0, "the number of elements (%lld) must not be negative", (long long)n);
  LSRM_CHECK_ARG(p >= 0.0 && p < 1.0, "p (%g) must be in [0, 1)", p);
  LSRM_CHECK_ARG(dtype == LSRM_DTYPE_BF16 || dtype == LSRM_DTYPE_F16 || dtype == LSRM_DTYPE_F32,
                 "dtype must be bf16, fp16 or fp32");
  LSRM_CHECK_ARG(((uintptr_t)x & 15) == 0 && ((uintptr_t)y & 15) == 0, "x and y must be 16-byte aligned");
  if (n == 0) return LSRM_OK;
  LSRM_CHECK_ARG(x && y, "x and y must not be NULL");
  const DropoutParams d = make_dropout(p, seed, offset);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  ProfScope ps("dropout", s);
  return dtype == LSRM_DTYPE_BF16  ? launch_dropout<__nv_bfloat16>(x, y, n, d, s)
         : dtype == LSRM_DTYPE_F16 ? launch_dropout<__half>(x, y, n, d, s)
                                   : launch_dropout<float>(x, y, n, d, s);
}
