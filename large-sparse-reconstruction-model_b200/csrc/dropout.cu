// Dropout whose mask is never stored: y = x / (1 - p) where the element's
// Philox word (philox.cuh) is kept, else 0.  The backward pass is the same
// call on the gradient.  A thread takes eight elements (two counter blocks).
#include <algorithm>

#include "host_util.h"
#include "philox.cuh"
#include "vec8.cuh"

namespace lsrm {
namespace {

template <typename T>
__global__ void __launch_bounds__(256) dropout_kernel(const T* __restrict__ x, T* __restrict__ y, long long n,
                                                      const DropoutParams d) {
  const long long full = n >> 3;
  const long long stride = (long long)gridDim.x * blockDim.x;
  long long c = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  for (; c < full; c += stride) {
    float f[8];
    load8(x, c, f);
    const uint32_t keep = dropout_keep8(d, c);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (keep >> i & 1u) ? f[i] * d.scale : 0.f;
    store8(y, c, f);
  }
  if (c == full && (n & 7)) {
    float f[8];
    const int rest = (int)(n & 7);
    load8_part(x, c, 0, rest, f);
    const uint32_t keep = dropout_keep8(d, c);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (keep >> i & 1u) ? f[i] * d.scale : 0.f;
    store8_part(y, c, 0, rest, f);
  }
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
  const int grid = (int)std::min<long long>((n / 8 + 256) / 256, (long long)num_sms() * 8);
  if (dtype == LSRM_DTYPE_BF16)
    dropout_kernel<<<grid, 256, 0, s>>>(static_cast<const __nv_bfloat16*>(x), static_cast<__nv_bfloat16*>(y), n, d);
  else if (dtype == LSRM_DTYPE_F16)
    dropout_kernel<<<grid, 256, 0, s>>>(static_cast<const __half*>(x), static_cast<__half*>(y), n, d);
  else
    dropout_kernel<<<grid, 256, 0, s>>>(static_cast<const float*>(x), static_cast<float*>(y), n, d);
  LSRM_LAUNCH_CHECK();
  return LSRM_OK;
}
