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
  for (; c + stride < full; c += 2 * stride) {  // two loads in flight
    float f[8], g[8];
    load8(x, c, f);
    load8(x, c + stride, g);
    dropout8(d, c, f);
    store8(y, c, f);
    dropout8(d, c + stride, g);
    store8(y, c + stride, g);
  }
  for (; c <= full; c += stride) {
    float f[8];
    if (c < full) {
      load8(x, c, f);
      dropout8(d, c, f);
      store8(y, c, f);
    } else if (n & 7) {
      load8_part(x, c, 0, (int)(n & 7), f);
      dropout8(d, c, f);
      store8_part(y, c, 0, (int)(n & 7), f);
    }
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
