// The single-token form of the windowed attention with sinks over a ring
// cache.  Sequence b holds n = lengths[b] tokens; the new token takes position
// n.  Position j is kept in slot j while j < sinks, else in slot
// sinks + (j - sinks) % (capacity - sinks): the ring holds the last
// capacity - sinks positions past the sinks.  The call writes the new key and
// value to their slot and attends to positions [0, sinks) and (n - window, n].
// A negative length marks an idle row: nothing is written, its output is 0.
//
// A warp owns a (sequence, query head): lanes take 32 keys at a time.
#include <algorithm>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "host_util.h"

namespace lsrm {
namespace {

struct DecodeParams {
  int batch, hq, hkv, g, capacity, window, sinks;
  float scale;
  long long q_stride, kn_stride, vn_stride;            // elements between sequences of q, k_new, v_new
  long long kc_batch, kc_slot, vc_batch, vc_slot;      // elements between sequences / slots of the caches
  const void *q, *k_new, *v_new;
  void *k_cache, *v_cache, *out;
  const int32_t* lengths;
};

__device__ __forceinline__ int slot_of(int pos, int sinks, int ring) {
  return pos < sinks ? pos : sinks + (pos - sinks) % ring;
}

template <typename T, int D>
__global__ void __launch_bounds__(32) window_decode_kernel(const DecodeParams p) {
  __shared__ float sq[D];
  const int lane = threadIdx.x, h = blockIdx.x, b = blockIdx.y, hk = h / p.g;
  const int n = p.lengths[b], ring = p.capacity - p.sinks;
  T* out = static_cast<T*>(p.out) + ((long long)b * p.hq + h) * D;
  if (n < 0) {
    for (int d = lane; d < D; d += 32) out[d] = (T)0.f;
    return;
  }
  const T* q = static_cast<const T*>(p.q) + b * p.q_stride + h * D;
  const T* kn = static_cast<const T*>(p.k_new) + b * p.kn_stride + hk * D;
  const T* vn = static_cast<const T*>(p.v_new) + b * p.vn_stride + hk * D;
  T* kc = static_cast<T*>(p.k_cache) + b * p.kc_batch + hk * D;
  T* vc = static_cast<T*>(p.v_cache) + b * p.vc_batch + hk * D;
  const int slot_n = slot_of(n, p.sinks, ring);
  float m = 0.f, l = 1.f, acc[D / 32];
  float s0 = 0.f;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    const int d = lane + 32 * i;
    sq[d] = (float)q[d] * p.scale;
    s0 = fmaf(sq[d], (float)kn[d], s0);
    acc[i] = (float)vn[d];
    if (h % p.g == 0) {
      kc[slot_n * p.kc_slot + d] = kn[d];
      vc[slot_n * p.vc_slot + d] = vn[d];
    }
  }
  for (int o = 16; o > 0; o >>= 1) s0 += __shfl_xor_sync(0xffffffffu, s0, o);
  m = s0;
  __syncwarp();
  // the cached positions: [0, sink) and [lo, n)
  const int lo = max(min(p.sinks, n), n + 1 - p.window), sink = min(p.sinks, n), cnt = sink + max(0, n - lo);
  for (int base = 0; base < cnt; base += 32) {
    const int idx = base + lane;
    const int slot = slot_of(idx < sink ? idx : lo + idx - sink, p.sinks, ring);
    float s = -INFINITY;
    if (idx < cnt) {
      s = 0.f;
      for (int d = 0; d < D; ++d) s = fmaf(sq[d], (float)kc[slot * p.kc_slot + d], s);
    }
    float mx = s;
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float m_new = fmaxf(m, mx), r = expf(m - m_new), e = expf(s - m_new);
    float es = e;
    for (int o = 16; o > 0; o >>= 1) es += __shfl_xor_sync(0xffffffffu, es, o);
    l = l * r + es;
    m = m_new;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] *= r;
    const int here = min(32, cnt - base);
    for (int t = 0; t < here; ++t) {
      const float pt = __shfl_sync(0xffffffffu, e, t);
      const int st = __shfl_sync(0xffffffffu, slot, t);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) acc[i] = fmaf(pt, (float)vc[st * p.vc_slot + lane + 32 * i], acc[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < D / 32; ++i) out[lane + 32 * i] = (T)(acc[i] / l);
}

}  // namespace
}  // namespace lsrm

using namespace lsrm;

extern "C" int lsrm_window_decode(const lsrm_window_decode_shape* shape, const void* q, const void* k_new,
                                  const void* v_new, void* k_cache, void* v_cache, const int32_t* lengths, void* out,
                                  void* stream) {
  LSRM_CHECK_ARG(shape, "shape must not be NULL");
  const lsrm_window_decode_shape& d = *shape;
  LSRM_CHECK_ARG(d.batch >= 0 && d.batch <= 65535, "batch (%d) must be in [0, 65535]", d.batch);
  LSRM_CHECK_ARG(d.num_kv_heads >= 1 && d.num_q_heads >= 1 && d.num_q_heads % d.num_kv_heads == 0,
                 "num_q_heads (%d) must be a multiple of num_kv_heads (%d)", d.num_q_heads, d.num_kv_heads);
  LSRM_CHECK_ARG(d.num_q_heads / d.num_kv_heads <= 64, "at most 64 query heads per kv head");
  LSRM_CHECK_ARG(d.head_dim == 32 || d.head_dim == 64 || d.head_dim == 128, "head_dim (%d) must be 32, 64 or 128",
                 d.head_dim);
  LSRM_CHECK_ARG(d.dtype == LSRM_DTYPE_BF16 || d.dtype == LSRM_DTYPE_F16, "dtype must be bf16 or fp16");
  LSRM_CHECK_ARG(d.window >= 1 && d.sinks >= 0, "window (%d) must be at least 1 and sinks (%d) not negative", d.window,
                 d.sinks);
  LSRM_CHECK_ARG(d.capacity > d.sinks && d.capacity - d.sinks >= d.window,
                 "capacity (%d) must hold the sinks (%d) and the window (%d)", d.capacity, d.sinks, d.window);
  const int64_t qr = (int64_t)d.num_q_heads * d.head_dim, kr = (int64_t)d.num_kv_heads * d.head_dim;
  LSRM_CHECK_ARG(d.q_stride >= qr && d.k_new_stride >= kr && d.v_new_stride >= kr && d.k_slot_stride >= kr &&
                     d.v_slot_stride >= kr && d.k_batch_stride >= 0 && d.v_batch_stride >= 0,
                 "strides must cover the heads");
  LSRM_CHECK_ARG(((d.q_stride | d.k_new_stride | d.v_new_stride | d.k_slot_stride | d.v_slot_stride |
                   d.k_batch_stride | d.v_batch_stride) & 7) == 0, "strides must be multiples of 8 elements");
  LSRM_CHECK_ARG((((uintptr_t)q | (uintptr_t)k_new | (uintptr_t)v_new | (uintptr_t)k_cache | (uintptr_t)v_cache |
                   (uintptr_t)out) & 15) == 0, "tensors must be 16-byte aligned");
  if (d.batch == 0) return LSRM_OK;
  LSRM_CHECK_ARG(q && k_new && v_new && k_cache && v_cache && lengths && out, "pointers must not be NULL");
  DecodeParams p;
  p.batch = d.batch, p.hq = d.num_q_heads, p.hkv = d.num_kv_heads, p.g = p.hq / p.hkv;
  p.capacity = d.capacity, p.window = d.window, p.sinks = d.sinks;
  p.scale = d.softmax_scale > 0.f ? d.softmax_scale : 1.f / sqrtf((float)d.head_dim);
  p.q_stride = d.q_stride, p.kn_stride = d.k_new_stride, p.vn_stride = d.v_new_stride;
  p.kc_batch = d.k_batch_stride, p.kc_slot = d.k_slot_stride, p.vc_batch = d.v_batch_stride;
  p.vc_slot = d.v_slot_stride;
  p.q = q, p.k_new = k_new, p.v_new = v_new, p.k_cache = k_cache, p.v_cache = v_cache, p.out = out;
  p.lengths = lengths;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  ProfScope ps("window_decode", s);
  const dim3 grid(p.hq, p.batch);
#define CALL(T, D) window_decode_kernel<T, D><<<grid, 32, 0, s>>>(p)
  if (d.dtype == LSRM_DTYPE_BF16) {
    if (d.head_dim == 32) CALL(__nv_bfloat16, 32);
    else if (d.head_dim == 64) CALL(__nv_bfloat16, 64);
    else CALL(__nv_bfloat16, 128);
  } else {
    if (d.head_dim == 32) CALL(__half, 32);
    else if (d.head_dim == 64) CALL(__half, 64);
    else CALL(__half, 128);
  }
#undef CALL
  LSRM_LAUNCH_CHECK();
  return LSRM_OK;
}
