// Attention with a sliding window and a few first tokens that stay visible
// (sinks): forward and backward over packed sequences, grouped query heads.
//   s_ij = scale q_i . k_j over the keys that window_common.cuh names,
//   lse_i = log sum_j exp s_ij,  o_i = sum_j exp(s_ij - lse_i) v_j
// (a query that sees no key: o = 0, lse = -inf).  Backward:
//   delta_i = o_i . do_i,  p = exp(s - lse),  ds = p (do_i . v_j - delta_i)
//   dq_i = scale sum_j ds k_j,  dk_j = scale sum_i ds q_i,  dv_j = sum_i p do_i
// with the query heads of a group summed into their kv head.
//
// A warp owns a query (forward, dq) or a key (dk, dv); its lanes take 32 keys
// (queries) at a time for the scores and the channels for the sums.
#include <algorithm>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "window_host.h"

namespace lsrm {
namespace {

template <typename T>
__device__ __forceinline__ float dot_row(const float* a, const T* b, int d) {
  float s = 0.f;
  for (int c = 0; c < d; c += 8) {
    const uint4 u = *reinterpret_cast<const uint4*>(b + c);
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fmaf(a[c + i], (float)e[i], s);
  }
  return s;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct WindowBwdParams : WindowParams {
  const void* dout;  // [total_q, hq, D]
  float* delta;      // [total_q, hq]
  void *dq, *dk, *dv;
};

template <typename T, int D>
__global__ void __launch_bounds__(128) window_dq_kernel(const WindowBwdParams p) {
  __shared__ float sq[4][D], sdo[4][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * 4 + warp;
  if (row >= (long long)p.total_q * p.hq) return;
  const int tok = (int)(row / p.hq), h = (int)(row % p.hq), hk = h / p.g;
  const int b = seq_of_token(p.cu_q, p.num_seqs, tok);
  const Seq s_ = seq_of(p, b);
  const int pos = tok - s_.q0 + s_.lk - s_.lq;
  const Seen seen = keys_of(p, pos, s_.lk, b < p.num_seqs);
  const T* q = static_cast<const T*>(p.q) + tok * p.q_stride + h * D;
  const T* dout = static_cast<const T*>(p.dout) + row * D;
  const T* out = static_cast<const T*>(p.out) + row * D;
  float delta = 0.f;
  for (int d = lane; d < D; d += 32) {
    sq[warp][d] = (float)q[d] * p.scale;
    sdo[warp][d] = (float)dout[d];
    delta += (float)dout[d] * (float)out[d];
  }
  delta = warp_sum(delta);
  if (lane == 0) p.delta[row] = delta;
  __syncwarp();
  const float lse = p.lse[row];
  const T* k = static_cast<const T*>(p.k) + s_.k0 * p.k_stride + hk * D;
  const T* v = static_cast<const T*>(p.v) + s_.k0 * p.v_stride + hk * D;
  float acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) acc[i] = 0.f;
  const int n = lse == -INFINITY ? 0 : seen.sink + seen.hi - seen.lo;
  for (int base = 0; base < n; base += 32) {
    const int idx = base + lane;
    const int j = idx < seen.sink ? idx : seen.lo + idx - seen.sink;
    float ds = 0.f;
    if (idx < n) {
      const float pr = expf(dot_row(sq[warp], k + j * p.k_stride, D) - lse);
      ds = pr * (dot_row(sdo[warp], v + j * p.v_stride, D) - delta);
    }
    const int cnt = min(32, n - base);
    for (int t = 0; t < cnt; ++t) {
      const float dt = __shfl_sync(0xffffffffu, ds, t);
      const int jt = __shfl_sync(0xffffffffu, j, t);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) acc[i] = fmaf(dt, (float)k[jt * p.k_stride + lane + 32 * i], acc[i]);
    }
  }
  T* dq = static_cast<T*>(p.dq) + row * D;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) dq[lane + 32 * i] = (T)(acc[i] * p.scale);
}

template <typename T, int D>
__global__ void __launch_bounds__(128) window_dkv_kernel(const WindowBwdParams p) {
  __shared__ float sk[4][D], sv[4][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * 4 + warp;
  if (row >= (long long)p.total_k * p.hkv) return;
  const int tok = (int)(row / p.hkv), hk = (int)(row % p.hkv);
  const int b = seq_of_token(p.cu_k, p.num_seqs, tok);
  const Seq s_ = seq_of(p, b);
  const int j = tok - s_.k0, shift = s_.lk - s_.lq;
  // queries at positions [j - right, j + left] see key j; a sink is seen by all (causal: from j on)
  int i0 = max(0, j - p.right - shift), i1 = min(s_.lq, j + p.left + 1 - shift);
  if (j < p.sinks) {
    if (!p.causal) i0 = 0;
    i1 = s_.lq;
  }
  if (b >= p.num_seqs) i1 = i0;
  const T* k = static_cast<const T*>(p.k) + tok * p.k_stride + hk * D;
  const T* v = static_cast<const T*>(p.v) + tok * p.v_stride + hk * D;
  for (int d = lane; d < D; d += 32) sk[warp][d] = (float)k[d] * p.scale, sv[warp][d] = (float)v[d];
  __syncwarp();
  float dk[D / 32], dv[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) dk[i] = dv[i] = 0.f;
  for (int base = i0; base < i1; base += 32) {
    const int i = base + lane, cnt = min(32, i1 - base);
    for (int h = hk * p.g; h < (hk + 1) * p.g; ++h) {
      float pr = 0.f, ds = 0.f;
      if (i < i1) {
        const long long r = (long long)(s_.q0 + i) * p.hq + h;
        pr = expf(dot_row(sk[warp], static_cast<const T*>(p.q) + (s_.q0 + i) * p.q_stride + h * D, D) - p.lse[r]);
        ds = pr * (dot_row(sv[warp], static_cast<const T*>(p.dout) + r * D, D) - p.delta[r]);
      }
      for (int t = 0; t < cnt; ++t) {
        const float pt = __shfl_sync(0xffffffffu, pr, t), dt = __shfl_sync(0xffffffffu, ds, t);
        const T* q = static_cast<const T*>(p.q) + (s_.q0 + base + t) * p.q_stride + h * D;
        const T* dout = static_cast<const T*>(p.dout) + ((long long)(s_.q0 + base + t) * p.hq + h) * D;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          dk[c] = fmaf(dt, (float)q[lane + 32 * c], dk[c]);
          dv[c] = fmaf(pt, (float)dout[lane + 32 * c], dv[c]);
        }
      }
    }
  }
#pragma unroll
  for (int c = 0; c < D / 32; ++c) {
    static_cast<T*>(p.dk)[row * D + lane + 32 * c] = (T)(dk[c] * p.scale);
    static_cast<T*>(p.dv)[row * D + lane + 32 * c] = (T)dv[c];
  }
}

}  // namespace
}  // namespace lsrm

using namespace lsrm;

extern "C" size_t lsrm_window_attn_workspace_bytes(const lsrm_window_shape* shape) {
  if (!shape || shape->total_q < 0 || shape->num_q_heads < 1) return 0;
  return align_up((size_t)shape->total_q * shape->num_q_heads * sizeof(float), 256) + 256;
}

extern "C" int lsrm_window_attn_bwd(const lsrm_window_shape* shape, const int32_t* cu_seqlens_q,
                                    const int32_t* cu_seqlens_k, const void* q, const void* k, const void* v,
                                    const void* out, const float* lse, const void* dout, void* dq, void* dk, void* dv,
                                    void* workspace, size_t workspace_bytes, int* err_flags, void* stream) {
  int rc = check_window(shape, cu_seqlens_q, cu_seqlens_k, q, k, v);
  if (rc) return rc;
  LSRM_CHECK_ARG((shape->total_q == 0 || (out && lse && dout && dq)) && (shape->total_k == 0 || (dk && dv)),
                 "out, lse, dout and the gradients must not be NULL");
  LSRM_CHECK_ARG((((uintptr_t)out | (uintptr_t)dout | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) & 15) == 0,
                 "out, dout and the gradients must be 16-byte aligned");
  if (!workspace || workspace_bytes < lsrm_window_attn_workspace_bytes(shape)) {
    set_error("workspace too small: %zu bytes, %zu needed", workspace_bytes, lsrm_window_attn_workspace_bytes(shape));
    return LSRM_ERR_WORKSPACE;
  }
  WindowBwdParams p;
  static_cast<WindowParams&>(p) = window_params(shape, cu_seqlens_q, cu_seqlens_k, q, k, v, const_cast<void*>(out),
                                                const_cast<float*>(lse), err_flags);
  p.dout = dout, p.dq = dq, p.dk = dk, p.dv = dv;
  p.delta = static_cast<float*>(workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (p.total_q > 0) {
    ProfScope ps("window_attn_dq", s);
    const unsigned grid = (unsigned)(((long long)p.total_q * p.hq + 3) / 4);
#define CALL(BF, D) window_dq_kernel<std::conditional_t<BF, __nv_bfloat16, __half>, D><<<grid, 128, 0, s>>>(p);
    WINDOW_TYPES(CALL)
#undef CALL
    LSRM_LAUNCH_CHECK();
  }
  if (p.total_k > 0) {
    ProfScope ps("window_attn_dkv", s);
    const unsigned grid = (unsigned)(((long long)p.total_k * p.hkv + 3) / 4);
#define CALL(BF, D) window_dkv_kernel<std::conditional_t<BF, __nv_bfloat16, __half>, D><<<grid, 128, 0, s>>>(p);
    WINDOW_TYPES(CALL)
#undef CALL
    LSRM_LAUNCH_CHECK();
  }
  return LSRM_OK;
}
