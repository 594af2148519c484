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

#include "host_util.h"
#include "window_common.cuh"

namespace lsrm {
namespace {

constexpr int kMaxD = 128;
constexpr int kMaxSinks = 128;

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

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T, int D>
__global__ void __launch_bounds__(128) window_fwd_kernel(const WindowParams p) {
  __shared__ float sq[4][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * 4 + warp;
  if (row >= (long long)p.total_q * p.hq) return;
  const int tok = (int)(row / p.hq), h = (int)(row % p.hq), hk = h / p.g;
  const int b = seq_of_token(p.cu_q, p.num_seqs, tok);
  const Seq sq_ = seq_of(p, b);
  const int pos = tok - sq_.q0 + sq_.lk - sq_.lq;
  const Seen seen = keys_of(p, pos, sq_.lk, b < p.num_seqs);
  const T* q = static_cast<const T*>(p.q) + tok * p.q_stride + h * D;
  for (int d = lane; d < D; d += 32) sq[warp][d] = (float)q[d] * p.scale;
  __syncwarp();
  const T* k = static_cast<const T*>(p.k) + sq_.k0 * p.k_stride + hk * D;
  const T* v = static_cast<const T*>(p.v) + sq_.k0 * p.v_stride + hk * D;
  float m = -INFINITY, l = 0.f, acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) acc[i] = 0.f;
  const int n = seen.sink + seen.hi - seen.lo;
  for (int base = 0; base < n; base += 32) {
    const int idx = base + lane;
    const int j = idx < seen.sink ? idx : seen.lo + idx - seen.sink;
    const float s = idx < n ? dot_row(sq[warp], k + j * p.k_stride, D) : -INFINITY;
    const float m_new = fmaxf(m, warp_max(s));
    const float off = m_new == -INFINITY ? 0.f : m_new;
    const float r = expf(m - off), e = expf(s - off);
    l = l * r + warp_sum(e);
    m = m_new;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] *= r;
    const int cnt = min(32, n - base);
    for (int t = 0; t < cnt; ++t) {
      const float pt = __shfl_sync(0xffffffffu, e, t);
      const int jt = __shfl_sync(0xffffffffu, j, t);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) acc[i] = fmaf(pt, (float)v[jt * p.v_stride + lane + 32 * i], acc[i]);
    }
  }
  T* out = static_cast<T*>(p.out) + row * D;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) out[lane + 32 * i] = (T)(l == 0.f ? 0.f : acc[i] / l);
  if (lane == 0) p.lse[row] = l == 0.f ? -INFINITY : m + logf(l);
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

int check_window(const lsrm_window_shape* s, const int32_t* cu_q, const int32_t* cu_k, const void* q, const void* k,
                 const void* v) {
  LSRM_CHECK_ARG(s, "shape must not be NULL");
  LSRM_CHECK_ARG(s->num_seqs >= 0 && s->total_q >= 0 && s->total_k >= 0, "sizes must not be negative");
  LSRM_CHECK_ARG(s->num_kv_heads >= 1 && s->num_q_heads >= 1 && s->num_q_heads % s->num_kv_heads == 0,
                 "num_q_heads (%d) must be a multiple of num_kv_heads (%d)", s->num_q_heads, s->num_kv_heads);
  LSRM_CHECK_ARG(s->num_q_heads / s->num_kv_heads <= 64, "at most 64 query heads per kv head");
  LSRM_CHECK_ARG(s->head_dim == 32 || s->head_dim == 64 || s->head_dim == 128, "head_dim (%d) must be 32, 64 or 128",
                 s->head_dim);
  LSRM_CHECK_ARG(s->dtype == LSRM_DTYPE_BF16 || s->dtype == LSRM_DTYPE_F16, "dtype must be bf16 or fp16");
  LSRM_CHECK_ARG(s->window >= 1, "window (%d) must be at least 1", s->window);
  LSRM_CHECK_ARG(s->sinks >= 0 && s->sinks <= kMaxSinks, "sinks (%d) must be in [0, %d]", s->sinks, kMaxSinks);
  const int64_t qr = (int64_t)s->num_q_heads * s->head_dim, kr = (int64_t)s->num_kv_heads * s->head_dim;
  LSRM_CHECK_ARG(s->q_token_stride >= qr && s->k_token_stride >= kr && s->v_token_stride >= kr,
                 "token strides must cover the heads");
  LSRM_CHECK_ARG(s->q_token_stride % 8 == 0 && s->k_token_stride % 8 == 0 && s->v_token_stride % 8 == 0,
                 "token strides must be multiples of 8 elements");
  LSRM_CHECK_ARG((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) & 15) == 0, "q, k and v must be 16-byte aligned");
  LSRM_CHECK_ARG(cu_q && cu_k, "the sequence offsets must not be NULL");
  LSRM_CHECK_ARG((s->total_q == 0 || q) && (s->total_k == 0 || (k && v)), "q, k and v must not be NULL");
  return LSRM_OK;
}

WindowParams window_params(const lsrm_window_shape* s, const int32_t* cu_q, const int32_t* cu_k, const void* q,
                           const void* k, const void* v, void* out, float* lse, int* err) {
  WindowParams p{};
  p.num_seqs = s->num_seqs, p.total_q = s->total_q, p.total_k = s->total_k;
  p.hq = s->num_q_heads, p.hkv = s->num_kv_heads, p.g = p.hq / p.hkv;
  p.left = s->causal ? s->window - 1 : s->window / 2;
  p.right = s->causal ? 0 : s->window / 2;
  // reaches past every key are the same reach: keeps the index arithmetic in range
  p.left = std::min(p.left, std::max(p.total_q, p.total_k));
  p.right = std::min(p.right, std::max(p.total_q, p.total_k));
  p.sinks = s->sinks, p.causal = s->causal;
  p.scale = s->softmax_scale > 0.f ? s->softmax_scale : 1.f / sqrtf((float)s->head_dim);
  p.cu_q = cu_q, p.cu_k = cu_k;
  p.q_stride = s->q_token_stride, p.k_stride = s->k_token_stride, p.v_stride = s->v_token_stride;
  p.q = q, p.k = k, p.v = v, p.out = out, p.lse = lse, p.err = err;
  return p;
}

}  // namespace
}  // namespace lsrm

using namespace lsrm;

#define WINDOW_TYPES(CALL)                                             \
  if (shape->dtype == LSRM_DTYPE_BF16) {                               \
    if (shape->head_dim == 32) CALL(__nv_bfloat16, 32)                 \
    else if (shape->head_dim == 64) CALL(__nv_bfloat16, 64)            \
    else CALL(__nv_bfloat16, 128)                                      \
  } else {                                                             \
    if (shape->head_dim == 32) CALL(__half, 32)                        \
    else if (shape->head_dim == 64) CALL(__half, 64)                   \
    else CALL(__half, 128)                                             \
  }

extern "C" int lsrm_window_attn_fwd(const lsrm_window_shape* shape, const int32_t* cu_seqlens_q,
                                    const int32_t* cu_seqlens_k, const void* q, const void* k, const void* v,
                                    void* out, float* lse, int* err_flags, void* stream) {
  int rc = check_window(shape, cu_seqlens_q, cu_seqlens_k, q, k, v);
  if (rc) return rc;
  if (shape->total_q == 0) return LSRM_OK;
  LSRM_CHECK_ARG(out && lse, "out and lse must not be NULL");
  const WindowParams p = window_params(shape, cu_seqlens_q, cu_seqlens_k, q, k, v, out, lse, err_flags);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  ProfScope ps("window_attn_fwd", s);
  const unsigned grid = (unsigned)(((long long)p.total_q * p.hq + 3) / 4);
#define CALL(T, D) window_fwd_kernel<T, D><<<grid, 128, 0, s>>>(p);
  WINDOW_TYPES(CALL)
#undef CALL
  LSRM_LAUNCH_CHECK();
  return LSRM_OK;
}

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
#define CALL(T, D) window_dq_kernel<T, D><<<grid, 128, 0, s>>>(p);
    WINDOW_TYPES(CALL)
#undef CALL
    LSRM_LAUNCH_CHECK();
  }
  if (p.total_k > 0) {
    ProfScope ps("window_attn_dkv", s);
    const unsigned grid = (unsigned)(((long long)p.total_k * p.hkv + 3) / 4);
#define CALL(T, D) window_dkv_kernel<T, D><<<grid, 128, 0, s>>>(p);
    WINDOW_TYPES(CALL)
#undef CALL
    LSRM_LAUNCH_CHECK();
  }
  return LSRM_OK;
}
