// Host side of the windowed attention's entry points: argument checks, the
// parameters that the kernels share.
#pragma once

#include <algorithm>
#include <cmath>

#include "host_util.h"
#include "window_common.cuh"

namespace lsrm {

constexpr int kMaxSinks = 128;       // one key tile
constexpr int kMaxGroup = 64;        // query heads per kv head

inline int check_window(const lsrm_window_shape* s, const int32_t* cu_q, const int32_t* cu_k, const void* q, const void* k,
                 const void* v) {
  LSRM_CHECK_ARG(s, "shape must not be NULL");
  LSRM_CHECK_ARG(s->num_seqs >= 0 && s->total_q >= 0 && s->total_k >= 0, "sizes must not be negative");
  LSRM_CHECK_ARG(s->num_kv_heads >= 1 && s->num_q_heads >= 1 && s->num_q_heads % s->num_kv_heads == 0,
                 "num_q_heads (%d) must be a multiple of num_kv_heads (%d)", s->num_q_heads, s->num_kv_heads);
  LSRM_CHECK_ARG(s->num_q_heads / s->num_kv_heads <= kMaxGroup, "at most %d query heads per kv head", kMaxGroup);
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

inline WindowParams window_params(const lsrm_window_shape* s, const int32_t* cu_q, const int32_t* cu_k, const void* q,
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

#define WINDOW_TYPES(CALL)                                             \
  if (shape->dtype == LSRM_DTYPE_BF16) {                               \
    if (shape->head_dim == 32) CALL(true, 32)                          \
    else if (shape->head_dim == 64) CALL(true, 64)                     \
    else CALL(true, 128)                                               \
  } else {                                                             \
    if (shape->head_dim == 32) CALL(false, 32)                         \
    else if (shape->head_dim == 64) CALL(false, 64)                    \
    else CALL(false, 128)                                              \
  }

}  // namespace lsrm
