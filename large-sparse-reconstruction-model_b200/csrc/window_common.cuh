// What the windowed attention kernels share: which keys a query sees.
//
// Query i of a sequence with Lq queries and Lk keys stands at position
// pos = i + Lk - Lq.  It sees key j (0 <= j < Lk) when
//   causal:     j <= pos and (pos - j < window or j < sinks)
//   symmetric:  |pos - j| <= window / 2 or j < sinks.
#pragma once

#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "lsrm_sparse.h"

namespace lsrm {

// The two 16-bit values of a packed word.
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if constexpr (BF16) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
  } else {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
  }
}

struct WindowParams {
  int num_seqs, total_q, total_k;
  int hq, hkv, g;        // query heads, kv heads, query heads per kv head
  int left, right;       // the window's reach on both sides of pos
  int sinks, causal;
  float scale;           // softmax scale
  const int32_t *cu_q, *cu_k;
  long long q_stride, k_stride, v_stride;  // elements between tokens
  const void *q, *k, *v;
  void *out, *out_rest;  // out_rest: what out's rounding left over, may be null
  float* lse;            // [total_q, hq], natural log
  int* err;
};

// One sequence's tokens.  Index -1 stands for the tokens before the first
// sequence and num_seqs for those after the last one, which see and are seen by
// nothing (their outputs are zero).
struct Seq {
  int q0, lq, k0, lk;
};

__device__ __forceinline__ Seq seq_of(const WindowParams& p, int b) {
  const bool head = b < 0, tail = b >= p.num_seqs;
  int q0 = head ? 0 : p.cu_q[b], k0 = head ? 0 : p.cu_k[b];
  int q1 = tail ? p.total_q : p.cu_q[b + 1], k1 = tail ? p.total_k : p.cu_k[b + 1];
  // offsets outside the tensors or out of order: report and touch nothing
  if (q0 < 0 || q1 < q0 || q1 > p.total_q || k0 < 0 || k1 < k0 || k1 > p.total_k) {
    if (p.err) atomicOr(p.err, LSRM_ERR_BAD_INDEX);
    return Seq{0, 0, 0, 0};
  }
  return Seq{q0, q1 - q0, k0, k1 - k0};
}

// Tiles of `rows` tokens of ragged sequences: sequence b's tiles start at slot
// cu[b] / rows + b + 1 (those of the tokens before the first one at slot 0),
// which leaves each as many slots as it has tiles; total / rows + num_seqs + 2
// slots cover all, the tokens after the last sequence included.
__host__ __device__ __forceinline__ int tile_slots(int total, int num_seqs, int rows) {
  return total / rows + num_seqs + 2;
}

__device__ __forceinline__ int first_slot(const int32_t* cu, int b, int rows) { return b < 0 ? 0 : cu[b] / rows + b + 1; }

__device__ __forceinline__ int seq_of_slot(const int32_t* cu, int num_seqs, int rows, int slot) {
  int lo = -1, hi = num_seqs;  // the last index whose first slot is <= slot
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first_slot(cu, mid, rows) <= slot) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

}  // namespace lsrm
