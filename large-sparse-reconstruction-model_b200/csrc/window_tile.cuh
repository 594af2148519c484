// Device pieces of the windowed attention's tensor-core kernels: packed query
// rows, operand tiles in shared memory, the work items and their hand-over.
//
// Rows.  The query heads of one kv head read the same keys, so a tile's rows
// are packed (token, head) pairs: a TMA box of TT = R / G tokens x G heads
// lands as rows t * G + g (R = 128 or 64 rows; TT * G of them are used).  A
// window of W keys then spans W + TT rather than W + R keys a tile.
//
// Tiles.  A [rows][D] operand is stored as D / 64 sub-tiles of 64 channels
// (128-byte rows, 128-byte swizzle), or one of 32 channels (64-byte rows).
#pragma once

#include "common.cuh"
#include "window_common.cuh"

namespace lsrm {

template <int D>
struct TileShape {
  static constexpr int kSubs = D > 64 ? D / 64 : 1;    // sub-tiles
  static constexpr int kCols = D > 64 ? 64 : D;        // channels of one
  static constexpr int RB = 2 * kCols;                 // bytes of its row
  static constexpr uint64_t SWZ = swz_for_row_bytes(RB);
  static constexpr int bytes(int rows) { return rows * 2 * D; }
};

// Waits for a barrier's phase, bounded like common.cuh's waits (kWaitLimitNs at
// 2 GHz) but on the cycle counter: %globaltimer takes some 500 cycles to read,
// which every wait that is not over at once would pay before it looks again.
// All lanes of a warp call it; false when this or another wait of the CTA ran out.
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err) {
  bool ok = mbar_test(bar, parity);
  if (!ok) {
    const long long t0 = clock64();
    while (!(ok = mbar_test(bar, parity))) {
      if (*abort_flag) break;
      if (clock64() - t0 > 2 * (long long)kWaitLimitNs) {
        *abort_flag = 1;
        if (err) atomicOr(err, LSRM_ERR_TIMEOUT);
        break;
      }
    }
  }
  return __all_sync(0xffffffffu, ok);
}

// Descriptors of a [rows][D] tile at shared address `base`: as a K-major
// operand (the contraction runs over D; step ks takes 16 channels), and as an
// MN-major one (the contraction runs over the rows; step ks takes 16 of them).
template <int D>
__device__ __forceinline__ uint64_t desc_k(uint32_t base, int rows, int ks) {
  using S = TileShape<D>;
  constexpr int per = S::kCols / 16;
  return make_sdesc(base + (ks / per) * rows * S::RB + (ks % per) * 32, 16, 8 * S::RB, S::SWZ);
}
template <int D>
__device__ __forceinline__ uint64_t desc_mn(uint32_t base, int rows, int ks) {
  using S = TileShape<D>;
  return make_sdesc(base + ks * 16 * S::RB, rows * S::RB, 8 * S::RB, S::SWZ);
}

// TMA of one operand tile: rows of `heads` heads x tokens from (head, token).
template <int D>
__device__ __forceinline__ void load_tile(uint8_t* dst, int rows, const CUtensorMap* map, int head, int token,
                                          uint64_t* bar) {
  using S = TileShape<D>;
#pragma unroll
  for (int i = 0; i < S::kSubs; ++i) tma_load_3d(dst + i * rows * S::RB, map, i * S::kCols, head, token, bar);
}

// Zeroes rows [from, rows) of a tile that TMA has filled (one warp), and makes
// the zeros visible to the tensor core: what lies past a sequence's end must
// not reach a product, not even times zero.
template <int D>
__device__ __forceinline__ void zero_rows(uint8_t* tile, int rows, int from) {
  using S = TileShape<D>;
  constexpr int per = S::RB / 16;
  const int n = (rows - from) * per;
  for (int i = threadIdx.x & 31; i < n * S::kSubs; i += 32) {
    const int sub = i / n, r = i - sub * n;
    reinterpret_cast<uint4*>(tile + sub * rows * S::RB + from * S::RB)[r] = make_uint4(0u, 0u, 0u, 0u);
  }
  fence_proxy_async_smem();
  __syncwarp();
}

// 32 visibility bits (columns c0 .. c0 + 31 of a key tile): columns [lo, hi)
// and [0, sink).
__device__ __forceinline__ uint32_t range_bits(int lo, int hi) {
  lo = max(lo, 0);
  hi = min(hi, 32);
  if (hi <= lo) return 0u;
  return (0xffffffffu >> (32 - (hi - lo))) << lo;
}
__device__ __forceinline__ uint32_t seen_bits(int lo, int hi, int sink, int c0) {
  return range_bits(lo - c0, hi - c0) | range_bits(-1, sink - c0);
}

// Two-lane fp32 arithmetic (one issue slot for two results).
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(r))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)),
        "l"(reinterpret_cast<const uint64_t&>(c)));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(r))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(r))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
  return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ float max32(const float* s) {
  float m[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    m[j] = fmaxf(s[j], s[j + 4]);
#pragma unroll
    for (int i = 8; i < 32; i += 8) m[j] = max3(m[j], s[i + j], s[i + j + 4]);
  }
  return fmaxf(max3(m[0], m[1], m[2]), m[3]);
}

// Scores outside `bits` to -inf (whatever they hold).
__device__ __forceinline__ void mask32(float* s, uint32_t bits) {
#pragma unroll
  for (int i = 0; i < 32; ++i) s[i] = (bits >> i & 1u) ? s[i] : -INFINITY;
}

// Keys that one row sees, before the window and the sinks are merged: [lo, hi)
// and [0, sink).
struct RowKeys {
  int lo, hi, sink;
};
__device__ __forceinline__ RowKeys row_keys(const WindowParams& p, int pos, int lk) {
  RowKeys r;
  r.lo = max(0, pos - p.left);
  r.hi = min(lk, pos + p.right + 1);
  r.sink = min(min(p.sinks, lk), p.causal ? pos + 1 : lk);
  return r;
}

// Waits for the outstanding TMEM loads, and ties the N values of one of them
// to the wait: nothing that reads them may be scheduled ahead of it.
template <int N>
__device__ __forceinline__ void tmem_wait_values(float* v) {
  tmem_wait_ld();
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+f"(v[i]));
}

template <int N>
__device__ __forceinline__ void tmem_store_cols(uint32_t taddr, const uint32_t* v) {
  static_assert(N % 16 == 0, "whole sixteens");
#pragma unroll
  for (int c = 0; c < N; c += 16) tmem_st16(taddr + c, v + c);
}

}  // namespace lsrm
