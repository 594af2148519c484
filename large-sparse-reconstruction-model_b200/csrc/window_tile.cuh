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

// Waits for the outstanding TMEM loads, and ties the 32 values of one of them
// to the wait: nothing that reads them may be scheduled ahead of it.
__device__ __forceinline__ void tmem_wait_ld32(float* v) {
  tmem_wait_ld();
  asm volatile(""
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
               "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]),
               "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]),
               "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]),
               "+f"(v[29]), "+f"(v[30]), "+f"(v[31]));
}

template <int N>
__device__ __forceinline__ void tmem_store_cols(uint32_t taddr, const uint32_t* v) {
  static_assert(N % 16 == 0, "whole sixteens");
#pragma unroll
  for (int c = 0; c < N; c += 16) tmem_st16(taddr + c, v + c);
}

}  // namespace lsrm
