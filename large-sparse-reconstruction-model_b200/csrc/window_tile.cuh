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
// which every wait that is not over at once would pay before it looks again.  The
// loop is out of line: some thirty copies of it in a kernel cost its instruction
// fetch 1 to 2 % of the time (131072 tokens, 16 heads of 64 channels: forward 722
// us against 710, dQ 884 against 866, dK/dV 1016 against 1002).
// All lanes of a warp call wait_phase; false when this or another wait of the CTA
// ran out.
static __device__ __noinline__ bool wait_loop(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err) {
  bool ok;
  const long long t0 = clock64();
  while (!(ok = mbar_test(bar, parity))) {
    if (*abort_flag) break;
    if (clock64() - t0 > 2 * (long long)kWaitLimitNs) {
      *abort_flag = 1;
      if (err) atomicOr(err, LSRM_ERR_TIMEOUT);
      break;
    }
  }
  return ok;
}
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err) {
  const bool ok = mbar_test(bar, parity) || wait_loop(bar, parity, abort_flag, err);
  return __all_sync(0xffffffffu, ok);
}

// Operand descriptors of a [ROWS][D] tile, as their two words.  The upper one is
// a constant, and the lower one of a later step is the first one's plus a
// constant, so that one thread issues a product in a few instructions (building
// each descriptor from its fields took some 60 cycles a product, and the
// issuing warp bounded the kernels).
template <int D>
__device__ __forceinline__ constexpr uint32_t desc_hi() {
  using S = TileShape<D>;
  return (uint32_t)((8 * S::RB) >> 4) | (1u << 14) | ((uint32_t)S::SWZ << 29);
}
// K-major (the contraction runs over D, step ks takes 16 channels).
template <int D>
__device__ __forceinline__ uint32_t desc_k(uint32_t base) {
  return (base >> 4) | (1u << 16);
}
template <int D, int ROWS>
__device__ __forceinline__ constexpr uint32_t step_k(int ks) {
  using S = TileShape<D>;
  constexpr int per = S::kCols / 16;
  return (uint32_t)((ks / per) * ROWS * S::RB + (ks % per) * 32) >> 4;
}
// MN-major (the contraction runs over the rows, step ks takes 16 of them).
template <int D, int ROWS>
__device__ __forceinline__ uint32_t desc_mn(uint32_t base) {
  return (base >> 4) | ((uint32_t)(ROWS * TileShape<D>::RB >> 4) << 16);
}
template <int D>
__device__ __forceinline__ constexpr uint32_t step_mn(int ks) {
  return (uint32_t)(ks * 16 * TileShape<D>::RB) >> 4;
}

// D[tmem] (+)= A B, as umma_f16 / umma_f16_ts of common.cuh; ACC is known at
// compile time, or `acc` says.
template <int HI>
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %4};\n\tmov.b64 db, {%2, %4};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "n"(HI), "r"((uint32_t)acc)
      : "memory");
}
template <int HI>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
      "mov.b64 db, {%2, %4};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
      "r"(a_tmem), "r"(b), "r"(idesc), "n"(HI), "r"((uint32_t)acc)
      : "memory");
}

// D = A B^T over the D channels of an [A_ROWS][D] and a [B_ROWS][D] tile.
template <int D, int A_ROWS, int B_ROWS>
__device__ __forceinline__ void mma_rows(uint32_t d, uint32_t a_base, uint32_t b_base, uint32_t idesc) {
  const uint32_t a = desc_k<D>(a_base), b = desc_k<D>(b_base);
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks)
    mma_ss<(int)desc_hi<D>()>(d, a + step_k<D, A_ROWS>(ks), b + step_k<D, B_ROWS>(ks), idesc, ks > 0);
}
// D (+)= A B for A [128][ROWS] in TMEM and B a [ROWS][D] tile.  GAP columns lie
// between A's first 32 values and its next 32 (and so on).
template <int D, int ROWS, int GAP = 0>
__device__ __forceinline__ void mma_sum(uint32_t d, uint32_t a_tmem, uint32_t b_base, uint32_t idesc, bool acc,
                                        int steps = ROWS / 16) {
  const uint32_t b = desc_mn<D, ROWS>(b_base);
#pragma unroll
  for (int ks = 0; ks < ROWS / 16; ++ks)
    if (ks < steps)
      mma_ts<(int)desc_hi<D>()>(d, a_tmem + ks * 8 + (ks / 2) * GAP, b + step_mn<D>(ks), idesc, acc || ks > 0);
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

// Bits [lo, hi) of 32.
__device__ __forceinline__ uint32_t range_bits(int lo, int hi) {
  lo = max(lo, 0);
  hi = min(hi, 32);
  if (hi <= lo) return 0u;
  return (0xffffffffu >> (32 - (hi - lo))) << lo;
}

// Writes 32 channels of a warp's 32 rows (packed in w[16], a row a lane) to
// out + row * ld + c, `row` negative: none.  Straight from the lanes each store
// would touch 32 lines, which took longer than an item's last products; through
// `buf` (2 KB of the warp's own) four lanes write a row's 64 bytes.
constexpr int kRowBuf = 32 * 64;
__device__ __forceinline__ void store_rows32(uint32_t buf, const uint32_t* w, long long row, uint16_t* out, int ld,
                                             int c) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    st_shared_v4(buf + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4), w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = i * 8 + (lane >> 2), ch = lane & 3;
    uint32_t v[4];
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                 : "r"(buf + r * 64 + ((ch ^ ((r >> 1) & 3)) << 4))
                 : "memory");
    const long long at = __shfl_sync(0xffffffffu, row, r);
    if (at >= 0) *reinterpret_cast<uint4*>(out + at * ld + c + ch * 8) = make_uint4(v[0], v[1], v[2], v[3]);
  }
  __syncwarp();
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

// ---------------------------------------------------------------------------
// Work items of the kernels that keep query rows (forward, dQ): two
// tiles of TT tokens x G heads, one kv head, and the key tiles (KT keys) that
// either sees.  The producer plans them; the other warps read them from a ring.
// ---------------------------------------------------------------------------
constexpr int kItems = 4;

struct RowItem {
  int stop;         // 1: no more items
  int tok;          // first query token (global)
  int n[2];         // query tokens of each row tile
  int hk, pos, lk;  // kv head, position of the first query, keys of the sequence
  int key0;         // first key of the sequence (global)
  int tiles, sep;   // key tiles; the first `sep` of them hold the sinks alone, apart from the window
  int w0;           // first key of the window's first tile
  int a[2], b[2];   // key tiles [a, b) of each row tile

  template <int KT>
  __device__ __forceinline__ int key(int t) const {
    return t < sep ? KT * t : w0 + KT * (t - sep);
  }
  // Keys of tile t that exist (the rest of the tile lies past the sequence).
  template <int KT>
  __device__ __forceinline__ int valid(int t) const {
    return min(KT, lk - key<KT>(t));
  }
};

// Plans work item `w`; false when it holds no query.
template <int KT>
__device__ __forceinline__ bool row_item(const WindowParams& p, int w, int tt, RowItem& it) {
  const int slot = w / p.hkv;
  it.hk = w - slot * p.hkv;
  const int b = seq_of_slot(p.cu_q, p.num_seqs, 2 * tt, slot);
  const Seq s = seq_of(p, b);
  const int i0 = (slot - first_slot(p.cu_q, b, 2 * tt)) * 2 * tt;
  if (i0 < 0 || i0 >= s.lq) return false;
  it.tok = s.q0 + i0;
  it.n[0] = min(tt, s.lq - i0);
  it.n[1] = max(0, min(tt, s.lq - i0 - tt));
  it.lk = b >= 0 && b < p.num_seqs ? s.lk : 0;
  it.pos = i0 + s.lk - s.lq;
  it.key0 = s.k0;
  int lo[2], hi[2], sink[2], first = 0x7fffffff, end = 0, top = 0;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    lo[u] = hi[u] = sink[u] = 0;
    if (it.n[u] <= 0) continue;
    const RowKeys r0 = row_keys(p, it.pos + u * tt, it.lk), r1 = row_keys(p, it.pos + u * tt + it.n[u] - 1, it.lk);
    sink[u] = max(r1.sink, 0);
    top = max(top, sink[u]);
    if (r1.hi <= r0.lo) continue;
    lo[u] = r0.lo;
    hi[u] = r1.hi;
    first = min(first, lo[u]);
    end = max(end, hi[u]);
  }
  const bool apart = top > 0 && end > 0 && first > top;
  it.sep = apart ? (top + KT - 1) / KT : 0;
  if (end == 0) first = 0;
  if (!apart && top > 0) first = 0, end = max(end, top);
  it.w0 = first;
  it.tiles = (end - first + KT - 1) / KT + it.sep;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    int x = it.tiles, y = 0;
    if (hi[u] > lo[u]) x = (lo[u] - first) / KT + it.sep, y = (hi[u] - first + KT - 1) / KT + it.sep;
    if (sink[u] > 0) x = 0, y = max(y, (sink[u] + KT - 1) / KT);
    it.a[u] = y > x ? x : 0;
    it.b[u] = y > x ? y : 0;
  }
  return true;
}

// What one row of an item sees of its key tiles, and which of the tiles every
// row of the warp sees whole (between a window's edges: two comparisons a tile;
// spelling the masks out for each took longer than the exponentials).
template <int KT>
struct RowView {
  int lo, hi, sink;  // columns of the window's first tile (`sink`: of the item's first tile)
  int sep;
  int full0, full1;  // tiles [full0, full1) need no mask
  bool live;

  __device__ __forceinline__ RowView(const WindowParams& p, const RowItem& it, int pos, bool is_live, int col0, int cols) {
    const RowKeys k = row_keys(p, pos, it.lk);
    live = is_live;
    sep = it.sep;
    lo = k.lo - it.w0;
    hi = k.hi - it.w0;
    sink = k.sink;
    const int all_lo = __reduce_max_sync(0xffffffffu, live ? lo : 0) - col0;
    const int all_hi = __reduce_min_sync(0xffffffffu, live ? hi : 0x3fffffff) - col0 - cols;
    full0 = sep + (max(all_lo, 0) + KT - 1) / KT;
    full1 = all_hi < 0 ? 0 : sep + all_hi / KT + 1;
  }
  __device__ __forceinline__ bool full(int t) const { return t >= full0 && t < full1; }
  // Visibility of columns c0 .. c0 + 31 of tile t.
  __device__ __forceinline__ uint32_t bits(int t, int c0) const {
    if (!live) return 0u;
    if (t < sep) return range_bits(-1, sink - KT * t - c0);
    const int at = KT * (t - sep) + c0;
    return range_bits(lo - at, hi - at) | (sep ? 0u : range_bits(-1, sink - at));
  }
};

// This warp's 32 lanes x 4 TMEM columns from v[0..4) (see tmem_st16).
__device__ __forceinline__ void tmem_st4(uint32_t taddr, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(taddr), "r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3])
               : "memory");
}

}  // namespace lsrm
