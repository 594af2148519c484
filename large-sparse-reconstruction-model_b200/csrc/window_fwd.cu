// Forward of the attention with a sliding window and sinks (window_common.cuh
// says which keys a query sees):
//   s_ij = scale q_i . k_j,  lse_i = log sum_j exp s_ij,
//   o_i = sum_j exp(s_ij - lse_i) v_j      (no key: o = 0, lse = -inf)
//
// One pass over a query's keys with a running maximum and sum.  A persistent
// CTA per multiprocessor walks work items (two tiles of 128 packed query rows
// of one kv head and the keys that either sees):
//   warps 0-3, 4-7  softmax of row tile 0 and 1, a row a thread: S from TMEM,
//                   mask, running maximum, P = exp2(S - m) back over S as
//                   16-bit operand, at the end O / l to global memory
//   warps 8, 9      tensor-core issue for row tile 0 and 1: S = Q K^T, O += P V
//                   (P from TMEM); while one tile is in its softmax the other
//                   one's products run
//   warp 10         producer: work items, TMA of Q, K and V
// K and V tiles (128 keys) go through one ring and serve both row tiles, which
// halves the L2 reads per product.  Rounding: S, m, l and O are fp32; P is
// rounded to the operand type (the sum l takes it unrounded), O once at the end.
#include "window_host.h"
#include "window_tile.cuh"

namespace lsrm {
namespace {

constexpr int kFwThreads = 352;
constexpr int kFwItems = 4;  // work items in flight between the producer and the other warps

struct FwItem {
  int stop;         // 1: no more items
  int tok;          // first query token (global)
  int n[2];         // query tokens of each row tile
  int hk, pos, lk;  // kv head, position of the first query, keys of the sequence
  int key0;         // first key of the sequence (global)
  int tiles, sep;   // key tiles; 1: tile 0 holds the sinks alone, ahead of the window
  int w0;           // first key of the window's first tile
  int a[2], b[2];   // key tiles [a, b) of each row tile
};

template <int D>
struct FwSmem {
  static constexpr int TILE = TileShape<D>::bytes(128);
  static constexpr int NQ = D == 128 ? 1 : 2;  // Q buffers of each row tile
  static constexpr int NS = D == 128 ? 5 : 8;  // K / V ring
  static constexpr int OFF_KV = 2 * NQ * TILE;
  static constexpr int OFF_ITEM = OFF_KV + NS * TILE;
  static constexpr int OFF_BAR = OFF_ITEM + kFwItems * (int)sizeof(FwItem);
  // q_full[2][NQ], q_empty[2][NQ], kv_full[NS], kv_empty[NS], s_full[2], p_full[2], pv_done[2], item_full[],
  // item_empty[], mma_done[2]
  static constexpr int NBAR = 4 * NQ + 2 * NS + 6 + 2 * kFwItems + 2;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int BYTES = OFF_MISC + 16 + 1024;
  static constexpr int ALLOC = BYTES > kOneCtaPerSmSmem ? BYTES : kOneCtaPerSmSmem;
  static_assert(OFF_BAR % 8 == 0 && ALLOC <= 227 * 1024, "shared memory budget");
};

// First key of key tile t.
__device__ __forceinline__ int tile_key(const FwItem& it, int t) {
  return it.sep ? (t == 0 ? 0 : it.w0 + 128 * (t - 1)) : it.w0 + 128 * t;
}
// Keys of tile t that exist (the rest of the tile lies past the sequence).
__device__ __forceinline__ int tile_valid(const FwItem& it, int t) { return min(128, it.lk - tile_key(it, t)); }

// The keys that the row tiles of an item see, as key tiles.
__device__ __forceinline__ void plan_tiles(const WindowParams& p, FwItem& it, int tt) {
  int lo[2], hi[2], sink[2], first = 0x7fffffff, end = 0, top = 0;
  for (int u = 0; u < 2; ++u) {
    lo[u] = hi[u] = sink[u] = 0;
    if (it.n[u] <= 0) continue;
    const RowKeys r0 = row_keys(p, it.pos + u * tt, it.lk), r1 = row_keys(p, it.pos + u * tt + it.n[u] - 1, it.lk);
    lo[u] = r0.lo;
    hi[u] = max(r1.hi, 0);
    sink[u] = max(r1.sink, 0);
    if (hi[u] > lo[u]) first = min(first, lo[u]), end = max(end, hi[u]);
    else lo[u] = hi[u] = 0;
    top = max(top, sink[u]);
  }
  it.sep = top > 0 && end > 0 && first > top;  // window and sinks apart: the sinks get a tile of their own
  if (end == 0) first = 0;
  if (!it.sep && top > 0) first = 0, end = max(end, top);
  it.w0 = first;
  const int wt = (end - first + 127) / 128;
  it.tiles = wt + it.sep;
  for (int u = 0; u < 2; ++u) {
    int a = it.tiles, b = 0;
    if (hi[u] > lo[u]) a = (lo[u] - first) / 128 + it.sep, b = (hi[u] - first + 127) / 128 + it.sep;
    if (sink[u] > 0) a = 0, b = max(b, it.sep ? 1 : (sink[u] + 127) / 128);
    it.a[u] = b > a ? a : 0;
    it.b[u] = b > a ? b : 0;
  }
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kFwThreads, 1)
    window_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const WindowParams p, const int n_items) {
  using L = FwSmem<D>;
  constexpr uint32_t AB = BF16 ? 1u : 0u;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sKV = smem + L::OFF_KV;
  FwItem* items = reinterpret_cast<FwItem*>(smem + L::OFF_ITEM);
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* q_empty = q_full + 2 * L::NQ;
  uint64_t* kv_full = q_empty + 2 * L::NQ;
  uint64_t* kv_empty = kv_full + L::NS;
  uint64_t* s_full = kv_empty + L::NS;
  uint64_t* p_full = s_full + 2;
  uint64_t* pv_done = p_full + 2;
  uint64_t* item_full = pv_done + 2;
  uint64_t* item_empty = item_full + kFwItems;
  uint64_t* mma_done = item_empty + kFwItems;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::OFF_MISC + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = p.g, TT = 128 / G;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2 * L::NQ; ++i) mbar_init(&q_full[i], 1), mbar_init(&q_empty[i], 1);
    for (int i = 0; i < L::NS; ++i) mbar_init(&kv_full[i], 1), mbar_init(&kv_empty[i], 2);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&pv_done[i], 1);
      mbar_init(&mma_done[i], 1);
    }
    for (int i = 0; i < kFwItems; ++i) mbar_init(&item_full[i], 1), mbar_init(&item_empty[i], 10);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 10) {
    // ------------------------------ producer ------------------------------
    if (lane == 0) {
      tma_prefetch_desc(&tm_q);
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
      const uint32_t q_bytes = (uint32_t)(G * TT * D * 2);
      int n_it = 0, J = 0, nq[2] = {0, 0};
      bool ok = true;
      for (int w = blockIdx.x; ok; w += gridDim.x) {
        FwItem it;
        it.stop = w >= n_items;
        if (!it.stop) {
          const int slot = w / p.hkv;
          it.hk = w - slot * p.hkv;
          const int b = seq_of_slot(p.cu_q, p.num_seqs, 2 * TT, slot);
          const Seq s = seq_of(p, b);
          const int i0 = (slot - (p.cu_q[b] / (2 * TT) + b)) * 2 * TT;
          if (i0 < 0 || i0 >= s.lq) continue;
          it.tok = s.q0 + i0;
          it.n[0] = min(TT, s.lq - i0);
          it.n[1] = max(0, min(TT, s.lq - i0 - TT));
          it.lk = b < p.num_seqs ? s.lk : 0;
          it.pos = i0 + s.lk - s.lq;
          it.key0 = s.k0;
          plan_tiles(p, it, TT);
        }
        const int r = n_it % kFwItems;
        if (!mbar_wait(&item_empty[r], ((n_it / kFwItems) & 1) ^ 1, abort_flag, p.err)) { ok = false; break; }
        items[r] = it;
        mbar_arrive(&item_full[r]);
        ++n_it;
        if (it.stop) break;
        for (int u = 0; u < 2 && ok; ++u) {
          if (it.b[u] <= it.a[u]) continue;
          const int st = u * L::NQ + nq[u] % L::NQ;
          if (!mbar_wait(&q_empty[st], ((nq[u] / L::NQ) & 1) ^ 1, abort_flag, p.err)) { ok = false; break; }
          mbar_arrive_expect_tx(&q_full[st], q_bytes);
          load_tile<D>(sQ + st * L::TILE, 128, &tm_q, it.hk * G, it.tok + u * TT, &q_full[st]);
          ++nq[u];
        }
        for (int t = 0; t < it.tiles && ok; ++t) {
          const int key = it.key0 + tile_key(it, t);
          for (int kv = 0; kv < 2; ++kv, ++J) {
            const int st = J % L::NS;
            if (!mbar_wait(&kv_empty[st], ((J / L::NS) & 1) ^ 1, abort_flag, p.err)) { ok = false; break; }
            mbar_arrive_expect_tx(&kv_full[st], L::TILE);
            load_tile<D>(sKV + st * L::TILE, 128, kv ? &tm_v : &tm_k, it.hk, key, &kv_full[st]);
          }
        }
      }
      // after an abort: copies in flight land before the CTA exits
      if (*abort_flag) {
        for (int u = 0; u < 2; ++u)
          for (int k = max(0, nq[u] - L::NQ); k < nq[u]; ++k)
            mbar_wait_drain(&q_full[u * L::NQ + k % L::NQ], (k / L::NQ) & 1);
        for (int j = max(0, J - L::NS); j < J; ++j) mbar_wait_drain(&kv_full[j % L::NS], (j / L::NS) & 1);
      }
    }
    __syncwarp();
  } else if (warp >= 8) {
    // --------------------------- tensor-core issue ---------------------------
    const int u = warp - 8;
    const uint32_t tm_s = tmem + u * 128, tm_o = tmem + 256 + u * D;
    const uint32_t idesc_o = make_idesc(AB, 0, 1, 128, D);
    int n_it = 0, J = 0, nq = 0, np = 0;
    bool ok = true;
    while (ok) {
      const int r = n_it % kFwItems;
      if (!warp_wait(&item_full[r], (n_it / kFwItems) & 1, abort_flag, p.err)) break;
      const FwItem& it = items[r];
      ++n_it;
      if (it.stop) break;
      const int st_q = u * L::NQ + nq % L::NQ;
      const uint32_t q_base = smem_u32(sQ + st_q * L::TILE);
      const int a = it.a[u], b = it.b[u];
      if (b > a && !warp_wait(&q_full[st_q], (nq / L::NQ) & 1, abort_flag, p.err)) break;
      for (int t = 0; t < it.tiles; ++t, J += 2) {
        const int sk = J % L::NS, sv = (J + 1) % L::NS;
        if (!warp_wait(&kv_full[sk], (J / L::NS) & 1, abort_flag, p.err)) { ok = false; break; }
        if (t < a || t >= b) {  // the other row tile's keys only
          if (!warp_wait(&kv_full[sv], ((J + 1) / L::NS) & 1, abort_flag, p.err)) { ok = false; break; }
          if (lane == 0) {
            mbar_arrive(&kv_empty[sk]);
            mbar_arrive(&kv_empty[sv]);
          }
          continue;
        }
        // sinks of their own tile: only as many columns as they need
        const int cols = it.sep && t == 0 ? (p.sinks + 31) / 32 * 32 : 128;
        // P lies over S: the last product that reads it has to be over
        if (np > 0 && !warp_wait(&pv_done[u], (np - 1) & 1, abort_flag, p.err)) { ok = false; break; }
        tc_fence_after();
        if (lane == 0) {
          const uint32_t k_base = smem_u32(sKV + sk * L::TILE);
          const uint32_t idesc_s = make_idesc(AB, 0, 0, 128, cols);
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks)
            umma_f16(tm_s, desc_k<D>(q_base, 128, ks), desc_k<D>(k_base, 128, ks), idesc_s, ks > 0);
          umma_commit(&s_full[u]);
          umma_commit(&kv_empty[sk]);
          if (t == b - 1) umma_commit(&q_empty[st_q]);
        }
        __syncwarp();
        if (!warp_wait(&kv_full[sv], ((J + 1) / L::NS) & 1, abort_flag, p.err)) { ok = false; break; }
        const int valid = tile_valid(it, t);
        if (valid < cols) zero_rows<D>(sKV + sv * L::TILE, 128, valid);
        if (!warp_wait(&p_full[u], np & 1, abort_flag, p.err)) { ok = false; break; }
        ++np;
        tc_fence_after();
        if (lane == 0) {
          const uint32_t v_base = smem_u32(sKV + sv * L::TILE);
          for (int ks = 0; ks < cols / 16; ++ks)
            umma_f16_ts(tm_o, tm_s + ks * 8, desc_mn<D>(v_base, 128, ks), idesc_o, (t > a || ks > 0) ? 1u : 0u);
          umma_commit(&pv_done[u]);
          umma_commit(&kv_empty[sv]);
        }
        __syncwarp();
      }
      if (b > a) ++nq;
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[r]);
    }
    if (lane == 0) {
      umma_commit(&mma_done[u]);
      mbar_wait_drain(&mma_done[u], 0);
    }
    __syncwarp();
  } else {
    // ------------------------------ softmax -------------------------------
    // A thread owns a row.  The maximum is lazy: P = exp2(s - m) may reach 2^8
    // before O and l are rescaled to a new one (fp32 sums, and a 16-bit P keeps
    // its relative precision), so after a row's first tiles O is hardly ever
    // touched.
    constexpr float kLazy = 8.f;
    const int u = warp >> 2, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const int t_row = row / G, g = row - t_row * G;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const uint32_t tm_s = tmem + u * 128 + lanes, tm_o = tmem + 256 + u * D + lanes;
    const float sl2 = p.scale * 1.4426950408889634f;
    int n_it = 0, ns = 0;
    bool ok = true;
    while (ok) {
      const int r = n_it % kFwItems;
      if (!warp_wait(&item_full[r], (n_it / kFwItems) & 1, abort_flag, p.err)) break;
      const FwItem& it = items[r];
      ++n_it;
      if (it.stop) break;
      const int a = it.a[u], b = it.b[u];
      const bool live = t_row < it.n[u] && t_row < TT;
      const RowKeys keys = row_keys(p, it.pos + u * TT + t_row, it.lk);
      float m = -INFINITY;
      float2 l2 = make_float2(0.f, 0.f);
      for (int t = a; t < b; ++t) {
        const int key = tile_key(it, t);
        const bool sinks_only = it.sep && t == 0;
        const int lo = sinks_only ? 0 : keys.lo - key, hi = sinks_only ? 0 : keys.hi - key;
        const int sink = it.sep && t > 0 ? 0 : keys.sink - key;
        const int nch = sinks_only ? (p.sinks + 31) / 32 : 4;
        if (!warp_wait(&s_full[u], ns & 1, abort_flag, p.err)) { ok = false; break; }
        ++ns;
        tc_fence_after();
        // two sweeps over S, 32 columns at a time with the next ones in flight:
        // the maximum, then P (holding all 128 columns of a row spills)
        float s[2][32];
        const bool full = __all_sync(0xffffffffu, !live || (lo <= 0 && hi >= 128));
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        tmem_ld32(tm_s, s[0]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (c < nch) {
            tmem_wait_ld32(s[c & 1]);
            if (c < 3 && c + 1 < nch) tmem_ld32(tm_s + 32 * (c + 1), s[(c + 1) & 1]);
            float* v = s[c & 1];
            if (!full) {
              const uint32_t bits = seen_bits(lo, hi, sink, 32 * c);
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = (bits >> i & 1u) ? v[i] : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) mx[i & 3] = fmaxf(mx[i & 3], v[i]);
          }
        }
        tmem_ld32(tm_s, s[0]);  // the second sweep's first columns, in flight over what follows
        const float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sl2;
        const bool move = mt > m + kLazy || (m == -INFINITY && mt > -INFINITY);
        if (__any_sync(0xffffffffu, move)) {
          const float m_new = move ? mt : m;
          const float f = m == -INFINITY ? 0.f : ex2(m - m_new);
          m = m_new;
          l2.x *= f;
          l2.y *= f;
          if (t > a) {  // O holds the tiles before this one (their products precede this S)
#pragma unroll
            for (int c = 0; c < D; c += 16) {
              float o[16];
              tmem_ld16(tm_o + c, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] *= f;
              tmem_st16(tm_o + c, reinterpret_cast<const uint32_t*>(o));
            }
          }
        }
        const float off = m == -INFINITY ? 0.f : m;
        const float2 sc = make_float2(sl2, sl2), no2 = make_float2(-off, -off);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (c < nch) {
            tmem_wait_ld32(s[c & 1]);
            if (c < 3 && c + 1 < nch) tmem_ld32(tm_s + 32 * (c + 1), s[(c + 1) & 1]);
            float* v = s[c & 1];
            if (!full) {
              const uint32_t bits = seen_bits(lo, hi, sink, 32 * c);
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = (bits >> i & 1u) ? v[i] : -INFINITY;
            }
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              float2 e = fma2(make_float2(v[i], v[i + 1]), sc, no2);
              e.x = ex2(e.x);
              e.y = ex2(e.y);
              l2 = add2(l2, e);
              w[i / 2] = pack2<BF16>(e.x, e.y);
            }
            tmem_st16(tm_s + 16 * c, w);  // P's columns lie in S's first half, which this sweep has passed
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[u]);
      }
      if (!ok) break;
      if (b > a) {
        if (!warp_wait(&pv_done[u], (ns - 1) & 1, abort_flag, p.err)) break;
        tc_fence_after();
      }
      const float l = l2.x + l2.y;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const long long orow = (long long)(it.tok + u * TT + t_row) * p.hq + it.hk * G + g;
      uint4* out = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + orow * D);
#pragma unroll
      for (int c = 0; c < D; c += 32) {
        float o[32];
        if (b > a) {
          tmem_ld32(tm_o + c, o);
          tmem_wait_ld32(o);
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = l == 0.f ? 0.f : o[i] * inv;
        if (live) {
#pragma unroll
          for (int i = 0; i < 32; i += 8)
            out[(c + i) / 8] = make_uint4(pack2<BF16>(o[i], o[i + 1]), pack2<BF16>(o[i + 2], o[i + 3]),
                                          pack2<BF16>(o[i + 4], o[i + 5]), pack2<BF16>(o[i + 6], o[i + 7]));
        }
      }
      if (live) p.lse[orow] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
      tc_fence_before();  // O is read before this warp's next P lets the next item overwrite it
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[r]);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

template <int D, bool BF16>
int launch_fwd(const WindowParams& p, cudaStream_t s) {
  using L = FwSmem<D>;
  using S = TileShape<D>;
  CUtensorMap mq, mk, mv;
  const int tt = 128 / p.g;
  int rc = make_tmap_3d(&mq, p.q, D, p.hq, p.total_q, p.q_stride, p.g, tt, S::kCols);
  if (rc) return rc;
  // no key at all: the maps are never read
  const void* k = p.total_k ? p.k : p.q;
  const void* v = p.total_k ? p.v : p.q;
  if ((rc = make_tmap_3d(&mk, k, D, p.hkv, p.total_k, p.total_k ? p.k_stride : p.q_stride, 1, 128, S::kCols))) return rc;
  if ((rc = make_tmap_3d(&mv, v, D, p.hkv, p.total_k, p.total_k ? p.v_stride : p.q_stride, 1, 128, S::kCols))) return rc;
  const int n_items = tile_slots(p.total_q, p.num_seqs, 2 * tt) * p.hkv;
  const int grid = std::min(n_items, num_sms());
  LSRM_CUDA_TRY(cudaFuncSetAttribute(window_fwd_kernel<D, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::ALLOC));
  window_fwd_kernel<D, BF16><<<grid, kFwThreads, L::ALLOC, s>>>(mq, mk, mv, p, n_items);
  LSRM_LAUNCH_CHECK();
  return LSRM_OK;
}

}  // namespace
}  // namespace lsrm

using namespace lsrm;

extern "C" int lsrm_window_attn_fwd(const lsrm_window_shape* shape, const int32_t* cu_seqlens_q,
                                    const int32_t* cu_seqlens_k, const void* q, const void* k, const void* v,
                                    void* out, float* lse, int* err_flags, void* stream) {
  int rc = check_window(shape, cu_seqlens_q, cu_seqlens_k, q, k, v);
  if (rc) return rc;
  if (shape->total_q == 0) return LSRM_OK;
  LSRM_CHECK_ARG(out && lse, "out and lse must not be NULL");
  LSRM_CHECK_ARG(((uintptr_t)out & 15) == 0, "out must be 16-byte aligned");
  const WindowParams p = window_params(shape, cu_seqlens_q, cu_seqlens_k, q, k, v, out, lse, err_flags);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  ProfScope ps("window_attn_fwd", s);
#define CALL(BF, D) return launch_fwd<D, BF>(p, s);
  WINDOW_TYPES(CALL)
#undef CALL
}
