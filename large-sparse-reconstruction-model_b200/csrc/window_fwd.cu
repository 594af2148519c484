// Forward of the attention with a sliding window and sinks (window_common.cuh
// says which keys a query sees):
//   s_ij = scale q_i . k_j,  lse_i = log sum_j exp s_ij,
//   o_i = sum_j exp(s_ij - lse_i) v_j      (no key: o = 0, lse = -inf)
//
// One pass over a query's keys with a running maximum and sum.  A persistent
// CTA per multiprocessor walks work items (two tiles of 128 packed query rows
// of one kv head and the keys that either sees):
//   warps 0-3, 4-7  softmax of row tile 0 and 1, a row a thread: S from TMEM,
//                   mask, running maximum, P = exp2(S - m) to TMEM as 16-bit
//                   operand, at the end O / l to global memory
//   warps 8, 9      tensor-core issue for row tile 0 and 1: S = Q K^T, O += P V
//                   (P from TMEM)
//   warp 10         producer: work items, TMA of Q, K and V
// K and V tiles (64 keys) go through one ring and serve both row tiles, which
// halves the L2 reads per product (a ring for each row tile: 131072 tokens, 16
// heads of 64 channels, window 512, 766 us against 730).  S has two buffers of 64
// columns a row tile and P lies over its S, so that the products of the tiles
// before and after run under a tile's softmax.  Rounding: S, m, l and O are fp32;
// P is rounded to the operand type (the sum l takes it unrounded, and rows of few
// keys keep the remainder: few_keys), O once at the end.  Error against 64 bits 0.0023
// in bf16 at most, 0.0017 from O's rounding alone.
//
// What bounds it: 16384 tokens in two sequences, 32 / 8 heads of 128 channels,
// causal window 2048: 530 us, 900 TFLOP/s (0.54 of the library's GEMM rate; 560 us
// with what O's rounding leaves over, which training keeps); the tensor pipe is
// active 41 % of the time, the exponentials' pipe 40 %, and no other unit more.
// 131072 tokens, 16 heads of 64 channels, symmetric window 512: 710 us (752).  The
// softmax warps' chain of a tile (wait, TMEM read, maximum, exponentials, TMEM
// write, arrive) takes 1.5 times the exponentials alone; the two row tiles hide
// half of it.  Without the exponentials the time stays within 3 % at 128
// channels, and falls by 15 % at 64.  Tried without gain: tiles of 128 keys with a
// row's scores in registers (575 us at 128 channels), P in a place of its own
// (639), two threads a row (999), the row tiles taking turns at the exponentials
// (633), two CTAs a multiprocessor that read S twice (847 us at 64 channels).
#include "window_host.h"
#include "window_tile.cuh"

namespace lsrm {
namespace {

constexpr int kFwThreads = 352;
constexpr int kFwKeys = 64;

// Rows that see at most this many keys (one tile) enter the product with P and
// with what P's rounding left over: over a few keys the roundings do not average,
// and through the output they move delta, which showed in dq and dk (error against
// 64 bits up to 1.56 times a 32-bit form's; with the remainder, as in longer rows,
// sqrt(2) from dS alone, and a little).  It costs such a forward 18 % (131072 tokens,
// 16 heads of 64 channels, 68 keys a row: 393 to 462 us).  A kernel of its own (FEW),
// since its registers cost long rows 3 to 5 % (131072 tokens 774 us against 751, 16384
// of 128 channels 577 against 551): taken where the window is that short, or the
// sequences are on average.
constexpr int kFewKeys = kFwKeys;
__host__ __device__ __forceinline__ bool few_keys(const WindowParams& p, long long lk) {
  const long long reach = (long long)p.left + p.right + 1 + p.sinks;
  return (lk < reach ? lk : reach) <= kFewKeys;
}

template <int D>
struct FwSmem {
  static constexpr int QT = TileShape<D>::bytes(128), KT = TileShape<D>::bytes(kFwKeys);
  static constexpr int NQ = D == 128 ? 1 : 2;  // Q buffers of each row tile
  static constexpr int NS = D == 128 ? 9 : 12;  // K / V ring
  static constexpr int OFF_KV = 2 * NQ * QT;
  static constexpr int OFF_ROWS = OFF_KV + NS * KT;
  static constexpr int OFF_ITEM = OFF_ROWS + 8 * kRowBuf;
  static constexpr int OFF_BAR = OFF_ITEM + kItems * (int)sizeof(RowItem);
  // q_full[2][NQ], q_empty[2][NQ], kv_full[NS], kv_empty[NS], s_full[2][2], p_full[2][2],
  // pv_done[2][2], item_full[], item_empty[], mma_done[2]
  static constexpr int NBAR = 4 * NQ + 2 * NS + 12 + 2 * kItems + 2;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int BYTES = OFF_MISC + 16 + 1024;
  static constexpr int ALLOC = BYTES > kOneCtaPerSmSmem ? BYTES : kOneCtaPerSmSmem;
  static_assert(OFF_BAR % 8 == 0 && ALLOC <= 227 * 1024, "shared memory budget");
};

template <int D, bool BF16, bool FEW>
__global__ void __launch_bounds__(kFwThreads, 1)
    window_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const WindowParams p, const int n_items) {
  using L = FwSmem<D>;
  constexpr uint32_t AB = BF16 ? 1u : 0u;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sKV = smem + L::OFF_KV;
  RowItem* items = reinterpret_cast<RowItem*>(smem + L::OFF_ITEM);
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* q_empty = q_full + 2 * L::NQ;
  uint64_t* kv_full = q_empty + 2 * L::NQ;
  uint64_t* kv_empty = kv_full + L::NS;
  uint64_t* s_full = kv_empty + L::NS;
  // [row tile][buffer]: two tiles are under way, so each has its own phases
  uint64_t* p_full = s_full + 4;
  uint64_t* pv_done = p_full + 4;
  uint64_t* item_full = pv_done + 4;
  uint64_t* item_empty = item_full + kItems;
  uint64_t* mma_done = item_empty + kItems;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::OFF_MISC + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = p.g, TT = 128 / G;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2 * L::NQ; ++i) mbar_init(&q_full[i], 1), mbar_init(&q_empty[i], 1);
    for (int i = 0; i < L::NS; ++i) mbar_init(&kv_full[i], 1), mbar_init(&kv_empty[i], 2);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[2 * i], 1);
      mbar_init(&s_full[2 * i + 1], 1);
      mbar_init(&p_full[2 * i], 4);
      mbar_init(&p_full[2 * i + 1], 4);
      mbar_init(&pv_done[2 * i], 1);
      mbar_init(&pv_done[2 * i + 1], 1);
      mbar_init(&mma_done[i], 1);
    }
    for (int i = 0; i < kItems; ++i) mbar_init(&item_full[i], 1), mbar_init(&item_empty[i], 10);
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
  // TMEM columns: S of row tile u, buffer i [128 u + 64 i, +64) with P over its first half (and its remainder over the
  // second, few_keys); O [256 + u D, +D)

  if (warp == 10) {
    // ------------------------------ producer ------------------------------
    // The whole warp walks the items; one elected lane issues (under elect.sync
    // the compiler knows that one lane is active and issues TMA and tensor-core
    // instructions from uniform registers; under `lane == 0` each took some 120
    // cycles).
    if (elect_one()) {
      tma_prefetch_desc(&tm_q);
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
    }
    const uint32_t q_bytes = (uint32_t)(G * TT * D * 2);
    int n_it = 0, J = 0, nq[2] = {0, 0};
    bool ok = true;
    for (int w = blockIdx.x; ok; w += gridDim.x) {
      RowItem it;
      it.stop = w >= n_items;
      if (!it.stop) {
        if (!row_item<kFwKeys>(p, w, TT, it)) continue;
      }
      const int r = n_it % kItems;
      if (!wait_phase(&item_empty[r], ((n_it / kItems) & 1) ^ 1, abort_flag, p.err)) break;
      if (lane == 0) {
        items[r] = it;
        mbar_arrive(&item_full[r]);
      }
      __syncwarp();
      ++n_it;
      if (it.stop) break;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (!ok || it.b[i] <= it.a[i]) continue;
        const int st = i * L::NQ + nq[i] % L::NQ;
        if (!(ok = wait_phase(&q_empty[st], ((nq[i] / L::NQ) & 1) ^ 1, abort_flag, p.err))) continue;
        if (elect_one()) {
          mbar_arrive_expect_tx(&q_full[st], q_bytes);
          load_tile<D>(sQ + st * L::QT, 128, &tm_q, it.hk * G, it.tok + i * TT, &q_full[st]);
        }
        __syncwarp();
        ++nq[i];
      }
      for (int t = 0; t < it.tiles && ok; ++t) {
        const int key = it.key0 + it.key<kFwKeys>(t);
        for (int kv = 0; kv < 2; ++kv) {
          const int st = J % L::NS;
          if (!(ok = wait_phase(&kv_empty[st], ((J / L::NS) & 1) ^ 1, abort_flag, p.err))) break;
          if (elect_one()) {
            mbar_arrive_expect_tx(&kv_full[st], L::KT);
            load_tile<D>(sKV + st * L::KT, kFwKeys, kv ? &tm_v : &tm_k, it.hk, key, &kv_full[st]);
          }
          __syncwarp();
          ++J;
        }
      }
    }
    // after an abort: copies in flight land before the CTA exits
    if (lane == 0 && *abort_flag) {
      for (int i = 0; i < 2; ++i)
        for (int k = max(0, nq[i] - L::NQ); k < nq[i]; ++k)
          mbar_wait_drain(&q_full[i * L::NQ + k % L::NQ], (k / L::NQ) & 1);
      for (int j = max(0, J - L::NS); j < J; ++j) mbar_wait_drain(&kv_full[j % L::NS], (j / L::NS) & 1);
    }
    __syncwarp();
  } else if (warp >= 8) {
    // --------------------------- tensor-core issue ---------------------------
    const int u = warp - 8;
    const uint32_t tm_s = tmem + u * 128, tm_o = tmem + 256 + u * D;
    const uint32_t idesc_o = make_idesc(AB, 0, 1, 128, D);
    int n_it = 0, J = 0, nq = 0;         // items, ring slots, Q tiles so far
    int ns = 0, np = 0;                  // S and P V products issued
    while (true) {
      const int r = n_it % kItems;
      if (!wait_phase(&item_full[r], (n_it / kItems) & 1, abort_flag, p.err)) break;
      const RowItem& it = items[r];
      ++n_it;
      if (it.stop) break;
      const int st_q = u * L::NQ + nq % L::NQ;
      const uint32_t q_base = smem_u32(sQ + st_q * L::QT);
      const int a = it.a[u], b = it.b[u];
      const bool few = FEW && few_keys(p, it.lk);
      // sinks of their own tile: only as many columns as they need
      auto cols_of = [&](int t) { return t < it.sep ? min(kFwKeys, (p.sinks - t * kFwKeys + 31) / 32 * 32) : kFwKeys; };
      auto wait_slot = [&](int j) { return wait_phase(&kv_full[j % L::NS], (j / L::NS) & 1, abort_flag, p.err); };
      // keys that only the other row tile sees
      auto pass = [&](int t) {
        if (!wait_slot(J + 2 * t) || !wait_slot(J + 2 * t + 1)) return false;
        if (lane == 0) {
          mbar_arrive(&kv_empty[(J + 2 * t) % L::NS]);
          mbar_arrive(&kv_empty[(J + 2 * t + 1) % L::NS]);
        }
        __syncwarp();
        return true;
      };
      auto issue_s = [&](int t) {
        const int j = J + 2 * t, st = j % L::NS, buf = ns & 1;
        if (!wait_slot(j)) return false;
        // the product that reads the buffer's last P is over
        if (ns >= 2 && !wait_phase(&pv_done[2 * u + buf], ((ns >> 1) & 1) ^ 1, abort_flag, p.err)) return false;
        ++ns;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t k_base = smem_u32(sKV + st * L::KT);
          const uint32_t idesc_s = make_idesc(AB, 0, 0, 128, cols_of(t));
          mma_rows<D, 128, kFwKeys>(tm_s + 64 * buf, q_base, k_base, idesc_s);
          umma_commit(&s_full[2 * u + buf]);
          umma_commit(&kv_empty[st]);
          if (t == b - 1) umma_commit(&q_empty[st_q]);
        }
        __syncwarp();
        return true;
      };
      bool ok = true;
      for (int t = 0; t < a && ok; ++t) ok = pass(t);
      if (ok && b > a) {
        ok = wait_phase(&q_full[st_q], (nq / L::NQ) & 1, abort_flag, p.err) && issue_s(a) && (b < a + 2 || issue_s(a + 1));
        ++nq;
      }
      for (int t = a; t < b && ok; ++t) {
        const int j = J + 2 * t + 1, st = j % L::NS, cols = cols_of(t), valid = it.valid<kFwKeys>(t);
        if (!(ok = wait_slot(j))) break;
        if (valid < cols) zero_rows<D>(sKV + st * L::KT, kFwKeys, valid);
        if (!(ok = wait_phase(&p_full[2 * u + (np & 1)], (np >> 1) & 1, abort_flag, p.err))) break;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t v_base = smem_u32(sKV + st * L::KT);
          mma_sum<D, kFwKeys>(tm_o, tm_s + 64 * (np & 1), v_base, idesc_o, t > a, cols / 16);
          if (few) mma_sum<D, kFwKeys>(tm_o, tm_s + 64 * (np & 1) + 32, v_base, idesc_o, true, cols / 16);
          umma_commit(&pv_done[2 * u + (np & 1)]);
          umma_commit(&kv_empty[st]);
        }
        __syncwarp();
        ++np;
        if (t + 2 < b) ok = issue_s(t + 2);
      }
      for (int t = b > a ? b : a; t < it.tiles && ok; ++t) ok = pass(t);
      if (!ok) break;
      J += 2 * it.tiles;
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[r]);
    }
    if (elect_one()) {
      umma_commit(&mma_done[u]);
      mbar_wait_drain(&mma_done[u], 0);
    }
    __syncwarp();
  } else {
    // ------------------------------ softmax -------------------------------
    // A thread owns a row.  The maximum is lazy: P = exp2(s - m) may reach 2^8
    // before O and l are rescaled to a new one (fp32 sums, and a 16-bit P keeps
    // its relative precision), so after a row's first tiles O is hardly ever
    // touched.  A chunk of 32 columns that no row of the warp sees is skipped and
    // one that all see is not masked, which leaves one masked chunk of a window's
    // slanted edge.
    constexpr float kLazy = 8.f;
    const int u = warp >> 2, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const int t_row = row / G, g = row - t_row * G;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const uint32_t tm_s0 = tmem + u * 128 + lanes, tm_o = tmem + 256 + u * D + lanes;
    const float sl2 = p.scale * 1.4426950408889634f;
    int n_it = 0, ns = 0;  // items, tiles so far
    // An item's rows leave while the next one's first products run (1 to 5 % of the time, against at its own end).
    struct {
      bool due;
      float m, l;
      long long row;
    } last = {};
    auto write_rows = [&](bool any) -> bool {
      last.due = false;
      if (any) {
        if (!wait_phase(&pv_done[2 * u + ((ns - 1) & 1)], ((ns - 1) >> 1) & 1, abort_flag, p.err)) return false;
        tc_fence_after();
      }
      const bool none = !any || last.l == 0.f;
      const float inv = none ? 0.f : 1.f / last.l;
#pragma unroll
      for (int c = 0; c < D; c += 32) {
        float o[32];
        uint32_t w[16];
        if (any) {
          tmem_ld32(tm_o + c, o);
          tmem_wait_values<32>(o);
        }
#pragma unroll
        for (int i = 0; i < 32; i += 2) w[i / 2] = none ? 0u : pack2<BF16>(o[i] * inv, o[i + 1] * inv);
        const uint32_t buf = smem_u32(smem + L::OFF_ROWS + warp * kRowBuf);
        store_rows32(buf, w, last.row, static_cast<uint16_t*>(p.out), D, c);
        if (p.out_rest) {
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 r = unpack2<BF16>(w[i / 2]);
            w[i / 2] = none ? 0u : pack2<BF16>(fmaf(o[i], inv, -r.x), fmaf(o[i + 1], inv, -r.y));
          }
          store_rows32(buf, w, last.row, static_cast<uint16_t*>(p.out_rest), D, c);
        }
      }
      tc_fence_before();  // O is read before this warp's next P lets the next item overwrite it
      if (last.row >= 0) p.lse[last.row] = none ? -INFINITY : (last.m + log2f(last.l)) * 0.6931471805599453f;
      return true;
    };
    while (true) {
      const int r = n_it % kItems;
      if (!wait_phase(&item_full[r], (n_it / kItems) & 1, abort_flag, p.err)) break;
      const RowItem& it = items[r];
      ++n_it;
      if (it.stop) {
        if (last.due) write_rows(true);
        break;
      }
      const int a = it.a[u], b = it.b[u];
      const bool few = FEW && few_keys(p, it.lk);
      const bool live = t_row < it.n[u] && t_row < TT;
      const long long orow = live ? (long long)(it.tok + u * TT + t_row) * p.hq + it.hk * G + g : -1;
      const RowView<kFwKeys> view(p, it, it.pos + u * TT + t_row, live, 0, kFwKeys);
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[r]);
      if (last.due && !write_rows(true)) break;
      float m = -INFINITY;
      float2 l2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      bool ok = true;
      float s[2][32];
      for (int t = a; t < b; ++t) {
        // columns 32 c .. + 31: which of them this row sees; per warp, whether some and whether all rows see them
        uint32_t bits[2];
        bool some[2] = {true, true}, all[2] = {true, true};
        if (!view.full(t)) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            bits[c] = view.bits(t, 32 * c);
            some[c] = __any_sync(0xffffffffu, bits[c] != 0u);
            all[c] = __all_sync(0xffffffffu, !live || bits[c] == 0xffffffffu);
          }
        }
        const uint32_t tm_s = tm_s0 + 64 * (ns & 1);
        if (!(ok = wait_phase(&s_full[2 * u + (ns & 1)], (ns >> 1) & 1, abort_flag, p.err))) break;
        ++ns;
        tc_fence_after();
        if (some[0]) tmem_ld32(tm_s, s[0]);
        if (some[1]) tmem_ld32(tm_s + 32, s[1]);
        tmem_wait_values<32>(s[0]);
        tmem_wait_values<32>(s[1]);
        float mt = -INFINITY;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (some[c]) {
            if (!all[c]) mask32(s[c], bits[c]);
            mt = fmaxf(mt, max32(s[c]));
          }
        }
        mt *= sl2;
        const bool move = mt > m + kLazy || (m == -INFINITY && mt > -INFINITY);
        if (__any_sync(0xffffffffu, move)) {
          const float m_new = move ? mt : m;
          const float f = m == -INFINITY ? 0.f : ex2(m - m_new);
          m = m_new;
#pragma unroll
          for (int j = 0; j < 2; ++j) l2[j] = mul2(l2[j], make_float2(f, f));
          if (t > a) {
            // O is whole once the product of the tile before is over
            if (!(ok = wait_phase(&pv_done[2 * u + (ns & 1)], ((ns - 2) >> 1) & 1, abort_flag, p.err))) break;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < D; c += 16) {
              float o[16];
              tmem_ld16(tm_o + c, o);
              tmem_wait_values<16>(o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] *= f;
              tmem_st16(tm_o + c, reinterpret_cast<const uint32_t*>(o));
            }
          }
        }
        const float off = m == -INFINITY ? 0.f : m;
        const float2 sc = make_float2(sl2, sl2), no2 = make_float2(-off, -off);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t w[16];
          if (some[c]) {
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              float2 e = fma2(make_float2(s[c][i], s[c][i + 1]), sc, no2);
              e.x = ex2(e.x);
              e.y = ex2(e.y);
              l2[(i >> 1) & 1] = add2(l2[(i >> 1) & 1], e);
              w[i / 2] = pack2<BF16>(e.x, e.y);
              if (FEW) s[c][i] = e.x, s[c][i + 1] = e.y;
            }
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = 0u;
          }
          tmem_st16(tm_s + 16 * c, w);
          if (few) {
            if (some[c]) {
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                const float2 h = unpack2<BF16>(w[i / 2]);
                w[i / 2] = pack2<BF16>(s[c][i] - h.x, s[c][i + 1] - h.y);
              }
            }
            tmem_st16(tm_s + 32 + 16 * c, w);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * u + ((ns - 1) & 1)]);
      }
      if (!ok) break;
      last.row = orow;
      if (b > a) {
        last.due = true;
        last.m = m;
        last.l = l2[0].x + l2[0].y + l2[1].x + l2[1].y;
      } else {
        write_rows(false);
      }
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
  if ((rc = make_tmap_3d(&mk, k, D, p.hkv, p.total_k, p.total_k ? p.k_stride : p.q_stride, 1, kFwKeys, S::kCols))) return rc;
  if ((rc = make_tmap_3d(&mv, v, D, p.hkv, p.total_k, p.total_k ? p.v_stride : p.q_stride, 1, kFwKeys, S::kCols))) return rc;
  const int n_items = tile_slots(p.total_q, p.num_seqs, 2 * tt) * p.hkv;
  const int grid = std::min(n_items, num_sms());
  auto launch = [&](auto kernel) {
    LSRM_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::ALLOC));
    kernel<<<grid, kFwThreads, L::ALLOC, s>>>(mq, mk, mv, p, n_items);
    LSRM_LAUNCH_CHECK();
    return LSRM_OK;
  };
  const bool few = few_keys(p, p.total_k / std::max(p.num_seqs, 1));
  return few ? launch(window_fwd_kernel<D, BF16, true>) : launch(window_fwd_kernel<D, BF16, false>);
}

}  // namespace
}  // namespace lsrm

using namespace lsrm;

extern "C" int lsrm_window_attn_fwd(const lsrm_window_shape* shape, const int32_t* cu_seqlens_q,
                                    const int32_t* cu_seqlens_k, const void* q, const void* k, const void* v,
                                    void* out, void* out_rest, float* lse, int* err_flags, void* stream) {
  int rc = check_window(shape, cu_seqlens_q, cu_seqlens_k, q, k, v);
  if (rc) return rc;
  if (shape->total_q == 0) return LSRM_OK;
  LSRM_CHECK_ARG(out && lse, "out and lse must not be NULL");
  LSRM_CHECK_ARG((((uintptr_t)out | (uintptr_t)out_rest) & 15) == 0, "out and out_rest must be 16-byte aligned");
  WindowParams p = window_params(shape, cu_seqlens_q, cu_seqlens_k, q, k, v, out, lse, err_flags);
  p.out_rest = out_rest;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  ProfScope ps("window_attn_fwd", s);
#define CALL(BF, D) return launch_fwd<D, BF>(p, s);
  WINDOW_TYPES(CALL)
#undef CALL
}
