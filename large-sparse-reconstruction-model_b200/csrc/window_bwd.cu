// Backward of the attention with a sliding window and sinks:
//   delta_i = o_i . do_i,  p_ij = exp(s_ij - lse_i),  ds_ij = p_ij (do_i . v_j - delta_i)
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i
// with the query heads of a group summed into their kv head.  Scores are
// recomputed from q, k and the forward's lse.
//
// Two passes, one that keeps query rows (dQ, built like the forward) and one
// that keeps key rows (dK, dV), so that every sum is taken by one CTA in a
// fixed order: no atomics, the same bits every time, at the price of computing
// S and dP twice (seven products in place of five).
//
// Rounding: P and dS are rounded once to the operand type, everything else is
// fp32.  The products take operands of one 16-bit type; the remainders would be two
// more products, with operands in TMEM, which is full.  The gradients' error
// against 64 bits grows by sqrt(2) over that of rounding the results (bf16 0.0024
// for 0.0017, fp16 0.0003 for 0.0002).  dS is not scaled: fp16 gradients of the
// output far below 0.01 fall into the type's subnormal range there, so fp16 training
// wants its usual loss scale.
//
// Sinks are seen by every later query.  The key tile that holds them sums the
// queries that its window reaches; the queries past it are cut into chunks
// that are items of their own, with fp32 partial sums that sink_sum_kernel adds
// in ascending order.
#include "window_host.h"
#include "window_tile.cuh"

namespace lsrm {
namespace {

struct WindowBwdParams : WindowParams {
  const void* dout;    // [total_q, hq, D]
  float* delta;        // [total_q, hq]
  void *dq, *dk, *dv;
  // sinks past the window's reach
  int chunk;           // query tokens per partial sum (0: no sinks)
  int chunk_slots;
  float* part0;        // [num_seqs][hkv][sinks][2][D] fp32: dv, dk of the sinks' own tile
  float* part;         // [chunk_slots][hkv][sinks][2][D]
};

// delta = rowsum(o * do), D / 8 lanes a row.  o is the forward's output and what
// its rounding left over (`rest`, may be null): from the rounded output alone
// delta's error is half of ds's own rounding and shows in dq and dk.  Bound by
// HBM: 131072 tokens, 16 heads of 64 channels, 136 us, 5.9 TB/s.
template <typename T, int D>
__global__ void __launch_bounds__(256) window_delta_kernel(const uint4* __restrict__ o, const uint4* __restrict__ rest,
                                                           const uint4* __restrict__ d, float* __restrict__ delta,
                                                           long long rows) {
  constexpr int GL = D / 8;
  const long long stride = (long long)gridDim.x * blockDim.x;
  const long long n = rows * GL, top = (n + 31) / 32 * 32;  // whole warps take part in the shuffles
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < top; i += stride) {
    float s = 0.f;
    if (i < n) {
      const uint4 a = o[i], b = d[i];
      const T *x = reinterpret_cast<const T*>(&a), *y = reinterpret_cast<const T*>(&b);
#pragma unroll
      for (int j = 0; j < 8; ++j) s = fmaf((float)x[j], (float)y[j], s);
      if (rest) {
        const uint4 c = rest[i];
        const T* z = reinterpret_cast<const T*>(&c);
#pragma unroll
        for (int j = 0; j < 8; ++j) s = fmaf((float)z[j], (float)y[j], s);
      }
    }
#pragma unroll
    for (int k = GL / 2; k > 0; k >>= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
    if (i < n && i % GL == 0) delta[i / GL] = s;
  }
}

// ------------------------------- dQ ----------------------------------------
// As the forward: a persistent CTA, two tiles of 128 packed query rows, key
// tiles of 64 (S, dP and dQ of both row tiles fill TMEM at 128 channels).  One
// thread a row: with two, the waits of a tile count twice (16384 tokens, 32 / 8 heads
// of 128 channels: 904 us against 1037 in the first form).
//
// What bounds it: a row tile's chain of a key tile, of which the two row tiles
// hide each other's.  S and dP have barriers of their own: the next S is formed
// under the exponentials, and dS lies over dP, whose next product follows dQ's
// under the next exponentials: 685 us there, 1.0 PFLOP/s, against 913 with both
// waiting for dS; 131072 tokens, 16 heads of 64 channels, symmetric window 512:
// 866 us (884 then) against 922.

constexpr int kBwThreads = 352;
constexpr int kDqKeys = 64;

template <int D>
struct DqSmem {
  static constexpr int QT = TileShape<D>::bytes(128), KT = TileShape<D>::bytes(kDqKeys);
  static constexpr int NQ = D == 128 ? 1 : 2;  // Q and dO buffers of each row tile
  static constexpr int NS = D == 128 ? 5 : 8;  // K / V ring
  static constexpr int OFF_KV = 4 * NQ * QT;   // [row tile][buffer][Q, dO]
  static constexpr int OFF_ROWS = OFF_KV + NS * KT;
  static constexpr int OFF_ITEM = OFF_ROWS + 8 * kRowBuf;
  static constexpr int OFF_BAR = OFF_ITEM + kItems * (int)sizeof(RowItem);
  // q_full[2][NQ], q_empty[2][NQ], kv_full[NS], kv_empty[NS], s_full[2], s_free[2], dp_full[2], ds_full[2],
  // dq_done[2], item_full[], item_empty[], mma_done[2]
  static constexpr int NBAR = 4 * NQ + 2 * NS + 10 + 2 * kItems + 2;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int BYTES = OFF_MISC + 16 + 1024;
  static constexpr int ALLOC = BYTES > kOneCtaPerSmSmem ? BYTES : kOneCtaPerSmSmem;
  static_assert(OFF_BAR % 8 == 0 && ALLOC <= 227 * 1024, "shared memory budget");
};

template <int D, bool BF16>
__global__ void __launch_bounds__(kBwThreads, 1)
    window_dq_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do,
                     const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                     const WindowBwdParams p, const int n_items) {
  using L = DqSmem<D>;
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
  uint64_t* s_free = s_full + 2;
  uint64_t* dp_full = s_free + 2;
  uint64_t* ds_full = dp_full + 2;
  uint64_t* dq_done = ds_full + 2;
  uint64_t* item_full = dq_done + 2;
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
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 4);
      mbar_init(&dp_full[i], 1);
      mbar_init(&ds_full[i], 4);
      mbar_init(&dq_done[i], 1);
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
  // TMEM columns per row tile u: S [128 u, +64), dP [128 u + 64, +64) with dS over it, dQ [256 + u D, +D)

  if (warp == 10) {
    // ------------------------------ producer ------------------------------
    if (elect_one()) {
      tma_prefetch_desc(&tm_q);
      tma_prefetch_desc(&tm_do);
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
    }
    const uint32_t q_bytes = (uint32_t)(2 * G * TT * D * 2);
    int n_it = 0, J = 0, nq[2] = {0, 0};
    bool ok = true;
    for (int w = blockIdx.x; ok; w += gridDim.x) {
      RowItem it;
      it.stop = w >= n_items;
      if (!it.stop && !row_item<kDqKeys>(p, w, TT, it)) continue;
      const int r = n_it % kItems;
      if (!wait_phase(&item_empty[r], ((n_it / kItems) & 1) ^ 1, abort_flag, p.err)) break;
      if (lane == 0) {
        items[r] = it;
        mbar_arrive(&item_full[r]);
      }
      __syncwarp();
      ++n_it;
      if (it.stop) break;
      for (int u = 0; u < 2 && ok; ++u) {
        if (it.b[u] <= it.a[u]) continue;
        const int st = u * L::NQ + nq[u] % L::NQ;
        if (!(ok = wait_phase(&q_empty[st], ((nq[u] / L::NQ) & 1) ^ 1, abort_flag, p.err))) break;
        if (elect_one()) {
          mbar_arrive_expect_tx(&q_full[st], q_bytes);
          load_tile<D>(sQ + 2 * st * L::QT, 128, &tm_q, it.hk * G, it.tok + u * TT, &q_full[st]);
          load_tile<D>(sQ + (2 * st + 1) * L::QT, 128, &tm_do, it.hk * G, it.tok + u * TT, &q_full[st]);
        }
        __syncwarp();
        ++nq[u];
      }
      for (int t = 0; t < it.tiles && ok; ++t) {
        const int key = it.key0 + it.key<kDqKeys>(t);
        for (int kv = 0; kv < 2; ++kv) {
          const int st = J % L::NS;
          if (!(ok = wait_phase(&kv_empty[st], ((J / L::NS) & 1) ^ 1, abort_flag, p.err))) break;
          if (elect_one()) {
            mbar_arrive_expect_tx(&kv_full[st], L::KT);
            load_tile<D>(sKV + st * L::KT, kDqKeys, kv ? &tm_v : &tm_k, it.hk, key, &kv_full[st]);
          }
          __syncwarp();
          ++J;
        }
      }
    }
    if (lane == 0 && *abort_flag) {  // copies in flight land before the CTA exits
      for (int u = 0; u < 2; ++u)
        for (int k = max(0, nq[u] - L::NQ); k < nq[u]; ++k)
          mbar_wait_drain(&q_full[u * L::NQ + k % L::NQ], (k / L::NQ) & 1);
      for (int j = max(0, J - L::NS); j < J; ++j) mbar_wait_drain(&kv_full[j % L::NS], (j / L::NS) & 1);
    }
    __syncwarp();
  } else if (warp >= 8) {
    // --------------------------- tensor-core issue ---------------------------
    const int u = warp - 8;
    const uint32_t tm_s = tmem + u * 128, tm_dp = tm_s + 64, tm_dq = tmem + 256 + u * D;
    const uint32_t idesc_s = make_idesc(AB, 0, 0, 128, kDqKeys), idesc_q = make_idesc(AB, 0, 1, 128, D);
    int n_it = 0, J = 0, nq = 0, ns = 0, np = 0;  // items, ring slots, Q tiles, S and dQ products so far
    while (true) {
      const int r = n_it % kItems;
      if (!wait_phase(&item_full[r], (n_it / kItems) & 1, abort_flag, p.err)) break;
      const RowItem& it = items[r];
      ++n_it;
      if (it.stop) break;
      const int st_q = u * L::NQ + nq % L::NQ;
      const uint32_t q_base = smem_u32(sQ + 2 * st_q * L::QT), do_base = q_base + L::QT;
      const int a = it.a[u], b = it.b[u];
      auto wait_slot = [&](int j) { return wait_phase(&kv_full[j % L::NS], (j / L::NS) & 1, abort_flag, p.err); };
      auto pass = [&](int t) {  // keys that only the other row tile sees
        if (!wait_slot(J + 2 * t) || !wait_slot(J + 2 * t + 1)) return false;
        if (lane == 0) {
          mbar_arrive(&kv_empty[(J + 2 * t) % L::NS]);
          mbar_arrive(&kv_empty[(J + 2 * t + 1) % L::NS]);
        }
        __syncwarp();
        return true;
      };
      auto issue_s = [&](int t) {  // once the last S has been read
        const int sk = (J + 2 * t) % L::NS;
        if (!wait_slot(J + 2 * t)) return false;
        if (ns > 0 && !wait_phase(&s_free[u], (ns - 1) & 1, abort_flag, p.err)) return false;
        ++ns;
        tc_fence_after();
        if (elect_one()) {
          mma_rows<D, 128, kDqKeys>(tm_s, q_base, smem_u32(sKV + sk * L::KT), idesc_s);
          umma_commit(&s_full[u]);
        }
        __syncwarp();
        return true;
      };
      auto issue_dp = [&](int t) {  // once the product that reads the last dS is over
        const int sv = (J + 2 * t + 1) % L::NS;
        if (!wait_slot(J + 2 * t + 1)) return false;
        if (np > 0 && !wait_phase(&dq_done[u], (np - 1) & 1, abort_flag, p.err)) return false;
        tc_fence_after();
        if (elect_one()) {
          mma_rows<D, 128, kDqKeys>(tm_dp, do_base, smem_u32(sKV + sv * L::KT), idesc_s);
          umma_commit(&dp_full[u]);
          umma_commit(&kv_empty[sv]);
          if (t == b - 1) umma_commit(&q_empty[st_q]);
        }
        __syncwarp();
        return true;
      };
      bool ok = true;
      for (int t = 0; t < a && ok; ++t) ok = pass(t);
      if (ok && b > a) {
        ok = wait_phase(&q_full[st_q], (nq / L::NQ) & 1, abort_flag, p.err) && issue_s(a) && issue_dp(a);
        ++nq;
      }
      for (int t = a; t < b && ok; ++t) {
        if (t + 1 < b && !(ok = issue_s(t + 1))) break;
        const int st = (J + 2 * t) % L::NS, valid = it.valid<kDqKeys>(t);
        if (valid < kDqKeys) zero_rows<D>(sKV + st * L::KT, kDqKeys, valid);
        if (!(ok = wait_phase(&ds_full[u], np & 1, abort_flag, p.err))) break;
        ++np;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t k_base = smem_u32(sKV + st * L::KT);
          mma_sum<D, kDqKeys>(tm_dq, tm_dp, k_base, idesc_q, t > a);
          umma_commit(&dq_done[u]);
          umma_commit(&kv_empty[st]);
        }
        __syncwarp();
        if (t + 1 < b) ok = issue_dp(t + 1);
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
    // ------------------------------ dS -------------------------------------
    // A thread owns a row: p = exp2(s - lse), ds = p (dp - delta).
    const int u = warp >> 2, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const int t_row = row / G, g = row - t_row * G;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const uint32_t tm_s = tmem + u * 128 + lanes, tm_dp = tm_s + 64, tm_dq = tmem + 256 + u * D + lanes;
    const float sl2 = p.scale * 1.4426950408889634f;
    const float2 sc = make_float2(sl2, sl2);
    // An item's rows leave while the next one's lse, delta and first products are on their way.
    bool due = false, due_any = false;
    long long due_row = -1;
    int n_it = 0, ns = 0;
    auto write_rows = [&]() -> bool {
      if (due_any) {
        if (!wait_phase(&dq_done[u], (ns - 1) & 1, abort_flag, p.err)) return false;
        tc_fence_after();
      }
#pragma unroll
      for (int c = 0; c < D; c += 32) {
        float s[32];
        uint32_t w[16];
        if (due_any) {
          tmem_ld32(tm_dq + c, s);
          tmem_wait_values<32>(s);
        }
#pragma unroll
        for (int i = 0; i < 32; i += 2)
          w[i / 2] = due_any ? pack2<BF16>(s[i] * p.scale, s[i + 1] * p.scale) : 0u;
        store_rows32(smem_u32(smem + L::OFF_ROWS + warp * kRowBuf), w, due_row, static_cast<uint16_t*>(p.dq), D, c);
      }
      tc_fence_before();  // dQ is read before this warp's next dS lets the next item overwrite it
      return true;
    };
    while (true) {
      const int r = n_it % kItems;
      if (!wait_phase(&item_full[r], (n_it / kItems) & 1, abort_flag, p.err)) break;
      const RowItem& it = items[r];
      ++n_it;
      if (it.stop) {
        if (due) write_rows();
        break;
      }
      const int a = it.a[u], b = it.b[u];
      const bool live = t_row < it.n[u] && t_row < TT;
      const long long orow = (long long)(it.tok + u * TT + t_row) * p.hq + it.hk * G + g;
      float lse2 = live ? p.lse[orow] * 1.4426950408889634f : 0.f;
      const float delta = live ? p.delta[orow] : 0.f;
      const RowView<kDqKeys> view(p, it, it.pos + u * TT + t_row, live, 0, kDqKeys);
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[r]);
      if (due && !write_rows()) break;
      due = true;
      due_any = b > a;
      due_row = live ? orow : -1;
      if (lse2 == -INFINITY) lse2 = 0.f;  // a row that sees nothing: every column is masked
      const float2 nl = make_float2(-lse2, -lse2), nd = make_float2(-delta, -delta);
      bool ok = true;
      for (int t = a; t < b; ++t) {
        uint32_t bits[2] = {0xffffffffu, 0xffffffffu};
        const bool all = view.full(t);
        if (!all) bits[0] = view.bits(t, 0), bits[1] = view.bits(t, 32);
        const bool some[2] = {all || __any_sync(0xffffffffu, bits[0] != 0u), all || __any_sync(0xffffffffu, bits[1] != 0u)};
        if (!(ok = wait_phase(&s_full[u], ns & 1, abort_flag, p.err))) break;
        tc_fence_after();
        float s[2][32];
        if (some[0]) tmem_ld32(tm_s, s[0]);
        if (some[1]) tmem_ld32(tm_s + 32, s[1]);
        tmem_wait_values<32>(s[0]);
        tmem_wait_values<32>(s[1]);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[u]);  // the next tile's S is formed under this one's exponentials
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (some[c]) {
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const float2 e = fma2(make_float2(s[c][i], s[c][i + 1]), sc, nl);
              s[c][i] = ex2(e.x);
              s[c][i + 1] = ex2(e.y);
            }
          }
        }
        if (!(ok = wait_phase(&dp_full[u], ns & 1, abort_flag, p.err))) break;
        ++ns;
        tc_fence_after();
        uint32_t w[2][16];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (some[c]) {
            const bool full = all || __all_sync(0xffffffffu, !live || bits[c] == 0xffffffffu);
#pragma unroll
            for (int h = 0; h < 32; h += 16) {
              float d[16];
              tmem_ld16(tm_dp + 32 * c + h, d);
              tmem_wait_values<16>(d);
#pragma unroll
              for (int i = 0; i < 16; i += 2) {
                const float2 e = mul2(make_float2(s[c][h + i], s[c][h + i + 1]), add2(make_float2(d[i], d[i + 1]), nd));
                s[c][h + i] = e.x;
                s[c][h + i + 1] = e.y;
              }
            }
            if (!full) {
#pragma unroll
              for (int i = 0; i < 32; ++i) s[c][i] = (bits[c] >> i & 1u) ? s[c][i] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < 32; i += 2) w[c][i / 2] = pack2<BF16>(s[c][i], s[c][i + 1]);
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) w[c][i] = 0u;
          }
        }
        tmem_st16(tm_dp, w[0]);  // over dP
        tmem_st16(tm_dp + 16, w[1]);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ds_full[u]);
      }
      if (!ok) break;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

// ----------------------------- dK and dV ------------------------------------
// A persistent CTA keeps 128 keys of a kv head and walks the queries that see
// them, 64 packed rows at a time:
//   S^T = K Q^T, dP^T = V dO^T (128 keys x 64 rows; three TMEM stages up to 64 channels, two at 128)
//   warps 0-7 (even query tiles), 8-15 (odd ones): two threads a key, 32 rows each;
//   P^T and dS^T as 16-bit operands in TMEM, over S^T and dP^T;  dV += P^T dO, dK += dS^T Q
//   warp 16 issues the first two products, warp 19 the sums (one warp for all
//   four spends longer on issuing than they take), warp 17 loads, warp 18 gathers
//   the rows' lse and delta.
//
// What bounds it: a tile's chain (products, exponentials, sums), of which two or
// three are in flight.  131072 tokens, 16 heads of 64 channels, symmetric window
// 512: 1002 us; with two stages, whose P^T and dS^T have places of their own, 1083
// against 1018.  16384 tokens, 32 / 8 heads of 128 channels, causal window 2048: 991 us,
// the tensor pipe's own time about 650.  The scores come from TMEM eight columns
// at a time: with sixteen 1050 us there against 1005, with all 32 up front 1183 (the
// registers then leave the exponentials no slack).  Four threads a key, all 16 warps on one
// tile, gives 1008 us there and loses elsewhere (ragged sequences, 32 / 2 heads of
// 32 channels: 320 us against 273); S^T and dP^T on barriers of their own, as in dQ,
// keep a tile's exponentials in registers that are not there (1108 us against 1016;
// with one thread a key 1037 against 994).  An item's sums leave under the next one's
// first tiles: 1125 us against 1244 before the other steps (131072 tokens).

constexpr int kKvRows = 64;  // packed query rows of a tile
constexpr int kKvThreads = 640;

struct KvItem {
  int stop;
  int hk, key;         // kv head, first key (global)
  int nk, j0;          // keys, position of the first
  int tok, ntok, pos;  // first query token (global), their number, the position of the first
  int sinks_only;      // 1: a chunk of queries past the window's reach, for the sinks alone
  float* part;         // where the sinks' sums go (fp32), or null
};

template <int D>
struct KvSmem {
  static constexpr int KT = TileShape<D>::bytes(128), QT = TileShape<D>::bytes(kKvRows);
  static constexpr int NK = D == 128 ? 1 : 2;  // K and V buffers
  static constexpr int NS = D == 128 ? 3 : 5;  // ring of (Q, dO, lse, delta)
  static constexpr int NT = D == 128 ? 2 : 3;  // TMEM stages of S^T and dP^T
  static constexpr int OFF_Q = 2 * NK * KT;
  static constexpr int OFF_ROWS = OFF_Q + 2 * NS * QT;
  static constexpr int OFF_STAT = OFF_ROWS + (D >= 64 ? 16 * kRowBuf : 0);
  static constexpr int OFF_ITEM = OFF_STAT + NS * 2 * kKvRows * 4;
  static constexpr int OFF_BAR = OFF_ITEM + kItems * (int)sizeof(KvItem);
  // k_full[NK], k_empty[NK], q_full[NS], q_empty[NS], s_full[NT], p_full[NT], acc_done[NT], acc_full,
  // acc_free, item_full[], item_empty[], mma_done[2]
  static constexpr int NBAR = 2 * NK + 2 * NS + 3 * NT + 2 + 2 * kItems + 2;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int BYTES = OFF_MISC + 16 + 1024;
  static constexpr int ALLOC = BYTES > kOneCtaPerSmSmem ? BYTES : kOneCtaPerSmSmem;
  static_assert(OFF_BAR % 8 == 0 && OFF_STAT % 16 == 0 && ALLOC <= 227 * 1024, "shared memory budget");
};

// The queries that the window of keys [j0, j0 + nk) reaches, as token range
// [first, last) of the sequence; from token 0 on for the tile of the sinks
// (queries ahead of its window see them too).
__device__ __forceinline__ void window_queries(const WindowParams& p, const Seq& s, int j0, int nk, int& first,
                                               int& last) {
  const int shift = s.lk - s.lq;
  first = max(0, j0 - p.right - shift);
  last = min(s.lq, j0 + nk + p.left - shift);
  if (j0 == 0 && p.sinks > 0) first = 0;
  if (last < first) last = first;
}

// Query tokens of chunk `c` of a sequence that see nothing of it but the sinks.
__device__ __forceinline__ void sink_queries(const WindowParams& p, const Seq& s, int chunk, int c, int& first,
                                             int& last) {
  int a, b;
  window_queries(p, s, 0, min(128, s.lk), a, b);
  first = max(c * chunk, b);
  last = s.lk > 0 ? min(s.lq, (c + 1) * chunk) : 0;
  if (last < first) last = first;
}

__device__ __forceinline__ bool kv_item(const WindowBwdParams& p, int w, int D, KvItem& it) {
  const int n_sink = p.chunk_slots * p.hkv;
  const long long row = (long long)p.sinks * 2 * D;
  it.sinks_only = w < n_sink;
  it.part = nullptr;
  if (it.sinks_only) {
    const int slot = w / p.hkv;
    it.hk = w - slot * p.hkv;
    const int b = seq_of_slot(p.cu_q, p.num_seqs, p.chunk, slot);
    if (b < 0 || b >= p.num_seqs) return false;
    const Seq s = seq_of(p, b);
    int first, last;
    sink_queries(p, s, p.chunk, slot - first_slot(p.cu_q, b, p.chunk), first, last);
    if (last <= first) return false;
    it.key = s.k0;
    it.nk = min(p.sinks, s.lk);
    it.j0 = 0;
    it.tok = s.q0 + first;
    it.ntok = last - first;
    it.pos = first + s.lk - s.lq;
    it.part = p.part + w * row;
    return true;
  }
  w -= n_sink;
  const int slot = w / p.hkv;
  it.hk = w - slot * p.hkv;
  const int b = seq_of_slot(p.cu_k, p.num_seqs, 128, slot);
  const Seq s = seq_of(p, b);
  const bool real = b >= 0 && b < p.num_seqs;
  it.j0 = (slot - first_slot(p.cu_k, b, 128)) * 128;
  if (it.j0 < 0 || it.j0 >= s.lk) return false;
  it.key = s.k0 + it.j0;
  it.nk = min(128, s.lk - it.j0);
  int first = 0, last = 0;
  if (real) window_queries(p, s, it.j0, it.nk, first, last);
  it.tok = s.q0 + first;
  it.ntok = last - first;
  it.pos = first + s.lk - s.lq;
  if (it.j0 == 0 && p.sinks > 0 && real) it.part = p.part0 + (long long)(b * p.hkv + it.hk) * row;
  return true;
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kKvThreads, 1)
    window_dkv_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do,
                      const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                      const WindowBwdParams p, const int n_items) {
  using L = KvSmem<D>;
  constexpr uint32_t AB = BF16 ? 1u : 0u;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sK = smem;                 // [NK][K, V]
  uint8_t* sQ = smem + L::OFF_Q;      // [NS][Q, dO]
  float* stat = reinterpret_cast<float*>(smem + L::OFF_STAT);  // [NS][lse (log2), delta][64], negated
  KvItem* items = reinterpret_cast<KvItem*>(smem + L::OFF_ITEM);
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* k_empty = k_full + L::NK;
  uint64_t* q_full = k_empty + L::NK;
  uint64_t* q_empty = q_full + L::NS;
  uint64_t* s_full = q_empty + L::NS;
  uint64_t* p_full = s_full + L::NT;
  uint64_t* acc_done = p_full + L::NT;
  uint64_t* acc_full = acc_done + L::NT;
  uint64_t* acc_free = acc_full + 1;
  uint64_t* item_full = acc_free + 1;
  uint64_t* item_empty = item_full + kItems;
  uint64_t* mma_done = item_empty + kItems;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::OFF_MISC + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = p.g, TT = kKvRows / G;

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::NK; ++i) mbar_init(&k_full[i], 1), mbar_init(&k_empty[i], 1);
    for (int i = 0; i < L::NS; ++i) mbar_init(&q_full[i], 2), mbar_init(&q_empty[i], 1);
    for (int i = 0; i < L::NT; ++i) mbar_init(&s_full[i], 1), mbar_init(&p_full[i], 8), mbar_init(&acc_done[i], 1);
    mbar_init(acc_full, 1);
    mbar_init(acc_free, 16);
    for (int i = 0; i < kItems; ++i) mbar_init(&item_full[i], 1), mbar_init(&item_empty[i], 19);
    mbar_init(&mma_done[0], 1);
    mbar_init(&mma_done[1], 1);
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
  // TMEM columns: stage st: S^T [128 st, +64), dP^T [128 st + 64, +64), P^T and dS^T over them; then dV, dK
  constexpr int NT = L::NT;
  const uint32_t tacc = tmem + NT * 128;

  if (warp == 17) {
    // ------------------------------ producer ------------------------------
    if (elect_one()) {
      tma_prefetch_desc(&tm_q);
      tma_prefetch_desc(&tm_do);
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
    }
    const uint32_t q_bytes = (uint32_t)(2 * G * TT * D * 2);
    int n_it = 0, J = 0, nk = 0;
    bool ok = true;
    for (int w = blockIdx.x; ok; w += gridDim.x) {
      KvItem it;
      it.stop = w >= n_items;
      if (!it.stop && !kv_item(p, w, D, it)) continue;
      const int r = n_it % kItems;
      if (!wait_phase(&item_empty[r], ((n_it / kItems) & 1) ^ 1, abort_flag, p.err)) break;
      if (lane == 0) {
        items[r] = it;
        mbar_arrive(&item_full[r]);
      }
      __syncwarp();
      ++n_it;
      if (it.stop) break;
      if (it.ntok <= 0) continue;
      const int sk = nk % L::NK;
      if (!(ok = wait_phase(&k_empty[sk], ((nk / L::NK) & 1) ^ 1, abort_flag, p.err))) break;
      if (elect_one()) {
        mbar_arrive_expect_tx(&k_full[sk], 2 * L::KT);
        load_tile<D>(sK + 2 * sk * L::KT, 128, &tm_k, it.hk, it.key, &k_full[sk]);
        load_tile<D>(sK + (2 * sk + 1) * L::KT, 128, &tm_v, it.hk, it.key, &k_full[sk]);
      }
      __syncwarp();
      ++nk;
      for (int t = 0; t * TT < it.ntok; ++t) {
        const int st = J % L::NS;
        if (!(ok = wait_phase(&q_empty[st], ((J / L::NS) & 1) ^ 1, abort_flag, p.err))) break;
        if (elect_one()) {
          mbar_arrive_expect_tx(&q_full[st], q_bytes);
          load_tile<D>(sQ + 2 * st * L::QT, kKvRows, &tm_q, it.hk * G, it.tok + t * TT, &q_full[st]);
          load_tile<D>(sQ + (2 * st + 1) * L::QT, kKvRows, &tm_do, it.hk * G, it.tok + t * TT, &q_full[st]);
        }
        __syncwarp();
        ++J;
      }
    }
    if (lane == 0 && *abort_flag) {  // copies in flight land before the CTA exits
      for (int k = max(0, nk - L::NK); k < nk; ++k) mbar_wait_drain(&k_full[k % L::NK], (k / L::NK) & 1);
      for (int j = max(0, J - L::NS); j < J; ++j) mbar_wait_drain(&q_full[j % L::NS], (j / L::NS) & 1);
    }
    __syncwarp();
  } else if (warp == 18) {
    // -------------------- lse and delta of the query rows --------------------
    int tr[2], off[2], n_it = 0, J = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      tr[i] = (lane + 32 * i) / G;
      off[i] = tr[i] * p.hq + lane + 32 * i - tr[i] * G;
    }
    bool ok = true;
    while (ok) {
      const int r = n_it % kItems;
      if (!wait_phase(&item_full[r], (n_it / kItems) & 1, abort_flag, p.err)) break;
      const KvItem& it = items[r];
      ++n_it;
      if (it.stop) break;
      const int ntok = it.ntok;
      const long long base = (long long)it.tok * p.hq + it.hk * G;
      float l[2], d[2];
      auto fetch = [&](int t) {  // the next tile's are on their way while this one waits for its slot
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          l[i] = d[i] = 0.f;
          if (tr[i] < TT && t * TT + tr[i] < ntok) {
            const long long at = base + (long long)t * TT * p.hq + off[i];
            l[i] = p.lse[at];
            d[i] = p.delta[at];
          }
        }
      };
      fetch(0);
      for (int t = 0; t * TT < ntok; ++t, ++J) {
        const int st = J % L::NS;
        if (!(ok = wait_phase(&q_empty[st], ((J / L::NS) & 1) ^ 1, abort_flag, p.err))) break;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          // a query that sees nothing (lse = -inf): every key is masked
          stat[(2 * st) * kKvRows + lane + 32 * i] = l[i] == -INFINITY ? 0.f : l[i] * -1.4426950408889634f;
          stat[(2 * st + 1) * kKvRows + lane + 32 * i] = -d[i];
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[st]);
        fetch(t + 1);
      }
      if (!ok) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[r]);
    }
  } else if (warp == 16) {
    // --------------------- tensor-core issue: S^T and dP^T -------------------
    const uint32_t idesc = make_idesc(AB, 0, 0, 128, kKvRows);
    int n_it = 0, J = 0, nk = 0;  // items, query tiles, K tiles so far
    while (true) {
      const int r = n_it % kItems;
      if (!wait_phase(&item_full[r], (n_it / kItems) & 1, abort_flag, p.err)) break;
      const KvItem& it = items[r];
      ++n_it;
      if (it.stop) break;
      const int n = (it.ntok + TT - 1) / TT, ntok = it.ntok;
      bool ok = true;
      if (n > 0) {
        const int sk = nk % L::NK;
        const uint32_t k_base = smem_u32(sK + 2 * sk * L::KT), v_base = k_base + L::KT;
        if (!wait_phase(&k_full[sk], (nk / L::NK) & 1, abort_flag, p.err)) break;
        ++nk;
        for (int t = 0; t < n; ++t, ++J) {
          const int st = J % L::NS, stage = J % NT;
          if (!(ok = wait_phase(&q_full[st], (J / L::NS) & 1, abort_flag, p.err))) break;
          // rows that hold no query of the sequence must not reach the sums, not even times zero
          const int rows = min(TT, ntok - t * TT) * G;
          if (rows < kKvRows) {
            zero_rows<D>(sQ + 2 * st * L::QT, kKvRows, rows);
            zero_rows<D>(sQ + (2 * st + 1) * L::QT, kKvRows, rows);
          }
          // the sums that read the stage's last P^T and dS^T are over
          if (J >= NT && !(ok = wait_phase(&acc_done[stage], ((J / NT) & 1) ^ 1, abort_flag, p.err))) break;
          tc_fence_after();
          if (elect_one()) {
            const uint32_t q_base = smem_u32(sQ + 2 * st * L::QT), do_base = q_base + L::QT;
            const uint32_t tm_s = tmem + stage * 128;
            mma_rows<D, 128, kKvRows>(tm_s, k_base, q_base, idesc);
            mma_rows<D, 128, kKvRows>(tm_s + 64, v_base, do_base, idesc);
            umma_commit(&s_full[stage]);
            if (t == n - 1) umma_commit(&k_empty[sk]);
          }
          __syncwarp();
        }
      }
      if (!ok) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[r]);
    }
    if (elect_one()) {
      umma_commit(&mma_done[0]);
      mbar_wait_drain(&mma_done[0], 0);
    }
    __syncwarp();
  } else if (warp == 19) {
    // ------------------------ tensor-core issue: dV and dK --------------------
    // (S^T's issue has seen the tile's Q and dO, and zeroed what is no query, before P^T can be announced)
    const uint32_t idesc = make_idesc(AB, 0, 1, 128, D);
    const uint32_t tm_dv = tacc, tm_dk = tacc + D;
    int n_it = 0, J = 0, n_acc = 0;  // items, query tiles, items with sums so far
    while (true) {
      const int r = n_it % kItems;
      if (!wait_phase(&item_full[r], (n_it / kItems) & 1, abort_flag, p.err)) break;
      const KvItem& it = items[r];
      ++n_it;
      if (it.stop) break;
      const int n = (it.ntok + TT - 1) / TT;
      bool ok = true;
      for (int t = 0; t < n; ++t, ++J) {
        const int st = J % L::NS, stage = J % NT;
        // the last item's sums have been read
        if (t == 0 && n_acc > 0 && !(ok = wait_phase(acc_free, (n_acc - 1) & 1, abort_flag, p.err))) break;
        if (!(ok = wait_phase(&q_full[st], (J / L::NS) & 1, abort_flag, p.err))) break;
        if (!(ok = wait_phase(&p_full[stage], (J / NT) & 1, abort_flag, p.err))) break;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t q_base = smem_u32(sQ + 2 * st * L::QT), do_base = q_base + L::QT;
          const uint32_t tm_p = tmem + 128 * stage;
          mma_sum<D, kKvRows, 16>(tm_dv, tm_p, do_base, idesc, t > 0);
          mma_sum<D, kKvRows, 16>(tm_dk, tm_p + 64, q_base, idesc, t > 0);
          umma_commit(&acc_done[stage]);
          umma_commit(&q_empty[st]);
          if (t == n - 1) umma_commit(acc_full);
        }
        __syncwarp();
      }
      if (!ok) break;
      if (n > 0) ++n_acc;
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[r]);
    }
    if (elect_one()) {
      umma_commit(&mma_done[1]);
      mbar_wait_drain(&mma_done[1], 0);
    }
    __syncwarp();
  } else {
    // --------------------------- P^T and dS^T --------------------------------
    const int wg = warp >> 3, half = (warp >> 2) & 1, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const float sl2 = p.scale * 1.4426950408889634f;
    const float2 sc = make_float2(sl2, sl2);
    const float mul = wg ? p.scale : 1.f;
    uint16_t* out = static_cast<uint16_t*>(wg ? p.dk : p.dv);
    constexpr int DH = D / 2, CH = DH < 32 ? DH : 32;
    // An item's sums leave after the group's first tile of the next one: what they wait for runs under that tile.
    bool due = false;
    long long due_row = -1;   // row of dK / dV, or none
    float* due_part = nullptr;  // place of a sink's sums, or none
    int n_it = 0, J = 0, n_acc = 0;
    // warps 0-7 write dV, warps 8-15 dK, a half of the channels each
    auto write_sums = [&](bool any) -> bool {
      if (any) {
        if (!wait_phase(acc_full, n_acc & 1, abort_flag, p.err)) return false;
        ++n_acc;
        tc_fence_after();
      }
#pragma unroll
      for (int c = 0; c < DH; c += CH) {
        float s[CH];
        uint32_t w[CH / 2];
        if (any) {
          tmem_load_cols<CH>(tacc + wg * D + half * DH + c + lanes, s);
          tmem_wait_values<CH>(s);
          if (c + CH == DH) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_free);
          }
        }
#pragma unroll
        for (int i = 0; i < CH; ++i) s[i] = any ? s[i] * mul : 0.f;
#pragma unroll
        for (int i = 0; i < CH; i += 2) w[i / 2] = pack2<BF16>(s[i], s[i + 1]);
        if constexpr (CH == 32) {
          store_rows32(smem_u32(smem + L::OFF_ROWS + warp * kRowBuf), w, due_row, out, D, half * DH + c);
        } else if (due_row >= 0) {
#pragma unroll
          for (int i = 0; i < CH; i += 8)
            *reinterpret_cast<uint4*>(out + due_row * D + half * DH + c + i) =
                make_uint4(w[i / 2], w[i / 2 + 1], w[i / 2 + 2], w[i / 2 + 3]);
        }
        if (due_part) {
#pragma unroll
          for (int i = 0; i < CH; i += 4)
            *reinterpret_cast<float4*>(due_part + c + i) = make_float4(s[i], s[i + 1], s[i + 2], s[i + 3]);
        }
      }
      return true;
    };
    while (true) {
      const int r = n_it % kItems;
      if (!wait_phase(&item_full[r], (n_it / kItems) & 1, abort_flag, p.err)) break;
      const KvItem& it = items[r];
      ++n_it;
      if (it.stop) {
        if (due) write_sums(true);
        break;
      }
      const int n = (it.ntok + TT - 1) / TT;
      // queries that see this thread's key, as a token range of the item
      const int j = it.j0 + row;
      int lo = j - p.right - it.pos, hi = j + p.left + 1 - it.pos;
      if (j < p.sinks) {
        if (!p.causal) lo = 0;
        hi = it.ntok;
      } else if (it.sinks_only) {
        hi = lo;
      }
      lo = max(lo, 0);
      hi = min(hi, it.ntok);
      const bool live = row < it.nk;
      if (!live) hi = lo;
      const bool to_part = live && it.part && j < p.sinks;
      const long long row_out = live && !it.sinks_only && !to_part ? (long long)(it.key + row) * p.hkv + it.hk : -1;
      float* const part = to_part ? it.part + (long long)(j * 2 + wg) * D + half * DH : nullptr;
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[r]);
      bool ok = true;
      for (int t = (J & 1) ^ wg; t < n; t += 2) {
        const int jt = J + t, st = jt % L::NS, sg = jt % NT;
        // P^T and dS^T go over S^T and dP^T: the halves' places do not touch what the other one may still read
        const uint32_t tm_s = tmem + sg * 128 + 32 * half + lanes, tm_dp = tm_s + 64;
        const uint32_t bits = range_bits((lo - t * TT) * G - 32 * half, (min(hi, (t + 1) * TT) - t * TT) * G - 32 * half);
        const bool some = __any_sync(0xffffffffu, bits != 0u);
        const bool full = __all_sync(0xffffffffu, !live || bits == 0xffffffffu);
        if (!(ok = wait_phase(&s_full[sg], (jt / NT) & 1, abort_flag, p.err))) break;
        tc_fence_after();
        const float* nl = stat + (2 * st) * kKvRows + 32 * half;
        const float* nd = nl + kKvRows;
        if (some) {
#pragma unroll
          for (int c = 0; c < 32; c += 8) {
            float s[8], d[8];
            uint32_t wp[4], wd[4];
            tmem_ld8(tm_s + c, s);
            tmem_wait_values<8>(s);
            tmem_ld8(tm_dp + c, d);
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
              const float4 l4 = *reinterpret_cast<const float4*>(nl + c + i);
              float2 e0 = fma2(make_float2(s[i], s[i + 1]), sc, make_float2(l4.x, l4.y));
              float2 e1 = fma2(make_float2(s[i + 2], s[i + 3]), sc, make_float2(l4.z, l4.w));
              s[i] = ex2(e0.x);
              s[i + 1] = ex2(e0.y);
              s[i + 2] = ex2(e1.x);
              s[i + 3] = ex2(e1.y);
            }
            tmem_wait_values<8>(d);
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
              const float4 d4 = *reinterpret_cast<const float4*>(nd + c + i);
              float2 e0 = make_float2(s[i], s[i + 1]), e1 = make_float2(s[i + 2], s[i + 3]);
              float2 f0 = mul2(e0, add2(make_float2(d[i], d[i + 1]), make_float2(d4.x, d4.y)));
              float2 f1 = mul2(e1, add2(make_float2(d[i + 2], d[i + 3]), make_float2(d4.z, d4.w)));
              if (!full) {
                const uint32_t b4 = bits >> (c + i);
                e0.x = (b4 & 1u) ? e0.x : 0.f, f0.x = (b4 & 1u) ? f0.x : 0.f;
                e0.y = (b4 & 2u) ? e0.y : 0.f, f0.y = (b4 & 2u) ? f0.y : 0.f;
                e1.x = (b4 & 4u) ? e1.x : 0.f, f1.x = (b4 & 4u) ? f1.x : 0.f;
                e1.y = (b4 & 8u) ? e1.y : 0.f, f1.y = (b4 & 8u) ? f1.y : 0.f;
              }
              wp[i / 2] = pack2<BF16>(e0.x, e0.y);
              wp[i / 2 + 1] = pack2<BF16>(e1.x, e1.y);
              wd[i / 2] = pack2<BF16>(f0.x, f0.y);
              wd[i / 2 + 1] = pack2<BF16>(f1.x, f1.y);
            }
            tmem_st4(tm_s + c / 2, wp);  // over S^T and dP^T, the columns are ones that have been read
            tmem_st4(tm_dp + c / 2, wd);
          }
        } else {
          const uint32_t z[16] = {};
          tmem_st16(tm_s, z);
          tmem_st16(tm_dp, z);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[sg]);
        if (due) {
          due = false;
          if (!(ok = write_sums(true))) break;
        }
      }
      if (!ok) break;
      J += n;
      if (due) {  // the group had no tile of this item
        due = false;
        if (!write_sums(true)) break;
      }
      due_row = row_out;
      due_part = part;
      if (n > 0) due = true;
      else write_sums(false);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

// dv and dk of the sinks: their own tile's sum, then the chunks' in ascending
// order (four interleaved runs, joined in order).  A block a sink; bound by the
// chain of loads (131072 tokens, 16 heads of 64 channels, 16 sinks: 21 us).
template <typename T, int D>
__global__ void __launch_bounds__(4 * 2 * D) sink_sum_kernel(const WindowBwdParams p) {
  __shared__ float sum[4][2 * D];
  const int b = blockIdx.x, hk = blockIdx.y, j = blockIdx.z, e = threadIdx.x;
  const Seq s = seq_of(p, b);
  if (j >= min(p.sinks, s.lk)) return;
  const long long row = (long long)p.sinks * 2 * D;
  const int slot0 = first_slot(p.cu_q, b, p.chunk);
  float a = 0.f;
  for (int c = threadIdx.y; c * p.chunk < s.lq; c += 4) {
    int first, last;
    sink_queries(p, s, p.chunk, c, first, last);
    if (last > first) a += p.part[((long long)(slot0 + c) * p.hkv + hk) * row + j * 2 * D + e];
  }
  sum[threadIdx.y][e] = a;
  __syncthreads();
  if (threadIdx.y) return;
  a = p.part0[(long long)(b * p.hkv + hk) * row + j * 2 * D + e];
  for (int i = 0; i < 4; ++i) a += sum[i][e];
  T* out = static_cast<T*>(e < D ? p.dv : p.dk);
  out[((long long)(s.k0 + j) * p.hkv + hk) * D + e % D] = (T)a;
}

// Query tokens of a sink chunk: at least as many as a key tile's window
// reaches, so that its item is no longer than they are, and never under 1024,
// which bounds the partial sums' memory.
int sink_chunk(const WindowParams& p) { return std::max(1024, 128 + p.left + p.right); }

struct BwdLayout {
  size_t delta, part0, part, bytes;
  int chunk, slots;
};

BwdLayout bwd_layout(const WindowParams& p, int D) {
  BwdLayout l{};
  l.delta = 0;
  size_t at = align_up((size_t)p.total_q * p.hq * sizeof(float), 256);
  if (p.sinks > 0 && p.num_seqs > 0) {
    l.chunk = sink_chunk(p);
    l.slots = tile_slots(p.total_q, p.num_seqs, l.chunk);
    const size_t row = (size_t)p.hkv * p.sinks * 2 * D * sizeof(float);
    l.part0 = at;
    at = align_up(at + p.num_seqs * row, 256);
    l.part = at;
    at = align_up(at + l.slots * row, 256);
  }
  l.bytes = at + 256;
  return l;
}

template <int D, bool BF16>
int launch_bwd(const WindowBwdParams& p, cudaStream_t s) {
  using T = std::conditional_t<BF16, __nv_bfloat16, __half>;
  using S = TileShape<D>;
  const int tt = 128 / p.g, tk = kKvRows / p.g;
  int rc;
  if (p.total_q > 0) {
    ProfScope ps("window_attn_delta", s);
    const long long rows = (long long)p.total_q * p.hq;
    const int grid = (int)std::min<long long>((rows * (D / 8) + 255) / 256, (long long)num_sms() * 8);
    window_delta_kernel<T, D><<<grid, 256, 0, s>>>(static_cast<const uint4*>(p.out),
                                                   static_cast<const uint4*>(p.out_rest),
                                                   static_cast<const uint4*>(p.dout), p.delta, rows);
    LSRM_LAUNCH_CHECK();
  }
  // no query or no key at all: the maps are never read
  const void* q = p.total_q ? p.q : p.k;
  const void* d = p.total_q ? p.dout : p.k;
  const void* k = p.total_k ? p.k : p.q;
  const void* v = p.total_k ? p.v : p.q;
  const long long qs = p.total_q ? p.q_stride : p.k_stride, ds = p.total_q ? (long long)p.hq * D : p.k_stride;
  const long long ks = p.total_k ? p.k_stride : p.q_stride, vs = p.total_k ? p.v_stride : p.q_stride;
  CUtensorMap mq, md, mk, mv;
  if (p.total_q > 0) {
    if ((rc = make_tmap_3d(&mq, q, D, p.hq, p.total_q, qs, p.g, tt, S::kCols))) return rc;
    if ((rc = make_tmap_3d(&md, d, D, p.hq, p.total_q, ds, p.g, tt, S::kCols))) return rc;
    if ((rc = make_tmap_3d(&mk, k, D, p.hkv, p.total_k, ks, 1, kDqKeys, S::kCols))) return rc;
    if ((rc = make_tmap_3d(&mv, v, D, p.hkv, p.total_k, vs, 1, kDqKeys, S::kCols))) return rc;
    ProfScope ps("window_attn_dq", s);
    const int n_items = tile_slots(p.total_q, p.num_seqs, 2 * tt) * p.hkv;
    LSRM_CUDA_TRY(cudaFuncSetAttribute(window_dq_kernel<D, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       DqSmem<D>::ALLOC));
    window_dq_kernel<D, BF16><<<std::min(n_items, num_sms()), kBwThreads, DqSmem<D>::ALLOC, s>>>(mq, md, mk, mv, p,
                                                                                                 n_items);
    LSRM_LAUNCH_CHECK();
  }
  if (p.total_k > 0) {
    if ((rc = make_tmap_3d(&mq, q, D, p.hq, p.total_q, qs, p.g, tk, S::kCols))) return rc;
    if ((rc = make_tmap_3d(&md, d, D, p.hq, p.total_q, ds, p.g, tk, S::kCols))) return rc;
    if ((rc = make_tmap_3d(&mk, k, D, p.hkv, p.total_k, ks, 1, 128, S::kCols))) return rc;
    if ((rc = make_tmap_3d(&mv, v, D, p.hkv, p.total_k, vs, 1, 128, S::kCols))) return rc;
    {
      ProfScope ps("window_attn_dkv", s);
      const int n_items = (tile_slots(p.total_k, p.num_seqs, 128) + p.chunk_slots) * p.hkv;
      LSRM_CUDA_TRY(cudaFuncSetAttribute(window_dkv_kernel<D, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         KvSmem<D>::ALLOC));
      window_dkv_kernel<D, BF16><<<std::min(n_items, num_sms()), kKvThreads, KvSmem<D>::ALLOC, s>>>(mq, md, mk, mv, p,
                                                                                                    n_items);
      LSRM_LAUNCH_CHECK();
    }
    if (p.chunk) {
      ProfScope ps("window_attn_sinks", s);
      sink_sum_kernel<T, D><<<dim3(p.num_seqs, p.hkv, p.sinks), dim3(2 * D, 4), 0, s>>>(p);
      LSRM_LAUNCH_CHECK();
    }
  }
  return LSRM_OK;
}

}  // namespace
}  // namespace lsrm

using namespace lsrm;

extern "C" size_t lsrm_window_attn_workspace_bytes(const lsrm_window_shape* shape) {
  if (!shape || shape->total_q < 0 || shape->total_k < 0 || shape->num_seqs < 0 || shape->num_kv_heads < 1 ||
      shape->num_q_heads < 1 || shape->window < 1)
    return 0;
  return bwd_layout(window_params(shape, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr),
                    shape->head_dim)
      .bytes;
}

extern "C" int lsrm_window_attn_bwd(const lsrm_window_shape* shape, const int32_t* cu_seqlens_q,
                                    const int32_t* cu_seqlens_k, const void* q, const void* k, const void* v,
                                    const void* out, const void* out_rest, const float* lse, const void* dout,
                                    void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes,
                                    int* err_flags, void* stream) {
  int rc = check_window(shape, cu_seqlens_q, cu_seqlens_k, q, k, v);
  if (rc) return rc;
  LSRM_CHECK_ARG((shape->total_q == 0 || (out && lse && dout && dq)) && (shape->total_k == 0 || (dk && dv)),
                 "out, lse, dout and the gradients must not be NULL");
  LSRM_CHECK_ARG((((uintptr_t)out | (uintptr_t)out_rest | (uintptr_t)dout | (uintptr_t)dq | (uintptr_t)dk |
                   (uintptr_t)dv) & 15) == 0, "out, out_rest, dout and the gradients must be 16-byte aligned");
  if (!workspace || workspace_bytes < lsrm_window_attn_workspace_bytes(shape)) {
    set_error("workspace too small: %zu bytes, %zu needed", workspace_bytes, lsrm_window_attn_workspace_bytes(shape));
    return LSRM_ERR_WORKSPACE;
  }
  LSRM_CHECK_ARG(((uintptr_t)workspace & 255) == 0, "the workspace must be 256-byte aligned");
  if (shape->total_q == 0 && shape->total_k == 0) return LSRM_OK;
  WindowBwdParams p;
  static_cast<WindowParams&>(p) = window_params(shape, cu_seqlens_q, cu_seqlens_k, q, k, v, const_cast<void*>(out),
                                                const_cast<float*>(lse), err_flags);
  p.out_rest = const_cast<void*>(out_rest), p.dout = dout, p.dq = dq, p.dk = dk, p.dv = dv;
  const BwdLayout l = bwd_layout(p, shape->head_dim);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.delta = reinterpret_cast<float*>(ws + l.delta);
  p.chunk = l.chunk, p.chunk_slots = l.slots;
  p.part0 = reinterpret_cast<float*>(ws + l.part0);
  p.part = reinterpret_cast<float*>(ws + l.part);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define CALL(BF, D) return launch_bwd<D, BF>(p, s);
  WINDOW_TYPES(CALL)
#undef CALL
}
