// The single-token form of the windowed attention with sinks over a ring
// cache.  Sequence b holds n = lengths[b] tokens; the new token takes position
// n.  Position j is kept in slot j while j < sinks, else in slot
// sinks + (j - sinks) % (capacity - sinks): the ring holds the last
// capacity - sinks positions past the sinks.  The call writes the new key and
// value to their slot and attends to positions [0, sinks) and (n - window, n].
// A negative length marks an idle row: nothing is written, its output is 0.
//
// The work is reading the visible keys and values once: bound by HBM.  Up to
// sixteen query heads of a kv head share one read (rows of an m16n8k16 product;
// at a few heads a row the products are hardly used, and still far from the
// limit).  A (sequence, kv head)'s positions are cut over the CTAs of a
// thread-block cluster, so that few rows fill the GPU too; each CTA streams its
// slice through a cp.async ring, 64 positions a stage, a quarter of a stage a
// warp, every warp with its own running maximum and sum.  The warps' and then
// the cluster's partial results are joined through shared memory in one launch.
// Probabilities enter the product as the sum of two 16-bit values (the
// remainder of the first one's rounding in the second), which costs tensor
// work that is idle and leaves the output's rounding the only one (5 % of the
// time where the caches are large).  Measured: 64 sequences of up to 20000
// tokens, window 8192, 8 kv heads of 128 read 1.59 GB in 298 us, 5.35 TB/s or
// 82 % of a plain copy's rate (reads alone, without the products: 242 us); one
// row takes 5.4 us, which is the launch, two round trips to HBM and the join.
#include <algorithm>

#include "common.cuh"
#include "host_util.h"
#include "window_common.cuh"

namespace lsrm {
namespace {

struct DecodeParams {
  int batch, hq, hkv, g, capacity, window, sinks;
  float scale;
  long long q_stride, kn_stride, vn_stride;            // elements between sequences of q, k_new, v_new
  long long kc_batch, kc_slot, vc_batch, vc_slot;      // elements between sequences / slots of the caches
  const void *q, *k_new, *v_new;
  void *k_cache, *v_cache, *out;
  const int32_t* lengths;
};

constexpr int kDcRows = 16;      // query heads of a CTA
constexpr int kDcKeys = 64;      // positions of a stage
constexpr int kDcThreads = 128;
constexpr int kDcMaxSplit = 8;   // CTAs of a cluster (the portable limit)

template <int D>
struct DcSmem {
  static constexpr int TILE = kDcKeys * D * 2;
  // Two stages leave room for three CTAs a multiprocessor, which hide each other's products better than a deeper ring
  // of two CTAs: 298 us against 332 (64 sequences, window 8192, 8 kv heads of 128), 17.0 against 19.4 (16, 1024, 16 of 64).
  static constexpr int NS = 2;
  static constexpr int RING = 2 * NS * TILE;
  // after the ring: per warp m, l and O; the first one's slot ends up with the CTA's
  static constexpr int PART = (2 * kDcRows + kDcRows * D) * 4;
  static constexpr int BYTES = RING > 4 * PART ? RING : 4 * PART;
};

// 16-byte chunk `c` of row `r` of a [rows][D] tile: the low bits are swizzled so
// that eight rows of one chunk fall into different banks.
template <int D>
__device__ __forceinline__ uint32_t dc_offset(int r, int c) {
  if constexpr (D >= 64) return r * (2 * D) + ((c ^ (r & 7)) << 4);
  else return r * (2 * D) + ((c ^ ((r >> 1) & 3)) << 4);
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
// c += a (16 x 16) b (16 x 8)
template <bool BF16>
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, const uint32_t* b) {
  if constexpr (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

// cp.async of 16 bytes, or of zeros where `live` is false.
__device__ __forceinline__ void cp_async_16_or_zero(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The float at this CTA's shared address `addr`, in the cluster's CTA `rank`.
__device__ __forceinline__ float ld_cluster(uint32_t addr, uint32_t rank) {
  uint32_t remote;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
  return v;
}

// grid (splits, kv heads x blocks of 16 query heads, batch), clusters of `splits`
template <int D, bool BF16>
__global__ void __launch_bounds__(kDcThreads) window_decode_kernel(const DecodeParams p) {
  using L = DcSmem<D>;
  constexpr int CH = D / 8;  // 16-byte chunks of a row
  extern __shared__ __align__(16) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int splits = gridDim.x, split = splits > 1 ? (int)cluster_rank() : 0;
  const int blocks = (p.g + kDcRows - 1) / kDcRows;
  const int hk = blockIdx.y / blocks, row0 = (blockIdx.y - hk * blocks) * kDcRows, b = blockIdx.z;
  const int rows = min(kDcRows, p.g - row0), h0 = hk * p.g + row0;
  const int n = p.lengths[b], ring = p.capacity - p.sinks;
  const uint16_t* kn = static_cast<const uint16_t*>(p.k_new) + b * p.kn_stride + hk * D;
  const uint16_t* vn = static_cast<const uint16_t*>(p.v_new) + b * p.vn_stride + hk * D;
  uint16_t* kc = static_cast<uint16_t*>(p.k_cache) + b * p.kc_batch + hk * D;
  uint16_t* vc = static_cast<uint16_t*>(p.v_cache) + b * p.vc_batch + hk * D;
  uint16_t* out = static_cast<uint16_t*>(p.out) + ((long long)b * p.hq + h0) * D;

  // visible positions, numbered 0 .. cnt - 1: the sinks, then the window's; the last one is the new token
  // (n itself may be the largest int: no n + 1)
  const int sink = n < 0 ? 0 : n < p.sinks ? n + 1 : p.sinks;
  const int lo = max(p.sinks, n - p.window + 1);
  const int cnt = n < 0 ? 0 : sink + (n < lo ? 0 : n - lo + 1);
  const int first_slot = lo > p.sinks ? (lo - p.sinks) % ring : 0;  // the window's first position in the ring
  auto slot_of = [&](int i) {
    if (i < sink) return i;
    const int s = first_slot + i - sink;
    return p.sinks + (s >= ring ? s - ring : s);
  };
  // this CTA's slice, whole stages
  const int stages = (cnt + kDcKeys - 1) / kDcKeys;
  const int t0 = (int)((long long)stages * split / splits), t1 = (int)((long long)stages * (split + 1) / splits);

  if (split == 0 && row0 == 0 && cnt > 0 && tid < 2 * CH) {  // the new token enters the cache (its slot is read by nobody)
    const bool is_v = tid >= CH;
    const int c = is_v ? tid - CH : tid, slot = slot_of(cnt - 1);
    reinterpret_cast<uint4*>(is_v ? vc + slot * p.vc_slot : kc + slot * p.kc_slot)[c] =
        reinterpret_cast<const uint4*>(is_v ? vn : kn)[c];
  }

  const uint32_t s_base = smem_u32(smem);
  auto load_stage = [&](int t) {
    if (t < t1) {
      const uint32_t dst = s_base + (t - t0) % L::NS * 2 * L::TILE;
#pragma unroll
      for (int i = tid; i < kDcKeys * CH; i += kDcThreads) {
        const int r = i / CH, c = i % CH, pos = t * kDcKeys + r;
        const bool live = pos < cnt, is_new = pos == cnt - 1;
        const int slot = live ? slot_of(pos) : 0;
        const uint16_t* ks = is_new ? kn : kc + slot * p.kc_slot;
        const uint16_t* vs = is_new ? vn : vc + slot * p.vc_slot;
        cp_async_16_or_zero(dst + dc_offset<D>(r, c), ks + 8 * c, live);
        cp_async_16_or_zero(dst + L::TILE + dc_offset<D>(r, c), vs + 8 * c, live);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < L::NS - 1; ++i) load_stage(t0 + i);

  // Q as A operand: rows lane / 4 and + 8
  const int r0 = lane >> 2, cq = (lane & 3) * 2;
  uint32_t aq[D / 16][4];
  const uint16_t* q = static_cast<const uint16_t*>(p.q) + b * p.q_stride + (long long)h0 * D;
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = r0 + (i & 1) * 8, c = ks * 16 + cq + (i >> 1) * 8;
      aq[ks][i] = r < rows ? *reinterpret_cast<const uint32_t*>(q + r * D + c) : 0u;
    }
  }
  float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
  const float sl2 = p.scale * 1.4426950408889634f;
  const int mat = lane >> 3, mrow = lane & 7;  // the ldmatrix tile and row whose address this lane gives

  for (int t = t0; t < t1; ++t) {
    cp_async_wait<L::NS - 2>();
    __syncthreads();
    load_stage(t + L::NS - 1);
    const uint32_t k_base = s_base + (t - t0) % L::NS * 2 * L::TILE, v_base = k_base + L::TILE;
    const int kr = warp * 16;  // this warp's rows of the stage
    if (t * kDcKeys + kr >= cnt) continue;
    float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      uint32_t kb[4];
      ldsm4(k_base + dc_offset<D>(kr + (mat >> 1) * 8 + mrow, 2 * ks + (mat & 1)), kb);
      mma16816<BF16>(s[0], aq[ks], kb);
      mma16816<BF16>(s[1], aq[ks], kb + 2);
    }
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int pos = t * kDcKeys + kr + 8 * j + cq + (i & 1);
        s[j][i] = pos < cnt ? s[j][i] * sl2 : -INFINITY;
        mx[i >> 1] = fmaxf(mx[i >> 1], s[j][i]);
      }
    float off[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
      const float m_new = fmaxf(m[i], mx[i]);
      off[i] = m_new == -INFINITY ? 0.f : m_new;
      const float f = ex2(m[i] - off[i]);
      m[i] = m_new;
      if (f != 1.f) {
        l[i] *= f;
#pragma unroll
        for (int c = 0; c < D / 8; ++c) o[c][2 * i] *= f, o[c][2 * i + 1] *= f;
      }
    }
    uint32_t ph[4], pl[4];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {  // rows r0 and r0 + 8
        const float e0 = ex2(s[j][2 * i] - off[i]), e1 = ex2(s[j][2 * i + 1] - off[i]);
        l[i] += e0 + e1;
        ph[2 * j + i] = pack2<BF16>(e0, e1);
        const float2 h = unpack2<BF16>(ph[2 * j + i]);
        pl[2 * j + i] = pack2<BF16>(e0 - h.x, e1 - h.y);
      }
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      uint32_t vb[4];
      ldsm4_t(v_base + dc_offset<D>(kr + (mat & 1) * 8 + mrow, 2 * c + (mat >> 1)), vb);
      mma16816<BF16>(o[2 * c], ph, vb);
      mma16816<BF16>(o[2 * c], pl, vb);
      mma16816<BF16>(o[2 * c + 1], ph, vb + 2);
      mma16816<BF16>(o[2 * c + 1], pl, vb + 2);
    }
  }
  cp_async_wait<0>();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
  }
  __syncthreads();  // the ring is free
  // partial results [warp]: m[16], l[16], O[16][D]
  float* part = reinterpret_cast<float*>(smem);
  constexpr int PF = L::PART / 4;
  {
    float* w = part + warp * PF;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = r0 + 8 * i;
      if (r >= rows) continue;
      if ((lane & 3) == 0) w[r] = m[i], w[kDcRows + r] = l[i];
#pragma unroll
      for (int c = 0; c < D / 8; ++c)
        *reinterpret_cast<float2*>(w + 2 * kDcRows + r * D + 8 * c + cq) = make_float2(o[c][2 * i], o[c][2 * i + 1]);
    }
  }
  __syncthreads();
  // Joins parts as fetch(i, offset) gives them, i < n, for element e of row r.
  auto join = [&](int parts, int r, int e, float& mj, float& lj, auto fetch) {
    mj = -INFINITY;
    for (int i = 0; i < parts; ++i) mj = fmaxf(mj, fetch(i, r));
    const float off = mj == -INFINITY ? 0.f : mj;
    float acc = 0.f;
    lj = 0.f;
    for (int i = 0; i < parts; ++i) {
      const float f = ex2(fetch(i, r) - off);
      lj = fmaf(f, fetch(i, kDcRows + r), lj);
      acc = fmaf(f, fetch(i, 2 * kDcRows + r * D + e), acc);
    }
    return acc;
  };
  auto put = [&](int r, int e, float acc, float lj) {
    const float v = lj == 0.f ? 0.f : acc / lj;
    out[r * D + e] = BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
  };
  auto local = [&](int i, int at) { return part[i * PF + at]; };
  if (splits == 1) {
    for (int i = tid; i < rows * D; i += kDcThreads) {
      float mj, lj;
      const float acc = join(4, i / D, i % D, mj, lj, local);
      put(i / D, i % D, acc, lj);
    }
    return;
  }
  // the CTA's own result replaces warp 0's (every element is read by the thread that writes it, m and l last)
  for (int i = tid; i < rows * D; i += kDcThreads) {
    float mj, lj;
    const float acc = join(4, i / D, i % D, mj, lj, local);
    part[2 * kDcRows + i] = acc;
  }
  __syncthreads();
  float mj = 0.f, lj = 0.f;
  if (tid < rows) join(4, tid, 0, mj, lj, local);
  __syncthreads();
  if (tid < rows) part[tid] = mj, part[kDcRows + tid] = lj;
  cluster_sync();
  auto remote = [&](int i, int at) { return ld_cluster(s_base + at * 4, (uint32_t)i); };
  for (int i = split * kDcThreads + tid; i < rows * D; i += splits * kDcThreads) {
    float mc, lc;
    const float acc = join(splits, i / D, i % D, mc, lc, remote);
    put(i / D, i % D, acc, lc);
  }
  cluster_sync();  // no CTA leaves while another reads its shared memory
}

template <int D, bool BF16>
int launch_decode(const DecodeParams& p, cudaStream_t s) {
  const int blocks = (p.g + kDcRows - 1) / kDcRows;
  const long long ctas = (long long)p.batch * p.hkv * blocks;
  // Cut a row's positions while fewer than two CTAs a multiprocessor run and each keeps a stage; past that only long
  // rows, whose ragged lengths then even out over a few rounds.  At one, two, four and eight cuts, * the rule's: 64
  // sequences, window 8192, 8 kv heads of 128: 331, 322, 318*, 344 us; 16 sequences, window 1024, 16 kv heads of 64:
  // 21.6, 15.1*, 16.6, 20.6; 32 of window 512: 14.6*, 16.1, 19.9, 31.8; one sequence, window 8192, 8 kv heads of 128: 188,
  // 98, 52, 29.1* (34 MB, 5.2 us at a copy's rate: 64 CTAs with a stage each in flight do not fill HBM).
  const int stages = (int)((std::min<long long>((long long)p.window + p.sinks, p.capacity) + kDcKeys - 1) / kDcKeys);
  int splits = 1;
  while (splits < kDcMaxSplit && splits < stages &&
         (ctas * splits < 2LL * num_sms() || (ctas * splits < 8LL * num_sms() && stages >= 32 * splits)))
    splits *= 2;
  auto kernel = window_decode_kernel<D, BF16>;
  LSRM_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, DcSmem<D>::BYTES));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(splits, p.hkv * blocks, p.batch);
  cfg.blockDim = dim3(kDcThreads);
  cfg.dynamicSmemBytes = DcSmem<D>::BYTES;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  LSRM_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, p));
  LSRM_LAUNCH_CHECK();
  return LSRM_OK;
}

}  // namespace
}  // namespace lsrm

using namespace lsrm;

extern "C" int lsrm_window_decode(const lsrm_window_decode_shape* shape, const void* q, const void* k_new,
                                  const void* v_new, void* k_cache, void* v_cache, const int32_t* lengths, void* out,
                                  void* stream) {
  LSRM_CHECK_ARG(shape, "shape must not be NULL");
  const lsrm_window_decode_shape& d = *shape;
  LSRM_CHECK_ARG(d.batch >= 0 && d.batch <= 65535, "batch (%d) must be in [0, 65535]", d.batch);
  LSRM_CHECK_ARG(d.num_kv_heads >= 1 && d.num_q_heads >= 1 && d.num_q_heads % d.num_kv_heads == 0,
                 "num_q_heads (%d) must be a multiple of num_kv_heads (%d)", d.num_q_heads, d.num_kv_heads);
  LSRM_CHECK_ARG(d.num_q_heads / d.num_kv_heads <= 64 && d.num_q_heads <= 65535,
                 "at most 64 query heads per kv head");
  LSRM_CHECK_ARG(d.head_dim == 32 || d.head_dim == 64 || d.head_dim == 128, "head_dim (%d) must be 32, 64 or 128",
                 d.head_dim);
  LSRM_CHECK_ARG(d.dtype == LSRM_DTYPE_BF16 || d.dtype == LSRM_DTYPE_F16, "dtype must be bf16 or fp16");
  LSRM_CHECK_ARG(d.window >= 1 && d.sinks >= 0, "window (%d) must be at least 1 and sinks (%d) not negative", d.window,
                 d.sinks);
  LSRM_CHECK_ARG(d.capacity > d.sinks && d.capacity - d.sinks >= d.window,
                 "capacity (%d) must hold the sinks (%d) and the window (%d)", d.capacity, d.sinks, d.window);
  const int64_t qr = (int64_t)d.num_q_heads * d.head_dim, kr = (int64_t)d.num_kv_heads * d.head_dim;
  LSRM_CHECK_ARG(d.q_stride >= qr && d.k_new_stride >= kr && d.v_new_stride >= kr && d.k_slot_stride >= kr &&
                     d.v_slot_stride >= kr && d.k_batch_stride >= 0 && d.v_batch_stride >= 0,
                 "strides must cover the heads");
  LSRM_CHECK_ARG(((d.q_stride | d.k_new_stride | d.v_new_stride | d.k_slot_stride | d.v_slot_stride |
                   d.k_batch_stride | d.v_batch_stride) & 7) == 0, "strides must be multiples of 8 elements");
  LSRM_CHECK_ARG((((uintptr_t)q | (uintptr_t)k_new | (uintptr_t)v_new | (uintptr_t)k_cache | (uintptr_t)v_cache |
                   (uintptr_t)out) & 15) == 0, "tensors must be 16-byte aligned");
  if (d.batch == 0) return LSRM_OK;
  LSRM_CHECK_ARG(q && k_new && v_new && k_cache && v_cache && lengths && out, "pointers must not be NULL");
  DecodeParams p;
  p.batch = d.batch, p.hq = d.num_q_heads, p.hkv = d.num_kv_heads, p.g = p.hq / p.hkv;
  p.capacity = d.capacity, p.window = d.window, p.sinks = d.sinks;
  p.scale = d.softmax_scale > 0.f ? d.softmax_scale : 1.f / sqrtf((float)d.head_dim);
  p.q_stride = d.q_stride, p.kn_stride = d.k_new_stride, p.vn_stride = d.v_new_stride;
  p.kc_batch = d.k_batch_stride, p.kc_slot = d.k_slot_stride, p.vc_batch = d.v_batch_stride;
  p.vc_slot = d.v_slot_stride;
  p.q = q, p.k_new = k_new, p.v_new = v_new, p.k_cache = k_cache, p.v_cache = v_cache, p.out = out;
  p.lengths = lengths;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  ProfScope ps("window_decode", s);
#define CALL(BF, D) return launch_decode<D, BF>(p, s)
  if (d.dtype == LSRM_DTYPE_BF16) {
    if (d.head_dim == 32) CALL(true, 32);
    if (d.head_dim == 64) CALL(true, 64);
    CALL(true, 128);
  }
  if (d.head_dim == 32) CALL(false, 32);
  if (d.head_dim == 64) CALL(false, 64);
  CALL(false, 128);
#undef CALL
}
