// Root-mean-square norm with the residual's addition, the branch's dropout and
// an optional output in 8 bits:
//   h = residual + drop(x)            (the stream, kept in the residual's type)
//   y = h * r * w,  r = 1 / sqrt(mean_c h^2 + eps)
// Sums, statistics and y are formed from the fp32 h before it is rounded for
// storage.  Backward, with g = dy * w:
//   dh_total = r * (g - h * r^2 * mean_c(g * h)) + dh
//   dresidual = dh_total, dx = drop(dh_total), dw_c = sum_rows dy * h * r
// where drop regenerates the forward's mask from its counter (philox.cuh).
//
// The stored h is what the backward reads: its rounding to the stream's type
// enters the gradients once (a 16-bit stream: error against 64 bits 0.0023 where
// the results' own rounding is 0.0017); an fp32 h of its own, or x and the residual
// once more, would be a tensor more to move.
//
// What bounds the passes.  131072 x 1024 bf16: forward 174 us without dropout
// (6.2 TB/s, HBM: the warps wait for loads), 229 with it; backward 211 and 311
// with dw's sum (5.1 and 4.3 TB/s); 16384 x 4096 to int8 104 us (4.5 TB/s) and
// back 44.  In all but the first, instruction issue is busier than DRAM: issue
// slots 65 % in the forward with dropout, 74 and 66 % in the backward, 76 % to
// 8 bits, with DRAM at 51, 60, 51 and 51 % (65536 x 1024; 16384 x 4096).  Every
// tensor is read or written once, a row stays in registers between its
// statistics and its output.  A team of 32 to
// 512 threads owns a row; a thread holds NV chunks of eight consecutive
// elements.  Chunks are cut from the flat tensor (chunk = flat index / 8), so
// that rows of any width use 16-byte accesses: a row that does not start or
// end on a chunk shares its first and last one with its neighbours, reads
// them whole and writes its own elements one by one.
#include <algorithm>

#include <cuda_fp8.h>

#include "host_util.h"
#include "philox.cuh"
#include "vec8.cuh"

namespace lsrm {
namespace {

constexpr int kNormMaxCols = 16384;  // 512 threads x 4 chunks x 8 elements
constexpr int kRowWarps = 8;         // rows per block when a warp owns a row
// Chunks a thread holds at most.  131072 x 1024 bf16, forward with dropout:
// 264 us at one, 230 at two, 272 at four; backward, before its loads went a row
// ahead, 343, 388, 422 (three more tensors in registers: rows in flight count for
// more than barriers saved).
constexpr int kFwdChunks = 2, kBwdChunks = 1;

struct NormParams {
  long long rows;
  int cols, cols8;       // columns; chunks a row can touch
  long long total8;      // chunks that lie wholly inside the tensors
  float eps, inv_cols;
  const void* x;         // forward: the branch; backward: unused
  const void* residual;  // may be null
  const void* w;         // may be null
  int w_f32;
  void* y;
  void* h;
  float* rstd;           // [rows], may be null
  DropoutParams drop;
  // 8-bit output
  uint8_t* q;
  float* scales;
  int group, groups;     // columns per scale (cols: one scale per row), scales per row
  float q_inv;           // 1 / the format's largest magnitude
  // backward
  const void* dy;
  const void* dh;        // may be null
  void* dx;              // null when it equals dresidual
  void* dres;
  float* dw_part;        // [blocks, cols] or null
};

// The larger of two magnitudes; NaN when either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Sum / max over the TPR threads of a team.  Teams wider than a warp are whole
// blocks; `buf` has two slots that alternate between calls, so one barrier a
// call is enough.
template <bool MAX>
__device__ __forceinline__ float team_reduce(float v, int tpr, float (*buf)[16], int& turn) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float u = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? max_nan(v, u) : v + u;
  }
  if (tpr == 32) return v;
  const int warps = tpr >> 5;
  float* b = buf[turn];
  turn ^= 1;
  if ((threadIdx.x & 31) == 0) b[threadIdx.x >> 5] = v;
  __syncthreads();
  v = b[0];
  for (int i = 1; i < warps; ++i) v = MAX ? max_nan(v, b[i]) : v + b[i];
  return v;
}

// The part [lo, hi) of chunk `c` that belongs to row `row`.
struct Part {
  int lo, hi;
};
__device__ __forceinline__ Part part_of(long long c, long long e0, int cols) {
  const long long a = e0 - 8 * c, b = e0 + cols - 8 * c;
  return Part{a > 0 ? (int)a : 0, b < 8 ? (int)b : 8};
}

template <bool EVEN, typename T>
__device__ __forceinline__ void read_chunk(const T* base, long long c, long long total8, Part p, float* f) {
  if (EVEN || c < total8)
    load8(base, c, f);
  else
    load8_part(base, c, p.lo, p.hi, f);
}

template <bool EVEN, typename T>
__device__ __forceinline__ void write_chunk(T* base, long long c, Part p, const float* f) {
  if (EVEN || (p.lo == 0 && p.hi == 8))
    store8(base, c, f);
  else
    store8_part(base, c, p.lo, p.hi, f);
}

__device__ __forceinline__ float read_w(const NormParams& p, int col, bool is_bf16) {
  if (p.w_f32) return static_cast<const float*>(p.w)[col];
  return is_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.w)[col])
                 : __half2float(static_cast<const __half*>(p.w)[col]);
}

template <typename T>
__device__ __forceinline__ void read_w8(const NormParams& p, int col0, float* f) {
  if (p.w_f32)
    load8(static_cast<const float*>(p.w), col0 >> 3, f);
  else
    load8(static_cast<const T*>(p.w), col0 >> 3, f);
}

enum NormOut { kOutPlain = 0, kOutE4m3 = 1, kOutInt8 = 2 };

// A group's scale: its largest magnitude over the format's, 1 for a group of
// zeros, and never so small that its reciprocal overflows.  A group that holds
// a NaN or an infinity gets a NaN scale: int8 has no value for them, so the
// scale says that the group's values stand for no numbers.
__device__ __forceinline__ float scale_of(float amax, float q_inv) {
  if (amax == 0.f) return 1.f;
  return amax <= 3.4028235e38f ? fmaxf(amax * q_inv, 1.1754944e-38f) : __int_as_float(0x7fffffff);
}

// Eight values of at most q_max / inv to 8 bits, to nearest even: e4m3 by the
// conversion instruction; int8 by adding 1.5 * 2^23, which leaves the rounded
// integer in the low mantissa bits (the conversion instruction runs at an
// eighth of the addition's rate).
template <int OUT>
__device__ __forceinline__ uint64_t quantise8(const float* f, float inv) {
  uint32_t r[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float* v = f + 4 * h;
    if (OUT == kOutE4m3) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[0] * inv, v[1] * inv), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[2] * inv, v[3] * inv), __NV_SATFINITE, __NV_E4M3);
      r[h] = lo | hi << 16;
    } else {
      constexpr float kMagic = 12582912.f;
      const uint32_t lo = __byte_perm(__float_as_uint(__fadd_rn(__fmul_rn(v[0], inv), kMagic)),
                                      __float_as_uint(__fadd_rn(__fmul_rn(v[1], inv), kMagic)), 0x0040);
      const uint32_t hi = __byte_perm(__float_as_uint(__fadd_rn(__fmul_rn(v[2], inv), kMagic)),
                                      __float_as_uint(__fadd_rn(__fmul_rn(v[3], inv), kMagic)), 0x0040);
      r[h] = __byte_perm(lo, hi, 0x5410);
    }
  }
  return (uint64_t)r[1] << 32 | r[0];
}

__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// T: type of x, y (and dy, dx); S: type of the residual stream.
template <typename T, typename S, int NV, bool EVEN, int OUT, bool DROP>
__global__ void __launch_bounds__(512) residual_norm_kernel(const NormParams p) {
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  __shared__ float buf[2][16];
  extern __shared__ int s_amax[];  // 8-bit output of uneven rows: a maximum per group (as int bits)
  const int tpr = blockDim.y == 1 ? blockDim.x : 32;  // warp teams: one warp per y
  const int t = threadIdx.x;
  int turn = 0;
  PhiloxHigh ph;
  const T* x = static_cast<const T*>(p.x);
  const S* res = static_cast<const S*>(p.residual);
  T* y = static_cast<T*>(p.y);
  S* hs = static_cast<S*>(p.h);
  const long long team = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  const long long teams = (long long)gridDim.x * blockDim.y;
  // even rows, 8-bit output: the next row's loads are in flight while this one is worked on (16384 x 4096: 119 -> 106
  // us; without the rounding to 8 bits there is too little to hide: 131072 x 1024 174 -> 196 us)
  constexpr bool kAhead = EVEN && OUT != kOutPlain;
  Raw8<T> xr[NV];
  Raw8<S> rr[NV];
  auto fetch = [&](long long row) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = t + tpr * i;
      if (row < p.rows && k < p.cols8) {
        xr[i] = load8_raw(x, row * p.cols8 + k);
        if (res) rr[i] = load8_raw(res, row * p.cols8 + k);
      }
    }
  };
  if (kAhead) fetch(team);
  for (long long row = team; row < p.rows; row += teams) {
    const long long e0 = row * p.cols, c0 = e0 >> 3;
    const int n8 = EVEN ? p.cols8 : (int)(((e0 + p.cols - 1) >> 3) - c0 + 1);
    float v[NV][8];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = t + tpr * i;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
      if (k < n8) {
        const long long c = c0 + k;
        const Part pt = EVEN ? Part{0, 8} : part_of(c, e0, p.cols);
        if (kAhead) unpack8(xr[i], v[i]);
        else read_chunk<EVEN>(x, c, p.total8, pt, v[i]);
        if (DROP) dropout8(p.drop, ph, c, v[i]);
        if (res) {
          float r[8];
          if (kAhead) unpack8(rr[i], r);
          else read_chunk<EVEN>(res, c, p.total8, pt, r);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i][j] += r[j];
        }
        if (!EVEN) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (j < pt.lo || j >= pt.hi) v[i][j] = 0.f;
        }
        write_chunk<EVEN>(hs, c, pt, v[i]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(v[i][j], v[i][j], ss);
    }
    if (kAhead) fetch(row + teams);
    ss = team_reduce<false>(ss, tpr, buf, turn);
    const float rstd = 1.f / sqrtf(ss * p.inv_cols + p.eps);
    if (p.rstd && t == 0) p.rstd[row] = rstd;
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = t + tpr * i;
      if (!EVEN) {
        const int col0 = (int)(8 * (c0 + k) - e0);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int col = col0 + j;
          v[i][j] *= rstd;
          if (p.w && col >= 0 && col < p.cols) v[i][j] *= read_w(p, col, kBf16);
        }
      } else {
        float w[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
        if (p.w && k < n8) read_w8<T>(p, 8 * k, w);  // from L1: registers are better spent on more rows in flight
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] *= rstd * w[j];
      }
      if (OUT == kOutPlain) {
        if (k < n8) write_chunk<EVEN>(y, c0 + k, EVEN ? Part{0, 8} : part_of(c0 + k, e0, p.cols), v[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = max_nan(amax, fabsf(v[i][j]));
      }
    }
    if (OUT == kOutPlain) continue;
    // A scale per row, or per group of columns.  Even rows: a group is
    // group / 8 consecutive lanes.  Uneven rows: their chunks straddle the
    // groups, so the maxima meet in shared memory (an order-free maximum).
    const bool whole = p.groups == 1;
    if (whole) {
      amax = team_reduce<true>(amax, tpr, buf, turn);
    } else if (!EVEN) {
      for (int g = t; g < p.groups; g += tpr) s_amax[g] = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col0 = (int)(8 * (c0 + t + tpr * i) - e0);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int col = col0 + j;
          if (col >= 0 && col < p.cols) atomicMax(&s_amax[col / p.group], __float_as_int(fabsf(v[i][j])));
        }
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = t + tpr * i;
      if (EVEN) {
        float a = amax;
        if (!whole) {
          a = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) a = max_nan(a, fabsf(v[i][j]));
          for (int o = p.group >> 4; o > 0; o >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
        }
        const float scale = scale_of(a, p.q_inv);
        if (k < n8) {
          reinterpret_cast<uint64_t*>(p.q)[c0 + k] = quantise8<OUT>(v[i], reciprocal(scale));
          if (!whole && (8 * k) % p.group == 0) p.scales[row * p.groups + 8 * k / p.group] = scale;
          if (whole && k == 0) p.scales[row] = scale;
        }
      } else if (k < n8) {
        const long long c = c0 + k;
        const Part pt = part_of(c, e0, p.cols);
        const int col0 = (int)(8 * c - e0);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int col = col0 + j;
          if (j < pt.lo || j >= pt.hi) continue;
          const float a = whole ? amax : __int_as_float(s_amax[col / p.group]);
          const float scale = scale_of(a, p.q_inv);
          const float one[8] = {v[i][j], 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          p.q[8 * c + j] = (uint8_t)quantise8<OUT>(one, reciprocal(scale));
          if (col % p.group == 0) p.scales[row * p.groups + col / p.group] = scale;
        }
      }
    }
    if (!EVEN && !whole) __syncthreads();  // the maxima are cleared for the next row
  }
}

template <typename T, typename S, int NV, bool EVEN, bool DROP>
__global__ void __launch_bounds__(512) residual_norm_bwd_kernel(const NormParams p) {
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  __shared__ float buf[2][16];
  extern __shared__ float s_dw[];  // [cols] per team (uneven rows), or per block
  const int tpr = blockDim.y == 1 ? blockDim.x : 32;
  const int t = threadIdx.x;
  int turn = 0;
  PhiloxHigh ph;
  const S* hs = static_cast<const S*>(p.h);
  const T* dy = static_cast<const T*>(p.dy);
  const S* dh = static_cast<const S*>(p.dh);
  T* dx = static_cast<T*>(p.dx);
  S* dres = static_cast<S*>(p.dres);
  const long long team = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  const long long teams = (long long)gridDim.x * blockDim.y;
  float dw[EVEN ? NV : 1][8];
  float* s_row = s_dw + (EVEN ? 0 : threadIdx.y * p.cols);
#pragma unroll
  for (int i = 0; i < (EVEN ? NV : 1); ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[i][j] = 0.f;
  if (!EVEN && p.dw_part) {
    for (int c = t; c < p.cols; c += tpr) s_row[c] = 0.f;
    if (tpr == 32) __syncwarp();
    else __syncthreads();
  }
  Raw8<T> yr[NV];
  Raw8<S> hr[NV], dr[NV];
  float next_rstd = 0.f;
  auto fetch = [&](long long row) {
    if (row < p.rows) next_rstd = p.rstd[row];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = t + tpr * i;
      if (row < p.rows && k < p.cols8) {
        yr[i] = load8_raw(dy, row * p.cols8 + k);
        hr[i] = load8_raw(hs, row * p.cols8 + k);
        if (dh) dr[i] = load8_raw(dh, row * p.cols8 + k);
      }
    }
  };
  if (EVEN) fetch(team);
  for (long long row = team; row < p.rows; row += teams) {
    const long long e0 = row * p.cols, c0 = e0 >> 3;
    const int n8 = EVEN ? p.cols8 : (int)(((e0 + p.cols - 1) >> 3) - c0 + 1);
    const float rstd = EVEN ? next_rstd : p.rstd[row];
    float g[NV][8], h[NV][8], d0[EVEN ? NV : 1][8];
    float gh = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = t + tpr * i;
#pragma unroll
      for (int j = 0; j < 8; ++j) g[i][j] = h[i][j] = 0.f;
      if (k < n8) {
        const long long c = c0 + k;
        const Part pt = EVEN ? Part{0, 8} : part_of(c, e0, p.cols);
        if (EVEN) {
          unpack8(yr[i], g[i]);
          unpack8(hr[i], h[i]);
          if (dh) unpack8(dr[i], d0[i]);
        } else {
          read_chunk<EVEN>(dy, c, p.total8, pt, g[i]);
          read_chunk<EVEN>(hs, c, p.total8, pt, h[i]);
        }
        const int col0 = (int)(8 * c - e0);
        float w[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
        if (EVEN && p.w) read_w8<T>(p, 8 * k, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (!EVEN && (j < pt.lo || j >= pt.hi)) {
            g[i][j] = h[i][j] = 0.f;
            continue;
          }
          if (EVEN) {
            dw[i][j] = fmaf(g[i][j] * h[i][j], rstd, dw[i][j]);
            g[i][j] *= w[j];
          } else {
            // a column belongs to one thread of the team in a row; the team meets between rows
            if (p.dw_part) s_row[col0 + j] = fmaf(g[i][j] * h[i][j], rstd, s_row[col0 + j]);
            if (p.w) g[i][j] *= read_w(p, col0 + j, kBf16);
          }
          gh = fmaf(g[i][j], h[i][j], gh);
        }
      }
    }
    if (EVEN) fetch(row + teams);
    gh = team_reduce<false>(gh, tpr, buf, turn);
    const float k2 = gh * p.inv_cols * rstd * rstd;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = t + tpr * i;
      if (k < n8) {
        const long long c = c0 + k;
        const Part pt = EVEN ? Part{0, 8} : part_of(c, e0, p.cols);
        float d[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) d[j] = EVEN && dh ? d0[i][j] : 0.f;
        if (!EVEN && dh) read_chunk<EVEN>(dh, c, p.total8, pt, d);
#pragma unroll
        for (int j = 0; j < 8; ++j) d[j] = fmaf(rstd, g[i][j] - h[i][j] * k2, d[j]);
        write_chunk<EVEN>(dres, c, pt, d);
        if (dx) {
          if (DROP) dropout8(p.drop, ph, c, d);
          write_chunk<EVEN>(dx, c, pt, d);
        }
      }
    }
    if (!EVEN && tpr == 32) __syncwarp();
  }
  if (!p.dw_part) return;
  // This block's sum over its rows, teams in ascending order.
  float* part = p.dw_part + (long long)blockIdx.x * p.cols;
  if (EVEN && tpr > 32) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t + tpr * i < p.cols8) store8(part, t + tpr * i, dw[i]);
  } else if (EVEN) {
    for (int r = 0; r < (int)blockDim.y; ++r) {
      if ((int)threadIdx.y == r) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int c = t + tpr * i;
          if (c < p.cols8) {
#pragma unroll
            for (int j = 0; j < 8; ++j) s_dw[8 * c + j] = r ? s_dw[8 * c + j] + dw[i][j] : dw[i][j];
          }
        }
      }
      __syncthreads();
    }
    for (int c = threadIdx.y * 32 + t; c < p.cols; c += 32 * blockDim.y) part[c] = s_dw[c];
  } else {
    __syncthreads();
    for (int c = threadIdx.y * blockDim.x + t; c < p.cols; c += blockDim.x * blockDim.y) {
      float s = s_dw[c];
      for (int r = 1; r < (int)blockDim.y; ++r) s += s_dw[r * p.cols + c];
      part[c] = s;
    }
  }
}

// dw[c] = sum over the blocks' partial rows, in a fixed order: 32 interleaved
// runs of the rows per column, then the runs in order.
constexpr int kDwRuns = 32;
template <typename T>
__global__ void __launch_bounds__(32 * kDwRuns) norm_dw_kernel(const float* __restrict__ part, int blocks, int cols,
                                                               T* dw) {
  __shared__ float s[kDwRuns][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float a = 0.f;
  if (c < cols) {
#pragma unroll 4
    for (int b = threadIdx.y; b < blocks; b += kDwRuns) a += part[(long long)b * cols + c];
  }
  s[threadIdx.y][threadIdx.x] = a;
  __syncthreads();
  if (threadIdx.y == 0 && c < cols) {
    for (int i = 1; i < kDwRuns; ++i) a += s[i][threadIdx.x];
    dw[c] = (T)a;
  }
}

// y = value * scale.  WIDE > 0: rows and groups are whole runs of WIDE (8 or
// 16) elements, one run and one scale a thread; 0: eight elements anywhere.
template <typename T, bool E4M3, int WIDE>
__global__ void __launch_bounds__(256) dequantize8_kernel(const uint8_t* __restrict__ q, const float* __restrict__ sc,
                                                          T* __restrict__ y, long long rows, int cols, int group,
                                                          int groups) {
  const long long stride = (long long)gridDim.x * blockDim.x;
  auto value = [](uint64_t u, int i) {
    const uint32_t b = (uint32_t)(u >> (8 * i)) & 0xffu;
    return E4M3 ? __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)b, __NV_E4M3)))
                : (float)(int8_t)b;
  };
  long long c = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if constexpr (WIDE > 0) {
    const int row_runs = cols / WIDE, group_runs = group / WIDE;
    const long long runs = rows * row_runs;
    // row and run of the row advance without a division
    long long row = c / row_runs;
    int k = (int)(c - row * row_runs);
    const long long step_row = stride / row_runs;
    const int step_k = (int)(stride - step_row * row_runs);
    for (; c < runs; c += stride) {
      uint64_t u[WIDE / 8];
      if constexpr (WIDE == 16) {
        const ulonglong2 v = reinterpret_cast<const ulonglong2*>(q)[c];
        u[0] = v.x, u[1] = v.y;
      } else {
        u[0] = reinterpret_cast<const uint64_t*>(q)[c];
      }
      const float s = sc[row * groups + (groups == 1 ? 0 : k / group_runs)];
#pragma unroll
      for (int h = 0; h < WIDE / 8; ++h) {
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = value(u[h], i) * s;
        store8(y, c * (WIDE / 8) + h, f);
      }
      row += step_row;
      k += step_k;
      if (k >= row_runs) k -= row_runs, ++row;
    }
    return;
  }
  const long long n = rows * cols, full = n >> 3, chunks = (n + 7) >> 3;
  for (; c < chunks; c += stride) {
    const int hi = c < full ? 8 : (int)(n & 7);
    uint64_t u = 0;
    if (hi == 8)
      u = reinterpret_cast<const uint64_t*>(q)[c];
    else
      for (int i = 0; i < hi; ++i) u |= (uint64_t)q[8 * c + i] << (8 * i);
    long long row = 8 * c / cols;
    int col = (int)(8 * c - row * cols);
    float f[8], s = 0.f;
    int left = 0;  // elements until the next scale
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i < hi && left == 0) {
        if (col == cols) col = 0, ++row;
        const int g = col / group;
        s = sc[row * groups + g];
        left = min(cols, (g + 1) * group) - col;
      }
      f[i] = value(u, i) * s;
      --left;
      ++col;
    }
    if (hi == 8)
      store8(y, c, f);
    else
      store8_part(y, c, 0, hi, f);
  }
}

template <typename T, bool E4M3>
int launch_dequantize(const uint8_t* q, const float* scales, void* y, long long rows, int cols, int group, int groups,
                      cudaStream_t s) {
  constexpr auto k16 = dequantize8_kernel<T, E4M3, 16>;
  constexpr auto k8 = dequantize8_kernel<T, E4M3, 8>;
  constexpr auto k0 = dequantize8_kernel<T, E4M3, 0>;
  auto whole = [&](int wide) { return cols % wide == 0 && (groups == 1 || group % wide == 0); };
  auto grid = [&](int wide, int resident) {
    return (int)std::min<long long>((rows * cols / wide + 256) / 256, (long long)num_sms() * resident);
  };
  if (whole(16))
    k16<<<grid(16, resident_blocks<k16>(256)), 256, 0, s>>>(q, scales, static_cast<T*>(y), rows, cols, group, groups);
  else if (whole(8))
    k8<<<grid(8, resident_blocks<k8>(256)), 256, 0, s>>>(q, scales, static_cast<T*>(y), rows, cols, group, groups);
  else
    k0<<<grid(8, resident_blocks<k0>(256)), 256, 0, s>>>(q, scales, static_cast<T*>(y), rows, cols, group, groups);
  LSRM_LAUNCH_CHECK();
  return LSRM_OK;
}

struct NormLaunch {
  dim3 block;
  long long teams;  // blocks that the rows can fill
  int nv;
  bool even;
};

// Threads per row: the narrowest team that holds the row in at most `chunks`
// chunks a thread (a warp where that suffices: the row's sums need no barrier).
// Where there are not enough rows to fill the GPU (fewer than four a
// multiprocessor), a thread takes one chunk so that a row's loads are in
// flight at once.
NormLaunch norm_launch(long long rows, int cols, bool block_teams, int chunks) {
  const bool even = cols % 8 == 0;
  const int n8 = even ? cols / 8 : cols / 8 + 2;
  const int most = rows <= 4LL * num_sms() ? 1 : chunks;
  int tpr = block_teams ? 64 : 32;
  while (tpr < 512 && tpr * most < n8) tpr *= 2;
  const int per = (n8 + tpr - 1) / tpr;
  NormLaunch l;
  l.nv = per <= 1 ? 1 : per <= 2 ? 2 : per <= 4 ? 4 : 5;
  l.even = even;
  l.block = tpr == 32 ? dim3(32, kRowWarps) : dim3(tpr, 1);
  l.teams = tpr == 32 ? (rows + kRowWarps - 1) / kRowWarps : rows;
  return l;
}

// Blocks of a launch, at most: what the multiprocessors hold at once.
int norm_blocks(const NormLaunch& l, int resident) {
  return (int)std::min<long long>(l.teams, (long long)num_sms() * resident);
}
int norm_blocks_most(const NormLaunch& l) { return norm_blocks(l, 2048 / (int)(l.block.x * l.block.y)); }

#define NORM_NV(CALL)          \
  switch (l.nv) {              \
    case 1: CALL(1); break;    \
    case 2: CALL(2); break;    \
    case 4: CALL(4); break;    \
    default: CALL(5); break;   \
  }

template <typename T, typename S, int OUT, bool DROP>
int launch_norm(const NormParams& p, const NormLaunch& l, size_t smem, cudaStream_t s) {
#define NORM_CALL(NV)                                                                     \
  {                                                                                       \
    constexpr auto k0 = residual_norm_kernel<T, S, NV, true, OUT, DROP>;                  \
    constexpr auto k1 = residual_norm_kernel<T, S, NV, false, OUT, DROP>;                 \
    const int threads = l.block.x * l.block.y;                                            \
    if (l.even)                                                                           \
      k0<<<norm_blocks(l, resident_blocks<k0>(threads)), l.block, smem, s>>>(p);          \
    else                                                                                  \
      k1<<<norm_blocks(l, resident_blocks<k1>(threads)), l.block, smem, s>>>(p);          \
  }
  NORM_NV(NORM_CALL)
#undef NORM_CALL
  LSRM_LAUNCH_CHECK();
  return LSRM_OK;
}

template <typename T, typename S, bool DROP>
int launch_norm_bwd(const NormParams& p, const NormLaunch& l, size_t smem, cudaStream_t s, int* blocks) {
#define NORM_CALL(NV)                                                                                              \
  {                                                                                                                \
    constexpr auto k0 = residual_norm_bwd_kernel<T, S, NV, true, DROP>;                                            \
    constexpr auto k1 = residual_norm_bwd_kernel<T, S, NV, false, DROP>;                                           \
    const int threads = l.block.x * l.block.y;                                                                     \
    *blocks = norm_blocks(l, l.even ? resident_blocks<k0>(threads) : resident_blocks<k1>(threads));                \
    auto k = l.even ? k0 : k1;                                                                                     \
    if (smem > 48 * 1024) LSRM_CUDA_TRY(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)); \
    k<<<*blocks, l.block, smem, s>>>(p);                                                                           \
  }
  NORM_NV(NORM_CALL)
#undef NORM_CALL
  LSRM_LAUNCH_CHECK();
  return LSRM_OK;
}

int check_norm(int64_t rows, int32_t cols, int32_t dtype, int32_t stream_dtype, int32_t weight_dtype, const void* w) {
  LSRM_CHECK_ARG(rows >= 0 && rows < (1LL << 40), "rows (%lld) out of range", (long long)rows);
  LSRM_CHECK_ARG(cols >= 1 && cols <= kNormMaxCols, "cols (%d) must be in [1, %d]", cols, kNormMaxCols);
  LSRM_CHECK_ARG(dtype == LSRM_DTYPE_BF16 || dtype == LSRM_DTYPE_F16, "dtype must be bf16 or fp16");
  LSRM_CHECK_ARG(stream_dtype == dtype || stream_dtype == LSRM_DTYPE_F32,
                 "the residual must have x's type or fp32");
  LSRM_CHECK_ARG(!w || weight_dtype == dtype || weight_dtype == LSRM_DTYPE_F32, "the weight must have x's type or fp32");
  return LSRM_OK;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

NormParams norm_params(int64_t rows, int32_t cols, float eps, const void* w, int32_t weight_dtype) {
  NormParams p{};
  p.rows = rows;
  p.cols = cols;
  p.cols8 = cols / 8;
  p.total8 = rows * cols / 8;
  p.eps = eps;
  p.inv_cols = 1.f / (float)cols;
  p.w = w;
  p.w_f32 = weight_dtype == LSRM_DTYPE_F32;
  return p;
}

template <typename T, int OUT, bool DROP>
int launch_norm_s(bool s_f32, const NormParams& p, const NormLaunch& l, size_t smem, cudaStream_t s) {
  return s_f32 ? launch_norm<T, float, OUT, DROP>(p, l, smem, s) : launch_norm<T, T, OUT, DROP>(p, l, smem, s);
}

template <typename T>
int launch_norm_t(bool s_f32, int out, bool drop, const NormParams& p, const NormLaunch& l, size_t smem,
                  cudaStream_t s) {
  if (out == kOutE4m3) return launch_norm_s<T, kOutE4m3, false>(s_f32, p, l, smem, s);
  if (out == kOutInt8) return launch_norm_s<T, kOutInt8, false>(s_f32, p, l, smem, s);
  return drop ? launch_norm_s<T, kOutPlain, true>(s_f32, p, l, smem, s)
              : launch_norm_s<T, kOutPlain, false>(s_f32, p, l, smem, s);
}

template <typename T>
int launch_norm_bwd_t(bool s_f32, bool drop, const NormParams& p, const NormLaunch& l, size_t smem, cudaStream_t s,
                      int* blocks) {
  if (s_f32)
    return drop ? launch_norm_bwd<T, float, true>(p, l, smem, s, blocks)
                : launch_norm_bwd<T, float, false>(p, l, smem, s, blocks);
  return drop ? launch_norm_bwd<T, T, true>(p, l, smem, s, blocks) : launch_norm_bwd<T, T, false>(p, l, smem, s, blocks);
}

}  // namespace
}  // namespace lsrm

using namespace lsrm;

extern "C" int lsrm_residual_rms_norm_fwd(int64_t rows, int32_t cols, int32_t dtype, int32_t stream_dtype,
                                          int32_t weight_dtype, float eps, double p_drop, uint64_t seed,
                                          uint64_t offset, const void* x, const void* residual, const void* weight,
                                          void* y, void* h, float* rstd, void* stream) {
  int rc = check_norm(rows, cols, dtype, stream_dtype, weight_dtype, weight);
  if (rc) return rc;
  LSRM_CHECK_ARG(p_drop >= 0.0 && p_drop < 1.0, "p (%g) must be in [0, 1)", p_drop);
  LSRM_CHECK_ARG(aligned16(x) && aligned16(residual) && aligned16(weight) && aligned16(y) && aligned16(h),
                 "tensors must be 16-byte aligned");
  if (rows == 0) return LSRM_OK;
  LSRM_CHECK_ARG(x && y && h, "x, y and h must not be NULL");
  NormParams p = norm_params(rows, cols, eps, weight, weight_dtype);
  p.x = x, p.residual = residual, p.y = y, p.h = h, p.rstd = rstd;
  p.drop = make_dropout(p_drop, seed, offset);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  ProfScope ps("residual_rms_norm", s);
  const NormLaunch l = norm_launch(rows, cols, false, kFwdChunks);
  return dtype == LSRM_DTYPE_BF16
             ? launch_norm_t<__nv_bfloat16>(stream_dtype == LSRM_DTYPE_F32, kOutPlain, p_drop > 0, p, l, 0, s)
             : launch_norm_t<__half>(stream_dtype == LSRM_DTYPE_F32, kOutPlain, p_drop > 0, p, l, 0, s);
}

extern "C" int lsrm_residual_rms_norm_8bit(int64_t rows, int32_t cols, int32_t dtype, int32_t stream_dtype,
                                           int32_t weight_dtype, float eps, int32_t out_dtype, int32_t group,
                                           const void* x, const void* residual, const void* weight, void* values,
                                           float* scales, void* h, void* stream) {
  int rc = check_norm(rows, cols, dtype, stream_dtype, weight_dtype, weight);
  if (rc) return rc;
  LSRM_CHECK_ARG(out_dtype == LSRM_DTYPE_E4M3 || out_dtype == LSRM_DTYPE_INT8, "out_dtype must be e4m3 or int8");
  LSRM_CHECK_ARG(group == 0 || group == 32 || group == 64 || group == 128, "group (%d) must be 0, 32, 64 or 128",
                 group);
  LSRM_CHECK_ARG(aligned16(x) && aligned16(residual) && aligned16(weight) && aligned16(values) && aligned16(h),
                 "tensors must be 16-byte aligned");
  if (rows == 0) return LSRM_OK;
  LSRM_CHECK_ARG(x && values && scales && h, "x, values, scales and h must not be NULL");
  NormParams p = norm_params(rows, cols, eps, weight, weight_dtype);
  p.x = x, p.residual = residual, p.h = h;
  p.q = static_cast<uint8_t*>(values);
  p.scales = scales;
  p.group = group ? group : cols;
  p.groups = (cols + p.group - 1) / p.group;
  p.q_inv = out_dtype == LSRM_DTYPE_E4M3 ? 1.f / 448.f : 1.f / 127.f;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  ProfScope ps("residual_rms_norm_8bit", s);
  const bool uneven_groups = cols % 8 != 0 && p.groups > 1;
  const NormLaunch l = norm_launch(rows, cols, uneven_groups, kFwdChunks);
  const size_t smem = uneven_groups ? p.groups * sizeof(int) : 0;
  const int out = out_dtype == LSRM_DTYPE_E4M3 ? kOutE4m3 : kOutInt8;
  return dtype == LSRM_DTYPE_BF16
             ? launch_norm_t<__nv_bfloat16>(stream_dtype == LSRM_DTYPE_F32, out, false, p, l, smem, s)
             : launch_norm_t<__half>(stream_dtype == LSRM_DTYPE_F32, out, false, p, l, smem, s);
}

// The partial sums of dw: one row of fp32 per block of the backward kernel.
extern "C" size_t lsrm_residual_rms_norm_workspace_bytes(int64_t rows, int32_t cols) {
  if (rows <= 0 || cols < 1 || cols > kNormMaxCols) return 0;
  return (size_t)norm_blocks_most(norm_launch(rows, cols, false, kBwdChunks)) * cols * sizeof(float);
}

extern "C" int lsrm_residual_rms_norm_bwd(int64_t rows, int32_t cols, int32_t dtype, int32_t stream_dtype,
                                          int32_t weight_dtype, double p_drop, uint64_t seed, uint64_t offset,
                                          const void* h, const float* rstd, const void* weight, const void* dy,
                                          const void* dh, void* dx, void* dresidual, void* dweight, void* workspace,
                                          size_t workspace_bytes, void* stream) {
  int rc = check_norm(rows, cols, dtype, stream_dtype, weight_dtype, weight);
  if (rc) return rc;
  LSRM_CHECK_ARG(p_drop >= 0.0 && p_drop < 1.0, "p (%g) must be in [0, 1)", p_drop);
  LSRM_CHECK_ARG(aligned16(h) && aligned16(weight) && aligned16(dy) && aligned16(dh) && aligned16(dx) &&
                     aligned16(dresidual) && aligned16(workspace),
                 "tensors must be 16-byte aligned");
  LSRM_CHECK_ARG(!dweight || weight, "dweight needs the weight");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows == 0) {
    if (dweight) LSRM_CUDA_TRY(cudaMemsetAsync(dweight, 0, (size_t)cols * (weight_dtype == LSRM_DTYPE_F32 ? 4 : 2), s));
    return LSRM_OK;
  }
  LSRM_CHECK_ARG(h && rstd && dy && dresidual, "h, rstd, dy and dresidual must not be NULL");
  LSRM_CHECK_ARG(dx || (p_drop == 0.0 && stream_dtype == dtype), "dx may be NULL only where it equals dresidual");
  if (dweight && workspace_bytes < lsrm_residual_rms_norm_workspace_bytes(rows, cols)) {
    set_error("workspace too small: %zu bytes", workspace_bytes);
    return LSRM_ERR_WORKSPACE;
  }
  NormParams p = norm_params(rows, cols, 0.f, weight, weight_dtype);
  p.h = const_cast<void*>(h), p.rstd = const_cast<float*>(rstd), p.dy = dy, p.dh = dh, p.dx = dx, p.dres = dresidual;
  p.dw_part = dweight ? static_cast<float*>(workspace) : nullptr;
  p.drop = make_dropout(p_drop, seed, offset);
  const NormLaunch l = norm_launch(rows, cols, false, kBwdChunks);
  size_t smem = 0;
  if (dweight && (!l.even || l.block.y > 1)) smem = (size_t)cols * (l.even ? 1 : l.block.y) * sizeof(float);
  int blocks = 0;
  {
    ProfScope ps("residual_rms_norm_bwd", s);
    rc = dtype == LSRM_DTYPE_BF16
             ? launch_norm_bwd_t<__nv_bfloat16>(stream_dtype == LSRM_DTYPE_F32, p_drop > 0, p, l, smem, s, &blocks)
             : launch_norm_bwd_t<__half>(stream_dtype == LSRM_DTYPE_F32, p_drop > 0, p, l, smem, s, &blocks);
    if (rc) return rc;
  }
  if (!dweight) return LSRM_OK;
  ProfScope ps("residual_rms_norm_dw", s);
  const dim3 grid((cols + 31) / 32), block(32, kDwRuns);
  if (weight_dtype == LSRM_DTYPE_F32)
    norm_dw_kernel<<<grid, block, 0, s>>>(p.dw_part, blocks, cols, static_cast<float*>(dweight));
  else if (dtype == LSRM_DTYPE_BF16)
    norm_dw_kernel<<<grid, block, 0, s>>>(p.dw_part, blocks, cols, static_cast<__nv_bfloat16*>(dweight));
  else
    norm_dw_kernel<<<grid, block, 0, s>>>(p.dw_part, blocks, cols, static_cast<__half*>(dweight));
  LSRM_LAUNCH_CHECK();
  return LSRM_OK;
}

extern "C" int lsrm_dequantize_8bit(int64_t rows, int32_t cols, int32_t in_dtype, int32_t out_dtype, int32_t group,
                                    const void* values, const float* scales, void* y, void* stream) {
  LSRM_CHECK_ARG(rows >= 0 && cols >= 1, "bad sizes");
  LSRM_CHECK_ARG(in_dtype == LSRM_DTYPE_E4M3 || in_dtype == LSRM_DTYPE_INT8, "values must be e4m3 or int8");
  LSRM_CHECK_ARG(out_dtype == LSRM_DTYPE_BF16 || out_dtype == LSRM_DTYPE_F16 || out_dtype == LSRM_DTYPE_F32,
                 "y must be bf16, fp16 or fp32");
  LSRM_CHECK_ARG(group >= 0, "group (%d) must not be negative", group);
  LSRM_CHECK_ARG(aligned16(values) && aligned16(y), "values and y must be 16-byte aligned");
  if (rows == 0) return LSRM_OK;
  LSRM_CHECK_ARG(values && scales && y, "values, scales and y must not be NULL");
  const int g = group ? group : cols, groups = (cols + g - 1) / g;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  ProfScope ps("dequantize_8bit", s);
  const uint8_t* q = static_cast<const uint8_t*>(values);
#define DEQ(T)                                                                                               \
  return in_dtype == LSRM_DTYPE_E4M3 ? launch_dequantize<T, true>(q, scales, y, rows, cols, g, groups, s)     \
                                     : launch_dequantize<T, false>(q, scales, y, rows, cols, g, groups, s);
  if (out_dtype == LSRM_DTYPE_BF16) {
    DEQ(__nv_bfloat16)
  } else if (out_dtype == LSRM_DTYPE_F16) {
    DEQ(__half)
  } else {
    DEQ(float)
  }
#undef DEQ
}
