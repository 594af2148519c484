// Philox4x32-10, the counter-based generator of Salmon, Moraes, Dror and Shaw
// ("Parallel random numbers: as easy as 1, 2, 3", SC 2011): ten rounds of two
// 32 x 32 -> 64 bit products over a 128-bit counter, keyed by 64 bits.  A
// block of four 32-bit words depends on its counter and the key alone, so the
// backward pass of a dropout recomputes the mask that the forward applied.
//
// Element e of a tensor takes word e % 4 of block offset + e / 4 under the key
// `seed`, and is kept when the word is >= threshold = floor(p * 2^32).
//
// The rounds bound a dropout that streams through HBM (18 products, 36 logical
// operations per four elements, which keep two pipes busier than DRAM), so what does not change from block to block is
// taken out of them: the round keys come from the host as constants, and of a
// counter (low, high, 0, 0) the first round needs one product and the second
// one has one operand that depends on the upper word alone.
#pragma once

#include <cstdint>

namespace lsrm {

constexpr uint32_t kPhiloxM0 = 0xD2511F53u, kPhiloxM1 = 0xCD9E8D57u;

struct DropoutParams {
  uint32_t k0[10], k1[10];  // round keys
  uint64_t offset;          // first counter block
  uint32_t threshold;       // floor(p * 2^32); 0 keeps everything
  float scale;              // 1 / (1 - p)
};

inline DropoutParams make_dropout(double p, uint64_t seed, uint64_t offset) {
  DropoutParams d{};
  for (uint32_t r = 0; r < 10; ++r) {
    d.k0[r] = (uint32_t)seed + r * 0x9E3779B9u;
    d.k1[r] = (uint32_t)(seed >> 32) + r * 0xBB67AE85u;
  }
  d.offset = offset;
  d.threshold = (uint32_t)(p * 4294967296.0);
  d.scale = (float)(1.0 / (1.0 - p));
  return d;
}

// What the blocks of one upper counter word share: the second round's product
// of the first one's word 0 (its upper half with the round key).
struct PhiloxHigh {
  uint32_t high = 0, lo, hi_key;
  bool set = false;
  __device__ __forceinline__ void take(uint32_t h, const DropoutParams& d) {
    if (set && h == high) return;
    set = true;
    high = h;
    const uint32_t x0 = h ^ d.k0[0];
    lo = x0 * kPhiloxM0;
    hi_key = __umulhi(x0, kPhiloxM0) ^ d.k1[1];
  }
};

__device__ __forceinline__ uint4 philox4x32(uint32_t low, const PhiloxHigh& s, const DropoutParams& d) {
  // round one: words (high ^ k0, 0, upper half of low * M0 ^ k1, lower half); round two
  const uint32_t y = __umulhi(low, kPhiloxM0) ^ d.k1[0];
  uint32_t x0 = __umulhi(y, kPhiloxM1) ^ d.k0[1], x1 = y * kPhiloxM1;
  uint32_t x2 = s.hi_key ^ (low * kPhiloxM0), x3 = s.lo;
#pragma unroll
  for (int r = 2; r < 10; ++r) {
    const uint32_t ah = __umulhi(x0, kPhiloxM0), al = x0 * kPhiloxM0;
    const uint32_t bh = __umulhi(x2, kPhiloxM1), bl = x2 * kPhiloxM1;
    x0 = bh ^ x1 ^ d.k0[r];
    x1 = bl;
    x2 = ah ^ x3 ^ d.k1[r];
    x3 = al;
  }
  return make_uint4(x0, x1, x2, x3);
}

// The words of elements 8 * chunk .. 8 * chunk + 7.
__device__ __forceinline__ void dropout_words(const DropoutParams& d, PhiloxHigh& s, long long chunk, uint32_t* w) {
  const uint64_t b0 = d.offset + 2 * (uint64_t)chunk, b1 = b0 + 1;
  s.take((uint32_t)(b0 >> 32), d);
  const uint4 a = philox4x32((uint32_t)b0, s, d);
  if ((uint32_t)b1 == 0u) s.take((uint32_t)(b1 >> 32), d);
  const uint4 b = philox4x32((uint32_t)b1, s, d);
  w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
}

// Drops and scales the eight elements 8 * chunk .. 8 * chunk + 7 in place.
__device__ __forceinline__ void dropout8(const DropoutParams& d, PhiloxHigh& s, long long chunk, float* f) {
  uint32_t w[8];
  dropout_words(d, s, chunk, w);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = w[i] >= d.threshold ? f[i] * d.scale : 0.f;
}

}  // namespace lsrm
