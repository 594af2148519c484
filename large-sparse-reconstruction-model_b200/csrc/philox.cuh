// Philox4x32-10, the counter-based generator of Salmon, Moraes, Dror and Shaw
// ("Parallel random numbers: as easy as 1, 2, 3", SC 2011): ten rounds of two
// 32 x 32 -> 64 bit products over a 128-bit counter, keyed by 64 bits.  A
// block of four 32-bit words depends on its counter and the key alone, so the
// backward pass of a dropout recomputes the mask that the forward applied.
//
// Element e of a tensor takes word e % 4 of block offset + e / 4 under the key
// `seed`, and is kept when the word is >= threshold = floor(p * 2^32).
#pragma once

#include <cstdint>

namespace lsrm {

struct DropoutParams {
  uint32_t key0, key1;    // seed, low and high words
  uint64_t offset;        // first counter block
  uint32_t threshold;     // floor(p * 2^32); 0 keeps everything
  float scale;            // 1 / (1 - p)
};

inline DropoutParams make_dropout(double p, uint64_t seed, uint64_t offset) {
  return DropoutParams{(uint32_t)seed, (uint32_t)(seed >> 32), offset, (uint32_t)(p * 4294967296.0),
                       (float)(1.0 / (1.0 - p))};
}

__device__ __forceinline__ uint4 philox4x32(uint64_t block, uint32_t k0, uint32_t k1) {
  uint32_t x0 = (uint32_t)block, x1 = (uint32_t)(block >> 32), x2 = 0u, x3 = 0u;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)x0 * 0xD2511F53u, b = (uint64_t)x2 * 0xCD9E8D57u;
    x0 = (uint32_t)(b >> 32) ^ x1 ^ k0;
    x1 = (uint32_t)b;
    x2 = (uint32_t)(a >> 32) ^ x3 ^ k1;
    x3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(x0, x1, x2, x3);
}

// Drops and scales the eight elements 8 * chunk .. 8 * chunk + 7 in place.
__device__ __forceinline__ void dropout8(const DropoutParams& d, long long chunk, float* f) {
  const uint4 a = philox4x32(d.offset + 2 * (uint64_t)chunk, d.key0, d.key1);
  const uint4 b = philox4x32(d.offset + 2 * (uint64_t)chunk + 1, d.key0, d.key1);
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = w[i] >= d.threshold ? f[i] * d.scale : 0.f;
}

}  // namespace lsrm
