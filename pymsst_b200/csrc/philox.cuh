// Counter-based random bits for dropout: Philox4x32 with seven rounds
// (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3",
// SC 2011; seven is the smallest round count they report as passing their
// full test battery).  A mask is a pure function of (seed, step, site,
// element), so the backward and a recomputed forward draw the same one and
// nothing is stored.
//
//   key words      seed low, seed high ^ site
//   counter words  (c0, c1, c2, step low)
//   one call serves eight elements with 16 bits each: element e takes word
//   e / 2, its low half for even e, its high half for odd e
//   dropped when the 16 bits are below t = round(65536 p); kept values are
//   scaled by 65536 / (65536 - t), the exact inverse of the keep probability
//
// 16 bits per element: the probability is met to 2^-17 and one call (seven
// rounds of two 32 x 32 -> 64-bit products) serves a 16-byte vector of
// 16-bit values.  With 32 bits per element the integer products alone would
// cost an elementwise pass over HBM 2x, the attention kernels 8 instructions
// more per score.
#pragma once

#include "common.cuh"

namespace pmb {

// Everything a kernel needs to draw: `limit` is 65536 t - 1 (t in [1, 65536]);
// a 16-bit number u is kept when (u << 16) > limit, i.e. when u >= t.
struct DropArgs {
  const int64_t* key;  // device: seed, step
  uint32_t site;
  uint32_t limit;
  float scale;
};

inline DropArgs drop_args(const int64_t* key, uint32_t site, int threshold) {
  DropArgs d;
  d.key = key;
  d.site = site;
  d.limit = threshold > 0 ? (uint32_t)(((uint64_t)threshold << 16) - 1) : 0u;
  d.scale = threshold < 65536 ? (float)(65536.0 / (65536.0 - (double)threshold)) : 0.f;
  return d;
}

#ifdef __CUDACC__
struct Philox {
  uint32_t k0, k1, step;

  __device__ __forceinline__ explicit Philox(const DropArgs& d) {
    const uint64_t seed = (uint64_t)__ldg(reinterpret_cast<const long long*>(d.key));
    k0 = (uint32_t)seed;
    k1 = (uint32_t)(seed >> 32) ^ d.site;
    step = (uint32_t)__ldg(reinterpret_cast<const long long*>(d.key) + 1);
  }

  __device__ __forceinline__ uint4 operator()(uint32_t c0, uint32_t c1, uint32_t c2) const {
    uint32_t c3 = step, a = k0, b = k1;
#pragma unroll
    for (int r = 0; r < 7; ++r) {
      const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
      c0 = (uint32_t)(p1 >> 32) ^ c1 ^ a;
      c2 = (uint32_t)(p0 >> 32) ^ c3 ^ b;
      c1 = (uint32_t)p1;
      c3 = (uint32_t)p0;
      a += 0x9E3779B9u;
      b += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
  }
};

// Bit e of the result: element e of the group is kept.
__device__ __forceinline__ uint32_t keep_bits(uint4 r, uint32_t limit) {
  uint32_t m = 0;
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m |= (w[i] << 16) > limit ? 1u << (2 * i) : 0u;
    m |= w[i] > limit ? 2u << (2 * i) : 0u;
  }
  return m;
}
#endif

}  // namespace pmb
