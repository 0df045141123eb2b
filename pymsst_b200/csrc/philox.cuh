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

// Everything a kernel needs to draw.  A 16-bit number u is kept when u >= t:
// `limit` holds t - 1 in both halves for packed comparisons (t in [1, 65536]),
// `high` is 65536 t - 1 for one number in the upper half of a word, with
// anything in the lower one.
struct DropArgs {
  const int64_t* key;  // device: seed, step
  uint32_t site;
  uint32_t limit;
  uint32_t high;
  float scale;
};

inline DropArgs drop_args(const int64_t* key, uint32_t site, int threshold) {
  DropArgs d;
  d.key = key;
  d.site = site;
  d.limit = threshold > 0 ? (uint32_t)(threshold - 1) * 0x10001u : 0u;
  d.high = threshold > 0 ? (uint32_t)(((uint64_t)threshold << 16) - 1) : 0u;
  d.scale = threshold < 65536 ? (float)(65536.0 / (65536.0 - (double)threshold)) : 0.f;
  return d;
}

#ifdef __CUDACC__
// One call by itself.
__device__ __forceinline__ uint4 philox(const DropArgs& d, uint32_t c0, uint32_t c1, uint32_t c2) {
  const uint64_t seed = (uint64_t)__ldg(reinterpret_cast<const long long*>(d.key));
  uint32_t a = (uint32_t)seed, b = (uint32_t)(seed >> 32) ^ d.site;
  uint32_t c3 = (uint32_t)__ldg(reinterpret_cast<const long long*>(d.key) + 1);
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

// Many calls under one key.
struct Philox {
  uint32_t ka[7], kb[7], step;  // the rounds' keys, held in registers: 14 additions per call less

  __device__ __forceinline__ explicit Philox(const DropArgs& d) {
    if (d.key == nullptr) return;  // no dropout: never called
    const uint64_t seed = (uint64_t)__ldg(reinterpret_cast<const long long*>(d.key));
    step = (uint32_t)__ldg(reinterpret_cast<const long long*>(d.key) + 1);
#pragma unroll
    for (int r = 0; r < 7; ++r) {
      ka[r] = (uint32_t)seed + (uint32_t)r * 0x9E3779B9u;
      kb[r] = ((uint32_t)(seed >> 32) ^ d.site) + (uint32_t)r * 0xBB67AE85u;
      asm volatile("" : "+r"(ka[r]), "+r"(kb[r]));  // values of their own, so that they are not added up again
    }
  }

  __device__ __forceinline__ uint4 operator()(uint32_t c0, uint32_t c1, uint32_t c2) const {
    uint32_t c3 = step;
#pragma unroll
    for (int r = 0; r < 7; ++r) {
      const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
      c0 = (uint32_t)(p1 >> 32) ^ c1 ^ ka[r];
      c2 = (uint32_t)(p0 >> 32) ^ c3 ^ kb[r];
      c1 = (uint32_t)p1;
      c3 = (uint32_t)p0;
    }
    return make_uint4(c0, c1, c2, c3);
  }
};

// Whether element `odd` (0 or 1) of a word is kept.
__device__ __forceinline__ bool kept(uint32_t w, int odd, uint32_t high) { return (odd ? w : w << 16) > high; }

// 1 in each half of the word whose number is kept: max(u, t - 1) - (t - 1),
// which never borrows across the halves, capped at 1.
__device__ __forceinline__ uint32_t keep_ones(uint32_t w, uint32_t limit) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(limit));
  r -= limit;
  asm("min.u16x2 %0, %1, %2;" : "=r"(r) : "r"(r), "r"(0x00010001u));
  return r;
}

// All ones in each half of the word whose number is kept: an AND mask for two packed 16-bit values.
__device__ __forceinline__ uint32_t keep_mask2(uint32_t w, uint32_t limit) { return keep_ones(w, limit) * 0xffffu; }

// Bit e of the result: element e of the group is kept.
__device__ __forceinline__ uint32_t keep_bits(uint4 r, uint32_t limit) {
  const uint32_t m = keep_ones(r.x, limit) + keep_ones(r.y, limit) * 4u + keep_ones(r.z, limit) * 16u +
                     keep_ones(r.w, limit) * 64u;  // even elements in the low half, odd ones in the high half
  return (m | (m >> 15)) & 0xffu;
}
#endif

}  // namespace pmb
