// Packed fp32 pairs, for passes bound by instruction issue (the 16-bit GELU
// passes, the attention kernels' exponentials).  Internal linkage.
#pragma once

#include <stdint.h>

namespace pmb {
namespace {

// Pairs of fp32 values in one 64-bit register for the sm_100a packed
// instructions fma / mul / add .rn.f32x2: each half is the IEEE fp32
// operation of the scalar form, rounded the same way, so a paired evaluation
// gives the scalar one's results bit for bit with half the FMA-pipe
// instructions.
__device__ __forceinline__ uint64_t pk2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpk2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

}  // namespace
}  // namespace pmb
