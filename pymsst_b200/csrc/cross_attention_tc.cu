// Cross attention on the tcgen05 tensor cores (16-bit types, head dims up to
// 128 in multiples of 8); the formulas are at the top of cross_attention.cu.
//
// Rows.  Query heads that share a key / value head are packed: with gp the
// largest power of two (up to 64) that divides the group (and keeps a unit
// below 2^30 rows), gp heads form a
// unit and row R = position * gp + head of the unit, so a few queries of many
// heads fill a tile and each key / value head is read once for all of them.
// A 5-D TMA map (dim, gp, positions, units, batch) loads packed tiles as they
// lie; rows behind the last are zeros.  Head dims below 64 (or between 64 and
// 128) use the 64-wide tiles, the TMA filling the rest with zeros.
//
// All three kernels are persistent and warp-specialised: warp 0 feeds tiles
// by TMA, one lane of warp 1 issues tcgen05.mma, the row warps own one tensor
// memory lane per thread.  Waits are bounded (umma.cuh).  Nothing is summed
// with atomics, so results do not depend on the order of execution.
// What bounds them is the row warps' chain (tensor-memory reads, exponentials,
// random bits, barriers) with eight such warps an SM, no pipe: ncu has 0.38 to
// 0.52 of the issue slots, tensor pipe 17 to 33 %, special-function pipe 15 to
// 50 %.
//
// Keys at or behind a batch item's length are masked in the scores by a
// select, and their value (forward) or key (dQ) rows are zeroed in shared
// memory before the product that multiplies them by a zero weight, so NaN
// there stays there.
//
// Row statistics are base-2 logarithms (lse2 = max + log2(sum), of scores
// times scale * log2 e), kept negated, as the backward adds them; -inf for a
// row without keys, or with scores of -infinity alone, whose probabilities then
// come out as 0.  D is kept negated too.
#include "attention_tiles.cuh"
#include "cross_attention.cuh"
#include "f32x2.cuh"
#include "tma.cuh"
#include "umma.cuh"

namespace pmb {
unsigned int timeout_flag_cross(int reset) { return umma::flag_reader(reset); }

namespace xattn {
namespace {

constexpr int BM = 128;                // rows of a tile
constexpr int TILE = BM * 128;         // bytes of 128 rows x 64 16-bit elements
constexpr int kMaxSplits = 64;

// Division of numbers below 2^31 by a divisor known at launch: floor(n m / 2^(31 + s)) with s = ceil(log2 d) and m =
// ceil(2^(31 + s) / d) (Granlund and Montgomery, PLDI 1994).  Item decoding divides a few times per item and warp.
struct Divisor {
  uint32_t mul, shift, d;

  __device__ __forceinline__ int div(int n) const { return (int)(((uint64_t)(uint32_t)n * mul) >> shift); }
  __device__ __forceinline__ int split(int n, int& rest) const {  // quotient, and the remainder in rest
    const int q = div(n);
    rest = n - q * (int)d;
    return q;
  }
};

// What a kernel needs to find its tiles.
struct Geometry {
  int units, gp_shift, kv_units;       // units per batch item, log2 gp, units per key / value head
  int rows, ldr, nblk;                 // packed rows per unit, their pitch in lse, row tiles per unit
  int width, splits;                   // forward: keys per chunk, key ranges per row tile
  int total;                           // work items
  Divisor by_nblk, by_splits, by_units, by_width, by_kv_units, by_kblk, by_kv_heads;
};

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// 16-bit instruction descriptors, fp32 accumulate, M = 128.
template <typename T>
struct Desc {
  static constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  // A, B K-major, N columns
  __device__ __forceinline__ static uint32_t kk(int n) {
    return umma::idesc_f16(kBf16, false, false, BM, 16) + ((uint32_t)((n - 16) >> 3) << 17);
  }
  static constexpr uint32_t MN = umma::idesc_f16(kBf16, false, true, BM, 64);  // B MN-major, 64 head elements
};

// Descriptor of a 128-byte-swizzled tile in shared memory; tiles and K steps
// further on are 16-byte units added to it.
__device__ __forceinline__ uint64_t tile_desc(const void* smem) {
  return umma::smem_desc_sw128(umma::smem_u32(smem), 16, 1024);
}

// D (+)= A B^T, A and B K-major: DC sub-tiles of 64 elements, strides a_sub / b_sub bytes apart.
template <int DC>
__device__ __forceinline__ void mma_scores(uint32_t d, uint64_t a, uint32_t a_sub, uint64_t b, uint32_t b_sub,
                                           uint32_t idesc) {
#pragma unroll
  for (int dc = 0; dc < DC; ++dc)
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
      umma::mma_f16(d, a + (dc * a_sub + kk * 32) / 16, b + (dc * b_sub + kk * 32) / 16, idesc, (dc || kk) ? 1u : 0u);
}

// D (+)= A B with A in tensor memory, 16-bit pairs in 32-bit columns, and B MN-major: its rows are the K index, its
// 64 head elements the N index, DC sub-tiles b_sub bytes apart into accumulators 64 columns apart.
template <int DC>
__device__ __forceinline__ void mma_rows_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t b_sub, uint32_t idesc,
                                            int ksteps, bool accumulate) {
#pragma unroll
  for (int ks = 0; ks < 6; ++ks) {  // chunks hold 96 rows at most
    if (ks >= ksteps) break;
#pragma unroll
    for (int dc = 0; dc < DC; ++dc)
      umma::mma_f16_ts(d + dc * 64, a + ks * 8, b + (dc * b_sub + ks * 2048) / 16, idesc, (accumulate || ks) ? 1u : 0u);
  }
}

// Elements [n, 32) of 16 packed pairs to zero.
__device__ __forceinline__ void zero_tail(uint32_t (&p)[16], int n) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    if (2 * i + 1 >= n) p[i] &= 0x0000ffffu;
    if (2 * i >= n) p[i] = 0;
  }
}

// 32 accumulator columns (times mul) to head elements [d0, d0 + 32) of a global row, as far as the head goes.
template <typename T>
__device__ __forceinline__ void store_row(T* row, int d0, int dim, const uint32_t (&a)[32], float mul) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float* f = reinterpret_cast<const float*>(a) + 8 * i;
    if (d0 + 8 * i < dim)
      *reinterpret_cast<uint4*>(row + d0 + 8 * i) =
          make_uint4(pack2<T>(f[0] * mul, f[1] * mul), pack2<T>(f[2] * mul, f[3] * mul),
                     pack2<T>(f[4] * mul, f[5] * mul), pack2<T>(f[6] * mul, f[7] * mul));
  }
}

// Zero the 128-byte rows [first, rows) of DC sub-tiles, one row per thread.
template <int DC>
__device__ __forceinline__ void zero_rows(uint8_t* tile, uint32_t sub, int first, int rows, int thread) {
  const int r = thread;
  if (r < first || r >= rows) return;
#pragma unroll
  for (int dc = 0; dc < DC; ++dc)
#pragma unroll
    for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(tile + dc * sub + r * 128 + c * 16) = make_uint4(0, 0, 0, 0);
}

// max of three
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// ---------------------------------------------------------------- forward
// Item = 128 packed rows of a unit, over one of `splits` key ranges.  Keys
// come in chunks of `width` <= 96 (a multiple of 16 that divides the keys
// evenly): S (two buffers of 96 columns) and O (64 columns per 64 head
// elements) then fill 256 tensor memory columns and two CTAs fit an SM.
//
// A row thread owns a row: no exchange between threads.  It takes the row's
// maximum, then turns 32 scores at a time into probabilities and writes them,
// as 16-bit pairs, over the scores just read: P is the product's A operand
// straight from tensor memory (no shared memory and no proxy fence between
// the two products), and S of the next chunk sits in the other buffer, so the
// row warps wait for neither product.  Measured per chunk and CTA before this
// form, with P in shared memory and two threads per row: 4000 cycles, of
// which 1500 arithmetic, 550 the threads' exchange, 550 waiting for the
// previous product to release P, 360 fences.
//
// O stays in tensor memory; the running maximum moves only when a row's grows
// by more than 8 (a factor 256 in P, harmless in fp32 sums and 16-bit P; a
// known step of published attention kernels, as is sharing the exponentials
// between the two pipes),
// which after the first chunks is rare, and then the row threads rescale O
// themselves.  P is rounded to the input type (as in attention.cu); the row
// sums add the unrounded values before dropout, whose scale is applied once
// at the end.
namespace fw {
constexpr int kThreads = 192;
constexpr int kMaxW = 96;
constexpr int kStages = 3;        // K and V rings
constexpr int SUB = kMaxW * 128;  // one 64-element sub-tile of a K or V stage
template <int DC>
struct L {
  static constexpr int OFF_K = 2 * DC * TILE;               // two Q tiles
  static constexpr int OFF_V = OFF_K + kStages * DC * SUB;
  static constexpr int OFF_BAR = OFF_V + kStages * DC * SUB;
  static constexpr int SMEM = OFF_BAR + 256 + 1024;
  static constexpr uint32_t kTmemO = 2 * kMaxW;
  static constexpr uint32_t kCols = DC == 1 ? 256 : 512;
};
constexpr int kBars = 4 + 4 * kStages + 2 + 5;
constexpr float kRescale = 8.f;
}  // namespace fw

// Position in a ring of N stages.
template <int N>
struct Ring {
  int s = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int k = 1) {  // k <= N
    s += k;
    if (s >= N) {
      s -= N;
      phase ^= 1;
    }
  }
};

// Scores [n, 32) of a block to -inf: weights of zero.
__device__ __forceinline__ void mask_tail(uint32_t (&s)[32], int n) {
#pragma unroll
  for (int e = 0; e < 32; ++e)
    if (e >= n) s[e] = 0xff800000u;
}

__device__ __forceinline__ float max32(const uint32_t (&s)[32], float mx) {
  float m4[4] = {mx, mx, mx, mx};
#pragma unroll
  for (int e = 0; e < 32; e += 2)
    m4[(e >> 1) & 3] = max3(m4[(e >> 1) & 3], __uint_as_float(s[e]), __uint_as_float(s[e + 1]));
  return max3(fmaxf(m4[0], m4[1]), m4[2], m4[3]);
}

// 2^a and 2^b for a, b <= 127 on the FMA pipe, relative error 2^-22.5: n = round(x) falls out of the addition of 1.5
// 2^23 (range reduction as in Cody and Waite, 1980), and 2^(x - n) on [-1/2, 1/2] is a degree-five polynomial with the
// constant term 1 (pymsst_b200/exp2_fit.py fits it and emulates this arithmetic).  Powers below 2^-127 become 2^-127,
// whose exponent bits are those of zero, so masked scores give exactly 0; NaN passes through the maximum and the
// product.
__device__ __forceinline__ void exp2_pair(float& a, float& b) {
  constexpr float kRound = 12582912.f;
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(-127.f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(b) : "f"(-127.f));
  const uint64_t x = pk2(a, b), t = add2(x, pk2(kRound, kRound));
  const uint64_t f = fma2(add2(t, pk2(-kRound, -kRound)), pk2(-1.f, -1.f), x);
  uint64_t p = pk2(0.001326472731307149f, 0.001326472731307149f);
  p = fma2(p, f, pk2(0.009671512991189957f, 0.009671512991189957f));
  p = fma2(p, f, pk2(0.05550733581185341f, 0.05550733581185341f));
  p = fma2(p, f, pk2(0.24022242426872253f, 0.24022242426872253f));
  p = fma2(p, f, pk2(0.6931470036506653f, 0.6931470036506653f));
  p = fma2(p, f, pk2(1.f, 1.f));
  float u, v;
  unpk2(t, u, v);
  u = __uint_as_float((__float_as_uint(u) << 23) + 0x3f800000u);
  v = __uint_as_float((__float_as_uint(v) << 23) + 0x3f800000u);
  unpk2(mul2(p, pk2(u, v)), a, b);
}

// 2^(s sl2 - m) of 32 scores: added to the pair of sums, and rounded to pairs of T.  With MIX every fourth pair comes
// from the FMA pipe, the rest from the special-function pipe, which alone is busy for half the time: 4096 x 4096
// without dropout 119.5 us with none of 16 pairs, 116.8 with two, 113.9 with four, 126.5 with eight; one query over
// 8192 keys 81.4, 78.7, 78.0, 80.5.  With dropout instruction issue is the bound and all stay there.
template <typename T, bool MIX>
__device__ __forceinline__ void exp32(const uint32_t (&s)[32], uint64_t sl22, uint64_t m22, uint64_t& sum,
                                      uint32_t (&p2)[16]) {
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    float a, b;
    unpk2(fma2(pk2(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), sl22, m22), a, b);
    if (MIX && e % 4 == 1) {
      exp2_pair(a, b);
    } else {
      a = ex2(a);
      b = ex2(b);
    }
    sum = add2(sum, pk2(a, b));
    p2[e] = pack2<T>(a, b);
  }
}

struct Item {
  int b, u, blk, split;
};

__device__ __forceinline__ Item forward_item(int item, const Geometry& g) {
  Item it;
  it.b = g.by_units.split(g.by_splits.split(g.by_nblk.split(item, it.blk), it.split), it.u);
  return it;
}

// Chunks [c0, c1) of an item.
__device__ __forceinline__ void chunk_range(int len, const Item& it, const Geometry& g, int& c0, int& c1) {
  const int n = g.by_width.div(len + g.width - 1);
  c0 = 0;
  c1 = n;
  if (g.splits > 1) {  // n splits < 2^31: the host sees to it
    c0 = g.by_splits.div(n * it.split);
    c1 = g.by_splits.div(n * (it.split + 1));
  }
}

template <typename T, int DC, bool DROP>
__global__ void __launch_bounds__(fw::kThreads, DC == 1 ? 2 : 1)
    xattn_fwd(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
              const __grid_constant__ CUtensorMap tmV, T* __restrict__ o, float* __restrict__ lse,
              float* __restrict__ part_o, float* __restrict__ part_lse, Plane po, Shape sh, Geometry g,
              DropArgs drop) {
  using namespace fw;
  using Y = L<DC>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Y::OFF_BAR);
  uint64_t* q_full = bars;         // [2]
  uint64_t* q_empty = q_full + 2;  // [2]
  uint64_t* k_full = q_empty + 2;
  uint64_t* k_empty = k_full + kStages;
  uint64_t* v_full = k_empty + kStages;
  uint64_t* v_empty = v_full + kStages;
  uint64_t* s_full = v_empty + kStages;  // [2]
  uint64_t* p_full = s_full + 2;         // [2]: a warp may be one chunk ahead of another
  uint64_t* o_done = p_full + 2;         // [2], for the same reason
  uint64_t* o_empty = o_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kBars);
  __shared__ int abort_flag;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // uniform in a warp
  const int gp_mask = (1 << g.gp_shift) - 1;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      umma::mbar_init(&q_full[i], 1);
      umma::mbar_init(&q_empty[i], 1);
      umma::mbar_init(&s_full[i], 1);
      umma::mbar_init(&p_full[i], 4);
      umma::mbar_init(&o_done[i], 1);
    }
    for (int s = 0; s < kStages; ++s) {
      umma::mbar_init(&k_full[s], 1);
      umma::mbar_init(&k_empty[s], 1);
      umma::mbar_init(&v_full[s], 1);
      umma::mbar_init(&v_empty[s], 1);
    }
    umma::mbar_init(o_empty, 4);
    abort_flag = 0;
    umma::fence_barrier_init();
  }
  if (warp == 0) umma::tmem_alloc(tmem_slot, Y::kCols);
  umma::tc_fence_before();
  __syncthreads();
  umma::tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

  if (warp == 0) {
    if (lane == 0) {
      umma::tma_prefetch(&tmQ);
      umma::tma_prefetch(&tmK);
      umma::tma_prefetch(&tmV);
      Ring<kStages> kv;
      Ring<2> q;
      bool ok = true;
      auto load = [&](const CUtensorMap* map, uint64_t* full, uint64_t* empty, int off, int c, const Item& it) -> bool {
        if (!umma::mbar_wait(&empty[kv.s], kv.phase ^ 1, 0x92)) return false;
        umma::mbar_arrive_expect_tx(&full[kv.s], DC * g.width * 128);
#pragma unroll
        for (int dc = 0; dc < DC; ++dc)
          umma::tma_load_4d(smem + off + (kv.s * DC + dc) * SUB, map, &full[kv.s], dc * 64, c * g.width,
                            g.by_kv_units.div(it.u), it.b);
        return true;
      };
      for (int item = blockIdx.x; item < g.total && ok && !abort_flag; item += gridDim.x) {
        const Item it = forward_item(item, g);
        int c0, c1;
        chunk_range(sh.keys(it.b), it, g, c0, c1);
        if (c0 >= c1) continue;
        if (!umma::mbar_wait(&q_empty[q.s], q.phase ^ 1, 0x91)) {
          ok = false;
          break;
        }
        umma::mbar_arrive_expect_tx(&q_full[q.s], DC * TILE);
#pragma unroll
        for (int dc = 0; dc < DC; ++dc)
          umma::tma_load_5d(smem + (q.s * DC + dc) * TILE, &tmQ, &q_full[q.s], dc * 64, 0, (it.blk * BM) >> g.gp_shift,
                            it.u, it.b);
        for (int c = c0; c < c1 && ok; ++c, kv.next())
          ok = load(&tmK, k_full, k_empty, Y::OFF_K, c, it) && load(&tmV, v_full, v_empty, Y::OFF_V, c, it);
        q.next();
      }
      if (!ok) abort_flag = 1;
    }
  } else if (warp == 1) {
    {  // the whole warp, so that addresses and descriptors stay uniform; one lane issues
      const bool leader = umma::elect_one();
      // O += P V of the chunk whose scores were issued last
      struct Pending {
        bool live, first;
        int keys;
        uint32_t t;
      } prev{false, false, 0, 0};
      uint32_t cc = 0, t = 0;  // chunks and items so far
      Ring<kStages> kr, vr;
      Ring<2> q;
      auto issue_o = [&](uint32_t c) -> bool {
        if (!umma::mbar_wait(&p_full[c & 1], (c >> 1) & 1, 0x94) || !umma::mbar_wait(&v_full[vr.s], vr.phase, 0x95)) return false;
        if (prev.first && !umma::mbar_wait(o_empty, (prev.t & 1) ^ 1, 0x96)) return false;
        umma::tc_fence_after();
        if (leader) {
          mma_rows_ts<DC>(tmem + Y::kTmemO, tmem + (c & 1) * kMaxW, tile_desc(smem + Y::OFF_V + vr.s * DC * SUB), SUB,
                          Desc<T>::MN, (prev.keys + 15) >> 4, !prev.first);
          umma::mma_commit(&o_done[c & 1]);
          umma::mma_commit(&v_empty[vr.s]);
        }
        __syncwarp();
        vr.next();
        return true;
      };
      bool ok = true;
      for (int item = blockIdx.x; item < g.total && ok && !abort_flag; item += gridDim.x) {
        const Item it = forward_item(item, g);
        const int len = sh.keys(it.b);
        int c0, c1;
        chunk_range(len, it, g, c0, c1);
        if (c0 >= c1) continue;
        if (!umma::mbar_wait(&q_full[q.s], q.phase, 0x93)) {
          ok = false;
          break;
        }
        for (int c = c0; c < c1; ++c, ++cc) {
          const int keys = min(g.width, len - c * g.width);
          // the buffer still holds P of the chunk before the previous one until its product is done
          if (!umma::mbar_wait(&k_full[kr.s], kr.phase, 0x97) || (cc > 1 && !umma::mbar_wait(&o_done[cc & 1], ((cc >> 1) - 1) & 1, 0x9a))) {
            ok = false;
            break;
          }
          umma::tc_fence_after();
          if (leader) {
            mma_scores<DC>(tmem + (cc & 1) * kMaxW, tile_desc(smem + q.s * DC * TILE), TILE,
                           tile_desc(smem + Y::OFF_K + kr.s * DC * SUB), SUB, Desc<T>::kk((keys + 15) & ~15));
            umma::mma_commit(&s_full[cc & 1]);
            umma::mma_commit(&k_empty[kr.s]);
            if (c == c1 - 1) umma::mma_commit(&q_empty[q.s]);
          }
          __syncwarp();
          kr.next();
          if (prev.live && !issue_o(cc - 1)) {
            ok = false;
            break;
          }
          prev = Pending{true, c == c0, keys, t};
        }
        q.next();
        ++t;
      }
      if (ok && prev.live) ok = issue_o(cc - 1);
      if (!ok) abort_flag = 1;
    }
  } else {
    const int quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    const float sl2 = sh.scale * kLog2e;
    const Philox rng(DROP ? drop : DropArgs{});
    uint32_t cc = 0;
    Ring<kStages> vr;
    for (int item = blockIdx.x; item < g.total && !abort_flag; item += gridDim.x) {
      const Item it = forward_item(item, g);
      const int len = sh.keys(it.b);
      int c0, c1;
      chunk_range(len, it, g, c0, c1);
      const int R = it.blk * BM + row, pos = R >> g.gp_shift, head = (it.u << g.gp_shift) + (R & gp_mask);
      const bool valid = R < g.rows;
      const bool idle = it.blk * BM + quarter * 32 >= g.rows;  // no row of this warp exists
      // formed where they are used, not held in registers across the loop
      auto stat = [&] { return (int64_t)(it.b * g.units + it.u) * g.ldr + R; };
      auto prow = [&] { return ((int64_t)(it.b * g.units + it.u) * g.splits + it.split) * g.rows + R; };
      auto dst = [&] { return o + it.b * po.s_b + pos * po.s_n + head * po.s_h; };
      if (c0 >= c1) {
        if (valid) {
          if (g.splits > 1) {
            part_lse[prow()] = -INFINITY;
          } else {
            for (int d = 0; d < sh.dim; d += 8) *reinterpret_cast<uint4*>(dst() + d) = make_uint4(0, 0, 0, 0);
            lse[stat()] = -INFINITY;
          }
        }
        continue;
      }
      const uint32_t bh = (uint32_t)(it.b * sh.heads + head);
      float m = -INFINITY, l = 0.f;
      bool ok = true;
      for (int c = c0; c < c1; ++c, ++cc, vr.next()) {
        const int kc = c * g.width, keys = min(g.width, len - kc);
        if (!umma::mbar_wait(&s_full[cc & 1], (cc >> 1) & 1, 0x98)) {
          ok = false;
          break;
        }
        umma::tc_fence_after();
        const uint32_t src = lanes + (cc & 1) * kMaxW;
        if (!idle) {
          // Without dropout a chunk's scores stay in registers and its code is straight; with it (45 more
          // instructions per eight scores) a loop over 32 scores that reads them twice is ahead, as the code
          // stays small.  Measured rolled against straight when this was chosen: 258 keys 182 against 224 us with
          // dropout, 127 against 123 us without, 4096 keys 135 against 116 us without.
          uint32_t s[DROP ? 1 : 3][32];
          float mx = -INFINITY;
          if constexpr (DROP) {
#pragma unroll 1
            for (int first = 0; first < keys; first += 32) {
              tmem_ld32_nowait(src + first, s[0]);
              wait_ld();
              tie32(s[0]);
              if (first + 32 > keys) mask_tail(s[0], keys - first);
              mx = max32(s[0], mx);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 3; ++i) tmem_ld32_nowait(src + i * 32, s[i]);
            wait_ld();
#pragma unroll
            for (int i = 0; i < 3; ++i) {
              tie32(s[i]);
              if (i * 32 + 32 > keys) mask_tail(s[i], keys - i * 32);
              mx = max32(s[i], mx);
            }
          }
          mx *= sl2;
          if (c == c0) {
            m = fmaxf(mx, xattn::kLowest);  // finite: a chunk of scores of -infinity weighs nothing
          } else {
            const bool grows = mx > m + kRescale;
            if (__any_sync(0xffffffffu, grows)) {
              if (!umma::mbar_wait(&o_done[(cc - 1) & 1], ((cc - 1) >> 1) & 1, 0x99)) {
                ok = false;
                break;
              }
              umma::tc_fence_after();
              const float mn = grows ? mx : m, f = grows ? ex2(m - mn) : 1.f;
              l *= f;
              m = mn;
#pragma unroll 1
              for (int k = 0; k < 4 * DC; ++k) {
                uint32_t a[16];
                tmem_ld16_nowait(lanes + Y::kTmemO + k * 16, a);
                wait_ld();
                tie16(a);
#pragma unroll
                for (int e = 0; e < 16; ++e) a[e] = __float_as_uint(__uint_as_float(a[e]) * f);
                umma::tmem_st16(lanes + Y::kTmemO + k * 16, a);
              }
            }
          }
          uint64_t sum = pk2(0.f, 0.f);
          const uint64_t sl22 = pk2(sl2, sl2), m22 = pk2(-m, -m);
          uint32_t p2[16];
          if constexpr (DROP) {
#pragma unroll 1
            for (int first = 0; first < keys; first += 32) {
              tmem_ld32_nowait(src + first, s[0]);
              uint32_t mask[16];
#pragma unroll
              for (int gr = 0; gr < 4; ++gr) {  // drawn while the scores come
                const uint4 r = rng((uint32_t)(kc + first) / 8 + gr, (uint32_t)pos, bh);
                mask[gr * 4] = keep_mask2(r.x, drop.limit);
                mask[gr * 4 + 1] = keep_mask2(r.y, drop.limit);
                mask[gr * 4 + 2] = keep_mask2(r.z, drop.limit);
                mask[gr * 4 + 3] = keep_mask2(r.w, drop.limit);
              }
              wait_ld();
              tie32(s[0]);
              if (first + 32 > keys) mask_tail(s[0], keys - first);
              exp32<T, false>(s[0], sl22, m22, sum, p2);
#pragma unroll
              for (int e = 0; e < 16; ++e) p2[e] &= mask[e];
              umma::tmem_st16(src + first / 2, p2);  // over scores this warp has read
            }
          } else {
#pragma unroll
            for (int i = 0; i < 3; ++i) {
              if (i * 32 < keys) {
                exp32<T, true>(s[i], sl22, m22, sum, p2);
                umma::tmem_st16(src + i * 16, p2);
              }
            }
          }
          umma::tmem_wait_st();
          float a, b;
          unpk2(sum, a, b);
          l += a + b;
        }
        bool zeroed = false;
        if (keys < g.width && sh.lengths != nullptr) {  // values behind the length: zeros, whatever they were
          if (!umma::mbar_wait(&v_full[vr.s], vr.phase, 0x9b)) {
            ok = false;
            break;
          }
          zero_rows<DC>(smem + Y::OFF_V + vr.s * DC * SUB, SUB, keys, (keys + 15) & ~15, threadIdx.x - 64);
          zeroed = true;
        }
        warp_arrive(&p_full[cc & 1], zeroed);
      }
      if (!ok || !umma::mbar_wait(&o_done[(cc - 1) & 1], ((cc - 1) >> 1) & 1, 0x9c)) {
        abort_flag = 1;
        break;
      }
      umma::tc_fence_after();
      const float inv = l == 0.f ? 0.f : (DROP ? drop.scale : 1.f) / l;  // every score -infinity: as without keys
#pragma unroll 1
      for (int k = 0; k < 2 * DC; ++k) {
        if (idle || k * 32 >= sh.dim) break;
        uint32_t a[32];
        tmem_ld32_nowait(lanes + Y::kTmemO + k * 32, a);
        wait_ld();
        tie32(a);
        if (valid && g.splits == 1) store_row<T>(dst(), k * 32, sh.dim, a, inv);
        if (valid && g.splits > 1) {
          const float* f = reinterpret_cast<const float*>(a);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (k * 32 + i * 4 < sh.dim)
              *reinterpret_cast<float4*>(part_o + prow() * sh.dim + k * 32 + i * 4) =
                  make_float4(f[4 * i] * inv, f[4 * i + 1] * inv, f[4 * i + 2] * inv, f[4 * i + 3] * inv);
        }
      }
      warp_arrive(o_empty, false);
      if (valid) {
        const float stat2 = m + log2f(l);
        if (g.splits > 1) part_lse[prow()] = stat2;
        else lse[stat()] = l == 0.f ? -INFINITY : -stat2;
      }
    }
  }
  umma::tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    umma::tc_fence_after();
    umma::tmem_dealloc(tmem, Y::kCols);
  }
}

// Joins the key ranges of a row: O = sum_s w_s O_s / sum_s w_s, w_s = 2^(lse_s - max), in the order of s.  One thread
// per row and 8 head elements.
template <typename T>
__global__ void __launch_bounds__(256)
    xattn_join(const float* __restrict__ part_o, const float* __restrict__ part_lse, T* __restrict__ o,
               float* __restrict__ lse, Plane po, Shape sh, Geometry g, int64_t threads) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= threads) return;
  const int per_row = sh.dim / 8, d = (int)(id % per_row) * 8;
  const int64_t row = id / per_row;
  const int R = (int)(row % g.rows);
  const int64_t bu = row / g.rows;
  const int u = (int)(bu % g.units), b = (int)(bu / g.units);
  const float* ls = part_lse + bu * g.splits * g.rows + R;
  const float* src = part_o + (bu * g.splits * g.rows + R) * sh.dim + d;
  float mx = -INFINITY;
  for (int s = 0; s < g.splits; ++s) mx = fmaxf(mx, ls[(int64_t)s * g.rows]);
  float acc[8] = {}, w = 0.f;
  bool any = false;
  for (int s = 0; s < g.splits; ++s) {
    const float l2 = ls[(int64_t)s * g.rows];
    if (l2 == -INFINITY) continue;  // no keys there, or none that weighs anything
    any = true;
    const float ws = exp2f(l2 - mx);
    w += ws;
    const float4* v = reinterpret_cast<const float4*>(src + (int64_t)s * g.rows * sh.dim);
    const float4 x = v[0], y = v[1];
    const float f[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = fmaf(ws, f[e], acc[e]);
  }
  const float inv = any ? 1.f / w : 0.f;
  const int pos = R >> g.gp_shift, head = (u << g.gp_shift) + (R & ((1 << g.gp_shift) - 1));
  *reinterpret_cast<uint4*>(o + b * po.s_b + pos * po.s_n + head * po.s_h + d) =
      make_uint4(pack2<T>(acc[0] * inv, acc[1] * inv), pack2<T>(acc[2] * inv, acc[3] * inv),
                 pack2<T>(acc[4] * inv, acc[5] * inv), pack2<T>(acc[6] * inv, acc[7] * inv));
  if (d == 0) lse[bu * g.ldr + R] = any ? -(mx + log2f(w)) : -INFINITY;
}

// ---------------------------------------------------------------- backward
// One CTA per SM, its row warps two groups of four (one tensor memory lane
// per thread), NB pairs of 64-column accumulators (S and dP, or their
// transposes).  Chunk n of the CTA's stream uses pair n % NB and goes to group
// n % 2.  One warp issues the score products, another the products of the
// 16-bit operands that a group has written over the scores and dP it read: a
// wait that is already over still costs a warp about 115 cycles and eight
// tcgen05.mma about 500, so one warp for both was the bound (1825 cycles per
// chunk).  With three pairs the scores a group takes next are ready when it
// finishes a chunk.  (Time axis, 258 positions, dropout, dK / dV + dQ: one
// pair per CTA and two CTAs per SM 321 + 219 us, three groups with a pair each
// 355 + 290, two groups over three pairs 310 + 247 with one issuing warp, 288
// + 228 with two; now, with D from a warp of its own and item decoding without
// divisions, 269 + 191, and 196 + 144 without dropout.)
//
// Barriers that groups wait on out of step have turns: item t uses barrier
// t % NB.  A chunk's scores are complete only after the products of the chunk
// NB before it, so when a group that has seen the scores of item t's last
// chunk waits, the turn before (item t - NB, at least NB chunks back) is over.
// D has 2 NB turns: it is formed when an item's tiles are there, so while the
// scores of item t - 2 (two tiles) are complete, of which the last NB - 1
// chunks may still be worked on: item t - 2 NB is over.
namespace bw {
constexpr int BC = 64;                 // chunk rows
constexpr int CT = BC * 128;           // bytes of a chunk's 64-element sub-tile
constexpr int G = 2;                   // groups of row warps
}  // namespace bw

// ------------------------------------------------------------ backward: dQ
// Item = 128 packed rows of a unit, chunks of 64 keys: S = Q K^T, dP = dO V^T,
// dQ += dS K.  A warp of its own forms D = rowsum(dO * O) of the items ahead
// of the groups, from tiles (O's rows read from global memory took a group
// 3000 cycles per item), and keeps it for the dK / dV kernel; the group with
// an item's last chunk writes dQ.
//
// With ONE, at most one chunk of keys in all, the group forms D = rowsum(P dP)
// itself before it uses the scores.  O is rounded, and what that leaves in D is
// the same for all keys of a row: many keys average it out, few do not (errors
// of dQ and dK against 64 bits, in units of fp32 arithmetic with one rounding:
// 2.3 for two keys, 1.75 for four, 1.5 for 20, 1.45 for 100 and for all lengths
// with D so formed, where dS rounded to 16 bits is what remains).  A kernel of
// its own, as the longer form's registers would not hold it: decided within one
// kernel it cost the time axis with dropout 191 -> 234 us.
namespace bq {
constexpr int kThreads = 128 + 128 * bw::G;  // one more control warp, for D
template <int DC>
struct L {
  static constexpr int NB = 3;
  static constexpr int kTiles = DC == 1 ? 2 : 1;            // Q, dO, O tiles
  static constexpr int kN = DC == 1 ? 6 : 3;                // stages of DC K sub-tiles, DC V sub-tiles
  static constexpr int TILES = 3 * DC * TILE;
  static constexpr int STAGE = 2 * DC * bw::CT;
  static constexpr int OFF_KV = kTiles * TILES;
  static constexpr int OFF_D = OFF_KV + kN * STAGE;         // [2 NB][128] -D, then [2 NB][128] -lse2
  static constexpr int OFF_BAR = OFF_D + 4 * NB * 512;
  static constexpr int SMEM = OFF_BAR + 512 + 1024;
  static constexpr uint32_t kTmemDQ = 128 * NB;
};
}  // namespace bq

// One chunk of the stream of a CTA: items with keys, in order, chunk by chunk.
struct QueryCursor {
  int item, len, c, nch;
  Item it;
  bool live;

  __device__ __forceinline__ void seek(const Shape& sh, const Geometry& g) {  // from `item` on
    live = false;
    for (; item < g.total; item += gridDim.x) {
      it = forward_item(item, g);
      len = sh.keys(it.b);
      nch = (len + bw::BC - 1) / bw::BC;
      if (nch > 0) {
        live = true;
        return;
      }
    }
  }
  __device__ __forceinline__ QueryCursor(const Shape& sh, const Geometry& g) : item(blockIdx.x), c(0) { seek(sh, g); }
  // k chunks on; the number of items left behind
  __device__ __forceinline__ int next(const Shape& sh, const Geometry& g, int k = 1) {
    int items = 0;
    c += k;
    while (c >= nch && live) {
      c -= nch;
      item += gridDim.x;
      seek(sh, g);
      ++items;
    }
    return items;
  }
  __device__ __forceinline__ bool first() const { return c == 0; }
  __device__ __forceinline__ bool last() const { return c == nch - 1; }
  __device__ __forceinline__ int keys() const { return min(bw::BC, len - c * bw::BC); }
};

template <typename T, int DC, bool DROP, bool ONE>
__global__ void __launch_bounds__(bq::kThreads, 1)
    xattn_bwd_dq(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmDO,
                 const __grid_constant__ CUtensorMap tmO, const __grid_constant__ CUtensorMap tmK,
                 const __grid_constant__ CUtensorMap tmV, const float* __restrict__ lse, float* __restrict__ delta,
                 T* __restrict__ dq, Plane pdq, Shape sh, Geometry g, DropArgs drop) {
  using namespace bw;
  using Y = bq::L<DC>;
  constexpr int NB = Y::NB;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Y::OFF_BAR);
  uint64_t* qd_full = bars;                  // [kTiles]
  uint64_t* qd_empty = qd_full + Y::kTiles;  // [kTiles]
  uint64_t* kv_full = qd_empty + Y::kTiles;  // [kN]
  uint64_t* kv_empty = kv_full + Y::kN;      // [kN]
  uint64_t* sd_full = kv_empty + Y::kN;      // [NB]
  uint64_t* ds_full = sd_full + NB;           // [NB]
  uint64_t* ds_done = ds_full + NB;           // [NB]
  uint64_t* d_full = ds_done + NB;            // [2 NB]
  uint64_t* dq_full = d_full + 2 * NB;        // [NB]
  uint64_t* dq_empty = dq_full + NB;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(dq_empty + 1);
  float* nd_s = reinterpret_cast<float*>(smem + Y::OFF_D);
  float* nl_s = nd_s + 2 * NB * 128;
  __shared__ int abort_flag;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // uniform in a warp
  const int gp_mask = (1 << g.gp_shift) - 1;
  if (threadIdx.x == 0) {
    for (int i = 0; i < Y::kTiles; ++i) {
      umma::mbar_init(&qd_full[i], 1);
      umma::mbar_init(&qd_empty[i], 2);  // the scores' commit and the warp that forms D
    }
    for (int i = 0; i < Y::kN; ++i) {
      umma::mbar_init(&kv_full[i], 1);
      umma::mbar_init(&kv_empty[i], 1);
    }
    for (int i = 0; i < NB; ++i) {
      umma::mbar_init(&sd_full[i], 1);
      umma::mbar_init(&ds_full[i], 4);
      umma::mbar_init(&ds_done[i], 1);
      umma::mbar_init(&d_full[i], 1);
      umma::mbar_init(&d_full[NB + i], 1);
      umma::mbar_init(&dq_full[i], 1);
    }
    umma::mbar_init(dq_empty, 4);
    abort_flag = 0;
    umma::fence_barrier_init();
  }
  if (warp == 0) umma::tmem_alloc(tmem_slot, 512);
  umma::tc_fence_before();
  __syncthreads();
  umma::tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

  if (warp == 0) {
    if (lane == 0) {  // tiles of an item before its first chunk
      umma::tma_prefetch(&tmQ);
      umma::tma_prefetch(&tmDO);
      umma::tma_prefetch(&tmO);
      umma::tma_prefetch(&tmK);
      umma::tma_prefetch(&tmV);
      Ring<Y::kTiles> qd;
      Ring<Y::kN> kv;
      for (QueryCursor cu(sh, g); cu.live && !abort_flag; cu.next(sh, g), kv.next()) {
        if (cu.first()) {
          if (!umma::mbar_wait(&qd_empty[qd.s], qd.phase ^ 1, 0xa1)) {
            abort_flag = 1;
            break;
          }
          uint8_t* dst = smem + qd.s * Y::TILES;
          umma::mbar_arrive_expect_tx(&qd_full[qd.s], Y::TILES);
          const int pos = (cu.it.blk * BM) >> g.gp_shift;
#pragma unroll
          for (int dc = 0; dc < DC; ++dc) {
            umma::tma_load_5d(dst + dc * TILE, &tmQ, &qd_full[qd.s], dc * 64, 0, pos, cu.it.u, cu.it.b);
            umma::tma_load_5d(dst + (DC + dc) * TILE, &tmDO, &qd_full[qd.s], dc * 64, 0, pos, cu.it.u, cu.it.b);
            umma::tma_load_5d(dst + (2 * DC + dc) * TILE, &tmO, &qd_full[qd.s], dc * 64, 0, pos, cu.it.u, cu.it.b);
          }
          qd.next();
        }
        if (!umma::mbar_wait(&kv_empty[kv.s], kv.phase ^ 1, 0xa2)) {
          abort_flag = 1;
          break;
        }
        uint8_t* dst = smem + Y::OFF_KV + kv.s * Y::STAGE;
        umma::mbar_arrive_expect_tx(&kv_full[kv.s], Y::STAGE);
#pragma unroll
        for (int dc = 0; dc < DC; ++dc) {
          umma::tma_load_4d(dst + dc * CT, &tmK, &kv_full[kv.s], dc * 64, cu.c * BC, g.by_kv_units.div(cu.it.u), cu.it.b);
          umma::tma_load_4d(dst + (DC + dc) * CT, &tmV, &kv_full[kv.s], dc * 64, cu.c * BC, g.by_kv_units.div(cu.it.u),
                            cu.it.b);
        }
      }
    }
  } else if (warp == 1) {  // scores; the whole warp runs along, so that addresses and descriptors stay uniform
    const bool leader = umma::elect_one();
    Ring<Y::kTiles> qd;
    Ring<Y::kN> kv;
    Ring<NB> gr;
    for (QueryCursor cu(sh, g); cu.live && !abort_flag;) {
      if ((cu.first() && !umma::mbar_wait(&qd_full[qd.s], qd.phase, 0xa3)) ||
          !umma::mbar_wait(&kv_full[kv.s], kv.phase, 0xa4) || !umma::mbar_wait(&ds_done[gr.s], gr.phase ^ 1, 0xa5)) {
        abort_flag = 1;
        break;
      }
      umma::tc_fence_after();
      const uint64_t k = tile_desc(smem + Y::OFF_KV + kv.s * Y::STAGE), q = tile_desc(smem + qd.s * Y::TILES);
      const uint32_t idesc = Desc<T>::kk((cu.keys() + 15) & ~15), acc = tmem + gr.s * 128;
      if (leader) {
        mma_scores<DC>(acc, q, TILE, k, CT, idesc);
        mma_scores<DC>(acc + 64, q + DC * TILE / 16, TILE, k + DC * CT / 16, CT, idesc);
        umma::mma_commit(&sd_full[gr.s]);
        if (cu.last()) umma::mma_commit(&qd_empty[qd.s]);
      }
      __syncwarp();
      kv.next();
      gr.next();
      if (cu.next(sh, g)) qd.next();
    }
  } else if (warp == 2) {  // products
    const bool leader = umma::elect_one();
    Ring<Y::kN> kv;
    Ring<NB> gr, turn;
    uint32_t odd = 0;  // items so far, modulo 2
    for (QueryCursor cu(sh, g); cu.live && !abort_flag;) {
      const bool first = cu.first();
      if (!umma::mbar_wait(&ds_full[gr.s], gr.phase, 0xa6) || (first && !umma::mbar_wait(dq_empty, odd ^ 1, 0xa7))) {
        abort_flag = 1;
        break;
      }
      umma::tc_fence_after();
      if (leader) {
        mma_rows_ts<DC>(tmem + Y::kTmemDQ, tmem + gr.s * 128, tile_desc(smem + Y::OFF_KV + kv.s * Y::STAGE), CT,
                        Desc<T>::MN, (cu.keys() + 15) >> 4, !first);
        if (cu.last()) umma::mma_commit(&dq_full[turn.s]);  // before the pair is free: see the turns above
        umma::mma_commit(&ds_done[gr.s]);
        umma::mma_commit(&kv_empty[kv.s]);
      }
      __syncwarp();
      kv.next();
      gr.next();
      if (cu.next(sh, g)) {
        turn.next();
        odd ^= 1;
      }
    }
  } else if (warp == 3) {  // D and the statistics of the items
    Ring<Y::kTiles> qd;
    Ring<2 * NB> turn;
    for (QueryCursor cu(sh, g); cu.live && !abort_flag; cu.next(sh, g, cu.nch), qd.next(), turn.next()) {
      const int rows = min(BM, g.rows - cu.it.blk * BM);
      const int64_t stat = (int64_t)(cu.it.b * g.units + cu.it.u) * g.ldr + cu.it.blk * BM + lane;
      float nlse[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) nlse[i] = lane + 32 * i < rows ? lse[stat + 32 * i] : 0.f;
      if (!umma::mbar_wait(&qd_full[qd.s], qd.phase, 0xa8)) {
        abort_flag = 1;
        break;
      }
      const uint8_t* go = smem + qd.s * Y::TILES + DC * TILE;
      float nd[4] = {0.f, 0.f, 0.f, 0.f};  // four rows at a time hide one another's latencies
#pragma unroll 2
      for (int c = ONE ? 8 * DC : 0; c < 8 * DC; ++c) {
        uint4 o4[4], d4[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t at = (c >> 3) * TILE + sw128(lane + 32 * i, c & 7);
          d4[i] = *reinterpret_cast<const uint4*>(go + at);
          o4[i] = *reinterpret_cast<const uint4*>(go + DC * TILE + at);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const T* oe = reinterpret_cast<const T*>(&o4[i]);
          const T* de = reinterpret_cast<const T*>(&d4[i]);
#pragma unroll
          for (int e = 0; e < 8; ++e) nd[i] = fmaf(-Elem<T>::to_f(oe[e]), Elem<T>::to_f(de[e]), nd[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (!ONE && lane + 32 * i < rows) delta[stat + 32 * i] = nd[i];
        nd_s[turn.s * 128 + lane + 32 * i] = nd[i];
        nl_s[turn.s * 128 + lane + 32 * i] = nlse[i];
      }
      __syncwarp();
      if (lane == 0) {
        umma::mbar_arrive(&d_full[turn.s]);
        umma::mbar_arrive(&qd_empty[qd.s]);
      }
    }
  } else {
    const int grp = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const float sl2 = sh.scale * kLog2e, mult = DROP ? drop.scale : 1.f;
    const uint64_t sl22 = pk2(sl2, sl2), mult2 = pk2(mult, mult);
    const Philox rng(DROP ? drop : DropArgs{});
    // rows of items without keys: zeros
    if (grp == 0 && sh.lengths != nullptr)
      for (int item = blockIdx.x; item < g.total; item += gridDim.x) {
        const Item it = forward_item(item, g);
        const int R = it.blk * BM + row;
        if (sh.keys(it.b) > 0 || R >= g.rows) continue;
        T* dst = dq + it.b * pdq.s_b + (R >> g.gp_shift) * pdq.s_n + ((it.u << g.gp_shift) + (R & gp_mask)) * pdq.s_h;
        for (int d = 0; d < sh.dim; d += 8) *reinterpret_cast<uint4*>(dst + d) = make_uint4(0, 0, 0, 0);
        delta[(int64_t)(it.b * g.units + it.u) * g.ldr + R] = 0.f;
      }
    QueryCursor cu(sh, g);
    Ring<Y::kN> kv;
    Ring<NB> gr;     // accumulators of the cursor's chunk
    Ring<NB> turn;   // of the items
    Ring<2 * NB> dturn;
    auto advance = [&](int k) {
      kv.next(k);
      gr.next(k);
      for (int i = cu.next(sh, g, k); i > 0; --i) {
        turn.next();
        dturn.next();
      }
    };
    if (grp == 1) advance(1);
    int known = -1;  // item whose statistics these are
    uint64_t nd2 = 0, nlse2 = 0;
    for (; cu.live && !abort_flag; advance(G)) {
      {
        const bool last = cu.last();
        const uint32_t acc = tmem + lane_off + gr.s * 128;
        const Item& it = cu.it;
        const int R = it.blk * BM + row, pos = R >> g.gp_shift, head = (it.u << g.gp_shift) + (R & gp_mask);
        const bool valid = R < g.rows, idle = it.blk * BM + quarter * 32 >= g.rows;
        if (!umma::mbar_wait(&sd_full[gr.s], gr.phase, 0xaa)) {
          abort_flag = 1;
          break;
        }
        if (cu.item != known) {
          if (!umma::mbar_wait(&d_full[dturn.s], dturn.phase, 0xa9)) {
            abort_flag = 1;
            break;
          }
          known = cu.item;
          const float nd = nd_s[dturn.s * 128 + row], nlse = nl_s[dturn.s * 128 + row];
          nd2 = pk2(nd, nd);
          nlse2 = pk2(nlse, nlse);
        }
        umma::tc_fence_after();
        const int keys = cu.keys();
        if (!idle) {
          const uint32_t bh = (uint32_t)(it.b * sh.heads + head);
          uint64_t bits = ~0ull;  // of all keys, when they are one chunk
          if constexpr (ONE) {
            if (DROP) bits = 0;
            float sum = 0.f;
#pragma unroll 1
            for (int first = 0; first < keys; first += 16) {
              uint32_t su[16], du[16];
              tmem_ld16_nowait(acc + first, su);
              tmem_ld16_nowait(acc + 64 + first, du);
              if (DROP) {
                const uint32_t low = keep_bits(rng((uint32_t)first / 8, (uint32_t)pos, bh), drop.limit);
                const uint32_t high = keep_bits(rng((uint32_t)first / 8 + 1, (uint32_t)pos, bh), drop.limit);
                bits |= (uint64_t)(low | (high << 8)) << first;
              }
              const uint32_t live = (uint32_t)(bits >> first) & (0xffffffffu >> (32 - min(16, keys - first)));
              tmem_wait16(su, du);
#pragma unroll
              for (int i = 0; i < 16; i += 2) {
                float p0, p1;
                unpk2(fma2(pk2(__uint_as_float(su[i]), __uint_as_float(su[i + 1])), sl22, nlse2), p0, p1);
                sum += (live >> i) & 1u ? ex2(p0) * __uint_as_float(du[i]) : 0.f;
                sum += (live >> (i + 1)) & 1u ? ex2(p1) * __uint_as_float(du[i + 1]) : 0.f;
              }
            }
            const float nd = -mult * sum;
            nd2 = pk2(nd, nd);
            if (valid) delta[(int64_t)(it.b * g.units + it.u) * g.ldr + R] = nd;
          }
#pragma unroll 1
          for (int first = 0; first < keys; first += 32) {
            uint32_t su[32], du[32];
            tmem_ld32_nowait(acc + first, su);
            tmem_ld32_nowait(acc + 64 + first, du);
            tmem_wait2(su, du);
            const uint32_t now = (uint32_t)(bits >> first);
            uint32_t p2[16];
#pragma unroll
            for (int q8 = 0; q8 < 4; ++q8) {
              uint4 r = make_uint4(0, 0, 0, 0);
              if (DROP && !ONE) r = rng((uint32_t)(cu.c * BC + first) / 8 + q8, (uint32_t)pos, bh);
              const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int i = q8 * 4 + e;
                float d0 = __uint_as_float(du[2 * i]), d1 = __uint_as_float(du[2 * i + 1]), p0, p1;
                unpk2(fma2(pk2(__uint_as_float(su[2 * i]), __uint_as_float(su[2 * i + 1])), sl22, nlse2), p0, p1);
                uint64_t x;
                if (DROP) {
                  d0 = (ONE ? (now >> (2 * i)) & 1u : kept(w[e], 0, drop.high)) ? d0 : 0.f;
                  d1 = (ONE ? (now >> (2 * i + 1)) & 1u : kept(w[e], 1, drop.high)) ? d1 : 0.f;
                  x = fma2(pk2(d0, d1), mult2, nd2);
                } else {
                  x = add2(pk2(d0, d1), nd2);
                }
                unpk2(mul2(pk2(ex2(p0), ex2(p1)), x), p0, p1);
                p2[i] = pack2<T>(p0, p1);
              }
            }
            if (first + 32 > keys) zero_tail(p2, keys - first);
            umma::tmem_st16(acc + first / 2, p2);  // over scores this warp has read
          }
          umma::tmem_wait_st();
        }
        const bool pad = keys < BC && sh.lengths != nullptr;
        if (pad)  // S of this chunk is formed: its keys behind the length become zeros
          zero_rows<DC>(smem + Y::OFF_KV + kv.s * Y::STAGE, CT, keys, (keys + 15) & ~15, row);
        warp_arrive(&ds_full[gr.s], pad);
        if (last) {
          if (!umma::mbar_wait(&dq_full[turn.s], turn.phase, 0xac)) {
            abort_flag = 1;
            break;
          }
          umma::tc_fence_after();
          T* dst = dq + it.b * pdq.s_b + pos * pdq.s_n + head * pdq.s_h;
#pragma unroll
          for (int dc = 0; dc < DC; ++dc) {  // 64 columns read at once, the last before the stores
            uint32_t a0[32], a1[32];
            if (!idle) {
              tmem_ld32_nowait(tmem + lane_off + Y::kTmemDQ + dc * 64, a0);
              tmem_ld32_nowait(tmem + lane_off + Y::kTmemDQ + dc * 64 + 32, a1);
              tmem_wait2(a0, a1);
            }
            if (dc == DC - 1) warp_arrive(dq_empty, false);
            if (valid) {
              store_row<T>(dst, dc * 64, sh.dim, a0, sh.scale);
              store_row<T>(dst, dc * 64 + 32, sh.dim, a1, sh.scale);
            }
          }
        }
      }
    }
  }
  umma::tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    umma::tc_fence_after();
    umma::tmem_dealloc(tmem, 512);
  }
}

// -------------------------------------------------------- backward: dK, dV
// Item = 128 keys of a key / value head; the packed rows of all its units
// come in chunks of 64 with their lse2 and D.  S^T = K Q^T and dP^T = V dO^T
// put a key in each tensor memory lane; dV += P^T dO, dK += dS^T Q.  The
// dropout bits come in groups of eight keys of one query, that is of eight
// lanes: each lane draws the groups of four of 32 columns and the eight
// exchange the keep bits by shuffles, so a group is still drawn once.
namespace bk {
constexpr int kThreads = 96 + 128 * bw::G;
template <int DC>
struct L {
  static constexpr int NB = DC == 1 ? 3 : 2;                // 512 columns: 128 NB + dV + dK
  static constexpr int kTiles = DC == 1 ? 2 : 1;            // K, V tiles
  static constexpr int kN = DC == 1 ? 8 : 4;
  static constexpr int TILES = 2 * DC * TILE;
  static constexpr int OFF_STAT = 2 * DC * bw::CT;          // within a stage: -lse2[64], -D[64]
  static constexpr int STAGE = OFF_STAT + 1024;
  static constexpr int OFF_CH = kTiles * TILES;
  static constexpr int OFF_BAR = OFF_CH + kN * STAGE;
  static constexpr int SMEM = OFF_BAR + 512 + 1024;
  static constexpr uint32_t kTmemDV = 128 * NB, kTmemDK = 128 * NB + 64 * DC;
};
}  // namespace bk

// One chunk of the stream of a CTA: key blocks with keys, in order, unit by unit, chunk by chunk.
struct KeyCursor {
  int item, blk, kh, b, len, u, u0, u_end, r0, span;  // span: the chunks' rows of a unit
  bool live;

  __device__ __forceinline__ void at(const Shape& sh, const Geometry& g) {
    b = g.by_kv_heads.split(g.by_kblk.split(item, blk), kh);
    len = sh.keys(b);
  }
  __device__ __forceinline__ void seek(const Shape& sh, const Geometry& g) {  // from `item` on
    live = false;
    for (; item < g.total; item += gridDim.x) {
      at(sh, g);
      u = u0 = kh * g.kv_units;
      u_end = u + g.kv_units;
      if (blk * BM < len) {
        live = true;
        return;
      }
    }
  }
  __device__ __forceinline__ KeyCursor(const Shape& sh, const Geometry& g)
      : item(blockIdx.x), r0(0), span((g.rows + bw::BC - 1) / bw::BC * bw::BC) {
    seek(sh, g);
  }
  // k chunks on; the number of items left behind
  __device__ __forceinline__ int next(const Shape& sh, const Geometry& g, int k = 1) {
    int items = 0;
    r0 += k * bw::BC;
    while (r0 >= span && live) {
      r0 -= span;
      if (++u == u_end) {
        item += gridDim.x;
        seek(sh, g);
        ++items;
      }
    }
    return items;
  }
  __device__ __forceinline__ bool first() const { return r0 == 0 && u == u0; }
  __device__ __forceinline__ bool last() const { return r0 + bw::BC == span && u + 1 == u_end; }
};

template <typename T, int DC, bool DROP>
__global__ void __launch_bounds__(bk::kThreads, 1)
    xattn_bwd_dkdv(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmDO,
                   const float* __restrict__ lse, const float* __restrict__ delta, T* __restrict__ dk,
                   T* __restrict__ dv, Plane pdk, Plane pdv, Shape sh, Geometry g, DropArgs drop) {
  using namespace bw;
  using Y = bk::L<DC>;
  constexpr int NB = Y::NB;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Y::OFF_BAR);
  uint64_t* kv_full = bars;                  // [kTiles]
  uint64_t* kv_empty = kv_full + Y::kTiles;  // [kTiles]
  uint64_t* ch_full = kv_empty + Y::kTiles;  // [kN]
  uint64_t* ch_empty = ch_full + Y::kN;      // [kN]
  uint64_t* sd_full = ch_empty + Y::kN;      // [NB]
  uint64_t* ps_full = sd_full + NB;           // [NB]
  uint64_t* ps_done = ps_full + NB;           // [NB]
  uint64_t* acc_full = ps_done + NB;          // [NB]
  uint64_t* acc_empty = acc_full + NB;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 1);
  __shared__ int abort_flag;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // uniform in a warp
  const int gp_mask = (1 << g.gp_shift) - 1;
  if (threadIdx.x == 0) {
    for (int i = 0; i < Y::kTiles; ++i) {
      umma::mbar_init(&kv_full[i], 1);
      umma::mbar_init(&kv_empty[i], 1);
    }
    for (int i = 0; i < Y::kN; ++i) {
      umma::mbar_init(&ch_full[i], 1);
      umma::mbar_init(&ch_empty[i], 1);
    }
    for (int i = 0; i < NB; ++i) {
      umma::mbar_init(&sd_full[i], 1);
      umma::mbar_init(&ps_full[i], 4);
      umma::mbar_init(&ps_done[i], 1);
      umma::mbar_init(&acc_full[i], 1);
    }
    umma::mbar_init(acc_empty, 4);
    abort_flag = 0;
    umma::fence_barrier_init();
  }
  if (warp == 0) umma::tmem_alloc(tmem_slot, 512);
  umma::tc_fence_before();
  __syncthreads();
  umma::tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

  if (warp == 0) {
    if (lane == 0) {  // tiles of an item before its first chunk
      umma::tma_prefetch(&tmK);
      umma::tma_prefetch(&tmV);
      umma::tma_prefetch(&tmQ);
      umma::tma_prefetch(&tmDO);
      Ring<Y::kTiles> kv;
      Ring<Y::kN> ch;
      for (KeyCursor cu(sh, g); cu.live && !abort_flag; cu.next(sh, g), ch.next()) {
        if (cu.first()) {
          if (!umma::mbar_wait(&kv_empty[kv.s], kv.phase ^ 1, 0xb1)) {
            abort_flag = 1;
            break;
          }
          uint8_t* dst = smem + kv.s * Y::TILES;
          umma::mbar_arrive_expect_tx(&kv_full[kv.s], Y::TILES);
#pragma unroll
          for (int dc = 0; dc < DC; ++dc) {
            umma::tma_load_4d(dst + dc * TILE, &tmK, &kv_full[kv.s], dc * 64, cu.blk * BM, cu.kh, cu.b);
            umma::tma_load_4d(dst + (DC + dc) * TILE, &tmV, &kv_full[kv.s], dc * 64, cu.blk * BM, cu.kh, cu.b);
          }
          kv.next();
        }
        if (!umma::mbar_wait(&ch_empty[ch.s], ch.phase ^ 1, 0xb2)) {
          abort_flag = 1;
          break;
        }
        uint8_t* dst = smem + Y::OFF_CH + ch.s * Y::STAGE;
        umma::mbar_arrive_expect_tx(&ch_full[ch.s], 2 * DC * CT + 2 * BC * 4);
#pragma unroll
        for (int dc = 0; dc < DC; ++dc) {
          umma::tma_load_5d(dst + dc * CT, &tmQ, &ch_full[ch.s], dc * 64, 0, cu.r0 >> g.gp_shift, cu.u, cu.b);
          umma::tma_load_5d(dst + (DC + dc) * CT, &tmDO, &ch_full[ch.s], dc * 64, 0, cu.r0 >> g.gp_shift, cu.u, cu.b);
        }
        const int64_t stat = (int64_t)(cu.b * g.units + cu.u) * g.ldr + cu.r0;  // both end 64 values behind the last row
        umma::bulk_load(dst + Y::OFF_STAT, lse + stat, BC * 4, &ch_full[ch.s]);
        umma::bulk_load(dst + Y::OFF_STAT + BC * 4, delta + stat, BC * 4, &ch_full[ch.s]);
      }
    }
  } else if (warp == 1) {  // scores
    const bool leader = umma::elect_one();
    Ring<Y::kTiles> kv;
    Ring<Y::kN> ch;
    Ring<NB> gr;
    for (KeyCursor cu(sh, g); cu.live && !abort_flag;) {
      if ((cu.first() && !umma::mbar_wait(&kv_full[kv.s], kv.phase, 0xb3)) ||
          !umma::mbar_wait(&ch_full[ch.s], ch.phase, 0xb4) || !umma::mbar_wait(&ps_done[gr.s], gr.phase ^ 1, 0xb5)) {
        abort_flag = 1;
        break;
      }
      umma::tc_fence_after();
      const uint64_t q = tile_desc(smem + Y::OFF_CH + ch.s * Y::STAGE), k = tile_desc(smem + kv.s * Y::TILES);
      const uint32_t idesc = Desc<T>::kk((min(BC, g.rows - cu.r0) + 15) & ~15), acc = tmem + gr.s * 128;
      if (leader) {
        mma_scores<DC>(acc, k, TILE, q, CT, idesc);
        mma_scores<DC>(acc + 64, k + DC * TILE / 16, TILE, q + DC * CT / 16, CT, idesc);
        umma::mma_commit(&sd_full[gr.s]);
        if (cu.last()) umma::mma_commit(&kv_empty[kv.s]);
      }
      __syncwarp();
      ch.next();
      gr.next();
      if (cu.next(sh, g)) kv.next();
    }
  } else if (warp == 2) {  // products
    const bool leader = umma::elect_one();
    Ring<Y::kN> ch;
    Ring<NB> gr, turn;
    uint32_t odd = 0;  // items so far, modulo 2
    for (KeyCursor cu(sh, g); cu.live && !abort_flag;) {
      const bool first = cu.first();
      if (!umma::mbar_wait(&ps_full[gr.s], gr.phase, 0xb6) || (first && !umma::mbar_wait(acc_empty, odd ^ 1, 0xb7))) {
        abort_flag = 1;
        break;
      }
      umma::tc_fence_after();
      const uint64_t q = tile_desc(smem + Y::OFF_CH + ch.s * Y::STAGE);
      const uint32_t acc = tmem + gr.s * 128;
      const int ksteps = (min(BC, g.rows - cu.r0) + 15) >> 4;
      if (leader) {
        mma_rows_ts<DC>(tmem + Y::kTmemDV, acc, q + DC * CT / 16, CT, Desc<T>::MN, ksteps, !first);
        mma_rows_ts<DC>(tmem + Y::kTmemDK, acc + 64, q, CT, Desc<T>::MN, ksteps, !first);
        if (cu.last()) umma::mma_commit(&acc_full[turn.s]);
        umma::mma_commit(&ps_done[gr.s]);
        umma::mma_commit(&ch_empty[ch.s]);
      }
      __syncwarp();
      ch.next();
      gr.next();
      if (cu.next(sh, g)) {
        turn.next();
        odd ^= 1;
      }
    }
  } else {
    const int grp = (warp - 3) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const float sl2 = sh.scale * kLog2e, mult = DROP ? drop.scale : 1.f;
    const uint64_t sl22 = pk2(sl2, sl2), mult2 = pk2(mult, mult);
    const Philox rng(DROP ? drop : DropArgs{});
    auto zeros = [&](const KeyCursor& c) {
      const int j = c.blk * BM + row;
      T* ok_ = dk + c.b * pdk.s_b + j * pdk.s_n + c.kh * pdk.s_h;
      T* ov = dv + c.b * pdv.s_b + j * pdv.s_n + c.kh * pdv.s_h;
      for (int d = 0; d < sh.dim; d += 8) {
        *reinterpret_cast<uint4*>(ok_ + d) = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(ov + d) = make_uint4(0, 0, 0, 0);
      }
    };
    // keys at or behind the length: zeros
    if (grp == 0 && sh.lengths != nullptr) {
      KeyCursor c(sh, g);
      for (c.item = blockIdx.x; c.item < g.total; c.item += gridDim.x) {
        c.at(sh, g);
        if (c.blk * BM + row >= c.len && c.blk * BM + row < sh.nk) zeros(c);
      }
    }
    KeyCursor cu(sh, g);
    Ring<Y::kN> ch;
    Ring<NB> gr;     // accumulators of the cursor's chunk
    Ring<NB> turn;   // of the items
    auto advance = [&](int k) {
      ch.next(k);
      gr.next(k);
      for (int i = cu.next(sh, g, k); i > 0; --i) turn.next();
    };
    if (grp == 1) advance(1);
    for (; cu.live && !abort_flag; advance(G)) {
      {
        const bool last = cu.last();
        const uint32_t acc = tmem + lane_off + gr.s * 128;
        const int j = cu.blk * BM + row, rows = min(BC, g.rows - cu.r0);
        const bool live = j < cu.len, idle = cu.blk * BM + quarter * 32 >= cu.len;
        // the statistics are read from the stage: wait for its TMA as well as for the products
        if (!umma::mbar_wait(&ch_full[ch.s], ch.phase, 0xb8) || !umma::mbar_wait(&sd_full[gr.s], gr.phase, 0xb9)) {
          abort_flag = 1;
          break;
        }
        umma::tc_fence_after();
        if (!idle) {
          const float* stats = reinterpret_cast<const float*>(smem + Y::OFF_CH + ch.s * Y::STAGE + Y::OFF_STAT);
#pragma unroll 1
          for (int c0 = 0; c0 < rows; c0 += 32) {
            uint32_t word = 0;  // keep bits of four columns x eight keys, drawn by this lane for its eight
            if (DROP) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int r = cu.r0 + c0 + (lane & 7) * 4 + e;
                const uint32_t bh = (uint32_t)(cu.b * sh.heads + (cu.u << g.gp_shift) + (r & gp_mask));
                word |= keep_bits(rng((uint32_t)j >> 3, (uint32_t)(r >> g.gp_shift), bh), drop.limit) << (8 * e);
              }
            }
            uint32_t pp[16], pd[16];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t su[16], du[16];
              tmem_ld16_nowait(acc + c0 + h * 16, su);
              tmem_ld16_nowait(acc + 64 + c0 + h * 16, du);
              tmem_wait16(su, du);
#pragma unroll
              for (int q4 = 0; q4 < 4; ++q4) {
                uint32_t bits = 0;
                if (DROP) bits = __shfl_sync(0xffffffffu, word, (lane & 24) + h * 4 + q4) >> (lane & 7);
                const float4 l4 = *reinterpret_cast<const float4*>(stats + c0 + h * 16 + 4 * q4);
                const float4 d4 = *reinterpret_cast<const float4*>(stats + BC + c0 + h * 16 + 4 * q4);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const int i = 4 * q4 + 2 * e;
                  // p = 2^(s - lse2), ds = p (dp - D); the statistics come negated
                  float p0, p1, d0 = __uint_as_float(du[i]), d1 = __uint_as_float(du[i + 1]);
                  unpk2(fma2(pk2(__uint_as_float(su[i]), __uint_as_float(su[i + 1])), sl22,
                             e ? pk2(l4.z, l4.w) : pk2(l4.x, l4.y)), p0, p1);
                  p0 = ex2(p0);
                  p1 = ex2(p1);
                  const uint64_t nd = e ? pk2(d4.z, d4.w) : pk2(d4.x, d4.y);
                  uint64_t x;
                  float q0 = p0, q1 = p1;
                  if (DROP) {
                    const bool k0 = bits & (1u << (16 * e)), k1 = bits & (1u << (16 * e + 8));
                    d0 = k0 ? d0 : 0.f;
                    d1 = k1 ? d1 : 0.f;
                    q0 = k0 ? p0 : 0.f;
                    q1 = k1 ? p1 : 0.f;
                    x = fma2(pk2(d0, d1), mult2, nd);
                  } else {
                    x = add2(pk2(d0, d1), nd);
                  }
                  unpk2(mul2(pk2(p0, p1), x), d0, d1);
                  pp[h * 8 + 2 * q4 + e] = pack2<T>(q0, q1);
                  pd[h * 8 + 2 * q4 + e] = pack2<T>(d0, d1);
                }
              }
            }
            if (c0 + 32 > rows) {  // queries behind the last: their statistics are someone else's, so zeros outright
              zero_tail(pp, rows - c0);
              zero_tail(pd, rows - c0);
            }
            umma::tmem_st16(acc + c0 / 2, pp);  // over accumulators this warp has read
            umma::tmem_st16(acc + 64 + c0 / 2, pd);
          }
          umma::tmem_wait_st();
        }
        warp_arrive(&ps_full[gr.s], false);
        if (last) {
          if (!umma::mbar_wait(&acc_full[turn.s], turn.phase, 0xbb)) {
            abort_flag = 1;
            break;
          }
          umma::tc_fence_after();
          T* out_k = dk + cu.b * pdk.s_b + j * pdk.s_n + cu.kh * pdk.s_h;
          T* out_v = dv + cu.b * pdv.s_b + j * pdv.s_n + cu.kh * pdv.s_h;
#pragma unroll 1
          for (int k = 0; k < 4 * DC; ++k) {
            const int d0 = (k >> 1) * 32;
            if (idle || d0 >= sh.dim) break;
            uint32_t a[32];
            tmem_ld32_nowait(tmem + lane_off + ((k & 1) ? Y::kTmemDK : Y::kTmemDV) + d0, a);
            wait_ld();
            tie32(a);
            if (live) store_row<T>((k & 1) ? out_k : out_v, d0, sh.dim, a, (k & 1) ? sh.scale : mult);
          }
          warp_arrive(acc_empty, false);
        }
      }
    }
  }
  umma::tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    umma::tc_fence_after();
    umma::tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------ host
int64_t round_up(int64_t n, int64_t m) { return (n + m - 1) / m * m; }

// Key ranges per row tile: the count with the least estimated time, in
// chunk times: waves of two CTAs per SM, each of its chunks and about two more
// for a tile's start and end, and, with more than one range, the partial rows'
// way out and back (about 5 GB a millisecond against 0.7 us per chunk) and the
// second launch.
int split_count(int64_t items, int nch, double elements) {
  if (items == 0) return 1;
  const int64_t slots = (int64_t)num_sms() * 2;
  int best = 1;
  double least = 0.;
  for (int s = 1; s <= kMaxSplits && (s == 1 || 2 * s <= nch); ++s) {
    const int64_t waves = (items * s + slots - 1) / slots;
    double t = (double)waves * ((nch + s - 1) / s + 2);
    if (s > 1) t += elements * s * 8 / 5e6 / 0.7 + 6.;
    if (s == 1 || t < least) {
      least = t;
      best = s;
    }
  }
  return best;
}

Divisor divisor(int64_t d) {
  uint32_t s = 0;
  while (((int64_t)1 << s) < d) ++s;
  return Divisor{(uint32_t)((((uint64_t)1 << (31 + s)) + (uint64_t)d - 1) / (uint64_t)d), 31 + s, (uint32_t)d};
}

// Rows and tiles of a shape; `splits` from the tile count alone, so that the
// workspace size, the forward and its join agree.
Geometry geometry(const Shape& sh) {
  Geometry g;
  const int group = sh.heads / sh.kv_heads;
  g.gp_shift = 0;
  while (g.gp_shift < 6 && group % (2 << g.gp_shift) == 0 && (int64_t)sh.nq << (g.gp_shift + 1) < (1 << 30))
    ++g.gp_shift;
  g.units = sh.heads >> g.gp_shift;
  g.kv_units = group >> g.gp_shift;
  g.rows = sh.nq << g.gp_shift;
  g.ldr = (int)round_up(g.rows, 4);
  g.nblk = (g.rows + BM - 1) / BM;
  const int nch = (sh.nk + fw::kMaxW - 1) / fw::kMaxW;
  g.width = (int)round_up((sh.nk + nch - 1) / nch, 16);
  g.splits = split_count((int64_t)sh.batch * g.units * g.nblk, nch, (double)sh.batch * g.units * g.rows * sh.dim);
  while ((int64_t)nch * g.splits >= ((int64_t)1 << 30)) --g.splits;
  g.total = 0;
  g.by_nblk = divisor(g.nblk);
  g.by_splits = divisor(g.splits);
  g.by_units = divisor(g.units);
  g.by_width = divisor(g.width);
  g.by_kv_units = divisor(g.kv_units);
  g.by_kblk = divisor((sh.nk + BM - 1) / BM);
  g.by_kv_heads = divisor(sh.kv_heads);
  return g;
}

int check_planes(const Shape& sh, const Plane* planes, const void* const* ptrs, const bool* query_side, int count,
                 const char* name) {
  for (int i = 0; i < count; ++i) {
    const Plane& p = planes[i];
    const int n = query_side[i] ? sh.nq : sh.nk, h = query_side[i] ? sh.heads : sh.kv_heads;
    const bool aligned = (reinterpret_cast<uintptr_t>(ptrs[i]) & 15) == 0 && (sh.batch == 1 || p.s_b % 8 == 0) &&
                         (n == 1 || p.s_n % 8 == 0) && (h == 1 || p.s_h % 8 == 0);
    if (!aligned) {
      set_error("%s: 16-bit planes with head dims in multiples of 8 must be 16-byte aligned, with strides that are "
                "multiples of 8", name);
      return PMB_ERR_ALIGNMENT;
    }
    PMB_REQUIRE((sh.batch == 1 || p.s_b > 0) && (n == 1 || p.s_n > 0) && (h == 1 || p.s_h > 0),
                "%s: strides must be positive", name);
  }
  return PMB_OK;
}

uint64_t stride_bytes(int64_t stride, int extent) { return extent > 1 ? (uint64_t)stride * 2 : 16; }

// Packed rows of a query-side plane: box of `rows` packed rows x 64 elements.
int query_map(CUtensorMap& map, const void* base, const Plane& p, const Shape& sh, const Geometry& g, int dtype,
              int rows, const char* name) {
  const int gp = 1 << g.gp_shift;
  const uint64_t dims[5] = {(uint64_t)sh.dim, (uint64_t)gp, (uint64_t)sh.nq, (uint64_t)g.units, (uint64_t)sh.batch};
  const uint64_t strides[4] = {stride_bytes(p.s_h, gp), stride_bytes(p.s_n, sh.nq),
                               stride_bytes(p.s_h * gp, g.units), stride_bytes(p.s_b, sh.batch)};
  const uint32_t box[5] = {64, (uint32_t)gp, (uint32_t)(rows / gp), 1, 1};
  return tma::make_map_5d(map, base, dtype, dims, strides, box, name);
}

int key_map(CUtensorMap& map, const void* base, const Plane& p, const Shape& sh, int dtype, int rows,
            const char* name) {
  const uint64_t dims[4] = {(uint64_t)sh.dim, (uint64_t)sh.nk, (uint64_t)sh.kv_heads, (uint64_t)sh.batch};
  const uint64_t strides[3] = {stride_bytes(p.s_n, sh.nk), stride_bytes(p.s_h, sh.kv_heads),
                               stride_bytes(p.s_b, sh.batch)};
  const uint32_t box[4] = {64, (uint32_t)rows, 1, 1};
  return tma::make_map_4d(map, base, dtype, dims, strides, box, name);
}

int persistent_grid(int64_t items, int per_sm) {
  const int64_t g = (int64_t)num_sms() * per_sm;
  return (int)(g < items ? g : items);
}

template <typename T, int DC, bool DROP>
int forward_launch(const Shape& sh, const Forward& a, Geometry g, const char* name) {
  CUtensorMap mq, mk, mv;
  if (int st = query_map(mq, a.q, a.pq, sh, g, a.dtype, BM, name)) return st;
  if (int st = key_map(mk, a.k, a.pk, sh, a.dtype, g.width, name)) return st;
  if (int st = key_map(mv, a.v, a.pv, sh, a.dtype, g.width, name)) return st;
  const int64_t rows = (int64_t)sh.batch * g.units * g.rows;
  float* part_lse = static_cast<float*>(a.workspace);
  float* part_o = part_lse + round_up(rows * g.splits, 64);
  auto kernel = xattn_fwd<T, DC, DROP>;
  constexpr int smem = fw::L<DC>::SMEM;
  PMB_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), name);
  kernel<<<persistent_grid(g.total, DC == 1 ? 2 : 1), fw::kThreads, smem, a.stream>>>(
      mq, mk, mv, static_cast<T*>(a.o), a.lse, part_o, part_lse, a.po, sh, g, a.drop);
  PMB_CHECK_LAUNCH(name);
  if (g.splits > 1) {
    const int64_t threads = rows * (sh.dim / 8);
    xattn_join<T><<<(unsigned)((threads + 255) / 256), 256, 0, a.stream>>>(part_o, part_lse, static_cast<T*>(a.o),
                                                                          a.lse, a.po, sh, g, threads);
    PMB_CHECK_LAUNCH(name);
  }
  return PMB_OK;
}

template <typename T, int DC, bool DROP>
int backward_launch(const Shape& sh, const Backward& a, Geometry g, const char* name) {
  CUtensorMap q128, do128, o128, q64, do64, k64, v64, k128, v128;
  if (int st = query_map(q128, a.q, a.pq, sh, g, a.dtype, BM, name)) return st;
  if (int st = query_map(do128, a.go, a.pgo, sh, g, a.dtype, BM, name)) return st;
  if (int st = query_map(o128, a.o, a.po, sh, g, a.dtype, BM, name)) return st;
  if (int st = query_map(q64, a.q, a.pq, sh, g, a.dtype, bw::BC, name)) return st;
  if (int st = query_map(do64, a.go, a.pgo, sh, g, a.dtype, bw::BC, name)) return st;
  if (int st = key_map(k64, a.k, a.pk, sh, a.dtype, bw::BC, name)) return st;
  if (int st = key_map(v64, a.v, a.pv, sh, a.dtype, bw::BC, name)) return st;
  if (int st = key_map(k128, a.k, a.pk, sh, a.dtype, BM, name)) return st;
  if (int st = key_map(v128, a.v, a.pv, sh, a.dtype, BM, name)) return st;
  float* delta = static_cast<float*>(a.workspace);
  {
    auto kernel = sh.nk <= bw::BC ? xattn_bwd_dq<T, DC, DROP, true> : xattn_bwd_dq<T, DC, DROP, false>;
    constexpr int smem = bq::L<DC>::SMEM;
    PMB_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), name);
    kernel<<<persistent_grid(g.total, 1), bq::kThreads, smem, a.stream>>>(
        q128, do128, o128, k64, v64, a.lse, delta, static_cast<T*>(a.gq), a.pgq, sh, g, a.drop);
    PMB_CHECK_LAUNCH(name);
  }
  const int kblk = (sh.nk + BM - 1) / BM;
  const int64_t items = (int64_t)sh.batch * sh.kv_heads * kblk;
  PMB_REQUIRE(items < ((int64_t)1 << 31), "%s: too many keys", name);
  g.total = (int)items;
  auto kernel = xattn_bwd_dkdv<T, DC, DROP>;
  constexpr int smem = bk::L<DC>::SMEM;
  PMB_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), name);
  kernel<<<persistent_grid(items, 1), bk::kThreads, smem, a.stream>>>(
      k128, v128, q64, do64, a.lse, delta, static_cast<T*>(a.gk), static_cast<T*>(a.gv), a.pgk, a.pgv, sh, g, a.drop);
  PMB_CHECK_LAUNCH(name);
  return PMB_OK;
}

template <typename T, int DC>
int forward_drop(const Shape& sh, const Forward& a, const Geometry& g, const char* name) {
  return a.threshold > 0 ? forward_launch<T, DC, true>(sh, a, g, name) : forward_launch<T, DC, false>(sh, a, g, name);
}
template <typename T, int DC>
int backward_drop(const Shape& sh, const Backward& a, const Geometry& g, const char* name) {
  return a.threshold > 0 ? backward_launch<T, DC, true>(sh, a, g, name) : backward_launch<T, DC, false>(sh, a, g, name);
}

int64_t forward_bytes(const Shape& sh, const Geometry& g) {
  if (g.splits <= 1) return 0;
  const int64_t rows = (int64_t)sh.batch * g.units * g.rows * g.splits;
  return round_up(round_up(rows, 64) * 4 + rows * sh.dim * 4, 256);
}

int count_items(const Shape& sh, Geometry& g, const char* name) {
  const int64_t items = (int64_t)sh.batch * g.units * g.nblk * g.splits;
  PMB_REQUIRE(items < ((int64_t)1 << 31), "%s: too many rows", name);
  g.total = (int)items;
  return PMB_OK;
}

}  // namespace

int64_t tc_lse_floats(int64_t heads_total, int64_t nq) { return heads_total * round_up(nq, 4) + 64; }

int64_t tc_forward_workspace(const Shape& sh) { return forward_bytes(sh, geometry(sh)); }

int64_t tc_backward_workspace(const Shape& sh) {
  return round_up(tc_lse_floats((int64_t)sh.batch * sh.heads, sh.nq) * 4, 256);
}

int tc_forward(const Shape& sh, const Forward& a, const char* name) {
  Geometry g = geometry(sh);
  if (int st = count_items(sh, g, name)) return st;
  const Plane planes[4] = {a.pq, a.pk, a.pv, a.po};
  const void* ptrs[4] = {a.q, a.k, a.v, a.o};
  const bool side[4] = {true, false, false, true};
  if (int st = check_planes(sh, planes, ptrs, side, 4, name)) return st;
  const int64_t need = forward_bytes(sh, g);
  if (need > 0 && (a.workspace == nullptr || a.workspace_bytes < need ||
                   (reinterpret_cast<uintptr_t>(a.workspace) & 15))) {
    set_error("%s: needs a 16-byte aligned workspace of %lld bytes (got %lld)", name, (long long)need,
              (long long)a.workspace_bytes);
    return PMB_ERR_WORKSPACE;
  }
  if (a.dtype == PMB_BFLOAT16)
    return sh.dim <= 64 ? forward_drop<__nv_bfloat16, 1>(sh, a, g, name) : forward_drop<__nv_bfloat16, 2>(sh, a, g, name);
  return sh.dim <= 64 ? forward_drop<__half, 1>(sh, a, g, name) : forward_drop<__half, 2>(sh, a, g, name);
}

int tc_backward(const Shape& sh, const Backward& a, const char* name) {
  Geometry g = geometry(sh);
  g.splits = 1;
  g.by_splits = divisor(1);
  if (int st = count_items(sh, g, name)) return st;
  const Plane planes[8] = {a.pq, a.pk, a.pv, a.po, a.pgo, a.pgq, a.pgk, a.pgv};
  const void* ptrs[8] = {a.q, a.k, a.v, a.o, a.go, a.gq, a.gk, a.gv};
  const bool side[8] = {true, false, false, true, true, true, false, false};
  if (int st = check_planes(sh, planes, ptrs, side, 8, name)) return st;
  if ((reinterpret_cast<uintptr_t>(a.lse) | reinterpret_cast<uintptr_t>(a.workspace)) & 15) {
    set_error("%s: lse and workspace must be 16-byte aligned", name);
    return PMB_ERR_ALIGNMENT;
  }
  if (a.dtype == PMB_BFLOAT16)
    return sh.dim <= 64 ? backward_drop<__nv_bfloat16, 1>(sh, a, g, name)
                        : backward_drop<__nv_bfloat16, 2>(sh, a, g, name);
  return sh.dim <= 64 ? backward_drop<__half, 1>(sh, a, g, name) : backward_drop<__half, 2>(sh, a, g, name);
}

}  // namespace xattn
}  // namespace pmb
