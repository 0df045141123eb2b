// Attention of nq queries over nk keys of another length, with key counts per
// batch item, key / value heads shared by groups of query heads, and dropout
// on the probabilities from counter-based bits (philox.cuh):
//
//   P = softmax_rows(scale Q K^T over keys < len),  Pd = keep c P,  O = Pd V
//   D = rowsum(P dP) (= rowsum(dO * O), the form for more than one tile of keys),  dP = keep c (dO V^T),
//   dS = P (dP - D),  dV = Pd^T dO,  dQ = scale dS K,  dK = scale dS^T Q
//
// dK and dV sum over the query heads of a group.  A row without keys, or with
// scores of -infinity alone, has O = 0, P = 0 (its lse is stored so that the
// backward's exponentials are zeros: +inf in the row form) and no gradient;
// keys at or behind `len` are never read, and their gradients are zeros.
//
// The C entries, and the row form, all arithmetic fp32: it serves fp32 and
// head dims the tensor-core form (cross_attention_tc.cu) does not take.  A
// warp owns eight rows (queries in the forward and for dQ, keys for dK / dV);
// tiles of 32 rows of the other side come through shared memory for the four
// warps of a CTA.  For the dot products a lane takes one row of the tile and
// multiplies it with the eight owned rows, which all lanes read alike; for the
// sums a lane takes every 32nd head element.  Nearest limit: shared-memory
// reads (9 of 16 bytes for 32 fused multiply-adds; ncu: 59 to 67 % of the
// wavefronts, 0.59 to 0.68 of the issue slots, at three to four CTAs an SM).  Measured
// for 62 x 8 heads x 258 x 258, dim 64, fp32 with dropout: forward 0.58, dQ
// 0.87, dK / dV 0.92 ms, where a warp to one row without tiles took 10.7, 16.2
// and 17.0 ms.  Every output row is summed by one warp in the order of the
// tiles, so results do not depend on the order of execution.
#include <type_traits>

#include "cross_attention.cuh"

namespace pmb {
namespace {

using xattn::Plane;
using xattn::Shape;

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kOwn = 8;                 // rows of a warp
constexpr int kTile = 32;               // streamed rows
constexpr int kRows = kWarps * kOwn;    // owned rows of a CTA
constexpr int kMaxDim = 256;

__host__ __device__ inline int pitch_of(int dim) { return (dim + 3) / 4 * 4 + 4; }  // floats; rows start 16-byte aligned
__host__ __device__ inline int own_pitch_of(int dim) { return (dim + 3) / 4 * 4; }

// Shared memory: two streamed tiles, two owned row sets, the warps' weights [2][32][8].
inline int shared_bytes(int dim) {
  return (2 * kTile * pitch_of(dim) + 2 * kRows * own_pitch_of(dim) + kWarps * 2 * kTile * kOwn) * 4;
}

struct Shared {
  float *ta, *tb, *oa, *ob, *w;
  __device__ __forceinline__ Shared(float* base, int dim) {
    ta = base;
    tb = ta + kTile * pitch_of(dim);
    oa = tb + kTile * pitch_of(dim);
    ob = oa + kRows * own_pitch_of(dim);
    w = ob + kRows * own_pitch_of(dim);
  }
};

// The first `count` of 32 rows of a plane (zeros for the rest and for the rows' padding), times mul, into shared
// memory.  A warp takes eight rows whose loads are issued together: one row after the other, the forward of 62 x 8
// heads x 258 x 258, dim 64, with dropout took 1.21 ms, like this 0.58 ms.
template <typename T>
__device__ __forceinline__ void stage(float* dst, int pitch, const T* __restrict__ src, int64_t s_n, int count,
                                      int dim, float mul) {
  static_assert(kTile == kRows && kTile % kWarps == 0);
  const int width = own_pitch_of(dim), warp = threadIdx.x >> 5;
  for (int c = threadIdx.x & 31; c < width; c += 32) {
    float x[kTile / kWarps];
#pragma unroll
    for (int i = 0; i < kTile / kWarps; ++i) {
      const int r = warp + i * kWarps;
      x[i] = r < count && c < dim ? Elem<T>::to_f(src[r * s_n + c]) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < kTile / kWarps; ++i) dst[(warp + i * kWarps) * pitch + c] = x[i] * mul;
  }
}

// s[i] = sum_c own[i][c] tile[lane][c]
__device__ __forceinline__ void dots(float (&s)[kOwn], const float* own, int own_pitch, const float* tile, int pitch,
                                     int dim) {
#pragma unroll
  for (int i = 0; i < kOwn; ++i) s[i] = 0.f;
  const float* mine = tile + (threadIdx.x & 31) * pitch;
  for (int c = 0; c < dim; c += 4) {
    const float4 x = *reinterpret_cast<const float4*>(mine + c);
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const float4 y = *reinterpret_cast<const float4*>(own + i * own_pitch + c);
      s[i] = fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, s[i]))));
    }
  }
}

// acc[i][a] += sum_t w[t][i] tile[t][lane + 32 a]
template <int NA>
__device__ __forceinline__ void sums(float (&acc)[kOwn][NA], const float* w, const float* tile, int pitch, int dim,
                                     int count) {
  const int lane = threadIdx.x & 31;
  for (int t = 0; t < count; ++t) {
    const float4 p0 = *reinterpret_cast<const float4*>(w + t * kOwn);
    const float4 p1 = *reinterpret_cast<const float4*>(w + t * kOwn + 4);
    const float p[kOwn] = {p0.x, p0.y, p0.z, p0.w, p1.x, p1.y, p1.z, p1.w};
#pragma unroll
    for (int a = 0; a < NA; ++a) {
      const float x = lane + 32 * a < dim ? tile[t * pitch + lane + 32 * a] : 0.f;
#pragma unroll
      for (int i = 0; i < kOwn; ++i) acc[i][a] = fmaf(p[i], x, acc[i][a]);
    }
  }
}

// the lane's eight weights, one row of [32][8]
__device__ __forceinline__ void put_weights(float* w, const float (&p)[kOwn]) {
  float* mine = w + (threadIdx.x & 31) * kOwn;
  *reinterpret_cast<float4*>(mine) = make_float4(p[0], p[1], p[2], p[3]);
  *reinterpret_cast<float4*>(mine + 4) = make_float4(p[4], p[5], p[6], p[7]);
}

// Keep bits of a tile of 32 keys (j0 a multiple of eight) and the warp's eight queries from i0 on: one Philox call
// covers eight keys of one query, so lane l draws keys j0 + 8 (l / 8).. of query i0 + l % 8 and `kept_key` hands them out.
__device__ __forceinline__ uint32_t draw(const Philox& rng, uint32_t limit, int j0, int i0, int bh) {
  const int lane = threadIdx.x & 31;
  return keep_bits(rng((uint32_t)(j0 >> 3) + (lane >> 3), (uint32_t)(i0 + (lane & 7)), (uint32_t)bh), limit);
}

// the bit of the lane's key and query i0 + i; the whole warp calls it
__device__ __forceinline__ bool kept_key(uint32_t bits, int i) {
  const int lane = threadIdx.x & 31;
  return (__shfl_sync(0xffffffffu, bits, (lane & 24) | i) >> (lane & 7)) & 1u;
}

// Grid: (tiles of kRows queries) x batch x heads.
template <typename T, bool DROP, int NA>
__global__ void __launch_bounds__(kThreads)
    attn_rows_fwd(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, T* __restrict__ o,
                  float* __restrict__ lse, Plane pq, Plane pk, Plane pv, Plane po, Shape sh, int blocks,
                  DropArgs drop) {
  extern __shared__ float4 smem4[];
  const Shared m_(reinterpret_cast<float*>(smem4), sh.dim);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, pitch = pitch_of(sh.dim), own = own_pitch_of(sh.dim);
  const int bh = blockIdx.x / blocks, i0 = (blockIdx.x - bh * blocks) * kRows, h = bh % sh.heads, b = bh / sh.heads;
  const int kh = h / (sh.heads / sh.kv_heads), len = sh.keys(b);
  const Philox rng(DROP ? drop : DropArgs{});
  stage(m_.oa, own, q + b * pq.s_b + i0 * pq.s_n + h * pq.s_h, pq.s_n, sh.nq - i0, sh.dim, sh.scale);
  k += b * pk.s_b + kh * pk.s_h;
  v += b * pv.s_b + kh * pv.s_h;
  float m[kOwn], l[kOwn], acc[kOwn][NA] = {};
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
  }
  float* w = m_.w + warp * 2 * kTile * kOwn;
  for (int j0 = 0; j0 < len; j0 += kTile) {
    const int count = len - j0 < kTile ? len - j0 : kTile;
    __syncthreads();
    stage(m_.ta, pitch, k + j0 * pk.s_n, pk.s_n, count, sh.dim, 1.f);
    stage(m_.tb, pitch, v + j0 * pv.s_n, pv.s_n, count, sh.dim, 1.f);
    __syncthreads();
    float p[kOwn];
    dots(p, m_.oa + warp * kOwn * own, own, m_.ta, pitch, sh.dim);
    const uint32_t bits = DROP ? draw(rng, drop.limit, j0, i0 + warp * kOwn, bh) : 0u;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      float mx = lane < count ? p[i] : -INFINITY;
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      const float mn = fmaxf(fmaxf(m[i], mx), xattn::kLowest), corr = expf(m[i] - mn);
      p[i] = lane < count ? expf(p[i] - mn) : 0.f;
      l[i] = l[i] * corr + warp_sum(p[i]);
      m[i] = mn;
#pragma unroll
      for (int a = 0; a < NA; ++a) acc[i][a] *= corr;
      if (DROP) p[i] = kept_key(bits, i) ? p[i] * drop.scale : 0.f;
    }
    put_weights(w, p);
    __syncwarp();
    sums<NA>(acc, w, m_.tb, pitch, sh.dim, count);
    __syncwarp();
  }
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    const int r = i0 + warp * kOwn + i;
    if (r >= sh.nq) break;
    T* out = o + b * po.s_b + r * po.s_n + h * po.s_h;
    // no keys, or scores of -infinity alone: zeros.  (A sum without keys is 0 too; with the length in the test the
    // compiler stays at 128 registers and four CTAs an SM, without it at 139 and three: 0.58 against 0.67 ms.)
    const bool some = len > 0 && l[i] != 0.f;
    const float inv = some ? 1.f / l[i] : 0.f;
#pragma unroll
    for (int a = 0; a < NA; ++a)
      if (lane + 32 * a < sh.dim) out[lane + 32 * a] = Elem<T>::from_f(acc[i][a] * inv);
    if (lane == 0) lse[(int64_t)bh * sh.nq + r] = some ? m[i] + logf(l[i]) : INFINITY;
  }
}

// ONE: at most one tile of keys, D = rowsum(P dP) from it; O's rounding, which few keys do not average out, stays away.
template <typename T, bool DROP, int NA, bool ONE>
__global__ void __launch_bounds__(kThreads)
    attn_rows_dq(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, const T* __restrict__ o,
                 const T* __restrict__ go, const float* __restrict__ lse, T* __restrict__ gq,
                 float* __restrict__ delta, Plane pq, Plane pk, Plane pv, Plane po, Plane pgo, Plane pgq, Shape sh,
                 int blocks, DropArgs drop) {
  extern __shared__ float4 smem4[];
  const Shared m_(reinterpret_cast<float*>(smem4), sh.dim);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, pitch = pitch_of(sh.dim), own = own_pitch_of(sh.dim);
  const int bh = blockIdx.x / blocks, i0 = (blockIdx.x - bh * blocks) * kRows, h = bh % sh.heads, b = bh / sh.heads;
  const int kh = h / (sh.heads / sh.kv_heads), len = sh.keys(b);
  const Philox rng(DROP ? drop : DropArgs{});
  stage(m_.oa, own, q + b * pq.s_b + i0 * pq.s_n + h * pq.s_h, pq.s_n, sh.nq - i0, sh.dim, sh.scale);
  stage(m_.ob, own, go + b * pgo.s_b + i0 * pgo.s_n + h * pgo.s_h, pgo.s_n, sh.nq - i0, sh.dim, 1.f);
  __syncthreads();
  float d[kOwn], ls[kOwn];
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    const int r = i0 + warp * kOwn + i;
    float x = 0.f;
    if (!ONE && r < sh.nq) {
      const T* orow = o + b * po.s_b + r * po.s_n + h * po.s_h;
      for (int c = lane; c < sh.dim; c += 32)
        x = fmaf(m_.ob[(warp * kOwn + i) * own + c], Elem<T>::to_f(orow[c]), x);
    }
    d[i] = ONE ? 0.f : warp_sum(x);
    ls[i] = r < sh.nq ? lse[(int64_t)bh * sh.nq + r] : 0.f;
    if (!ONE && r < sh.nq && lane == 0) delta[(int64_t)bh * sh.nq + r] = d[i];
  }
  k += b * pk.s_b + kh * pk.s_h;
  v += b * pv.s_b + kh * pv.s_h;
  float acc[kOwn][NA] = {};
  float* w = m_.w + warp * 2 * kTile * kOwn;
  for (int j0 = 0; j0 < len; j0 += kTile) {
    const int count = len - j0 < kTile ? len - j0 : kTile;
    __syncthreads();
    stage(m_.ta, pitch, k + j0 * pk.s_n, pk.s_n, count, sh.dim, 1.f);
    stage(m_.tb, pitch, v + j0 * pv.s_n, pv.s_n, count, sh.dim, 1.f);
    __syncthreads();
    float p[kOwn], dp[kOwn];
    dots(p, m_.oa + warp * kOwn * own, own, m_.ta, pitch, sh.dim);
    dots(dp, m_.ob + warp * kOwn * own, own, m_.tb, pitch, sh.dim);
    const uint32_t bits = DROP ? draw(rng, drop.limit, j0, i0 + warp * kOwn, bh) : 0u;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      if (DROP) dp[i] = kept_key(bits, i) ? dp[i] * drop.scale : 0.f;
      if constexpr (ONE) {
        const float e = lane < count ? expf(p[i] - ls[i]) : 0.f;
        d[i] = warp_sum(lane < count ? e * dp[i] : 0.f);
        p[i] = lane < count ? e * (dp[i] - d[i]) : 0.f;
      } else {
        p[i] = lane < count ? expf(p[i] - ls[i]) * (dp[i] - d[i]) : 0.f;
      }
    }
    put_weights(w, p);
    __syncwarp();
    sums<NA>(acc, w, m_.ta, pitch, sh.dim, count);
    __syncwarp();
  }
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    const int r = i0 + warp * kOwn + i;
    if (r >= sh.nq) break;
    T* out = gq + b * pgq.s_b + r * pgq.s_n + h * pgq.s_h;
#pragma unroll
    for (int a = 0; a < NA; ++a)
      if (lane + 32 * a < sh.dim) out[lane + 32 * a] = Elem<T>::from_f(acc[i][a] * sh.scale);
    if (ONE && lane == 0) delta[(int64_t)bh * sh.nq + r] = d[i];
  }
}

// Grid: (tiles of kRows keys) x batch x key / value heads.
template <typename T, bool DROP, int NA>
__global__ void __launch_bounds__(kThreads)
    attn_rows_dkdv(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, const T* __restrict__ go,
                   const float* __restrict__ lse, const float* __restrict__ delta, T* __restrict__ gk,
                   T* __restrict__ gv, Plane pq, Plane pk, Plane pv, Plane pgo, Plane pgk, Plane pgv, Shape sh,
                   int blocks, DropArgs drop) {
  extern __shared__ float4 smem4[];
  const Shared m_(reinterpret_cast<float*>(smem4), sh.dim);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, pitch = pitch_of(sh.dim), own = own_pitch_of(sh.dim);
  const int bk = blockIdx.x / blocks, j0 = (blockIdx.x - bk * blocks) * kRows, kh = bk % sh.kv_heads, b = bk / sh.kv_heads;
  const int group = sh.heads / sh.kv_heads, len = sh.keys(b), live = len - j0 < 0 ? 0 : len - j0;
  const Philox rng(DROP ? drop : DropArgs{});
  float ak[kOwn][NA] = {}, av[kOwn][NA] = {};
  if (live > 0) {
    stage(m_.oa, own, k + b * pk.s_b + j0 * pk.s_n + kh * pk.s_h, pk.s_n, live, sh.dim, sh.scale);
    stage(m_.ob, own, v + b * pv.s_b + j0 * pv.s_n + kh * pv.s_h, pv.s_n, live, sh.dim, 1.f);
    float* w = m_.w + warp * 2 * kTile * kOwn;
    for (int h = kh * group; h < (kh + 1) * group; ++h) {
      const int bh = b * sh.heads + h;
      for (int i0 = 0; i0 < sh.nq; i0 += kTile) {
        const int count = sh.nq - i0 < kTile ? sh.nq - i0 : kTile, i = i0 + lane;
        __syncthreads();
        stage(m_.ta, pitch, q + b * pq.s_b + i0 * pq.s_n + h * pq.s_h, pq.s_n, count, sh.dim, 1.f);
        stage(m_.tb, pitch, go + b * pgo.s_b + i0 * pgo.s_n + h * pgo.s_h, pgo.s_n, count, sh.dim, 1.f);
        __syncthreads();
        const float ls = lane < count ? lse[(int64_t)bh * sh.nq + i] : 0.f;
        const float d = lane < count ? delta[(int64_t)bh * sh.nq + i] : 0.f;
        float p[kOwn], ds[kOwn];
        dots(p, m_.oa + warp * kOwn * own, own, m_.ta, pitch, sh.dim);
        dots(ds, m_.ob + warp * kOwn * own, own, m_.tb, pitch, sh.dim);
        // the eight keys of a warp are one group of the random bits: j0 and kOwn are multiples of eight
        uint32_t keep = 0xffu;
        if (DROP && lane < count)
          keep = keep_bits(rng((uint32_t)(j0 + warp * kOwn) >> 3, (uint32_t)i, (uint32_t)bh), drop.limit);
        const float mult = DROP ? drop.scale : 1.f;
#pragma unroll
        for (int r = 0; r < kOwn; ++r) {
          const bool on = (keep >> r) & 1u;
          const float e = lane < count ? expf(p[r] - ls) : 0.f;
          ds[r] = lane < count ? e * ((on ? ds[r] * mult : 0.f) - d) : 0.f;
          p[r] = on ? e * mult : 0.f;
        }
        put_weights(w, p);
        put_weights(w + kTile * kOwn, ds);
        __syncwarp();
        sums<NA>(av, w, m_.tb, pitch, sh.dim, count);
        sums<NA>(ak, w + kTile * kOwn, m_.ta, pitch, sh.dim, count);
        __syncwarp();
      }
    }
  }
#pragma unroll
  for (int r = 0; r < kOwn; ++r) {
    const int j = j0 + warp * kOwn + r;
    if (j >= sh.nk) break;
    const bool on = j < len;
    T* ok = gk + b * pgk.s_b + j * pgk.s_n + kh * pgk.s_h;
    T* ov = gv + b * pgv.s_b + j * pgv.s_n + kh * pgv.s_h;
#pragma unroll
    for (int a = 0; a < NA; ++a) {
      if (lane + 32 * a >= sh.dim) break;
      ok[lane + 32 * a] = Elem<T>::from_f(on ? ak[r][a] * sh.scale : 0.f);
      ov[lane + 32 * a] = Elem<T>::from_f(on ? av[r][a] : 0.f);
    }
  }
}

// ------------------------------------------------------------------ host
Plane plane_at(const int64_t* s, int i) { return Plane{s[3 * i], s[3 * i + 1], s[3 * i + 2]}; }

// Sizes that the kernels' 32-bit indices hold; products of them are formed only behind this.
bool indexable(int64_t batch, int64_t heads, int64_t nq, int64_t nk) {
  constexpr int64_t kMax = 1 << 30;
  return batch < kMax && heads < kMax && nq < kMax && nk < kMax && batch * heads < kMax;
}

int make_shape(Shape& sh, int64_t batch, int64_t heads, int64_t kv_heads, int64_t nq, int64_t nk, int64_t dim,
               const int32_t* lengths, float scale, int threshold, const int64_t* key, const char* name) {
  PMB_REQUIRE(batch >= 0 && nq >= 0 && nk >= 0 && heads > 0 && kv_heads > 0, "%s: bad shape", name);
  PMB_REQUIRE(heads % kv_heads == 0, "%s: %lld heads are not a multiple of %lld key / value heads", name,
              (long long)heads, (long long)kv_heads);
  PMB_REQUIRE(dim > 0 && dim <= kMaxDim, "%s: head dim %lld outside [1, %d]", name, (long long)dim, kMaxDim);
  PMB_REQUIRE(indexable(batch, heads, nq, nk), "%s: too large", name);
  PMB_REQUIRE(threshold >= 0 && threshold <= 65536, "%s: drop threshold %d outside [0, 65536]", name, threshold);
  PMB_REQUIRE(key || threshold == 0, "%s: NULL key", name);
  sh = Shape{(int)batch, (int)heads, (int)kv_heads, (int)nq, (int)nk, (int)dim, lengths, scale};
  return PMB_OK;
}

// CTAs of `sets` (batch, head) pairs of `rows` rows each, `blocks` per pair.
int row_grid(int64_t sets, int64_t rows, unsigned& grid, int& blocks, const char* name) {
  const int64_t n = (rows + kRows - 1) / kRows;
  PMB_REQUIRE(n * sets < ((int64_t)1 << 31), "%s: too many rows", name);
  blocks = (int)n;
  grid = (unsigned)(n * sets);
  return PMB_OK;
}

// Launch one of the row kernels with the shared memory the head dim needs.
template <typename... P, typename... A>
int launch_rows(void (*kernel)(P...), unsigned grid, int dim, cudaStream_t s, const char* name, A... args) {
  const int bytes = shared_bytes(dim);
  PMB_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), name);
  kernel<<<grid, kThreads, bytes, s>>>(args...);
  PMB_CHECK_LAUNCH(name);
  return PMB_OK;
}

int64_t delta_bytes(int64_t rows) { return (rows * 4 + 255) / 256 * 256; }

}  // namespace
}  // namespace pmb

using namespace pmb;

extern "C" int64_t pmb_cross_attention_lse_size(int64_t batch, int64_t heads, int64_t nq) {
  return batch > 0 && heads > 0 && nq > 0 && indexable(batch, heads, nq, 0) ? xattn::tc_lse_floats(batch * heads, nq)
                                                                            : 0;
}

namespace pmb {
namespace {
// Shape of a workspace query; false where the sizes make no call.
bool query_shape(Shape& sh, int64_t batch, int64_t heads, int64_t kv_heads, int64_t nq, int64_t nk, int64_t dim) {
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || nq <= 0 || nk < 0 || dim <= 0 || dim > kMaxDim ||
      !indexable(batch, heads, nq, nk))
    return false;
  sh = Shape{(int)batch, (int)heads, (int)kv_heads, (int)nq, (int)nk, (int)dim, nullptr, 1.f};
  return true;
}
}  // namespace
}  // namespace pmb

extern "C" int64_t pmb_cross_attention_forward_workspace_size(int64_t batch, int64_t heads, int64_t kv_heads,
                                                              int64_t nq, int64_t nk, int64_t dim, int dtype) {
  Shape sh;
  if (!query_shape(sh, batch, heads, kv_heads, nq, nk, dim) || !xattn::tc_takes(sh, dtype)) return 0;
  return xattn::tc_forward_workspace(sh);
}

extern "C" int pmb_cross_attention_forward(const void* q, const void* k, const void* v, void* o, float* lse,
                                           const int32_t* key_lengths, int64_t batch, int64_t heads, int64_t kv_heads,
                                           int64_t nq, int64_t nk, int64_t dim, const int64_t* strides, float scale,
                                           int threshold, const int64_t* key, uint32_t site, int dtype,
                                           void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  const char* name = "pmb_cross_attention_forward";
  Shape sh;
  if (int st = make_shape(sh, batch, heads, kv_heads, nq, nk, dim, key_lengths, scale, threshold, key, name)) return st;
  const int64_t rows = batch * heads * nq;
  if (rows == 0) return PMB_OK;
  PMB_REQUIRE(q && o && lse && strides && ((k && v) || nk == 0), "%s: NULL argument", name);
  const DropArgs drop = drop_args(key, site, threshold);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const Plane pq = plane_at(strides, 0), pk = plane_at(strides, 1), pv = plane_at(strides, 2),
              po = plane_at(strides, 3);
  if (xattn::tc_takes(sh, dtype))
    return xattn::tc_forward(sh,
                             xattn::Forward{q, k, v, o, lse, pq, pk, pv, po, dtype, threshold, drop, workspace,
                                            workspace_bytes, s},
                             name);
  unsigned grid;
  int blocks;
  if (int st = row_grid(batch * heads, nq, grid, blocks, name)) return st;
  return PMB_DISPATCH(dtype, T, name, [&] {
    auto run = [&](auto kernel) {
      return launch_rows(kernel, grid, sh.dim, s, name, static_cast<const T*>(q), static_cast<const T*>(k),
                         static_cast<const T*>(v), static_cast<T*>(o), lse, pq, pk, pv, po, sh, blocks, drop);
    };
    if (dim <= 64) return threshold > 0 ? run(attn_rows_fwd<T, true, 2>) : run(attn_rows_fwd<T, false, 2>);
    return threshold > 0 ? run(attn_rows_fwd<T, true, 8>) : run(attn_rows_fwd<T, false, 8>);
  });
}

extern "C" int64_t pmb_cross_attention_backward_workspace_size(int64_t batch, int64_t heads, int64_t kv_heads,
                                                               int64_t nq, int64_t nk, int64_t dim, int dtype) {
  Shape sh;
  if (!query_shape(sh, batch, heads, kv_heads, nq, nk, dim)) return 0;
  return xattn::tc_takes(sh, dtype) ? xattn::tc_backward_workspace(sh) : delta_bytes(batch * heads * nq);
}

extern "C" int pmb_cross_attention_backward(const void* q, const void* k, const void* v, const void* o,
                                            const void* grad_out, const float* lse, void* grad_q, void* grad_k,
                                            void* grad_v, const int32_t* key_lengths, int64_t batch, int64_t heads,
                                            int64_t kv_heads, int64_t nq, int64_t nk, int64_t dim,
                                            const int64_t* strides, float scale, int threshold, const int64_t* key,
                                            uint32_t site, int dtype, void* workspace, int64_t workspace_bytes,
                                            void* stream) {
  clear_error();
  const char* name = "pmb_cross_attention_backward";
  Shape sh;
  if (int st = make_shape(sh, batch, heads, kv_heads, nq, nk, dim, key_lengths, scale, threshold, key, name)) return st;
  const int64_t rows = batch * heads * nq, keys = batch * kv_heads * nk;
  if (rows == 0 && keys == 0) return PMB_OK;
  PMB_REQUIRE(strides, "%s: NULL strides", name);
  PMB_REQUIRE(rows == 0 || (q && o && grad_out && lse && grad_q), "%s: NULL query-side argument", name);
  PMB_REQUIRE(keys == 0 || (k && v && grad_k && grad_v), "%s: NULL key-side argument", name);
  const int64_t need = pmb_cross_attention_backward_workspace_size(batch, heads, kv_heads, nq, nk, dim, dtype);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) {
    set_error("%s: workspace of %lld bytes is smaller than the %lld required", name, (long long)workspace_bytes,
              (long long)need);
    return PMB_ERR_WORKSPACE;
  }
  const Plane pq = plane_at(strides, 0), pk = plane_at(strides, 1), pv = plane_at(strides, 2),
              po = plane_at(strides, 3), pgo = plane_at(strides, 4), pgq = plane_at(strides, 5),
              pgk = plane_at(strides, 6), pgv = plane_at(strides, 7);
  const DropArgs drop = drop_args(key, site, threshold);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (xattn::tc_takes(sh, dtype))
    return xattn::tc_backward(sh,
                              xattn::Backward{q, k, v, o, grad_out, lse, grad_q, grad_k, grad_v, pq, pk, pv, po, pgo,
                                              pgq, pgk, pgv, dtype, threshold, drop, workspace, workspace_bytes, s},
                              name);
  float* delta = static_cast<float*>(workspace);
  unsigned qgrid, kgrid;
  int qblocks, kblocks;
  if (int st = row_grid(batch * heads, nq, qgrid, qblocks, name)) return st;
  if (int st = row_grid(batch * kv_heads, nk, kgrid, kblocks, name)) return st;
  return PMB_DISPATCH(dtype, T, name, [&] {
    auto run_q = [&](auto kernel) {
      return launch_rows(kernel, qgrid, sh.dim, s, name, static_cast<const T*>(q), static_cast<const T*>(k),
                         static_cast<const T*>(v), static_cast<const T*>(o), static_cast<const T*>(grad_out), lse,
                         static_cast<T*>(grad_q), delta, pq, pk, pv, po, pgo, pgq, sh, qblocks, drop);
    };
    auto run_k = [&](auto kernel) {
      return launch_rows(kernel, kgrid, sh.dim, s, name, static_cast<const T*>(q), static_cast<const T*>(k),
                         static_cast<const T*>(v), static_cast<const T*>(grad_out), lse, (const float*)delta,
                         static_cast<T*>(grad_k), static_cast<T*>(grad_v), pq, pk, pv, pgo, pgk, pgv, sh, kblocks, drop);
    };
    if (rows > 0) {
      auto pick = [&](auto one) {
        constexpr bool ONE = decltype(one)::value;
        return dim <= 64 ? (threshold > 0 ? run_q(attn_rows_dq<T, true, 2, ONE>) : run_q(attn_rows_dq<T, false, 2, ONE>))
                         : (threshold > 0 ? run_q(attn_rows_dq<T, true, 8, ONE>) : run_q(attn_rows_dq<T, false, 8, ONE>));
      };
      if (const int st = nk <= kTile ? pick(std::true_type{}) : pick(std::false_type{})) return st;
    }
    if (keys == 0) return PMB_OK;
    return dim <= 64 ? (threshold > 0 ? run_k(attn_rows_dkdv<T, true, 2>) : run_k(attn_rows_dkdv<T, false, 2>))
                     : (threshold > 0 ? run_k(attn_rows_dkdv<T, true, 8>) : run_k(attn_rows_dkdv<T, false, 8>));
  });
}
