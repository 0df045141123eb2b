// Attention of nq queries over nk keys of another length, with key counts per
// batch item, key / value heads shared by groups of query heads, and dropout
// on the probabilities from counter-based bits (philox.cuh):
//
//   P = softmax_rows(scale Q K^T over keys < len),  Pd = keep c P,  O = Pd V
//   D = rowsum(dO * O) (= rowsum(P dP)),  dP = keep c (dO V^T),
//   dS = P (dP - D),  dV = Pd^T dO,  dQ = scale dS K,  dK = scale dS^T Q
//
// dK and dV sum over the query heads of a group.  A row without keys has
// O = 0, lse = -inf and no gradient; keys at or behind `len` are never read,
// and their gradients are zeros.
//
// The C entries, and the row form: one warp per query row (forward, dQ) or
// key row (dK / dV), all arithmetic fp32; every output row is written by one
// warp, so results do not depend on the order of execution.  It serves fp32
// and head dims the tensor-core form (cross_attention_tc.cu) does not take.
#include "cross_attention.cuh"

namespace pmb {
namespace {

using xattn::Plane;
using xattn::Shape;

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxDim = 256;
constexpr int kAcc = kMaxDim / 32;

// sum_c a[c] * row[c] with a in shared memory
template <typename T>
__device__ __forceinline__ float dot(const float* a, const T* __restrict__ row, int dim) {
  float s = 0.f;
  for (int c = 0; c < dim; ++c) s = fmaf(a[c], Elem<T>::to_f(row[c]), s);
  return s;
}

// 16-bit number of (key, query, batch head) against the drop limit
__device__ __forceinline__ bool kept(const Philox& rng, uint32_t limit, int key, int query, int bh) {
  return (keep_bits(rng((uint32_t)key >> 3, (uint32_t)query, (uint32_t)bh), limit) >> (key & 7)) & 1u;
}

template <typename T, bool DROP>
__global__ void __launch_bounds__(kThreads)
    attn_rows_fwd(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, T* __restrict__ o,
                  float* __restrict__ lse, Plane pq, Plane pk, Plane pv, Plane po, Shape sh, DropArgs drop) {
  __shared__ float qs[kWarps][kMaxDim];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * kWarps + warp;
  if (row >= (int64_t)sh.batch * sh.heads * sh.nq) return;
  const int i = (int)(row % sh.nq), bh = (int)(row / sh.nq), h = bh % sh.heads, b = bh / sh.heads;
  const int kh = h / (sh.heads / sh.kv_heads), len = sh.keys(b);
  const Philox rng(DROP ? drop : DropArgs{});
  const T* qr = q + b * pq.s_b + i * pq.s_n + h * pq.s_h;
  for (int c = lane; c < sh.dim; c += 32) qs[warp][c] = Elem<T>::to_f(qr[c]) * sh.scale;
  __syncwarp();
  k += b * pk.s_b + kh * pk.s_h;
  v += b * pv.s_b + kh * pv.s_h;
  float m = -INFINITY, l = 0.f, acc[kAcc] = {};
  for (int j0 = 0; j0 < len; j0 += 32) {
    const int j = j0 + lane;
    const float s = j < len ? dot(qs[warp], k + j * pk.s_n, sh.dim) : -INFINITY;
    float mx = s;
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
    const float mn = fmaxf(m, mx), corr = expf(m - mn);
    float p = j < len ? expf(s - mn) : 0.f;
    l = l * corr + warp_sum(p);
    m = mn;
    if (DROP && j < len) p = kept(rng, drop.limit, j, i, bh) ? p * drop.scale : 0.f;
#pragma unroll
    for (int a = 0; a < kAcc; ++a) acc[a] *= corr;
    const int n = len - j0 < 32 ? len - j0 : 32;
    for (int t = 0; t < n; ++t) {
      const float pt = __shfl_sync(0xffffffffu, p, t);
      const T* vr = v + (j0 + t) * pv.s_n;
#pragma unroll
      for (int a = 0; a < kAcc; ++a)
        if (lane + 32 * a < sh.dim) acc[a] = fmaf(pt, Elem<T>::to_f(vr[lane + 32 * a]), acc[a]);
    }
  }
  T* out = o + b * po.s_b + i * po.s_n + h * po.s_h;
  const float inv = len > 0 ? 1.f / l : 0.f;
#pragma unroll
  for (int a = 0; a < kAcc; ++a)
    if (lane + 32 * a < sh.dim) out[lane + 32 * a] = Elem<T>::from_f(acc[a] * inv);
  if (lane == 0) lse[row] = len > 0 ? m + logf(l) : -INFINITY;
}

template <typename T, bool DROP>
__global__ void __launch_bounds__(kThreads)
    attn_rows_dq(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, const T* __restrict__ o,
                 const T* __restrict__ go, const float* __restrict__ lse, T* __restrict__ gq,
                 float* __restrict__ delta, Plane pq, Plane pk, Plane pv, Plane po, Plane pgo, Plane pgq, Shape sh,
                 DropArgs drop) {
  __shared__ float qs[kWarps][kMaxDim], gs[kWarps][kMaxDim];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * kWarps + warp;
  if (row >= (int64_t)sh.batch * sh.heads * sh.nq) return;
  const int i = (int)(row % sh.nq), bh = (int)(row / sh.nq), h = bh % sh.heads, b = bh / sh.heads;
  const int kh = h / (sh.heads / sh.kv_heads), len = sh.keys(b);
  const Philox rng(DROP ? drop : DropArgs{});
  const T* qr = q + b * pq.s_b + i * pq.s_n + h * pq.s_h;
  const T* gr = go + b * pgo.s_b + i * pgo.s_n + h * pgo.s_h;
  const T* orow = o + b * po.s_b + i * po.s_n + h * po.s_h;
  float d = 0.f;
  for (int c = lane; c < sh.dim; c += 32) {
    qs[warp][c] = Elem<T>::to_f(qr[c]) * sh.scale;
    gs[warp][c] = Elem<T>::to_f(gr[c]);
    d = fmaf(gs[warp][c], Elem<T>::to_f(orow[c]), d);
  }
  d = warp_sum(d);
  if (lane == 0) delta[row] = d;
  __syncwarp();
  k += b * pk.s_b + kh * pk.s_h;
  v += b * pv.s_b + kh * pv.s_h;
  const float ls = lse[row];
  float acc[kAcc] = {};
  for (int j0 = 0; j0 < len; j0 += 32) {
    const int j = j0 + lane;
    float ds = 0.f;
    if (j < len) {
      float dp = dot(gs[warp], v + j * pv.s_n, sh.dim);
      if (DROP) dp = kept(rng, drop.limit, j, i, bh) ? dp * drop.scale : 0.f;
      ds = expf(dot(qs[warp], k + j * pk.s_n, sh.dim) - ls) * (dp - d);
    }
    const int n = len - j0 < 32 ? len - j0 : 32;
    for (int t = 0; t < n; ++t) {
      const float dt = __shfl_sync(0xffffffffu, ds, t);
      const T* kr = k + (j0 + t) * pk.s_n;
#pragma unroll
      for (int a = 0; a < kAcc; ++a)
        if (lane + 32 * a < sh.dim) acc[a] = fmaf(dt, Elem<T>::to_f(kr[lane + 32 * a]), acc[a]);
    }
  }
  T* out = gq + b * pgq.s_b + i * pgq.s_n + h * pgq.s_h;
#pragma unroll
  for (int a = 0; a < kAcc; ++a)
    if (lane + 32 * a < sh.dim) out[lane + 32 * a] = Elem<T>::from_f(acc[a] * sh.scale);
}

template <typename T, bool DROP>
__global__ void __launch_bounds__(kThreads)
    attn_rows_dkdv(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, const T* __restrict__ go,
                   const float* __restrict__ lse, const float* __restrict__ delta, T* __restrict__ gk,
                   T* __restrict__ gv, Plane pq, Plane pk, Plane pv, Plane pgo, Plane pgk, Plane pgv, Shape sh,
                   DropArgs drop) {
  __shared__ float ks[kWarps][kMaxDim], vs[kWarps][kMaxDim];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * kWarps + warp;
  if (row >= (int64_t)sh.batch * sh.kv_heads * sh.nk) return;
  const int j = (int)(row % sh.nk), bk = (int)(row / sh.nk), kh = bk % sh.kv_heads, b = bk / sh.kv_heads;
  const int group = sh.heads / sh.kv_heads;
  const Philox rng(DROP ? drop : DropArgs{});
  float ak[kAcc] = {}, av[kAcc] = {};
  if (j < sh.keys(b)) {
    const T* kr = k + b * pk.s_b + j * pk.s_n + kh * pk.s_h;
    const T* vr = v + b * pv.s_b + j * pv.s_n + kh * pv.s_h;
    for (int c = lane; c < sh.dim; c += 32) {
      ks[warp][c] = Elem<T>::to_f(kr[c]) * sh.scale;
      vs[warp][c] = Elem<T>::to_f(vr[c]);
    }
    __syncwarp();
    for (int h = kh * group; h < (kh + 1) * group; ++h) {
      const T* qh = q + b * pq.s_b + h * pq.s_h;
      const T* gh = go + b * pgo.s_b + h * pgo.s_h;
      const int bh = b * sh.heads + h;
      const float* lh = lse + (int64_t)bh * sh.nq;
      const float* dh = delta + (int64_t)bh * sh.nq;
      for (int i0 = 0; i0 < sh.nq; i0 += 32) {
        const int i = i0 + lane;
        float p = 0.f, ds = 0.f;
        if (i < sh.nq) {
          p = expf(dot(ks[warp], qh + i * pq.s_n, sh.dim) - lh[i]);
          float dp = dot(vs[warp], gh + i * pgo.s_n, sh.dim);
          float mult = 1.f;
          if (DROP) mult = kept(rng, drop.limit, j, i, bh) ? drop.scale : 0.f;
          ds = p * ((mult > 0.f ? dp * mult : 0.f) - dh[i]);
          p *= mult;
        }
        const int n = sh.nq - i0 < 32 ? sh.nq - i0 : 32;
        for (int t = 0; t < n; ++t) {
          const float pt = __shfl_sync(0xffffffffu, p, t), dt = __shfl_sync(0xffffffffu, ds, t);
          const T* qr = qh + (i0 + t) * pq.s_n;
          const T* gr = gh + (i0 + t) * pgo.s_n;
#pragma unroll
          for (int a = 0; a < kAcc; ++a) {
            if (lane + 32 * a >= sh.dim) break;
            ak[a] = fmaf(dt, Elem<T>::to_f(qr[lane + 32 * a]), ak[a]);
            av[a] = fmaf(pt, Elem<T>::to_f(gr[lane + 32 * a]), av[a]);
          }
        }
      }
    }
  }
  T* ok = gk + b * pgk.s_b + j * pgk.s_n + kh * pgk.s_h;
  T* ov = gv + b * pgv.s_b + j * pgv.s_n + kh * pgv.s_h;
#pragma unroll
  for (int a = 0; a < kAcc; ++a) {
    if (lane + 32 * a >= sh.dim) break;
    ok[lane + 32 * a] = Elem<T>::from_f(ak[a] * sh.scale);
    ov[lane + 32 * a] = Elem<T>::from_f(av[a]);
  }
}

// ------------------------------------------------------------------ host
Plane plane_at(const int64_t* s, int i) { return Plane{s[3 * i], s[3 * i + 1], s[3 * i + 2]}; }

int make_shape(Shape& sh, int64_t batch, int64_t heads, int64_t kv_heads, int64_t nq, int64_t nk, int64_t dim,
               const int32_t* lengths, float scale, int threshold, const int64_t* key, const char* name) {
  PMB_REQUIRE(batch >= 0 && nq >= 0 && nk >= 0 && heads > 0 && kv_heads > 0, "%s: bad shape", name);
  PMB_REQUIRE(heads % kv_heads == 0, "%s: %lld heads are not a multiple of %lld key / value heads", name,
              (long long)heads, (long long)kv_heads);
  PMB_REQUIRE(dim > 0 && dim <= kMaxDim, "%s: head dim %lld outside [1, %d]", name, (long long)dim, kMaxDim);
  PMB_REQUIRE(nq < (1 << 30) && nk < (1 << 30) && batch * heads < (1 << 30), "%s: too large", name);
  PMB_REQUIRE(threshold >= 0 && threshold <= 65536, "%s: drop threshold %d outside [0, 65536]", name, threshold);
  PMB_REQUIRE(key || threshold == 0, "%s: NULL key", name);
  sh = Shape{(int)batch, (int)heads, (int)kv_heads, (int)nq, (int)nk, (int)dim, lengths, scale};
  return PMB_OK;
}

int row_grid(int64_t rows, unsigned& grid, const char* name) {
  const int64_t g = (rows + kWarps - 1) / kWarps;
  PMB_REQUIRE(g < ((int64_t)1 << 31), "%s: too many rows", name);
  grid = (unsigned)g;
  return PMB_OK;
}

int64_t delta_bytes(int64_t rows) { return (rows * 4 + 255) / 256 * 256; }

}  // namespace
}  // namespace pmb

using namespace pmb;

extern "C" int64_t pmb_cross_attention_lse_size(int64_t batch, int64_t heads, int64_t nq) {
  return batch > 0 && heads > 0 && nq > 0 ? xattn::tc_lse_floats(batch * heads, nq) : 0;
}

namespace pmb {
namespace {
// Shape of a workspace query; false where the sizes make no call.
bool query_shape(Shape& sh, int64_t batch, int64_t heads, int64_t kv_heads, int64_t nq, int64_t nk, int64_t dim) {
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || nq <= 0 || nk < 0 || dim <= 0) return false;
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
  if (int st = row_grid(rows, grid, name)) return st;
  return PMB_DISPATCH(dtype, T, name, [&] {
    auto kernel = threshold > 0 ? attn_rows_fwd<T, true> : attn_rows_fwd<T, false>;
    kernel<<<grid, kThreads, 0, s>>>(static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v),
                                     static_cast<T*>(o), lse, pq, pk, pv, po, sh, drop);
    PMB_CHECK_LAUNCH(name);
    return PMB_OK;
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
  if (int st = row_grid(rows, qgrid, name)) return st;
  if (int st = row_grid(keys, kgrid, name)) return st;
  return PMB_DISPATCH(dtype, T, name, [&] {
    if (rows > 0) {
      auto kernel = threshold > 0 ? attn_rows_dq<T, true> : attn_rows_dq<T, false>;
      kernel<<<qgrid, kThreads, 0, s>>>(static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v),
                                        static_cast<const T*>(o), static_cast<const T*>(grad_out), lse,
                                        static_cast<T*>(grad_q), delta, pq, pk, pv, po, pgo, pgq, sh, drop);
      PMB_CHECK_LAUNCH(name);
    }
    if (keys > 0) {
      auto kernel = threshold > 0 ? attn_rows_dkdv<T, true> : attn_rows_dkdv<T, false>;
      kernel<<<kgrid, kThreads, 0, s>>>(static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v),
                                        static_cast<const T*>(grad_out), lse, delta, static_cast<T*>(grad_k),
                                        static_cast<T*>(grad_v), pq, pk, pv, pgo, pgk, pgv, sh, drop);
      PMB_CHECK_LAUNCH(name);
    }
    return PMB_OK;
  });
}
