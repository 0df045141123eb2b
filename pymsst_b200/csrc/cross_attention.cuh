// What the two forms of the cross attention share: its shape, the planes, and
// the entries of the tensor-core form (cross_attention_tc.cu) that the C
// entries of cross_attention.cu dispatch to.
#pragma once

#include "common.cuh"
#include "philox.cuh"

namespace pmb {
namespace xattn {

// Lower limit of a row's running maximum (the lowest fp32 value): scores of -infinity, from a dot product that
// overflows, then weigh exp(-infinity) = 0 where -infinity - (-infinity) would be NaN.
constexpr float kLowest = -3.402823466e38f;

struct Plane {
  int64_t s_b, s_n, s_h;  // element strides, the head elements contiguous
};

struct Shape {
  int batch, heads, kv_heads, nq, nk, dim;
  const int32_t* lengths;  // keys of each batch item, or NULL: nk
  float scale;

  __device__ __forceinline__ int keys(int b) const {
    if (lengths == nullptr) return nk;
    const int n = __ldg(lengths + b);
    return n < 0 ? 0 : (n < nk ? n : nk);
  }
};

struct Forward {
  const void *q, *k, *v;
  void* o;
  float* lse;
  Plane pq, pk, pv, po;
  int dtype;
  int threshold;
  DropArgs drop;
  void* workspace;
  int64_t workspace_bytes;
  cudaStream_t stream;
};

struct Backward {
  const void *q, *k, *v, *o, *go;
  const float* lse;
  void *gq, *gk, *gv;
  Plane pq, pk, pv, po, pgo, pgq, pgk, pgv;
  int dtype;
  int threshold;
  DropArgs drop;
  void* workspace;
  int64_t workspace_bytes;
  cudaStream_t stream;
};

// Whether the tensor-core form takes a call: 16-bit types, head dims that are
// multiples of 8 up to 128, something on both sides, and a positive scale (the
// maximum is taken before scaling, and masked scores are -inf before it).
inline bool tc_takes(const Shape& sh, int dtype) {
  return dtype_size(dtype) == 2 && sh.dim % 8 == 0 && sh.dim <= 128 && sh.nq > 0 && sh.nk > 0 && sh.scale > 0.f;
}

int64_t tc_lse_floats(int64_t heads_total, int64_t nq);
int64_t tc_forward_workspace(const Shape& sh);
int64_t tc_backward_workspace(const Shape& sh);
int tc_forward(const Shape& sh, const Forward& a, const char* name);
int tc_backward(const Shape& sh, const Backward& a, const char* name);

}  // namespace xattn
}  // namespace pmb
