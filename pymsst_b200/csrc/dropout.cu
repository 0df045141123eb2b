// Dropout from counter-based random bits (philox.cuh), elementwise:
//   y  = keep ? c x : 0                    (also its own backward on gy)
//   y  = residual + (keep ? c x : 0)       the sum behind a projection
//   y  = keep ? c gelu(x) : 0              the feed-forward's activation
//   gx = keep ? c gy gelu'(x) : 0
// c = 1 / (keep probability).  A dropped element is a select, so an infinity
// or NaN under the mask does not reach y.  Computed in fp32 and rounded once.
//
// One thread takes groups of eight consecutive elements: one Philox call, and
// for 16-bit types one 16-byte vector per tensor.  Nothing but the tensors
// themselves moves (a stored mask would add a byte per element to both
// passes).  One group per thread: many small CTAs keep more loads in flight
// than a loop does (the residual form over 63,984 x 192 bf16 takes 16.4 us so,
// 20.7 with two groups per thread, 22.4 in a loop that loads one group ahead;
// floor 11.4, its backward 13.0, floor 7.6: kernels so short are bound by their
// ramp and the latency of the loads behind it).  The GELU forms are bound by
// instruction issue (ncu: 0.74 of the slots, FMA pipe 55 %, HBM 29 to 42 %): 62
// and 75 us for 63,984 x 768 bf16, floors 30.5 and 45.7.
#include "common.cuh"
#include "gelu.cuh"
#include "philox.cuh"

namespace pmb {
namespace {

constexpr int kThreads = 256;

enum Mode { kPlain = 0, kResidual = 1, kGelu = 2, kGeluGrad = 3 };

template <typename T>
struct alignas(16) Pack8 {
  T v[8];
};

// Results of two neighbouring elements before the drop: a = x, b = residual or gy.
template <typename T, int MODE>
__device__ __forceinline__ void value2(float a0, float a1, float b0, float b1, float c, bool k0, bool k1, float& y0,
                                       float& y1) {
  if (MODE == kPlain || MODE == kResidual) {
    y0 = k0 ? a0 : 0.f;
    y1 = k1 ? a1 : 0.f;
    const uint64_t r = fma2(pk2(y0, y1), pk2(c, c), MODE == kResidual ? pk2(b0, b1) : pk2(0.f, 0.f));
    unpk2(r, y0, y1);
    return;
  }
  if constexpr (MODE == kGelu) {
    if constexpr (sizeof(T) == 2) {
      float p0, p1;
      uint64_t t;
      phi_cdf_fast2(a0, a1, p0, p1, t);
      unpk2(mul2(mul2(pk2(a0, a1), pk2(p0, p1)), pk2(c, c)), y0, y1);
    } else {
      y0 = gelu_of<T>(a0) * c;
      y1 = gelu_of<T>(a1) * c;
    }
  } else if constexpr (MODE == kGeluGrad) {
    float d0, d1;
    if constexpr (sizeof(T) == 2) {
      gelu_grad_fast2(a0, a1, d0, d1);
    } else {
      d0 = gelu_grad_of<T>(a0);
      d1 = gelu_grad_of<T>(a1);
    }
    unpk2(mul2(mul2(pk2(d0, d1), pk2(b0, b1)), pk2(c, c)), y0, y1);
  }
  y0 = k0 ? y0 : 0.f;
  y1 = k1 ? y1 : 0.f;
}

template <typename T, int MODE, bool DROP, bool VEC>
__global__ void __launch_bounds__(kThreads)
    dropout_kernel(const T* __restrict__ a, const T* __restrict__ b, T* __restrict__ y, int64_t n, DropArgs drop) {
  constexpr bool kTwo = MODE == kResidual || MODE == kGeluGrad;
  const int64_t stride = (int64_t)gridDim.x * kThreads;
  const int64_t groups = (n + 7) / 8, full = VEC ? n / 8 : 0;
  for (int64_t g = (int64_t)blockIdx.x * kThreads + threadIdx.x; g < groups; g += stride) {
    Pack8<T> pa, pb, out;
    if (g < full) {
      pa = reinterpret_cast<const Pack8<T>*>(a)[g];
      if (kTwo) pb = reinterpret_cast<const Pack8<T>*>(b)[g];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int64_t i = g * 8 + e;
        pa.v[e] = i < n ? a[i] : Elem<T>::from_f(0.f);
        if (kTwo) pb.v[e] = i < n ? b[i] : Elem<T>::from_f(0.f);
      }
    }
    uint4 r = make_uint4(0, 0, 0, 0);
    if (DROP) r = philox(drop, (uint32_t)g, (uint32_t)((uint64_t)g >> 32), 0xffffffffu);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      float y0, y1;
      value2<T, MODE>(Elem<T>::to_f(pa.v[e]), Elem<T>::to_f(pa.v[e + 1]), kTwo ? Elem<T>::to_f(pb.v[e]) : 0.f,
                      kTwo ? Elem<T>::to_f(pb.v[e + 1]) : 0.f, DROP ? drop.scale : 1.f,
                      !DROP || kept(w[e / 2], 0, drop.high), !DROP || kept(w[e / 2], 1, drop.high), y0, y1);
      if constexpr (sizeof(T) == 2) {
        reinterpret_cast<uint32_t*>(out.v)[e / 2] = Elem<T>::pack2(y0, y1);
      } else {
        out.v[e] = y0;
        out.v[e + 1] = y1;
      }
    }
    if (g < full) {
      reinterpret_cast<Pack8<T>*>(y)[g] = out;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (g * 8 + e < n) y[g * 8 + e] = out.v[e];
    }
  }
}

template <typename T, int MODE>
int launch(const void* a, const void* b, void* y, int64_t n, int threshold, const DropArgs& drop, cudaStream_t s,
           const char* name) {
  const bool vec = ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) |
                     reinterpret_cast<uintptr_t>(y)) & 15) == 0;
  int64_t grid = ((n + 7) / 8 + kThreads - 1) / kThreads;
  if (grid > (1 << 30)) grid = 1 << 30;
  auto kernel = threshold > 0 ? (vec ? dropout_kernel<T, MODE, true, true> : dropout_kernel<T, MODE, true, false>)
                              : (vec ? dropout_kernel<T, MODE, false, true> : dropout_kernel<T, MODE, false, false>);
  kernel<<<(unsigned)grid, kThreads, 0, s>>>(static_cast<const T*>(a), static_cast<const T*>(b), static_cast<T*>(y), n,
                                             drop);
  PMB_CHECK_LAUNCH(name);
  return PMB_OK;
}

template <int MODE>
int entry(const void* a, const void* b, void* y, int64_t n, int threshold, const int64_t* key, uint32_t site,
          int dtype, void* stream, const char* name) {
  PMB_REQUIRE(n >= 0, "%s: bad size", name);
  PMB_REQUIRE(threshold >= 0 && threshold <= 65536, "%s: drop threshold %d outside [0, 65536]", name, threshold);
  if (n == 0) return PMB_OK;
  PMB_REQUIRE(a && y && (b || MODE == kPlain || MODE == kGelu), "%s: NULL tensor argument", name);
  PMB_REQUIRE(key || threshold == 0, "%s: NULL key", name);
  const DropArgs drop = drop_args(key, site, threshold);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return PMB_DISPATCH(dtype, T, name, [&] { return launch<T, MODE>(a, b, y, n, threshold, drop, s, name); });
}

// out = state, then the state's step moves on: what one forward's dropout sites share.
__global__ void next_key_kernel(int64_t* state, int64_t* out) {
  out[0] = state[0];
  out[1] = state[1];
  state[1] = state[1] + 1;
}

}  // namespace
}  // namespace pmb

using namespace pmb;

extern "C" int pmb_dropout_next_key(int64_t* state, int64_t* key, void* stream) {
  clear_error();
  const char* name = "pmb_dropout_next_key";
  PMB_REQUIRE(state && key, "%s: NULL argument", name);
  next_key_kernel<<<1, 1, 0, static_cast<cudaStream_t>(stream)>>>(state, key);
  PMB_CHECK_LAUNCH(name);
  return PMB_OK;
}

extern "C" int pmb_dropout(const void* x, const void* residual, void* y, int64_t n, int threshold, const int64_t* key,
                           uint32_t site, int dtype, void* stream) {
  clear_error();
  const char* name = "pmb_dropout";
  return residual ? entry<kResidual>(x, residual, y, n, threshold, key, site, dtype, stream, name)
                  : entry<kPlain>(x, nullptr, y, n, threshold, key, site, dtype, stream, name);
}

extern "C" int pmb_gelu_dropout_forward(const void* x, void* y, int64_t n, int threshold, const int64_t* key,
                                        uint32_t site, int dtype, void* stream) {
  clear_error();
  return entry<kGelu>(x, nullptr, y, n, threshold, key, site, dtype, stream, "pmb_gelu_dropout_forward");
}

extern "C" int pmb_gelu_dropout_backward(const void* grad_out, const void* x, void* grad_x, int64_t n, int threshold,
                                         const int64_t* key, uint32_t site, int dtype, void* stream) {
  clear_error();
  return entry<kGeluGrad>(x, grad_out, grad_x, n, threshold, key, site, dtype, stream, "pmb_gelu_dropout_backward");
}
