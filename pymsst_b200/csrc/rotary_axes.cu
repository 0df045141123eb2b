// Rotary embedding of tokens that carry several positions (frame, band,
// channel ...): interleaved pair p of a head belongs to one axis a(p) and
//   angle = position[token, a(p)] * freqs[p]
//   (e, o) -> (e cos - o sin, o cos + e sin);  inverse: the opposite angle.
// Pairs behind the last axis' section are copied.
//
// The angle of a far position needs more than fp32 (position 10^6 times a
// frequency near 1 leaves 0.06 rad of fp32 rounding), so it is formed and
// reduced to one turn in fp64: turns = position * freq / 2 pi, minus its
// nearest integer.  Its sine and cosine are then fp32.
//
// Bound by HBM (each value read once, written once).  The angles are shared
// by the heads: a CTA takes a few tokens, computes their angles into shared
// memory once (a few hundred fp64 products per CTA), and rotates all heads'
// values of those tokens with 16-byte vectors, whose loads are issued before
// the angles are computed.  4 x 15,996 tokens of 16 heads x 64 bf16, three
// axes: 51.5 us a direction, floor 40.8; 84 us before threads kept their place
// in the head and divided no more.
#include "common.cuh"

namespace pmb {
namespace {

constexpr int kThreads = 256;
constexpr int kAngles = 1024;  // angle slots per CTA
constexpr int kUnroll = 4;     // vectors in flight per thread
constexpr int kMaxAxes = 4;

struct Axes {
  int count;
  int end[kMaxAxes];  // running ends of the sections, in pairs
};

struct View {
  int64_t s_b, s_n, s_h;  // element strides, head elements contiguous
};

template <typename T, int P>
struct alignas(sizeof(T) * 2 * P < 16 ? sizeof(T) * 2 * P : 16) Pairs {
  T v[2 * P];
};

// Rotated vector: P pairs, `live` of them (or all) by the angles at w.
template <typename T, int P>
__device__ __forceinline__ Pairs<T, P> rotated(const Pairs<T, P>& in, const float2* w, int live) {
  Pairs<T, P> out = in;
  if (live >= P) {
    float2 cv[P];
    if constexpr (P > 1) {
#pragma unroll
      for (int j = 0; j < P; j += 2) *reinterpret_cast<float4*>(cv + j) = *reinterpret_cast<const float4*>(w + j);
    } else {
      cv[0] = w[0];
    }
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const float e = Elem<T>::to_f(in.v[2 * j]), o = Elem<T>::to_f(in.v[2 * j + 1]);
      const float ye = e * cv[j].x - o * cv[j].y, yo = o * cv[j].x + e * cv[j].y;
      if constexpr (sizeof(T) == 2) {
        reinterpret_cast<uint32_t*>(out.v)[j] = Elem<T>::pack2(ye, yo);
      } else {
        out.v[2 * j] = ye;
        out.v[2 * j + 1] = yo;
      }
    }
  } else if (live > 0) {
#pragma unroll
    for (int j = 0; j < P; ++j) {
      if (j < live) {
        const float2 c = w[j];
        const float e = Elem<T>::to_f(in.v[2 * j]), o = Elem<T>::to_f(in.v[2 * j + 1]);
        out.v[2 * j] = Elem<T>::from_f(e * c.x - o * c.y);
        out.v[2 * j + 1] = Elem<T>::from_f(o * c.x + e * c.y);
      }
    }
  }
  return out;
}

// One CTA per (batch, token tile), `tiles` of them per batch; tile * pitch <= kAngles (pitch: rotated pairs, made even
// so that a token's angles start on 16 bytes).  ROWS: the CTA's threads are a multiple of the vectors of a token, so a
// thread keeps its head and its place in the head and steps over tokens; otherwise (tokens of more than kThreads
// vectors) each vector's place is divided out.
template <typename T, typename PosT, int P, bool ROWS>
__global__ void __launch_bounds__(kThreads)
    rotary_axes_kernel(const T* __restrict__ x, const PosT* __restrict__ pos, const float* __restrict__ freqs,
                       T* __restrict__ y, int tokens, int heads, int pairs, int tile, int tiles, int pitch, View vx,
                       View vy, int64_t pos_b, Axes axes, float sign) {
  __shared__ __align__(16) float2 cs[kAngles];
  const int rot = axes.end[axes.count - 1];
  const int64_t b = blockIdx.x / tiles;
  const int t0 = (int)(blockIdx.x - b * tiles) * tile, nt = tokens - t0 < tile ? tokens - t0 : tile;
  const int per_head = pairs / P, per_token = heads * per_head, total = nt * per_token;
  x += b * vx.s_b + (int64_t)t0 * vx.s_n;
  y += b * vy.s_b + (int64_t)t0 * vy.s_n;
  // this thread's first vector: token, head, place in the head
  const int tt = threadIdx.x / per_token, rr = threadIdx.x - tt * per_token, hh = rr / per_head, cc = rr - hh * per_head;
  const int step = ROWS ? (int)blockDim.x / per_token : 0;

  Pairs<T, P> buf[kUnroll];
  auto load = [&](int first) {  // ROWS: a token, else a vector of the tile
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if constexpr (ROWS) {
        const int t = first + u * step;
        if (t < nt) buf[u] = *reinterpret_cast<const Pairs<T, P>*>(x + t * vx.s_n + hh * vx.s_h + cc * 2 * P);
      } else {
        const int i = first + u * kThreads;
        if (i < total) {
          const int t = i / per_token, r = i - t * per_token, h = r / per_head, c = r - h * per_head;
          buf[u] = *reinterpret_cast<const Pairs<T, P>*>(x + t * vx.s_n + h * vx.s_h + c * 2 * P);
        }
      }
    }
  };
  load(ROWS ? tt : (int)threadIdx.x);
  for (int i = threadIdx.x; i < nt * rot; i += blockDim.x) {
    const int t = i / rot, p = i - t * rot;
    int a = 0;
#pragma unroll
    for (int k = 0; k + 1 < kMaxAxes; ++k) a += p >= axes.end[k] ? 1 : 0;
    const double where = (double)pos[b * pos_b + (int64_t)(t0 + t) * axes.count + a];
    double turns = where * (double)freqs[p] * 0.15915494309189533577;
    turns -= rint(turns);
    float s, c;
    sincospif(2.f * (float)turns, &s, &c);
    cs[t * pitch + p] = make_float2(c, s * sign);
  }
  __syncthreads();
  if constexpr (ROWS) {
    const int live = rot - cc * P;
    const float2* w = cs + cc * P;
    T* dst = y + hh * vy.s_h + cc * 2 * P;
    for (int first = tt; first < nt; first += kUnroll * step) {
      if (first != tt) load(first);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int t = first + u * step;
        if (t < nt) *reinterpret_cast<Pairs<T, P>*>(dst + t * vy.s_n) = rotated<T, P>(buf[u], w + t * pitch, live);
      }
    }
  } else {
    for (int first = threadIdx.x; first < total; first += kThreads * kUnroll) {
      if (first != (int)threadIdx.x) load(first);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int i = first + u * kThreads;
        if (i < total) {
          const int t = i / per_token, r = i - t * per_token, h = r / per_head, c = r - h * per_head;
          *reinterpret_cast<Pairs<T, P>*>(y + t * vy.s_n + h * vy.s_h + c * 2 * P) =
              rotated<T, P>(buf[u], cs + t * pitch + c * P, rot - c * P);
        }
      }
    }
  }
}

template <typename T, typename PosT>
int launch(const void* x, const void* pos, const float* freqs, void* y, int64_t batch, int tokens, int heads, int pairs,
           const View& vx, const View& vy, int64_t pos_b, const Axes& axes, float sign, cudaStream_t s,
           const char* name) {
  constexpr int P = sizeof(T) == 2 ? 4 : 2;  // 16 bytes
  constexpr int kVec = 2 * P;
  const bool vec = pairs % P == 0 &&
                   ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 15) == 0 &&
                   vx.s_b % kVec == 0 && vx.s_n % kVec == 0 && vx.s_h % kVec == 0 && vy.s_b % kVec == 0 &&
                   vy.s_n % kVec == 0 && vy.s_h % kVec == 0;
  const int rot = axes.end[axes.count - 1];
  // tokens per CTA: kUnroll vectors per thread, as many as the angle slots allow
  const int64_t per_token = (int64_t)heads * (vec ? pairs / P : pairs);
  const bool rows = per_token <= kThreads;
  const int block = rows ? (int)(kThreads / per_token * per_token) : kThreads;
  int64_t tile = (int64_t)block * kUnroll / per_token;
  const int pitch = (rot + 1) / 2 * 2;
  if (tile > kAngles / pitch) tile = kAngles / pitch;
  if (tile < 1) tile = 1;
  if (tile > tokens) tile = tokens;
  const int64_t tiles = (tokens + tile - 1) / tile;
  PMB_REQUIRE(tiles * batch < ((int64_t)1 << 31), "%s: too many tokens", name);
  const unsigned grid = (unsigned)(tiles * batch);
  auto kernel = vec ? (rows ? rotary_axes_kernel<T, PosT, P, true> : rotary_axes_kernel<T, PosT, P, false>)
                    : (rows ? rotary_axes_kernel<T, PosT, 1, true> : rotary_axes_kernel<T, PosT, 1, false>);
  kernel<<<grid, block, 0, s>>>(static_cast<const T*>(x), static_cast<const PosT*>(pos), freqs, static_cast<T*>(y),
                                tokens, heads, pairs, (int)tile, (int)tiles, pitch, vx, vy, pos_b, axes, sign);
  PMB_CHECK_LAUNCH(name);
  return PMB_OK;
}

}  // namespace
}  // namespace pmb

using namespace pmb;

extern "C" int pmb_rotary_axes(const void* x, const void* positions, const float* freqs, void* y, int64_t batch,
                               int64_t tokens, int64_t heads, int64_t dim, const int64_t* strides,
                               int64_t position_batch_stride, int position_type, int axes, const int64_t* sections,
                               int inverse, int dtype, void* stream) {
  clear_error();
  const char* name = "pmb_rotary_axes";
  PMB_REQUIRE(batch >= 0 && tokens >= 0 && heads >= 0 && dim > 0, "%s: bad shape", name);
  PMB_REQUIRE(dim % 2 == 0 && dim / 2 <= kAngles, "%s: head dim %lld must be even and at most %d", name,
              (long long)dim, 2 * kAngles);
  PMB_REQUIRE(axes >= 1 && axes <= kMaxAxes && sections, "%s: 1 to %d axes (got %d)", name, kMaxAxes, axes);
  Axes ax;
  ax.count = axes;
  int64_t end = 0;
  for (int a = 0; a < axes; ++a) {
    PMB_REQUIRE(sections[a] > 0 && sections[a] <= dim / 2, "%s: section %d has a bad size", name, a);
    end += sections[a];
    ax.end[a] = (int)end;
  }
  for (int a = axes; a < kMaxAxes; ++a) ax.end[a] = (int)end;
  PMB_REQUIRE(end <= dim / 2, "%s: sections hold %lld pairs, the head has %lld", name, (long long)end,
              (long long)(dim / 2));
  if (batch == 0 || tokens == 0 || heads == 0) return PMB_OK;
  PMB_REQUIRE(batch < (1 << 30) && tokens < (1 << 30) && heads < (1 << 20) && heads * (dim / 2) < (1 << 20),
              "%s: too large", name);
  PMB_REQUIRE(x && positions && freqs && y && strides, "%s: NULL argument", name);
  const View vx{strides[0], strides[1], strides[2]}, vy{strides[3], strides[4], strides[5]};
  // pairs are read and written whole: a pair is aligned to its size
  PMB_REQUIRE(dtype_size(dtype) == 0 || ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) %
                                         (2 * dtype_size(dtype))) == 0,
              "%s: tensors must be aligned to a pair of elements", name);
  for (int i = 0; i < 6; ++i) PMB_REQUIRE(strides[i] % 2 == 0, "%s: strides must be even", name);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const float sign = inverse ? -1.f : 1.f;
  return PMB_DISPATCH(dtype, T, name, [&] {
    switch (position_type) {
      case 0:
        return launch<T, int32_t>(x, positions, freqs, y, batch, (int)tokens, (int)heads, (int)(dim / 2), vx, vy,
                                  position_batch_stride, ax, sign, s, name);
      case 1:
        return launch<T, int64_t>(x, positions, freqs, y, batch, (int)tokens, (int)heads, (int)(dim / 2), vx, vy,
                                  position_batch_stride, ax, sign, s, name);
      case 2:
        return launch<T, float>(x, positions, freqs, y, batch, (int)tokens, (int)heads, (int)(dim / 2), vx, vy,
                                position_batch_stride, ax, sign, s, name);
      default:
        set_error("%s: unknown position type %d", name, position_type);
        return PMB_ERR_UNSUPPORTED_DTYPE;
    }
  });
}
