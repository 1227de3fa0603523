// Rotary positions of one or two (B, L, H, D) tensors (q and k of an attention layer), and the gradient, which is the
// rotation by the opposite angle.
//
//   y_a = m (x_a cos w - x_b sin w),  y_b = m (x_a sin w + x_b cos w),  w = position[axis(p)] * f_p
//
// for every rotation pair p = (a, b): (2p, 2p+1) in the interleaved layout, (p, p + n) in the half layout with n pairs; the
// elements behind the last pair are copied.
//
// Angles: sin and cos need w modulo one turn only.  turns[p] = round(2^64 f_p / (2 pi)) is the part of a turn that one step of
// position adds, in 64-bit fixed point, so that position * turns[p] modulo 2^64, one wrapping integer product, IS the angle
// modulo one turn: exact but for |position| * 2^-65 turns, whatever the position (2^31: 2^-34 turns).  A product in 32-bit
// floating point would be off by half a radian at position 2^23.  No table of angles exists, so there is no longest position.
// Products and sums are 32-bit, with one rounding to the tensors' type.
//
// Memory-bound: each element is read once and written once.  A thread owns 16 bytes of a row (half layout: 16 bytes of either
// half) of one token and walks over up to sixteen heads with eight loads in flight, so that the angles of its pairs are computed once for
// them.  q and k of 24 heads x 32,760 x 128 bf16: 0.128 ms, 6.3 TB/s, 0.96 of the copy rate (0.255 with guarded loads and 64-bit index
// arithmetic per head).  fp32, 2 x 4,095 x 20 heads x 144, 96 of them rotated: 41 us, 4.6 TB/s (part of it out of L2).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernels.cuh"
#include "ptx.cuh"

namespace mcs {
namespace {

constexpr int kThreadsR = 256;

template <int kType> struct Elem;                            // 0 bf16, 1 fp16, 2 fp32
template <> struct Elem<0> {
  using T = __nv_bfloat16;
  static __device__ __forceinline__ float get(T x) { return __bfloat162float(x); }
  static __device__ __forceinline__ T put(float x) { return __float2bfloat16_rn(x); }
};
template <> struct Elem<1> {
  using T = __half;
  static __device__ __forceinline__ float get(T x) { return __half2float(x); }
  static __device__ __forceinline__ T put(float x) { return __float2half_rn(x); }
};
template <> struct Elem<2> {
  using T = float;
  static __device__ __forceinline__ float get(T x) { return x; }
  static __device__ __forceinline__ T put(float x) { return x; }
};

template <typename T, int N>
struct alignas(N * sizeof(T)) Pack { T v[N]; };

// kVec: elements per access; the host picks 16 bytes, or single elements where a stride, an address or the size of the rotated
// part does not allow 16 bytes.  kHalf: pairs (p, p + n) instead of (2p, 2p + 1).
template <int kType, bool kHalf, int kVec>
struct Layout {
  using E = Elem<kType>;
  using T = typename E::T;
  using V = Pack<T, kVec>;
  static constexpr int kPairs = kHalf ? kVec : (kVec > 1 ? kVec / 2 : 1);   // pairs of one unit
  static constexpr bool kSplit = kHalf || kVec == 1;                        // the members of a pair come from two accesses
};

// `heads` rows of one token, `stride` elements apart: rotated by (c, s), or copied
template <int kType, bool kHalf, int kVec, bool kRotate>
__device__ __forceinline__ void walk_heads(const typename Elem<kType>::T* x, typename Elem<kType>::T* y, long long xs, long long ys, int heads, int n_pairs,
                                           const float* c, const float* s) {
  using Y = Layout<kType, kHalf, kVec>;
  using E = typename Y::E;
  using V = typename Y::V;
  const int second = kHalf ? n_pairs : 1;                    // where the other member of a pair is
  auto turn = [&](V& a, V& b) {
    if constexpr (!kRotate) return;
    if constexpr (Y::kSplit) {
#pragma unroll
      for (int j = 0; j < Y::kPairs; ++j) {
        const float f = E::get(a.v[j]), g = E::get(b.v[j]);
        a.v[j] = E::put(fmaf(f, c[j], -g * s[j]));
        b.v[j] = E::put(fmaf(f, s[j], g * c[j]));
      }
    } else {
#pragma unroll
      for (int j = 0; j < Y::kPairs; ++j) {
        const float f = E::get(a.v[2 * j]), g = E::get(a.v[2 * j + 1]);
        a.v[2 * j] = E::put(fmaf(f, c[j], -g * s[j]));
        a.v[2 * j + 1] = E::put(fmaf(f, s[j], g * c[j]));
      }
    }
  };
  constexpr bool kTwo = Y::kSplit && kRotate;
  constexpr int kUnroll = kTwo ? 4 : 8;                      // loads in flight: eight of up to 16 bytes per thread
  int h = 0;
  for (; h + kUnroll <= heads; h += kUnroll, x += kUnroll * xs, y += kUnroll * ys) {
    V a[kUnroll], b[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      a[u] = *reinterpret_cast<const V*>(x + u * xs);
      if constexpr (kTwo) b[u] = *reinterpret_cast<const V*>(x + u * xs + second);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      turn(a[u], b[u]);
      *reinterpret_cast<V*>(y + u * ys) = a[u];
      if constexpr (kTwo) *reinterpret_cast<V*>(y + u * ys + second) = b[u];
    }
  }
  for (; h < heads; ++h, x += xs, y += ys) {
    V a, b;
    a = *reinterpret_cast<const V*>(x);
    if constexpr (kTwo) b = *reinterpret_cast<const V*>(x + second);
    turn(a, b);
    *reinterpret_cast<V*>(y) = a;
    if constexpr (kTwo) *reinterpret_cast<V*>(y + second) = b;
  }
}

// A CTA takes `tokens_per_cta` tokens: their rotated units first, then the units that are copied, so that few warps do both.
// blockIdx.y is a run of heads of q and k together.
template <int kType, bool kHalf, int kVec>
__global__ void __launch_bounds__(kThreadsR) rotary_kernel(const __grid_constant__ RotaryParams p) {
  using Y = Layout<kType, kHalf, kVec>;
  using T = typename Y::T;
  constexpr int kPairs = Y::kPairs;
  const int h0 = blockIdx.y * p.heads_per_cta, h1 = min(h0 + p.heads_per_cta, p.H[0] + p.H[1]);
  const int turning = p.tokens_per_cta * p.rot_units, copied = p.units - p.rot_units;
  for (int i = threadIdx.x; i < p.tokens_per_cta * p.units; i += kThreadsR) {
    const bool rotates = i < turning;
    const int n = rotates ? p.rot_units : copied, at = rotates ? i : i - turning, sub = at / n;
    const int unit = (rotates ? 0 : p.rot_units) + at - sub * n;
    const long long token = (long long)blockIdx.x * p.tokens_per_cta + sub;
    if (token >= (long long)p.B * p.L) continue;
    const int b = (int)(token / p.L), row = (int)(token - (long long)b * p.L);
    float c[kPairs], s[kPairs];
    if (rotates) {
      const long long base = b * p.p_stride[0] + row * p.p_stride[1];
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        const int pr = unit * kPairs + j;
        const long long at = base + (long long)p.axis[pr] * p.p_stride[2];
        const long long pos = p.pos64 ? reinterpret_cast<const long long*>(p.positions)[at]
                                      : (long long)reinterpret_cast<const int*>(p.positions)[at];
        const unsigned long long turn = (unsigned long long)pos * p.turns[pr];
        // the upper 32 bits as a signed fraction of half a turn: [-1, 1), relative rounding 2^-25
        const float half_turns = (float)(int)(turn >> 32) * 4.656612873077393e-10f;
        sincospif(half_turns, &s[j], &c[j]);
        c[j] *= p.magnitude;
        s[j] *= p.inverse ? -p.magnitude : p.magnitude;
      }
    }
    const int e = rotates ? (kHalf ? unit * kVec : unit * (kVec > 1 ? kVec : 2)) : 2 * p.n_pairs + (unit - p.rot_units) * kVec;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      // this CTA's heads of tensor t
      const int first = t == 0 ? h0 : max(h0 - p.H[0], 0), end = t == 0 ? min(h1, p.H[0]) : h1 - p.H[0];
      if (first >= end) continue;
      const T* x = reinterpret_cast<const T*>(p.x[t]) + b * p.x_stride[t][0] + row * p.x_stride[t][1] + first * p.x_stride[t][2] + e;
      T* y = reinterpret_cast<T*>(p.y[t]) + b * p.y_stride[t][0] + row * p.y_stride[t][1] + first * p.y_stride[t][2] + e;
      if (rotates) walk_heads<kType, kHalf, kVec, true>(x, y, p.x_stride[t][2], p.y_stride[t][2], end - first, p.n_pairs, c, s);
      else walk_heads<kType, kHalf, kVec, false>(x, y, p.x_stride[t][2], p.y_stride[t][2], end - first, p.n_pairs, c, s);
    }
  }
}

template <int kType, bool kHalf, int kVec>
int launch_variant(RotaryParams& p, bool copy_rest, cudaStream_t stream) {
  p.rot_units = p.n_pairs / Layout<kType, kHalf, kVec>::kPairs;
  p.units = p.rot_units + (copy_rest ? (p.D - 2 * p.n_pairs) / kVec : 0);
  if (p.units == 0) return 0;
  p.tokens_per_cta = p.units < kThreadsR ? kThreadsR / p.units : 1;
  const int heads = p.H[0] + p.H[1];
  const long long tokens = (long long)p.B * p.L, ctas = (tokens + p.tokens_per_cta - 1) / p.tokens_per_cta;
  if (ctas > 0x7fffffffLL) return -10;
  // Up to kMaxHeads heads share one computation of the angles; a CTA takes fewer, eight at least, where that leaves four waves of
  // 148 x 8 CTAs or less, and single heads where the launch would not fill the GPU (one new token: latency is all).
  constexpr int kMaxHeads = 16;
  long long per = ctas * heads / (148 * 8 * 4);
  per = per > kMaxHeads ? kMaxHeads : (per < 8 ? 8 : per / 4 * 4);
  if (ctas * ((heads + per - 1) / per) < 148 * 8) per = 1;
  if ((heads + per - 1) / per > 65535) per = (heads + 65534) / 65535;
  p.heads_per_cta = (int)per;
  rotary_kernel<kType, kHalf, kVec><<<dim3((unsigned)ctas, (unsigned)((heads + per - 1) / per)), kThreadsR, 0, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? 0 : -8;
}

template <int kType>
int launch_type(RotaryParams& p, bool half, bool vec, bool copy_rest, cudaStream_t stream) {
  constexpr int kWide = 16 / (int)sizeof(typename Elem<kType>::T);
  if (half) return vec ? launch_variant<kType, true, kWide>(p, copy_rest, stream) : launch_variant<kType, true, 1>(p, copy_rest, stream);
  return vec ? launch_variant<kType, false, kWide>(p, copy_rest, stream) : launch_variant<kType, false, 1>(p, copy_rest, stream);
}

}  // namespace

int launch_rotary(RotaryParams& p, int type, bool half, cudaStream_t stream) {
  const int es = type == 2 ? 4 : 2, wide = 16 / es;
  // 16-byte accesses: addresses and strides allow them, and the rotated part (half layout: either half of it) and the rest are
  // whole 16-byte units
  bool vec = (half ? p.n_pairs : 2 * p.n_pairs) % wide == 0 && p.D % wide == 0;
  bool copy_rest = false;
  for (int t = 0; t < 2; ++t) {
    if (p.H[t] == 0) continue;
    vec = vec && ((reinterpret_cast<uintptr_t>(p.x[t]) | reinterpret_cast<uintptr_t>(p.y[t])) & 15) == 0;
    bool same = p.x[t] == p.y[t];
    for (int i = 0; i < 3; ++i) {
      vec = vec && p.x_stride[t][i] % wide == 0 && p.y_stride[t][i] % wide == 0;
      same = same && p.x_stride[t][i] == p.y_stride[t][i];
    }
    copy_rest = copy_rest || !same;
  }
  copy_rest = copy_rest && 2 * p.n_pairs < p.D;
  if (type == 0) return launch_type<0>(p, half, vec, copy_rest, stream);
  if (type == 1) return launch_type<1>(p, half, vec, copy_rest, stream);
  return launch_type<2>(p, half, vec, copy_rest, stream);
}

}  // namespace mcs
