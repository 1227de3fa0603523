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
// half) of one token and walks over heads, so that the angles of its pairs are computed once for all its heads.
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
__global__ void __launch_bounds__(kThreadsR) rotary_kernel(const __grid_constant__ RotaryParams p) {
  using E = Elem<kType>;
  using T = typename E::T;
  // pairs per unit, and the elements of either member that one unit reads
  constexpr int kPairs = kHalf ? kVec : (kVec > 1 ? kVec / 2 : 1);
  constexpr bool kSplit = kHalf || kVec == 1;                // the members of a pair come from two accesses
  using V = Pack<T, kVec>;
  const long long idx = (long long)blockIdx.x * kThreadsR + threadIdx.x;
  const int unit = (int)(idx % p.units);
  const long long rest = idx / p.units;
  const long long tokens = (long long)p.B * p.L;
  const long long chunk = rest / tokens;
  if (chunk >= p.head_chunks) return;
  const long long token = rest - chunk * tokens;
  const long long b = token / p.L, row = token - b * p.L;
  const bool rotates = unit < p.rot_units;

  float c[kPairs], s[kPairs];
  int ea, eb;                                                // first elements of the two accesses
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
    ea = kHalf ? unit * kVec : unit * (kVec > 1 ? kVec : 2);
    eb = kHalf ? ea + p.n_pairs : ea + 1;
  } else {
    ea = eb = 2 * p.n_pairs + (unit - p.rot_units) * kVec;
  }

  const int heads = p.H[0] + p.H[1];
  const int h_begin = (int)chunk * p.heads_per_chunk;
  const int h_end = min(heads, h_begin + p.heads_per_chunk);
  constexpr int kUnroll = kSplit ? 2 : 4;
  for (int h0 = h_begin; h0 < h_end; h0 += kUnroll) {
    V xa[kUnroll], xb[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int h = h0 + u;
      if (h < h_end) {
        const int t = h >= p.H[0];
        const T* x = reinterpret_cast<const T*>(p.x[t]) + b * p.x_stride[t][0] + row * p.x_stride[t][1] +
                     (long long)(h - (t ? p.H[0] : 0)) * p.x_stride[t][2];
        xa[u] = *reinterpret_cast<const V*>(x + ea);
        if (kSplit && rotates) xb[u] = *reinterpret_cast<const V*>(x + eb);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int h = h0 + u;
      if (h >= h_end) break;
      const int t = h >= p.H[0];
      T* y = reinterpret_cast<T*>(p.y[t]) + b * p.y_stride[t][0] + row * p.y_stride[t][1] +
             (long long)(h - (t ? p.H[0] : 0)) * p.y_stride[t][2];
      if (rotates) {
        if constexpr (kSplit) {
          V ya, yb;
#pragma unroll
          for (int j = 0; j < kPairs; ++j) {
            const float a = E::get(xa[u].v[j]), d = E::get(xb[u].v[j]);
            ya.v[j] = E::put(fmaf(a, c[j], -d * s[j]));
            yb.v[j] = E::put(fmaf(a, s[j], d * c[j]));
          }
          *reinterpret_cast<V*>(y + ea) = ya;
          *reinterpret_cast<V*>(y + eb) = yb;
        } else {
          V ya;
#pragma unroll
          for (int j = 0; j < kPairs; ++j) {
            const float a = E::get(xa[u].v[2 * j]), d = E::get(xa[u].v[2 * j + 1]);
            ya.v[2 * j] = E::put(fmaf(a, c[j], -d * s[j]));
            ya.v[2 * j + 1] = E::put(fmaf(a, s[j], d * c[j]));
          }
          *reinterpret_cast<V*>(y + ea) = ya;
        }
      } else {
        *reinterpret_cast<V*>(y + ea) = xa[u];
      }
    }
  }
}

template <int kType, bool kHalf, int kVec>
int launch_variant(RotaryParams& p, bool copy_rest, cudaStream_t stream) {
  constexpr int kPairs = kHalf ? kVec : (kVec > 1 ? kVec / 2 : 1);
  p.rot_units = p.n_pairs / kPairs;
  p.units = p.rot_units + (copy_rest ? (p.D - 2 * p.n_pairs) / kVec : 0);
  if (p.units == 0) return 0;
  const int heads = p.H[0] + p.H[1];
  const long long per_head = (long long)p.B * p.L * p.units;
  // Few tokens: a thread takes fewer heads, so that the launch still fills the GPU (148 SMs x 8 CTAs); many tokens: up to
  // kMaxHeads heads share one computation of the angles.
  constexpr int kMaxHeads = 16;
  const long long want = 148LL * 8 * kThreadsR;
  long long per = per_head >= want ? kMaxHeads : per_head * heads / want;
  if (per < 1) per = 1;
  if (per > kMaxHeads) per = kMaxHeads;
  p.heads_per_chunk = (int)per;
  p.head_chunks = (heads + p.heads_per_chunk - 1) / p.heads_per_chunk;
  const long long blocks = (per_head * p.head_chunks + kThreadsR - 1) / kThreadsR;
  if (blocks > 0x7fffffffLL) return -10;
  rotary_kernel<kType, kHalf, kVec><<<(unsigned)blocks, kThreadsR, 0, stream>>>(p);
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
