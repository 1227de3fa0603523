// What the kernels of the attention's backward pass share: tile geometry, operand descriptors, the copy of a resident tile and
// the two elementwise steps on score tiles.
//
//   P = exp(scale Q K^T - lse)      dV = P^T dO      dP = dO V^T      dS = P o (dP - delta)      delta = rowsum(dO o O)
//   dQ = scale dS K                 dK = scale dS^T Q
//
// P is recomputed from the forward pass's log-sum-exp.  Scores, P, dP and dS are fp32 up to the one rounding of P and of dS to
// the inputs' type that makes them operands of the next product; every sum is fp32.
//
// fp16 inputs: P and dS have to be fp16 operands, whose normal range ends at 2^-14.  P (at most 1) is taken times 2^14
// (kBiasFp16, added to the exponent), and dS further times a power of two per (batch, head) that keeps the bound
// |dS| <= 2 max|dO row| max|V row| (finite rows, keys that take part) below 2^15; the factors are taken out of the sums in the epilogue.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernels.cuh"
#include "ptx.cuh"

namespace mcs {
namespace bwd {

constexpr float kBiasFp16 = 14.f;
constexpr int kSoftmaxWarps = 8;       // warps 0-3 take the first half of a score tile's columns, 4-7 the second; lane == row

// Row of q, out, dout and dq at position pos < Sq of head bh's order; -1, a row that is not there, for an entry of perm out of range: what
// is written through it must stay inside dq.
__device__ __forceinline__ int query_row(const AttnBwdParams& p, int bh, int pos) {
  if (p.perm == nullptr) return pos;
  const int64_t row = p.perm[(size_t)bh * p.Sq + pos];
  return row >= 0 && row < p.Sq ? (int)row : -1;
}

// Power of two by which dS / 2^14 may be multiplied (see above), from the largest row norms; 1 for bf16.  A whole warp calls it.
constexpr int kMaxBlocks = 64;          // CTAs per head of the statistics, each of which leaves its own maxima
template <bool kFp16>
__device__ __forceinline__ float ds_scale(const AttnBwdParams& p, int bh) {
  if constexpr (!kFp16) return 1.f;
  const int lane = threadIdx.x & 31;
  const float2* parts = p.row_max + (size_t)bh * kMaxBlocks;
  float2 v = make_float2(0.f, 0.f);
  for (int i = lane; i < p.max_blocks; i += 32) {
    const float2 m = parts[i];
    v = make_float2(fmaxf(v.x, m.x), fmaxf(v.y, m.y));
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) {
    v.x = fmaxf(v.x, __shfl_xor_sync(0xffffffffu, v.x, off));
    v.y = fmaxf(v.y, __shfl_xor_sync(0xffffffffu, v.y, off));
  }
  const float m = 2.f * v.x * v.y;
  if (!(m > 0.f) || isinf(m)) return 1.f;
  int e;
  frexpf(m, &e);                        // m < 2^e
  e = 1 - e;
  e = e < -60 ? -60 : (e > 60 ? 60 : e);
  return ldexpf(1.f, e);
}

// Streamed tiles have TN rows, resident tiles 128; both are DB column blocks of 64 elements (128 bytes, swizzled).
template <int DB, int TN>
struct Geo {
  static constexpr int kResBytes = DB * 16384;
  static constexpr int kTileBytes = DB * TN * 128;
  static constexpr int kHalf = TN / 2;                       // score columns of one softmax thread
};

constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);     // SBO 1024, version 1, 128-byte swizzle
__device__ __forceinline__ uint64_t desc_lo(uint32_t lo) { return (static_cast<uint64_t>(kDescHi) << 32) | lo; }
__device__ __forceinline__ uint32_t lo_kmajor(uint32_t saddr) { return ((saddr & 0x3FFFFu) >> 4) | ((16u >> 4) << 16); }
// MN-major operand: `block_bytes` from one block of 64 columns to the next
__device__ __forceinline__ uint32_t lo_mnmajor(uint32_t saddr, uint32_t block_bytes) { return ((saddr & 0x3FFFFu) >> 4) | ((block_bytes >> 4) << 16); }

// One warp copies 32 rows (lane i's row from source row `mine`, or zeros if that is negative) of D elements into rows r0 .. r0 + 31 of a
// tile of column blocks of block_rows rows.  Columns from D on are zeros.
template <int DB>
__device__ __forceinline__ void warp_copy_rows(uint32_t tile, int block_rows, int r0, int mine, int D, const uint8_t* base, size_t row_bytes, const void* any) {
  const int lane = threadIdx.x & 31;
  constexpr int kChunks = DB * 8;                            // 16-byte chunks of a row
  if constexpr (32 % kChunks == 0) {
    // a lane keeps its chunk, 32 / kChunks rows at a time
    constexpr int kRows = 32 / kChunks;
    const int c = lane % kChunks, sub = lane / kChunks;
    const uint8_t* src = base + c * 16;
    const uint32_t dst = tile + (c >> 3) * (block_rows * 128);
    const bool in = c * 8 < D;
#pragma unroll 8
    for (int i = 0; i < kChunks; ++i) {
      const int rl = i * kRows + sub, r = r0 + rl;
      const int id = __shfl_sync(0xffffffffu, mine, rl);
      const uint32_t at = dst + r * 128 + (((c & 7) ^ (r & 7)) << 4);
      if (in && id >= 0) cp_async16(at, src + (size_t)(uint32_t)id * row_bytes);
      else cp_async16_zfill(at, any, 0);
    }
  } else {
#pragma unroll 4
    for (int i = 0; i < kChunks; ++i) {
      const int e = i * 32 + lane, rl = e / kChunks, c = e % kChunks, r = r0 + rl;
      const int id = __shfl_sync(0xffffffffu, mine, rl);
      const uint32_t at = tile + (c >> 3) * (block_rows * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
      if (id >= 0 && c * 8 < D) cp_async16(at, base + (size_t)(uint32_t)id * row_bytes + c * 16);
      else cp_async16_zfill(at, any, 0);
    }
  }
}

template <bool kFp16>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if constexpr (kFp16) return pack_f16x2(a, b);
  else return pack_bf16x2(a, b);
}

// N consecutive fp32 columns of this thread's lane (N a multiple of 32); complete after tmem_wait_ld
template <int N>
__device__ __forceinline__ void load_columns(uint32_t taddr, uint32_t* r) {
#pragma unroll
  for (int q = 0; q < N; q += 32) tmem_ld32(taddr + q, *reinterpret_cast<uint32_t(*)[32]>(r + q));
}
// lo += the lower, hi += the upper of two 16-bit values: fp32 additions that take the 16-bit operand as it is
template <bool kFp16>
__device__ __forceinline__ void add_pair(uint32_t u, float& lo, float& hi) {
  if constexpr (kFp16)
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tadd.rn.f32.f16 %0, l, %0;\n\tadd.rn.f32.f16 %1, h, %1;\n\t}\n" : "+f"(lo), "+f"(hi) : "r"(u));
  else
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tadd.rn.f32.bf16 %0, l, %0;\n\tadd.rn.f32.bf16 %1, h, %1;\n\t}\n" : "+f"(lo), "+f"(hi) : "r"(u));
}
// sixteen fp32 values, rounded, into eight tensor-memory columns of this thread's lane
template <bool kFp16>
__device__ __forceinline__ void store_packed(uint32_t taddr, const uint32_t* v) {
  uint32_t pk[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) pk[i] = pack16<kFp16>(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
  tmem_st8(taddr, pk);
}

// what rounding a and b to 16 bits leaves of them
template <bool kFp16>
__device__ __forceinline__ void keep_rest(float& a, float& b) {
  const uint32_t u = pack16<kFp16>(a, b);
  if constexpr (kFp16) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
    a -= f.x;
    b -= f.y;
  } else {
    a -= bf16_lo(u);
    b -= bf16_hi(u);
  }
}

// eight fp32 values as one 32-byte store: a row's thread fills whole sectors
__device__ __forceinline__ void store8(float* dst, const float* f) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]),
               "f"(f[6]), "f"(f[7])
               : "memory");
}

}  // namespace bwd
}  // namespace mcs
