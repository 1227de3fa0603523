// Backward pass of the attention for sm_100a (bf16 / fp16, head dimensions up to 256): row statistics, the kernel of dQ (dense
// and gathered keys), the kernel of dK and dV of the dense call, and the sums of split launches.  The kernel of dK and dV of
// gathered keys is in attn_bwd_gather.cu.
//
// Two kernels, one per side, instead of one that forms all five products of a tile pair: dQ sums over keys and dK, dV over
// queries, so a kernel that makes them all has to add one side's partial sums in global memory with atomics (order, and with it
// bits, would change from run to run) and needs one operand of dS transposed in shared memory.  Each kernel here keeps its own
// side's sums in tensor memory, takes P and dS straight out of tensor memory as the first operand of the next product, and
// writes every result once.  The price is two products more (7 instead of 5): S and dP are computed on either side.
#include "attn_bwd.cuh"

namespace mcs {

namespace {

using namespace bwd;

constexpr int kMaxSmem = 232448;

// ------------------------------------------------------------------------------------------------ row statistics
// One CTA of 256 threads takes 16 rows at a time, 16 lanes each: neg_delta = -sum(dout * out) and neg_lse2 of every tile row
// (memory-bound: dout and out are read once), and for fp16 the largest norms of rows of dout and of v.
template <bool kFp16>
__device__ __forceinline__ float dot8(uint4 a, uint4 b, float acc) {
  const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (kFp16) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x[i])), g = __half22float2(*reinterpret_cast<const __half2*>(&y[i]));
      acc = fmaf(f.x, g.x, fmaf(f.y, g.y, acc));
    } else {
      acc = fmaf(bf16_lo(x[i]), bf16_lo(y[i]), fmaf(bf16_hi(x[i]), bf16_hi(y[i]), acc));
    }
  }
  return acc;
}

template <bool kFp16>
__global__ void __launch_bounds__(256) attn_bwd_stats_kernel(const AttnBwdParams p) {
  const int bh = blockIdx.y, h = bh % p.H, b = bh / p.H;
  const int l16 = threadIdx.x & 15, sub = threadIdx.x >> 4;
  const int rows = p.M * 128;
  const int total = rows + (kFp16 ? p.Sk : 0);
  const int chunks = p.D / 8;
  float m_do = 0.f, m_v = 0.f;
  for (int base = blockIdx.x * 16; base < total; base += gridDim.x * 16) {
    const int i = base + sub;
    float dot = 0.f, sq = 0.f;
    int row = -1;
    if (i < rows) {
      const int r = i & 127, pos = (i >> 7) * p.group_rows + r;
      if (r < p.group_rows && pos < p.Sq) row = p.perm != nullptr ? (int)p.perm[(size_t)bh * p.Sq + pos] : pos;
      if (row >= 0) {
        const uint8_t* g = reinterpret_cast<const uint8_t*>(p.dout) + 2 * ((size_t)b * p.dout_stride[0] + (size_t)row * p.dout_stride[1] + (size_t)h * p.dout_stride[2]);
        const uint8_t* o = reinterpret_cast<const uint8_t*>(p.out) + 2 * ((size_t)b * p.out_stride[0] + (size_t)row * p.out_stride[1] + (size_t)h * p.out_stride[2]);
        for (int c = l16; c < chunks; c += 16) {
          const uint4 x = *reinterpret_cast<const uint4*>(g + c * 16), y = *reinterpret_cast<const uint4*>(o + c * 16);
          dot = dot8<kFp16>(x, y, dot);
          if constexpr (kFp16) sq = dot8<kFp16>(x, x, sq);
        }
      }
    } else if (i < total) {
      const uint8_t* v = reinterpret_cast<const uint8_t*>(p.v) + 2 * ((size_t)b * p.v_stride[0] + (size_t)(i - rows) * p.v_stride[1] + (size_t)h * p.v_stride[2]);
      for (int c = l16; c < chunks; c += 16) {
        const uint4 x = *reinterpret_cast<const uint4*>(v + c * 16);
        sq = dot8<kFp16>(x, x, sq);
      }
    }
#pragma unroll
    for (int off = 8; off >= 1; off >>= 1) {
      dot += __shfl_xor_sync(0xffffffffu, dot, off);
      if constexpr (kFp16) sq += __shfl_xor_sync(0xffffffffu, sq, off);
    }
    if (i < rows) {
      if (l16 == 0) {
        float nl = -INFINITY, nd = 0.f;                      // rows behind the last one: P = 0
        if (row >= 0) {
          const float l = p.lse[(size_t)bh * p.Sq + row];
          // (a row without keys has lse = -inf and no gradient)
          if (l != -INFINITY) nl = (kFp16 ? kBiasFp16 : 0.f) - l * 1.4426950408889634f;
          nd = -dot;
        }
        p.neg_lse2[(size_t)bh * rows + i] = nl;
        p.neg_delta[(size_t)bh * rows + i] = nd;
      }
      if constexpr (kFp16) m_do = fmaxf(m_do, sq);
    } else if constexpr (kFp16) {
      m_v = fmaxf(m_v, sq);
    }
  }
  if constexpr (kFp16) {
    __shared__ float red[2][8];
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
      m_do = fmaxf(m_do, __shfl_xor_sync(0xffffffffu, m_do, off));
      m_v = fmaxf(m_v, __shfl_xor_sync(0xffffffffu, m_v, off));
    }
    if ((threadIdx.x & 31) == 0) { red[0][threadIdx.x >> 5] = m_do; red[1][threadIdx.x >> 5] = m_v; }
    __syncthreads();
    if (threadIdx.x < 2) {
      float m = 0.f;
      for (int i = 0; i < 8; ++i) m = fmaxf(m, red[threadIdx.x][i]);
      // (non-negative floats compare as their bits; the largest of a set does not depend on the order)
      atomicMax(p.row_max + 2 * bh + threadIdx.x, __float_as_uint(sqrtf(m) * 1.0001f));
    }
  }
}

// ------------------------------------------------------------------------------------------------ dQ
// One CTA per SM walks items (head, tile of 128 query rows, split of the keys).  Q and dO of the tile stay in shared memory, K and
// V tiles of TN keys come through a ring (TMA boxes, or rows gathered by index).  Per key tile t:
//     S(t) = Q K^T -> tensor memory, one of two buffers      P = exp2(scale S - lse2) in registers
//     dP(t) = dO V^T                                          dS = P (dP - delta), stored over S(t) as the operand of
//     dQ += dS(t) K(t)                                        (K tile read a second time, as an MN-major operand)
// Issue order dP(t), S(t+1), dQ(t): the softmax of t+1 has its scores before dQ(t) ends.
template <int DB, int TN>
struct SmemQ {
  using G = Geo<DB, TN>;
  static constexpr int kRing = DB == 4 ? 3 : 5;
  static constexpr int kQ = 0, kDO = G::kResBytes;
  static constexpr int kRingOff = 2 * G::kResBytes;
  static constexpr int kBars = kRingOff + kRing * G::kTileBytes;
  static constexpr int kFull = 0, kEmpty = kRing, kQFull = 2 * kRing, kQEmpty = kQFull + 1, kSFull = kQEmpty + 1, kDPFull = kSFull + 2,
                       kDPFree = kDPFull + 1, kDSReady = kDPFree + 1, kOFull = kDSReady + 2, kOFree = kOFull + 1, kDrain = kOFree + 1, kCount = kDrain + 1;
  static constexpr int kSlot = kBars + kCount * 8;
  static constexpr int kDynamic = kSlot + 16 + 1024;
};
static_assert(SmemQ<2, 128>::kDynamic <= kMaxSmem && SmemQ<4, 64>::kDynamic <= kMaxSmem, "must fit 227 KB");

constexpr int kIssueWarp = 8, kLoadWarp0 = 9;                // issuer, two copies of resident tiles, then the ring's producers
constexpr int kRingWarp0 = 11;

template <int DB, int TN, bool kFp16, bool kGather>
__global__ void __launch_bounds__(kGather ? 480 : 384, 1) attn_bwd_dq_kernel(const AttnBwdParams p, const __grid_constant__ DenseTileMaps maps) {
  using L = SmemQ<DB, TN>;
  using G = Geo<DB, TN>;
  constexpr int R = L::kRing, HC = G::kHalf;
  constexpr uint32_t kColS = 0, kColDP = 2 * TN, kColO = 3 * TN;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t s_base = smem_u32(smem);
  auto bar = [&](int i) { return s_base + L::kBars + 8u * i; };
  auto sRing = [&](int slot) { return s_base + L::kRingOff + slot * G::kTileBytes; };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kSlot);
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int n_items = p.B * p.H * p.M * p.splits;
  const int nd = (p.D + 15) & ~15, kd = nd / 16;             // columns and k-steps that are not padding
  struct Item { int bh, b, h, m, split, t0, t1; };
  auto decode = [&](int item) {
    Item it;
    it.split = item % p.splits;
    const int rest = item / p.splits;
    it.m = rest % p.M;
    it.bh = rest / p.M;
    it.b = it.bh / p.H;
    it.h = it.bh % p.H;
    int T;
    if constexpr (kGather) {
      const int most = p.gather_len / 128;
      T = (p.gl != nullptr ? min(max(p.gl[(size_t)it.bh * p.M + it.m], 1), most) : most) * (128 / TN);
    } else {
      T = (p.Sk + TN - 1) / TN;
    }
    it.t0 = (int)((long long)T * it.split / p.splits);
    it.t1 = (int)((long long)T * (it.split + 1) / p.splits);
    return it;
  };
  // query row behind tile row r, or -1
  auto row_of = [&](const Item& it, int r) {
    const int pos = it.m * p.group_rows + r;
    if (r >= p.group_rows || pos >= p.Sq) return -1;
    return p.perm != nullptr ? (int)p.perm[(size_t)it.bh * p.Sq + pos] : pos;
  };

  if (tid == 0) {
    for (int i = 0; i < R; ++i) { mbar_init(bar(L::kFull + i), kGather ? 128 : 1); mbar_init(bar(L::kEmpty + i), 1); }
    mbar_init(bar(L::kQFull), 64);
    mbar_init(bar(L::kQEmpty), 1);
    for (int i = 0; i < 2; ++i) { mbar_init(bar(L::kSFull + i), 1); mbar_init(bar(L::kDSReady + i), kSoftmaxWarps); }
    mbar_init(bar(L::kDPFull), 1);
    mbar_init(bar(L::kDPFree), kSoftmaxWarps);
    mbar_init(bar(L::kOFull), 1);
    mbar_init(bar(L::kOFree), kSoftmaxWarps);
    mbar_init(bar(L::kDrain), 1);
    mbar_fence_init();
  }
  if (warp == kIssueWarp) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp < kSoftmaxWarps) {
    auto warp_arrive = [&](uint32_t b) {
      __syncwarp();
      if (lane == 0) mbar_arrive(b);
    };
    const int x = warp >> 2, r_in = (warp & 3) * 32 + lane;
    const uint32_t lane_addr = (static_cast<uint32_t>(warp & 3) * 32u) << 16;
    const unsigned long long scale2 = f2_pack(p.scale_log2, p.scale_log2);
    int g = 0, ic = 0;
    bool ok = true;
#pragma unroll 1
    for (int item = blockIdx.x; item < n_items && ok; item += gridDim.x) {
      const Item it = decode(item);
      const size_t si = ((size_t)it.bh * p.M + it.m) * 128 + r_in;
      const float nl = p.neg_lse2[si], ndl = p.neg_delta[si];
      const unsigned long long nl2 = f2_pack(nl, nl), nd2 = f2_pack(ndl, ndl);
      const float c = ds_scale<kFp16>(p.row_max, it.bh);
      const unsigned long long c2 = f2_pack(c, c);
#pragma unroll 1
      for (int t = it.t0; t < it.t1; ++t, ++g) {
        const uint32_t tS = tmem + kColS + (g & 1) * TN + x * HC + lane_addr;
        ok = mbar_wait(bar(L::kSFull + (g & 1)), (g >> 1) & 1, p.status, 130);
        if (!ok) break;
        tc_fence_after();
        uint32_t sc[HC];
#pragma unroll
        for (int q = 0; q < HC / 32; ++q) tmem_ld32(tS + q * 32, *reinterpret_cast<uint32_t(*)[32]>(&sc[q * 32]));
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < HC; i += 2) {
          const float2 y = f2_unpack(f2_fma(f2_pack(__uint_as_float(sc[i]), __uint_as_float(sc[i + 1])), scale2, nl2));
          sc[i] = __float_as_uint(ex2_approx(y.x));
          sc[i + 1] = __float_as_uint(ex2_approx(y.y));
        }
        if constexpr (!kGather) {
          // key positions behind the sequence end (zero rows of the last tile): exp2(-lse2) could be anything
          const int rem = p.Sk - t * TN - x * HC;
          if (rem < HC) {
#pragma unroll
            for (int i = 0; i < HC; ++i)
              if (i >= rem) sc[i] = 0;
          }
        }
        ok = mbar_wait(bar(L::kDPFull), g & 1, p.status, 131);
        if (!ok) break;
        tc_fence_after();
        uint32_t dp[HC];
#pragma unroll
        for (int q = 0; q < HC / 32; ++q) tmem_ld32(tmem + kColDP + x * HC + lane_addr + q * 32, *reinterpret_cast<uint32_t(*)[32]>(&dp[q * 32]));
        tmem_wait_ld();
        tc_fence_before();
        warp_arrive(bar(L::kDPFree));                        // dP of the next tile may overwrite it
#pragma unroll
        for (int q = 0; q < HC / 16; ++q) {
          uint32_t pk[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int e = q * 16 + 2 * i;
            unsigned long long d = f2_add(f2_pack(__uint_as_float(dp[e]), __uint_as_float(dp[e + 1])), nd2);
            if constexpr (kFp16) d = f2_mul(d, c2);
            const float2 y = f2_unpack(f2_mul(f2_pack(__uint_as_float(sc[e]), __uint_as_float(sc[e + 1])), d));
            pk[i] = pack16<kFp16>(y.x, y.y);
          }
          tmem_st8(tS + q * 8, pk);                          // each half stays inside its own columns
        }
        tmem_wait_st();
        tc_fence_before();
        warp_arrive(bar(L::kDSReady + (g & 1)));
      }
      if (!ok) break;
      // ---- dQ row: this thread's half of the columns (in steps of 16)
      ok = mbar_wait(bar(L::kOFull), ic & 1, p.status, 132);
      if (!ok) break;
      tc_fence_after();
      const int row = row_of(it, r_in);
      const float w = p.out_scale / c * (kFp16 ? 6.103515625e-05f : 1.f);      // 2^-14
      const int c_mid = ((kd + 1) / 2) * 16, c0 = x ? c_mid : 0, c1 = x ? nd : c_mid;
      uint8_t* optr = reinterpret_cast<uint8_t*>(p.dq) + 2 * ((size_t)it.b * p.dq_stride[0] + (size_t)(row < 0 ? 0 : row) * p.dq_stride[1] + (size_t)it.h * p.dq_stride[2]);
      float* part = p.parts + (((size_t)it.split * p.B * p.H + it.bh) * p.Sq + (row < 0 ? 0 : row)) * p.D;
#pragma unroll 1
      for (int cc = c0; cc < c1; cc += 16) {
        uint32_t r[16];
        tmem_ld16(tmem + kColO + lane_addr + cc, r);
        tmem_wait_ld();
        float f[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] = __uint_as_float(r[i]) * w;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          if (row < 0 || cc + q * 8 >= p.D) break;
          if (p.splits > 1) {
            float4* o = reinterpret_cast<float4*>(part + cc + q * 8);
            o[0] = make_float4(f[q * 8], f[q * 8 + 1], f[q * 8 + 2], f[q * 8 + 3]);
            o[1] = make_float4(f[q * 8 + 4], f[q * 8 + 5], f[q * 8 + 6], f[q * 8 + 7]);
          } else {
            *reinterpret_cast<uint4*>(optr + 2 * (cc + q * 8)) =
                make_uint4(pack16<kFp16>(f[q * 8], f[q * 8 + 1]), pack16<kFp16>(f[q * 8 + 2], f[q * 8 + 3]),
                           pack16<kFp16>(f[q * 8 + 4], f[q * 8 + 5]), pack16<kFp16>(f[q * 8 + 6], f[q * 8 + 7]));
          }
        }
        __syncwarp();
      }
      tc_fence_before();
      warp_arrive(bar(L::kOFree));
      ++ic;
    }
    tc_fence_before();
  } else if (warp == kIssueWarp) {
    // ---- issuer of every product
    constexpr uint32_t kFmt = kFp16 ? 0u : 1u;
    constexpr uint32_t idesc_s = mma_idesc(kFmt, kFmt, 0, 0, 128, TN);
    const uint32_t idesc_o = mma_idesc(kFmt, kFmt, 0, 1, 128, nd);
    const bool leader = elect_one();
    bool ok = true;
    int g = 0, ic = 0;
    int n = 0;                                               // ring position: K(t) is load 2 g, V(t) load 2 g + 1
    auto wait_full = [&](int load) {
      ok = ok && mbar_wait(bar(L::kFull + load % R), (load / R) & 1, p.status, 133);
      if (!ok) return;
      if constexpr (kGather) fence_proxy_async_smem();
      tc_fence_after();
    };
    // (unrolled, the k-steps of padding predicated off: with a rolled loop of kd steps one of the products in the kernel of dK and dV
    // had its last step accumulated nine times)
    auto qk = [&](uint32_t d, uint32_t a_tile, uint32_t b_tile) {
      const uint32_t alo = lo_kmajor(a_tile), blo = lo_kmajor(b_tile);
#pragma unroll
      for (int j = 0; j < DB * 4; ++j) {
        const uint32_t in = (j & 3) * 2;
        if (leader && j < kd) mma_f16_ss(d, desc_lo(alo + (j >> 2) * (16384 >> 4) + in), desc_lo(blo + (j >> 2) * (TN * 128 >> 4) + in), idesc_s, j > 0);
      }
    };
#pragma unroll 1
    for (int item = blockIdx.x; item < n_items && ok; item += gridDim.x) {
      const Item it = decode(item);
      ok = mbar_wait(bar(L::kQFull), ic & 1, p.status, 134);
      if (!ok) break;
      fence_proxy_async_smem();
      tc_fence_after();
      wait_full(n);
      if (!ok) break;
      qk(tmem + kColS + (g & 1) * TN, s_base + L::kQ, sRing(n % R));
      if (leader) tc_commit(bar(L::kSFull + (g & 1)));
#pragma unroll 1
      for (int t = it.t0; t < it.t1; ++t, ++g, n += 2) {
        wait_full(n + 1);
        if (ok && g > 0) ok = mbar_wait(bar(L::kDPFree), (g - 1) & 1, p.status, 135);
        if (!ok) break;
        tc_fence_after();
        qk(tmem + kColDP, s_base + L::kDO, sRing((n + 1) % R));
        if (leader) {
          tc_commit(bar(L::kDPFull));
          tc_commit(bar(L::kEmpty + (n + 1) % R));
          if (t == it.t1 - 1) tc_commit(bar(L::kQEmpty));
        }
        if (t + 1 < it.t1) {
          wait_full(n + 2);
          if (!ok) break;
          qk(tmem + kColS + ((g + 1) & 1) * TN, s_base + L::kQ, sRing((n + 2) % R));
          if (leader) tc_commit(bar(L::kSFull + ((g + 1) & 1)));
        }
        ok = mbar_wait(bar(L::kDSReady + (g & 1)), (g >> 1) & 1, p.status, 136);
        if (ok && t == it.t0 && ic > 0) ok = mbar_wait(bar(L::kOFree), (ic - 1) & 1, p.status, 137);
        if (!ok) break;
        tc_fence_after();
        const uint32_t blo = lo_mnmajor(sRing(n % R), TN * 128);
        const uint32_t a = tmem + kColS + (g & 1) * TN;
#pragma unroll
        for (int j = 0; j < TN / 16; ++j)
          if (leader) mma_f16_ts(tmem + kColO, a + (j / (TN / 32)) * HC + (j % (TN / 32)) * 8, desc_lo(blo + j * (2048 >> 4)), idesc_o, t > it.t0 || j > 0);
        if (leader) {
          tc_commit(bar(L::kEmpty + n % R));
          if (t == it.t1 - 1) tc_commit(bar(L::kOFull));
        }
      }
      ++ic;
    }
    if (!ok) {
      // error path: let outstanding products retire before tensor memory is released
      if (leader) tc_commit(bar(L::kDrain));
      mbar_wait_quiet(bar(L::kDrain), 0, 1 << 20);
    }
    __syncwarp();
    tc_fence_before();
  } else if (warp < kRingWarp0) {
    // ---- Q (first warp) and dO (second) of an item, rows through the permutation
    const bool is_do = warp != kLoadWarp0;
    const void* src = is_do ? p.dout : p.q;
    const int64_t* st = is_do ? p.dout_stride : p.q_stride;
    int ic = 0;
    bool ok = true;
#pragma unroll 1
    for (int item = blockIdx.x; item < n_items && ok; item += gridDim.x) {
      const Item it = decode(item);
      if (ic > 0) ok = mbar_wait(bar(L::kQEmpty), (ic - 1) & 1, p.status, 138);
      if (!ok) break;
      warp_copy_rows<DB>(s_base + (is_do ? L::kDO : L::kQ), 128, 0, 128, p.D,
                         reinterpret_cast<const uint8_t*>(src) + 2 * ((size_t)it.b * st[0] + (size_t)it.h * st[2]), 2 * (size_t)st[1], src,
                         [&](int r) { return row_of(it, r); });
      cp_async_arrive_noinc(bar(L::kQFull));
      ++ic;
    }
    cp_async_wait_all();
    tc_fence_before();
  } else {
    // ---- K and V tiles
    const bool leader = elect_one();
    int n = 0;
    bool ok = true;
#pragma unroll 1
    for (int item = blockIdx.x; item < n_items && ok; item += gridDim.x) {
      const Item it = decode(item);
      int ck[4] = {0, 0, 0, 0}, cv[4] = {0, 0, 0, 0};
      if constexpr (!kGather) {
        ck[maps.k_pos_h] = it.h; ck[maps.k_pos_b] = it.b;
        cv[maps.v_pos_h] = it.h; cv[maps.v_pos_b] = it.b;
      }
#pragma unroll 1
      for (int e = 2 * it.t0; e < 2 * it.t1 && ok; ++e, ++n) {
        const bool is_v = e & 1;
        const int slot = n % R;
        if (n >= R) ok = mbar_wait(bar(L::kEmpty + slot), (n / R - 1) & 1, p.status, 139);
        if (!ok) break;
        if constexpr (kGather) {
          constexpr int kRows = TN / 4;
          const int w = warp - kRingWarp0;
          const int32_t* gi = p.gi + ((size_t)it.bh * p.M + it.m) * p.gather_len + (size_t)(e >> 1) * TN;
          const int64_t* st = is_v ? p.v_stride : p.k_stride;
          const void* src = is_v ? p.v : p.k;
          warp_copy_rows<DB>(sRing(slot), TN, w * kRows, kRows, p.D,
                             reinterpret_cast<const uint8_t*>(src) + 2 * ((size_t)it.b * st[0] + (size_t)it.h * st[2]), 2 * (size_t)st[1], src,
                             [&](int r) { return min(max(gi[r], 0), p.Sk - 1); });
          cp_async_arrive_noinc(bar(L::kFull + slot));
        } else if (leader) {
          mbar_arrive_expect_tx(bar(L::kFull + slot), G::kTileBytes);
          const void* map = is_v ? static_cast<const void*>(maps.v) : static_cast<const void*>(maps.k);
          int co[4] = {0, is_v ? cv[1] : ck[1], is_v ? cv[2] : ck[2], is_v ? cv[3] : ck[3]};
          co[is_v ? maps.v_pos_row : maps.k_pos_row] = (e >> 1) * TN;
#pragma unroll
          for (int cb = 0; cb < DB; ++cb)
            tma_load_4d(sRing(slot) + cb * TN * 128, map, cb * 64, co[1], co[2], co[3], bar(L::kFull + slot));
        }
      }
    }
    if constexpr (kGather) {
      cp_async_wait_all();
    } else if (!ok) {
      for (int i = n > R ? n - R : 0; i < n; ++i) mbar_wait_quiet(bar(L::kFull + i % R), (i / R) & 1, 1 << 16);   // copies in flight
    }
    tc_fence_before();
  }

  __syncthreads();
  if (warp == kIssueWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------------------------------------ dK, dV of the dense call
// One CTA per SM walks items (head, tile of 128 keys, block of up to 128 output columns, split of the queries).  K and V of the
// tile stay in shared memory, Q and dO tiles of TN rows come through a ring by TMA with their row statistics.  Scores are
// transposed, a row is a key, so that P^T and dS^T lie in tensor memory as the first operands of
//     dV += P^T dO        dK += dS^T Q
// Issue order dV(t), S(t+1), dK(t), dP(t+1): P of t+1 is computed under dK(t) and dP(t+1), dS of t under dV(t) and S(t+1).
// P^T overwrites its scores and dS^T its dP; products of one thread execute in order, so S(t+1) may follow dV(t) and dP(t+1) may
// follow dK(t) without a wait.
template <int DB, int TN>
struct SmemK {
  using G = Geo<DB, TN>;
  static constexpr int kRing = DB == 4 ? 3 : (DB == 2 ? 4 : 6);
  static constexpr int kK = 0, kV = G::kResBytes;
  static constexpr int kRingOff = 2 * G::kResBytes;
  static constexpr int kStat = kRingOff + kRing * G::kTileBytes;           // TN floats per slot: lse2 with Q, delta with dO
  static constexpr int kBars = kStat + kRing * TN * 4;
  static constexpr int kFull = 0, kEmpty = kRing, kKVFull = 2 * kRing, kKVEmpty = kKVFull + 1, kSFull = kKVEmpty + 1, kDPFull = kSFull + 1,
                       kPReady = kDPFull + 1, kDSReady = kPReady + 1, kOFull = kDSReady + 1, kOFree = kOFull + 1, kDrain = kOFree + 1, kCount = kDrain + 1;
  static constexpr int kSlot = kBars + kCount * 8;
  static constexpr int kDynamic = kSlot + 16 + 1024;
};
static_assert(SmemK<2, 128>::kDynamic <= kMaxSmem && SmemK<4, 64>::kDynamic <= kMaxSmem && SmemK<1, 128>::kDynamic <= kMaxSmem, "must fit 227 KB");

template <int DB, int TN, bool kFp16>
__global__ void __launch_bounds__(384, 1) attn_bwd_dkv_kernel(const AttnBwdParams p, const __grid_constant__ DenseTileMaps maps) {
  using L = SmemK<DB, TN>;
  using G = Geo<DB, TN>;
  constexpr int R = L::kRing, HC = G::kHalf;
  constexpr uint32_t kColS = 0, kColDP = TN, kColDV = 2 * TN, kColDK = 2 * TN + 128;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t s_base = smem_u32(smem);
  auto bar = [&](int i) { return s_base + L::kBars + 8u * i; };
  auto sRing = [&](int slot) { return s_base + L::kRingOff + slot * G::kTileBytes; };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kSlot);
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int nd = (p.D + 15) & ~15, kd = nd / 16;
  const int key_tiles = (p.Sk + 127) / 128, T = (p.Sq + TN - 1) / TN;
  const int blocks = (nd + 127) / 128;                       // output column blocks
  const int n_items = p.B * p.H * key_tiles * blocks * p.splits;
  struct Item { int bh, b, h, kt, cb, split, t0, t1, ncol; };
  auto decode = [&](int item) {
    Item it;
    it.split = item % p.splits;
    int rest = item / p.splits;
    it.cb = rest % blocks;
    rest /= blocks;
    it.kt = rest % key_tiles;
    it.bh = rest / key_tiles;
    it.b = it.bh / p.H;
    it.h = it.bh % p.H;
    it.t0 = (int)((long long)T * it.split / p.splits);
    it.t1 = (int)((long long)T * (it.split + 1) / p.splits);
    it.ncol = min(128, nd - it.cb * 128);
    return it;
  };

  if (tid == 0) {
    for (int i = 0; i < R; ++i) { mbar_init(bar(L::kFull + i), 1); mbar_init(bar(L::kEmpty + i), 1); }
    mbar_init(bar(L::kKVFull), 64);
    mbar_init(bar(L::kKVEmpty), 1);
    mbar_init(bar(L::kSFull), 1);
    mbar_init(bar(L::kDPFull), 1);
    mbar_init(bar(L::kPReady), kSoftmaxWarps);
    mbar_init(bar(L::kDSReady), kSoftmaxWarps);
    mbar_init(bar(L::kOFull), 1);
    mbar_init(bar(L::kOFree), kSoftmaxWarps);
    mbar_init(bar(L::kDrain), 1);
    mbar_fence_init();
  }
  if (warp == kIssueWarp) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp < kSoftmaxWarps) {
    auto warp_arrive = [&](uint32_t b) {
      __syncwarp();
      if (lane == 0) mbar_arrive(b);
    };
    const int x = warp >> 2, r_in = (warp & 3) * 32 + lane;
    const uint32_t lane_addr = (static_cast<uint32_t>(warp & 3) * 32u) << 16;
    const uint32_t tS = tmem + kColS + x * HC + lane_addr, tDP = tmem + kColDP + x * HC + lane_addr;
    const unsigned long long scale2 = f2_pack(p.scale_log2, p.scale_log2);
    int g = 0, ic = 0;
    bool ok = true;
#pragma unroll 1
    for (int item = blockIdx.x; item < n_items && ok; item += gridDim.x) {
      const Item it = decode(item);
      const float c = ds_scale<kFp16>(p.row_max, it.bh);
      const unsigned long long c2 = f2_pack(c, c);
#pragma unroll 1
      for (int t = it.t0; t < it.t1; ++t, ++g) {
        const int nq = 2 * g, nO = 2 * g + 1;                // ring loads of Q(t), dO(t)
        const ulonglong2* lse = reinterpret_cast<const ulonglong2*>(smem + L::kStat + (nq % R) * TN * 4 + x * HC * 4);
        const ulonglong2* dlt = reinterpret_cast<const ulonglong2*>(smem + L::kStat + (nO % R) * TN * 4 + x * HC * 4);
        ok = mbar_wait(bar(L::kSFull), g & 1, p.status, 140) && mbar_wait(bar(L::kFull + nq % R), (nq / R) & 1, p.status, 141);
        if (!ok) break;
        tc_fence_after();
        uint32_t sc[HC];
#pragma unroll
        for (int q = 0; q < HC / 32; ++q) tmem_ld32(tS + q * 32, *reinterpret_cast<uint32_t(*)[32]>(&sc[q * 32]));
        tmem_wait_ld();
#pragma unroll
        for (int q = 0; q < HC / 16; ++q) {
          uint32_t pk[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int e = q * 16 + 4 * i;
            const ulonglong2 nl = lse[q * 4 + i];
            const float2 y0 = f2_unpack(f2_fma(f2_pack(__uint_as_float(sc[e]), __uint_as_float(sc[e + 1])), scale2, nl.x));
            const float2 y1 = f2_unpack(f2_fma(f2_pack(__uint_as_float(sc[e + 2]), __uint_as_float(sc[e + 3])), scale2, nl.y));
            const float p0 = ex2_approx(y0.x), p1 = ex2_approx(y0.y), p2 = ex2_approx(y1.x), p3 = ex2_approx(y1.y);
            sc[e] = __float_as_uint(p0);
            sc[e + 1] = __float_as_uint(p1);
            sc[e + 2] = __float_as_uint(p2);
            sc[e + 3] = __float_as_uint(p3);
            pk[2 * i] = pack16<kFp16>(p0, p1);
            pk[2 * i + 1] = pack16<kFp16>(p2, p3);
          }
          tmem_st8(tS + q * 8, pk);
        }
        tmem_wait_st();
        tc_fence_before();
        warp_arrive(bar(L::kPReady));
        ok = mbar_wait(bar(L::kDPFull), g & 1, p.status, 142) && mbar_wait(bar(L::kFull + nO % R), (nO / R) & 1, p.status, 143);
        if (!ok) break;
        tc_fence_after();
        uint32_t dp[HC];
#pragma unroll
        for (int q = 0; q < HC / 32; ++q) tmem_ld32(tDP + q * 32, *reinterpret_cast<uint32_t(*)[32]>(&dp[q * 32]));
        tmem_wait_ld();
#pragma unroll
        for (int q = 0; q < HC / 16; ++q) {
          uint32_t pk[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int e = q * 16 + 4 * i;
            const ulonglong2 nd2 = dlt[q * 4 + i];
            unsigned long long d0 = f2_add(f2_pack(__uint_as_float(dp[e]), __uint_as_float(dp[e + 1])), nd2.x);
            unsigned long long d1 = f2_add(f2_pack(__uint_as_float(dp[e + 2]), __uint_as_float(dp[e + 3])), nd2.y);
            if constexpr (kFp16) { d0 = f2_mul(d0, c2); d1 = f2_mul(d1, c2); }
            const float2 y0 = f2_unpack(f2_mul(f2_pack(__uint_as_float(sc[e]), __uint_as_float(sc[e + 1])), d0));
            const float2 y1 = f2_unpack(f2_mul(f2_pack(__uint_as_float(sc[e + 2]), __uint_as_float(sc[e + 3])), d1));
            pk[2 * i] = pack16<kFp16>(y0.x, y0.y);
            pk[2 * i + 1] = pack16<kFp16>(y1.x, y1.y);
          }
          tmem_st8(tDP + q * 8, pk);
        }
        tmem_wait_st();
        tc_fence_before();
        warp_arrive(bar(L::kDSReady));
      }
      if (!ok) break;
      // ---- first half of the warps: dV rows, second half: dK rows
      ok = mbar_wait(bar(L::kOFull), ic & 1, p.status, 144);
      if (!ok) break;
      tc_fence_after();
      const int key = it.kt * 128 + r_in;
      const float unbias = kFp16 ? 6.103515625e-05f : 1.f;                     // 2^-14
      const float w = x == 0 ? unbias : p.out_scale / c * unbias;
      const uint32_t tO = tmem + (x == 0 ? kColDV : kColDK) + lane_addr;
      const int64_t* st = x == 0 ? p.dv_stride : p.dk_stride;
      uint8_t* optr = reinterpret_cast<uint8_t*>(x == 0 ? p.dv : p.dk) + 2 * ((size_t)it.b * st[0] + (size_t)min(key, p.Sk - 1) * st[1] + (size_t)it.h * st[2]);
      float* part = p.parts + ((((size_t)it.split * p.B * p.H + it.bh) * p.Sk + min(key, p.Sk - 1)) * 2 + (x == 0 ? 1 : 0)) * p.D;
#pragma unroll 1
      for (int cc = 0; cc < it.ncol; cc += 16) {
        uint32_t r[16];
        tmem_ld16(tO + cc, r);
        tmem_wait_ld();
        float f[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] = __uint_as_float(r[i]) * w;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int col = it.cb * 128 + cc + q * 8;
          if (key >= p.Sk || col >= p.D) break;
          if (p.splits > 1) {
            float4* o = reinterpret_cast<float4*>(part + col);
            o[0] = make_float4(f[q * 8], f[q * 8 + 1], f[q * 8 + 2], f[q * 8 + 3]);
            o[1] = make_float4(f[q * 8 + 4], f[q * 8 + 5], f[q * 8 + 6], f[q * 8 + 7]);
          } else {
            *reinterpret_cast<uint4*>(optr + 2 * col) =
                make_uint4(pack16<kFp16>(f[q * 8], f[q * 8 + 1]), pack16<kFp16>(f[q * 8 + 2], f[q * 8 + 3]),
                           pack16<kFp16>(f[q * 8 + 4], f[q * 8 + 5]), pack16<kFp16>(f[q * 8 + 6], f[q * 8 + 7]));
          }
        }
        __syncwarp();
      }
      tc_fence_before();
      warp_arrive(bar(L::kOFree));
      ++ic;
    }
    tc_fence_before();
  } else if (warp == kIssueWarp) {
    constexpr uint32_t kFmt = kFp16 ? 0u : 1u;
    constexpr uint32_t idesc_s = mma_idesc(kFmt, kFmt, 0, 0, 128, TN);
    const bool leader = elect_one();
    bool ok = true;
    int g = 0, ic = 0;
    auto wait_full = [&](int load) {
      ok = ok && mbar_wait(bar(L::kFull + load % R), (load / R) & 1, p.status, 145);
      tc_fence_after();
    };
    auto scores = [&](uint32_t d, uint32_t a_tile, uint32_t b_tile) {
      const uint32_t alo = lo_kmajor(a_tile), blo = lo_kmajor(b_tile);
#pragma unroll
      for (int j = 0; j < DB * 4; ++j) {
        const uint32_t in = (j & 3) * 2;
        if (leader && j < kd) mma_f16_ss(d, desc_lo(alo + (j >> 2) * (16384 >> 4) + in), desc_lo(blo + (j >> 2) * (TN * 128 >> 4) + in), idesc_s, j > 0);
      }
    };
    auto sum = [&](uint32_t d, uint32_t a, uint32_t b_tile, const Item& it, uint32_t idesc, bool first) {
      const uint32_t blo = lo_mnmajor(b_tile + it.cb * 2 * TN * 128, TN * 128);
#pragma unroll
      for (int j = 0; j < TN / 16; ++j)
        if (leader) mma_f16_ts(d, a + (j / (TN / 32)) * HC + (j % (TN / 32)) * 8, desc_lo(blo + j * (2048 >> 4)), idesc, !first || j > 0);
    };
#pragma unroll 1
    for (int item = blockIdx.x; item < n_items && ok; item += gridDim.x) {
      const Item it = decode(item);
      const uint32_t idesc_o = mma_idesc(kFmt, kFmt, 0, 1, 128, it.ncol);
      ok = mbar_wait(bar(L::kKVFull), ic & 1, p.status, 146);
      if (!ok) break;
      fence_proxy_async_smem();
      tc_fence_after();
      wait_full(2 * g);
      if (!ok) break;
      scores(tmem + kColS, s_base + L::kK, sRing((2 * g) % R));
      if (leader) tc_commit(bar(L::kSFull));
      wait_full(2 * g + 1);
      if (!ok) break;
      scores(tmem + kColDP, s_base + L::kV, sRing((2 * g + 1) % R));
      if (leader) {
        tc_commit(bar(L::kDPFull));
        if (it.t1 - it.t0 == 1) tc_commit(bar(L::kKVEmpty));
      }
#pragma unroll 1
      for (int t = it.t0; t < it.t1; ++t, ++g) {
        const bool first = t == it.t0, last = t == it.t1 - 1;
        const int n = 2 * g;
        ok = mbar_wait(bar(L::kPReady), g & 1, p.status, 147);
        if (ok && first && ic > 0) ok = mbar_wait(bar(L::kOFree), (ic - 1) & 1, p.status, 148);
        if (!ok) break;
        tc_fence_after();
        sum(tmem + kColDV, tmem + kColS, sRing((n + 1) % R), it, idesc_o, first);
        if (leader) tc_commit(bar(L::kEmpty + (n + 1) % R));
        if (!last) {
          wait_full(n + 2);
          if (!ok) break;
          scores(tmem + kColS, s_base + L::kK, sRing((n + 2) % R));
          if (leader) tc_commit(bar(L::kSFull));
        }
        ok = mbar_wait(bar(L::kDSReady), g & 1, p.status, 149);
        if (!ok) break;
        tc_fence_after();
        sum(tmem + kColDK, tmem + kColDP, sRing(n % R), it, idesc_o, first);
        if (leader) {
          tc_commit(bar(L::kEmpty + n % R));
          if (last) tc_commit(bar(L::kOFull));
        }
        if (!last) {
          wait_full(n + 3);
          if (!ok) break;
          scores(tmem + kColDP, s_base + L::kV, sRing((n + 3) % R));
          if (leader) {
            tc_commit(bar(L::kDPFull));
            if (t + 2 == it.t1) tc_commit(bar(L::kKVEmpty));
          }
        }
      }
      ++ic;
    }
    if (!ok) {
      if (leader) tc_commit(bar(L::kDrain));
      mbar_wait_quiet(bar(L::kDrain), 0, 1 << 20);
    }
    __syncwarp();
    tc_fence_before();
  } else if (warp < kRingWarp0) {
    // ---- K (first warp) and V (second) of an item
    const bool is_v = warp != kLoadWarp0;
    const void* src = is_v ? p.v : p.k;
    const int64_t* st = is_v ? p.v_stride : p.k_stride;
    int ic = 0;
    bool ok = true;
#pragma unroll 1
    for (int item = blockIdx.x; item < n_items && ok; item += gridDim.x) {
      const Item it = decode(item);
      if (ic > 0) ok = mbar_wait(bar(L::kKVEmpty), (ic - 1) & 1, p.status, 150);
      if (!ok) break;
      warp_copy_rows<DB>(s_base + (is_v ? L::kV : L::kK), 128, 0, 128, p.D,
                         reinterpret_cast<const uint8_t*>(src) + 2 * ((size_t)it.b * st[0] + (size_t)it.h * st[2]), 2 * (size_t)st[1], src,
                         [&](int r) { const int key = it.kt * 128 + r; return key < p.Sk ? key : -1; });
      cp_async_arrive_noinc(bar(L::kKVFull));
      ++ic;
    }
    cp_async_wait_all();
    tc_fence_before();
  } else {
    // ---- Q and dO tiles with their row statistics
    const bool leader = elect_one();
    int n = 0;
    bool ok = true;
#pragma unroll 1
    for (int item = blockIdx.x; item < n_items && ok; item += gridDim.x) {
      const Item it = decode(item);
      int cq[4] = {0, 0, 0, 0}, cd[4] = {0, 0, 0, 0};
      cq[maps.k_pos_h] = it.h; cq[maps.k_pos_b] = it.b;
      cd[maps.v_pos_h] = it.h; cd[maps.v_pos_b] = it.b;
#pragma unroll 1
      for (int e = 2 * it.t0; e < 2 * it.t1 && ok; ++e, ++n) {
        const bool is_do = e & 1;
        const int slot = n % R;
        if (n >= R) ok = mbar_wait(bar(L::kEmpty + slot), (n / R - 1) & 1, p.status, 151);
        if (!ok) break;
        if (leader) {
          mbar_arrive_expect_tx(bar(L::kFull + slot), G::kTileBytes + TN * 4);
          const void* map = is_do ? static_cast<const void*>(maps.v) : static_cast<const void*>(maps.k);
          int co[4] = {0, is_do ? cd[1] : cq[1], is_do ? cd[2] : cq[2], is_do ? cd[3] : cq[3]};
          co[is_do ? maps.v_pos_row : maps.k_pos_row] = (e >> 1) * TN;
#pragma unroll
          for (int cb = 0; cb < DB; ++cb)
            tma_load_4d(sRing(slot) + cb * TN * 128, map, cb * 64, co[1], co[2], co[3], bar(L::kFull + slot));
          bulk_load(s_base + L::kStat + slot * TN * 4, (is_do ? p.neg_delta : p.neg_lse2) + (size_t)it.bh * p.M * 128 + (size_t)(e >> 1) * TN, TN * 4,
                    bar(L::kFull + slot));
        }
      }
    }
    if (!ok)
      for (int i = n > R ? n - R : 0; i < n; ++i) mbar_wait_quiet(bar(L::kFull + i % R), (i / R) & 1, 1 << 16);   // copies in flight
    tc_fence_before();
  }

  __syncthreads();
  if (warp == kIssueWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------------------------------------ sums of split launches
// parts: (splits, B*H, S, pitch) fp32; columns [col0, col0 + D) are added in the order of the splits, rounded once and stored.
template <bool kFp16>
__global__ void __launch_bounds__(256) attn_bwd_sum_kernel(const float* parts, int splits, long long split_pitch, int pitch, int col0, int D, int H, int S,
                                                           long long rows, void* out, long long sb, long long ss, long long sh) {
  const int chunks = D / 8;
  const long long n = rows * chunks;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const long long row = i / chunks;
    const int c = (int)(i - row * chunks) * 8;
    const float* src = parts + row * pitch + col0 + c;
    float f[8] = {};
    for (int s = 0; s < splits; ++s, src += split_pitch) {
      const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
      f[0] += a.x; f[1] += a.y; f[2] += a.z; f[3] += a.w;
      f[4] += b.x; f[5] += b.y; f[6] += b.z; f[7] += b.w;
    }
    const long long bh = row / S, r = row - bh * S, b = bh / H, h = bh - b * H;
    uint8_t* o = reinterpret_cast<uint8_t*>(out) + 2 * (b * sb + r * ss + h * sh + c);
    *reinterpret_cast<uint4*>(o) = make_uint4(pack16<kFp16>(f[0], f[1]), pack16<kFp16>(f[2], f[3]), pack16<kFp16>(f[4], f[5]), pack16<kFp16>(f[6], f[7]));
  }
}

int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

// Splits of the summed axis (T tiles) for `items` items without splits.  A launch takes waves of one item per SM; an item costs its
// tiles and about two tiles' time to fill and drain.  Splits that do not end the launch earlier are not made: they cost the
// partial sums' traffic.
int pick_splits(long long items, int T, int sms) {
  if (items >= 4LL * sms) return 1;
  long long best = -1;
  int pick = 1;
  for (int s = 1; s <= T && s <= 32; ++s) {
    const long long cost = ((items * s + sms - 1) / sms) * ((T + s - 1) / s + 2) + (s > 1 ? 2 : 0);
    if (best < 0 || cost < best) { best = cost; pick = s; }
  }
  return pick;
}

struct Plan { int dq_splits, kv_splits; size_t stats, row_max, parts, total; };

constexpr size_t kAlign = 256;
size_t up(size_t n) { return (n + kAlign - 1) / kAlign * kAlign; }

int padded_blocks(int D) { return D <= 64 ? 1 : (D <= 128 ? 2 : 4); }

Plan make_plan(const AttnBwdParams& p, bool gather) {
  // (the split rule uses the B200's 148 SMs, not the current device's: sizes must not depend on the device that asks)
  constexpr int kSms = 148;
  Plan w{};
  const int TN = padded_blocks(p.D) == 4 ? 64 : 128;
  const long long bh = (long long)p.B * p.H;
  w.dq_splits = gather ? 1 : pick_splits(bh * p.M, (p.Sk + TN - 1) / TN, kSms);
  w.kv_splits = gather ? 1 : pick_splits(bh * ((p.Sk + 127) / 128) * ((((p.D + 15) & ~15) + 127) / 128), (p.Sq + TN - 1) / TN, kSms);
  w.stats = up((size_t)bh * p.M * 128 * 4);
  w.row_max = up((size_t)bh * 8);
  size_t a = w.dq_splits > 1 ? (size_t)w.dq_splits * bh * p.Sq * p.D * 4 : 0, b = w.kv_splits > 1 ? (size_t)w.kv_splits * bh * p.Sk * 2 * p.D * 4 : 0;
  w.parts = up(a > b ? a : b);
  w.total = 2 * w.stats + w.row_max + w.parts;
  return w;
}

template <typename K>
int set_smem(K kern, int bytes) {
  return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess ? 0 : -8;
}

template <int DB, int TN, bool kFp16>
int launch_dense(AttnBwdParams& p, const Plan& w, cudaStream_t stream) {
  DenseTileMaps kv, qd;
  if (!encode_tile_map(p.k, p.k_stride, p.B, p.Sk, p.H, p.D, kv.k, kv.k_pos_h, kv.k_pos_row, kv.k_pos_b, TN) ||
      !encode_tile_map(p.v, p.v_stride, p.B, p.Sk, p.H, p.D, kv.v, kv.v_pos_h, kv.v_pos_row, kv.v_pos_b, TN) ||
      !encode_tile_map(p.q, p.q_stride, p.B, p.Sq, p.H, p.D, qd.k, qd.k_pos_h, qd.k_pos_row, qd.k_pos_b, TN) ||
      !encode_tile_map(p.dout, p.dout_stride, p.B, p.Sq, p.H, p.D, qd.v, qd.v_pos_h, qd.v_pos_row, qd.v_pos_b, TN))
    return -9;
  const int sms = sm_count();
  const long long bh = (long long)p.B * p.H;
  auto dq = attn_bwd_dq_kernel<DB, TN, kFp16, false>;
  auto dkv = attn_bwd_dkv_kernel<DB, TN, kFp16>;
  if (set_smem(dq, SmemQ<DB, TN>::kDynamic) || set_smem(dkv, SmemK<DB, TN>::kDynamic)) return -8;
  p.splits = w.dq_splits;
  long long items = bh * p.M * p.splits;
  dq<<<(unsigned)(items < sms ? items : sms), 384, SmemQ<DB, TN>::kDynamic, stream>>>(p, kv);
  if (p.splits > 1) {
    const long long n = bh * p.Sq * (p.D / 8);
    attn_bwd_sum_kernel<kFp16><<<(unsigned)(n / 256 + 1 < 148 * 8 ? n / 256 + 1 : 148 * 8), 256, 0, stream>>>(
        p.parts, p.splits, bh * p.Sq * p.D, p.D, 0, p.D, p.H, p.Sq, bh * p.Sq, p.dq, p.dq_stride[0], p.dq_stride[1], p.dq_stride[2]);
  }
  p.splits = w.kv_splits;
  items = bh * ((p.Sk + 127) / 128) * ((((p.D + 15) & ~15) + 127) / 128) * p.splits;
  dkv<<<(unsigned)(items < sms ? items : sms), 384, SmemK<DB, TN>::kDynamic, stream>>>(p, qd);
  if (p.splits > 1) {
    const long long n = bh * p.Sk * (p.D / 8);
    const unsigned grid = (unsigned)(n / 256 + 1 < 148 * 8 ? n / 256 + 1 : 148 * 8);
    attn_bwd_sum_kernel<kFp16><<<grid, 256, 0, stream>>>(p.parts, p.splits, bh * p.Sk * 2 * p.D, 2 * p.D, 0, p.D, p.H, p.Sk, bh * p.Sk, p.dk,
                                                         p.dk_stride[0], p.dk_stride[1], p.dk_stride[2]);
    attn_bwd_sum_kernel<kFp16><<<grid, 256, 0, stream>>>(p.parts, p.splits, bh * p.Sk * 2 * p.D, 2 * p.D, p.D, p.D, p.H, p.Sk, bh * p.Sk, p.dv,
                                                         p.dv_stride[0], p.dv_stride[1], p.dv_stride[2]);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -8;
}

template <bool kFp16>
int launch_type(AttnBwdParams& p, const Plan& w, cudaStream_t stream) {
  if (kFp16 && cudaMemsetAsync(p.row_max, 0, (size_t)p.B * p.H * 8, stream) != cudaSuccess) return -8;
  const int rows = p.M * 128 + (kFp16 ? p.Sk : 0);
  const int per = (rows + 15) / 16;
  attn_bwd_stats_kernel<kFp16><<<dim3((unsigned)(per < 256 ? per : 256), (unsigned)(p.B * p.H)), 256, 0, stream>>>(p);
  switch (padded_blocks(p.D)) {
    case 1: return launch_dense<1, 128, kFp16>(p, w, stream);
    case 2: return launch_dense<2, 128, kFp16>(p, w, stream);
    default: return launch_dense<4, 64, kFp16>(p, w, stream);
  }
}

}  // namespace

int64_t attn_bwd_workspace_bytes(const AttnBwdParams& p, bool gather, bool) { return (int64_t)make_plan(p, gather).total; }

int launch_attn_bwd(AttnBwdParams& p, bool gather, bool fp16, void* workspace, cudaStream_t stream) {
  const Plan w = make_plan(p, gather);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.neg_lse2 = reinterpret_cast<float*>(ws);
  p.neg_delta = reinterpret_cast<float*>(ws + w.stats);
  p.row_max = reinterpret_cast<unsigned int*>(ws + 2 * w.stats);
  p.parts = reinterpret_cast<float*>(ws + 2 * w.stats + w.row_max);
  return fp16 ? launch_type<true>(p, w, stream) : launch_type<false>(p, w, stream);
}

}  // namespace mcs
