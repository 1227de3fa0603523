// dK and dV of the gather-KV attention (bf16 / fp16, head dimensions up to 256) for sm_100a.
//
// A key's gradient sums over the query groups that selected it.  The groups of one head name different keys in different
// places, so the sums cannot stay in tensor memory as in the dense call: a group's 128 x D contributions to a tile of 128 gathered keys
// go to rows of an fp32 buffer, and a second kernel adds the rows of every key.  The buffer is laid out by key: the entries
// (group, slot) that name key j take consecutive rows, in the order of groups, so that the second kernel reads it once, in
// order, and the sums (and their bits) do not depend on which CTA came first, which with atomics in place would be left to chance.  Equal entries inside one group have equal contributions, so their order does not matter.
//
// Bound: the buffer is written and read once, 8 D bytes per entry either way (12.9 GB + 12.9 GB at 24 heads x 256 groups x 2,048
// keys x 128: 3.9 ms at the copy rate), against 10 x 128 x D operations (1.25 ms): memory.  Measured there: 2.99 ms for the
// contributions (4.3 TB/s of rows scattered by key; the copy out of tensor memory, through shared memory and the SM's store path,
// is the longest stage of a tile: 1.6 ms without it), 1.98 ms for the sums (6.5 TB/s, the copy rate).  Steps: every thread storing its own row 4.83 ms; 128
// contiguous bytes at a time through shared memory 4.44; by warps of their own, under the next tile's P and dS, 3.26; dV released
// before dK 2.99.  Measured and not kept: rows in the order of groups, contiguous for a tile, gathered by the sums instead: 3.79 ms
// (against 4.44 then) for the contributions, but 4.53 ms for the sums; dV copied by the softmax warps: 3.21.
#include "attn_bwd.cuh"

namespace mcs {

namespace {

using namespace bwd;

// ------------------------------------------------------------------------------------------------ rows of the entries
// Counting sort of the entries by key that keeps the order of groups: groups are cut into segments; counts per (segment, key) by
// atomics (whole numbers: any order), their exclusive sums in (key, segment) order, then every segment hands out the rows of its
// entries, one group after the other.
__device__ __forceinline__ int group_entries(const AttnBwdParams& p, int bh, int m) {
  const int most = p.gather_len / 128;
  return 128 * (p.gl != nullptr ? min(max(p.gl[(size_t)bh * p.M + m], 1), most) : most);
}

// (one CTA per group)
__global__ void __launch_bounds__(256) attn_bwd_count_kernel(const AttnBwdParams p, int segs) {
  const int bh = blockIdx.y, m = blockIdx.x;
  int seg = (int)((long long)m * segs / p.M);                // the segment with M seg / segs <= m < M (seg + 1) / segs
  while ((int)((long long)p.M * (seg + 1) / segs) <= m) ++seg;
  int32_t* count = p.seg_count + ((size_t)bh * segs + seg) * p.Sk;
  const int n = group_entries(p, bh, m);
  const int32_t* gi = p.gi + ((size_t)bh * p.M + m) * p.gather_len;
  for (int i = threadIdx.x; i < n; i += 256) atomicAdd(count + min(max(gi[i], 0), p.Sk - 1), 1);
}

// Entries of 1,024 keys at a time, then key_start[j] = entries of keys before j; seg_count becomes the first row of (segment, key).
__device__ __forceinline__ int block_scan_inclusive(int v, int* warp_sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += y;
  }
  if (lane == 31) warp_sum[warp] = v;
  __syncthreads();
  if (warp == 0) {
    int w = warp_sum[lane];
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, off);
      if (lane >= off) w += y;
    }
    warp_sum[lane] = w;
  }
  __syncthreads();
  return v + (warp > 0 ? warp_sum[warp - 1] : 0);
}

__device__ __forceinline__ int key_entries(const AttnBwdParams& p, int bh, int segs, int j) {
  int total = 0;
  if (j < p.Sk)
    for (int s = 0; s < segs; ++s) total += p.seg_count[((size_t)bh * segs + s) * p.Sk + j];
  return total;
}

__global__ void __launch_bounds__(1024) attn_bwd_block_sum_kernel(const AttnBwdParams p, int segs) {
  __shared__ int warp_sum[32];
  const int v = block_scan_inclusive(key_entries(p, blockIdx.y, segs, blockIdx.x * 1024 + threadIdx.x), warp_sum);
  if (threadIdx.x == 1023) p.block_sum[(size_t)blockIdx.y * gridDim.x + blockIdx.x] = v;
}

__global__ void __launch_bounds__(1024) attn_bwd_scan_kernel(const AttnBwdParams p, int segs) {
  __shared__ int warp_sum[32];
  const int bh = blockIdx.y, j = blockIdx.x * 1024 + threadIdx.x;
  // entries of the blocks before this one
  int before = 0;
  for (int i = threadIdx.x; i < (int)blockIdx.x; i += 1024) before += p.block_sum[(size_t)bh * gridDim.x + i];
  block_scan_inclusive(before, warp_sum);
  const int carry = warp_sum[31];
  __syncthreads();
  const int total = key_entries(p, bh, segs, j);
  int at = carry + block_scan_inclusive(total, warp_sum) - total;
  if (j >= p.Sk) return;
  p.key_start[(size_t)bh * (p.Sk + 1) + j] = at;
  if (j == p.Sk - 1) p.key_start[(size_t)bh * (p.Sk + 1) + p.Sk] = at + total;
  for (int s = 0; s < segs; ++s) {
    int32_t* c = p.seg_count + ((size_t)bh * segs + s) * p.Sk + j;
    const int n = *c;
    *c = at;
    at += n;
  }
}

__global__ void __launch_bounds__(1024) attn_bwd_rows_kernel(const AttnBwdParams p, int segs) {
  const int bh = blockIdx.y, seg = blockIdx.x;
  const int m0 = (int)((long long)p.M * seg / segs), m1 = (int)((long long)p.M * (seg + 1) / segs);
  int32_t* next = p.seg_count + ((size_t)bh * segs + seg) * p.Sk;
  for (int m = m0; m < m1; ++m) {
    const int n = group_entries(p, bh, m);
    const size_t at = ((size_t)bh * p.M + m) * p.gather_len;
    for (int i = threadIdx.x; i < n; i += 1024) p.entry_row[at + i] = atomicAdd(next + min(max(p.gi[at + i], 0), p.Sk - 1), 1);
    __syncthreads();                                         // the next group's rows come behind this one's
  }
}

// ------------------------------------------------------------------------------------------------ contributions of every group
// One CTA per SM walks groups.  Q and dO of the group stay in shared memory; gathered K and V tiles of 128 keys come through a ring in
// blocks of up to 128 columns.  Per tile:
//     S^T = K Q^T, dP^T = V dO^T (rows: gathered keys)  ->  P^T, dS^T in tensor memory, over their scores
//     dV = P^T dO, dK = dS^T Q, up to 128 columns at a time, copied to the entries' rows by four warps of their own
// The copy is the longest part of a tile; the next tile's P and dS are computed under it.
template <int DB>
struct SmemG {
  static constexpr int kResBytes = DB * 16384;
  static constexpr int kSlotBlocks = DB > 2 ? 2 : DB;        // 64-column blocks of one ring slot
  static constexpr int kSlotBytes = kSlotBlocks * 16384;
  static constexpr int kRing = DB > 2 ? 2 : (DB == 2 ? 4 : 8);
  static constexpr int kQ = 0, kDO = kResBytes, kRingOff = 2 * kResBytes;
  static constexpr int kStat = kRingOff + kRing * kSlotBytes;               // neg_lse2, neg_delta of the group's rows
  static constexpr int kStage = kStat + 1024;                               // 32 rows x 128 bytes of every copying warp
  static constexpr int kBars = kStage + 4 * 4096;
  static constexpr int kFull = 0, kEmpty = kRing, kAFull = 2 * kRing, kAEmpty = kAFull + 1, kSFull = kAEmpty + 1, kDPFull = kSFull + 1,
                       kPReady = kDPFull + 1, kDSReady = kPReady + 1, kOFull = kDSReady + 1, kOFree = kOFull + 2, kDrain = kOFree + 2, kCount = kDrain + 1;   // kOFull, kOFree: dV, dK
  static constexpr int kSlot = kBars + kCount * 8;
  static constexpr int kDynamic = kSlot + 16 + 1024;
};
static_assert(SmemG<1>::kDynamic <= 232448 && SmemG<2>::kDynamic <= 232448 && SmemG<4>::kDynamic <= 232448, "must fit 227 KB");

constexpr int kThreadsG = 512;                               // 8 softmax warps, the issuer, three producers, four warps that copy out
constexpr int kIssueWarp = 8, kLoadWarp0 = 9, kLoadWarps = 3, kOutWarp0 = 12;
constexpr uint32_t kColS = 0, kColDP = 128, kColDV = 256, kColDK = 384;

template <int DB, bool kFp16>
__global__ void __launch_bounds__(kThreadsG, 1) attn_bwd_gather_dkv_kernel(const AttnBwdParams p) {
  using L = SmemG<DB>;
  constexpr int R = L::kRing, SB = L::kSlotBlocks;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t s_base = smem_u32(smem);
  auto bar = [&](int i) { return s_base + L::kBars + 8u * i; };
  auto sRing = [&](int slot) { return s_base + L::kRingOff + slot * L::kSlotBytes; };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kSlot);
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int n_items = p.bh_count * p.M;
  const int nd = (p.D + 15) & ~15, kd = nd / 16;
  const int CB = DB > 2 ? (nd + 127) / 128 : 1;              // column blocks of up to 128
  struct Item { int bh, b, h, m, T; };
  auto decode = [&](int item) {
    Item it;
    it.m = item % p.M;
    it.bh = p.bh0 + item / p.M;
    it.b = it.bh / p.H;
    it.h = it.bh % p.H;
    it.T = group_entries(p, it.bh, it.m) / 128;
    return it;
  };
  auto row_of = [&](const Item& it, int r) {
    const int pos = it.m * p.group_rows + r;
    if (r >= p.group_rows || pos >= p.Sq) return -1;
    return query_row(p, it.bh, pos);
  };

  if (tid == 0) {
    for (int i = 0; i < R; ++i) { mbar_init(bar(L::kFull + i), 128); mbar_init(bar(L::kEmpty + i), 1); }
    mbar_init(bar(L::kAFull), 256);
    mbar_init(bar(L::kAEmpty), 1);
    mbar_init(bar(L::kSFull), 1);
    mbar_init(bar(L::kDPFull), 1);
    mbar_init(bar(L::kPReady), kSoftmaxWarps);
    mbar_init(bar(L::kDSReady), kSoftmaxWarps);
    for (int i = 0; i < 2; ++i) { mbar_init(bar(L::kOFull + i), 1); mbar_init(bar(L::kOFree + i), 4); }
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
    const int x = warp >> 2;
    const uint32_t lane_addr = (static_cast<uint32_t>(warp & 3) * 32u) << 16;
    const uint32_t tS = tmem + kColS + x * 64 + lane_addr, tDP = tmem + kColDP + x * 64 + lane_addr;
    const unsigned long long scale2 = f2_pack(p.scale_log2, p.scale_log2);
    const ulonglong2* lse = reinterpret_cast<const ulonglong2*>(smem + L::kStat + x * 256);
    const ulonglong2* dlt = reinterpret_cast<const ulonglong2*>(smem + L::kStat + 512 + x * 256);
    int g = 0, ic = 0;
    bool ok = true;
#pragma unroll 1
    for (int item = blockIdx.x; item < n_items && ok; item += gridDim.x, ++ic) {
      const Item it = decode(item);
      const float c = ds_scale<kFp16>(p, it.bh);
      const unsigned long long c2 = f2_pack(c, c);
      ok = mbar_wait(bar(L::kAFull), ic & 1, p.status, 150);
      if (!ok) break;
#pragma unroll 1
      for (int t = 0; t < it.T; ++t, ++g) {
        ok = mbar_wait(bar(L::kSFull), g & 1, p.status, 151);
        if (!ok) break;
        tc_fence_after();
        uint32_t sc[64];
#pragma unroll
        for (int q = 0; q < 2; ++q) tmem_ld32(tS + q * 32, *reinterpret_cast<uint32_t(*)[32]>(&sc[q * 32]));
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 64; i += 4) {
          const ulonglong2 l = lse[i / 4];
          const float2 y0 = f2_unpack(f2_fma(f2_pack(__uint_as_float(sc[i]), __uint_as_float(sc[i + 1])), scale2, l.x));
          const float2 y1 = f2_unpack(f2_fma(f2_pack(__uint_as_float(sc[i + 2]), __uint_as_float(sc[i + 3])), scale2, l.y));
          sc[i] = __float_as_uint(ex2_approx(y0.x));
          sc[i + 1] = __float_as_uint(ex2_approx(y0.y));
          sc[i + 2] = __float_as_uint(ex2_approx(y1.x));
          sc[i + 3] = __float_as_uint(ex2_approx(y1.y));
          if (i % 16 == 12) store_packed<kFp16>(tS + (i - 12) / 2, &sc[i - 12]);
        }
        tmem_wait_st();
        tc_fence_before();
        warp_arrive(bar(L::kPReady));
        ok = mbar_wait(bar(L::kDPFull), g & 1, p.status, 152);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int s0 = 0; s0 < 64; s0 += 32) {
          uint32_t dp[32];
          tmem_ld32(tDP + s0, dp);
          tmem_wait_ld();
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            uint32_t pk[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int e = q * 16 + 4 * i;
              const ulonglong2 l = dlt[(s0 + e) / 4];
              unsigned long long d0 = f2_add(f2_pack(__uint_as_float(dp[e]), __uint_as_float(dp[e + 1])), l.x);
              unsigned long long d1 = f2_add(f2_pack(__uint_as_float(dp[e + 2]), __uint_as_float(dp[e + 3])), l.y);
              if constexpr (kFp16) { d0 = f2_mul(d0, c2); d1 = f2_mul(d1, c2); }
              const float2 y0 = f2_unpack(f2_mul(f2_pack(__uint_as_float(sc[s0 + e]), __uint_as_float(sc[s0 + e + 1])), d0));
              const float2 y1 = f2_unpack(f2_mul(f2_pack(__uint_as_float(sc[s0 + e + 2]), __uint_as_float(sc[s0 + e + 3])), d1));
              pk[2 * i] = pack16<kFp16>(y0.x, y0.y);
              pk[2 * i + 1] = pack16<kFp16>(y1.x, y1.y);
            }
            tmem_st8(tDP + (s0 + q * 16) / 2, pk);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        warp_arrive(bar(L::kDSReady));
      }
    }
    tc_fence_before();
  } else if (warp == kIssueWarp) {
    constexpr uint32_t kFmt = kFp16 ? 0u : 1u;
    constexpr uint32_t idesc_s = mma_idesc(kFmt, kFmt, 0, 0, 128, 128);
    const bool leader = elect_one();
    bool ok = true;
    int g = 0, ic = 0, n = 0, blk = 0;
    // S^T or dP^T of the next tile: one ring slot per column block
    auto scores = [&](uint32_t d, uint32_t b_tile, uint32_t done) {
#pragma unroll 1
      for (int cb = 0; cb < CB; ++cb, ++n) {
        ok = ok && mbar_wait(bar(L::kFull + n % R), (n / R) & 1, p.status, 154);
        if (!ok) return;
        fence_proxy_async_smem();
        tc_fence_after();
        const uint32_t alo = lo_kmajor(sRing(n % R)), blo = lo_kmajor(b_tile + cb * SB * 16384);
#pragma unroll
        for (int j = 0; j < SB * 4; ++j) {
          const uint32_t off = (j >> 2) * (16384 >> 4) + (j & 3) * 2;
          if (leader && cb * 8 + j < kd) mma_f16_ss(d, desc_lo(alo + off), desc_lo(blo + off), idesc_s, cb > 0 || j > 0);
        }
        if (leader) {
          tc_commit(bar(L::kEmpty + n % R));
          if (cb == CB - 1) tc_commit(done);
        }
      }
    };
    auto out_product = [&](uint32_t d, uint32_t a, uint32_t b_tile, int cb) {
      const uint32_t idesc = mma_idesc(kFmt, kFmt, 0, 1, 128, min(128, nd - cb * 128));
      const uint32_t blo = lo_mnmajor(b_tile + cb * SB * 16384, 16384);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (leader) mma_f16_ts(d, a + (j / 4) * 64 + (j % 4) * 8, desc_lo(blo + j * (2048 >> 4)), idesc, j > 0);
    };
#pragma unroll 1
    for (int item = blockIdx.x; item < n_items && ok; item += gridDim.x, ++ic) {
      const Item it = decode(item);
      ok = mbar_wait(bar(L::kAFull), ic & 1, p.status, 155);
      if (!ok) break;
      fence_proxy_async_smem();
      tc_fence_after();
#pragma unroll 1
      for (int t = 0; t < it.T && ok; ++t, ++g) {
#pragma unroll 1
        for (int i = 0; i < 2 && ok; ++i)
          scores(tmem + (i == 0 ? kColS : kColDP), s_base + (i == 0 ? L::kQ : L::kDO), bar(i == 0 ? L::kSFull : L::kDPFull));
        if (!ok) break;
        ok = mbar_wait(bar(L::kPReady), g & 1, p.status, 156);
        if (!ok) break;
#pragma unroll 1
        for (int cb = 0; cb < CB; ++cb, ++blk) {
          if (blk > 0) ok = mbar_wait(bar(L::kOFree), (blk - 1) & 1, p.status, 157);
          if (!ok) break;
          tc_fence_after();
          out_product(tmem + kColDV, tmem + kColS, s_base + L::kDO, cb);
          if (leader) tc_commit(bar(L::kOFull));
          if (cb == 0) ok = mbar_wait(bar(L::kDSReady), g & 1, p.status, 158);
          if (ok && blk > 0) ok = mbar_wait(bar(L::kOFree + 1), (blk - 1) & 1, p.status, 162);
          if (!ok) break;
          tc_fence_after();
          out_product(tmem + kColDK, tmem + kColDP, s_base + L::kQ, cb);
          if (leader) tc_commit(bar(L::kOFull + 1));
        }
        if (!ok) break;
        if (t == it.T - 1 && leader) tc_commit(bar(L::kAEmpty));
      }
    }
    if (!ok) {
      if (leader) tc_commit(bar(L::kDrain));
      mbar_wait_quiet(bar(L::kDrain), 0, 1 << 20);
    }
    __syncwarp();
    tc_fence_before();
  } else if (warp < kOutWarp0) {
    // ---- gathered rows, K blocks, then V blocks, of every tile: the warps take batches of 32 rows in turn.  Q, dO and their
    // statistics follow the first block, which does not have to wait for the item before to be done with them.
    const int w = warp - kLoadWarp0;
    int n = 0, ic = 0, batch = 0;
    bool ok = true;
    int key[4], next[4];                                     // indices of the tile that is copied, and of the next one, in flight meanwhile
    auto fetch = [&](const int32_t* gi, int t, int (&dst)[4]) {
#pragma unroll
      for (int q = 0; q < 4; ++q) dst[q] = __ldg(gi + t * 128 + q * 32 + lane);
    };
#pragma unroll 1
    for (int item = blockIdx.x; item < n_items && ok; item += gridDim.x, ++ic) {
      const Item it = decode(item);
      const int32_t* gi = p.gi + ((size_t)it.bh * p.M + it.m) * p.gather_len;
      const uint8_t* kb = reinterpret_cast<const uint8_t*>(p.k) + 2 * ((size_t)it.b * p.k_stride[0] + (size_t)it.h * p.k_stride[2]);
      const uint8_t* vb = reinterpret_cast<const uint8_t*>(p.v) + 2 * ((size_t)it.b * p.v_stride[0] + (size_t)it.h * p.v_stride[2]);
      fetch(gi, 0, key);
#pragma unroll 1
      for (int t = 0; t < it.T && ok; ++t) {
        if (t + 1 < it.T) fetch(gi, t + 1, next);
#pragma unroll 1
        for (int e = 0; e < 2 * CB; ++e, ++n) {
          const bool is_v = e >= CB;
          const int cb = is_v ? e - CB : e, slot = n % R;
          if (n >= R) ok = mbar_wait(bar(L::kEmpty + slot), (n / R - 1) & 1, p.status, 161);
          if (!ok) break;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if (batch == w) {
              warp_copy_rows<SB>(sRing(slot), 128, q * 32, min(max(key[q], 0), p.Sk - 1), min(SB * 64, p.D - cb * 128), (is_v ? vb : kb) + cb * 256,
                                 2 * (size_t)(is_v ? p.v_stride[1] : p.k_stride[1]), p.k);
              cp_async_arrive_noinc(bar(L::kFull + slot));
            }
            batch = batch == kLoadWarps - 1 ? 0 : batch + 1;
          }
          if (t == 0 && e == 0) {
            if (ic > 0) ok = mbar_wait(bar(L::kAEmpty), (ic - 1) & 1, p.status, 160);
            if (!ok) break;
#pragma unroll 1
            for (int q = 0; q < 8; ++q) {
              if (batch == w) {
                const bool is_do = q >= 4;
                const int64_t* st = is_do ? p.dout_stride : p.q_stride;
                const uint8_t* src = reinterpret_cast<const uint8_t*>(is_do ? p.dout : p.q) + 2 * ((size_t)it.b * st[0] + (size_t)it.h * st[2]);
                warp_copy_rows<DB>(s_base + (is_do ? L::kDO : L::kQ), 128, (q & 3) * 32, row_of(it, (q & 3) * 32 + lane), p.D, src, 2 * (size_t)st[1], p.q);
                if ((q & 3) == 0)
                  cp_async16(s_base + L::kStat + (is_do ? 512 : 0) + lane * 16,
                             (is_do ? p.neg_delta_kv : p.neg_lse2) + (size_t)it.bh * p.stat_rows + it.m * 128 + lane * 4);
                cp_async_arrive_noinc(bar(L::kAFull));
              }
              batch = batch == kLoadWarps - 1 ? 0 : batch + 1;
            }
          }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) key[q] = next[q];
      }
    }
    cp_async_wait_all();
    tc_fence_before();
  } else {
    // ---- dV and dK rows of every tile to their entries' rows, 32 columns at a time through shared memory (16-byte chunks swizzled by
    // row), so that eight lanes store 128 contiguous bytes: with each lane storing its own row, a store touched 32 lines
    const int lg = warp & 3;
    const uint32_t lane_addr = (static_cast<uint32_t>(lg) * 32u) << 16;
    const uint32_t stage = s_base + L::kStage + lg * 4096;
    const float unbias = kFp16 ? 6.103515625e-05f : 1.f;                       // 2^-14
    int blk = 0;
    bool ok = true;
#pragma unroll 1
    for (int item = blockIdx.x; item < n_items && ok; item += gridDim.x) {
      const Item it = decode(item);
      const float w_k = p.out_scale / ds_scale<kFp16>(p, it.bh) * unbias;
      const int32_t* rows = p.entry_row + ((size_t)it.bh * p.M + it.m) * p.gather_len + lg * 32 + lane;
      // dK at columns [0, D) of a row, dV behind it
      float* base = p.parts + (size_t)(it.bh - p.bh0) * p.M * p.gather_len * (2 * p.D) + (lane & 7) * 4;
      int next = rows[0];
#pragma unroll 1
      for (int t = 0; t < it.T && ok; ++t) {
        const int mine = next;
        if (t + 1 < it.T) next = rows[(t + 1) * 128];
        int to[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) to[i] = __shfl_sync(0xffffffffu, mine, i * 4 + (lane >> 3));
#pragma unroll 1
        for (int cb = 0; cb < CB; ++cb, ++blk) {
          const int cols = min(128, p.D - cb * 128);
          // (dV of the next tile is computed while this one's dK is copied)
#pragma unroll 1
          for (int part = 0; part < 2; ++part) {
            ok = ok && mbar_wait(bar(L::kOFull + part), blk & 1, p.status, 153);
            if (!ok) break;
            tc_fence_after();
            const float w = part == 0 ? unbias : w_k;
            float* to_cols = base + (part == 0 ? p.D : 0) + cb * 128;
            const uint32_t tO = tmem + (part == 0 ? kColDV : kColDK) + lane_addr;
#pragma unroll 1
            for (int cc = 0; cc < cols; cc += 32) {
              uint32_t r[32];
              tmem_ld32(tO + cc, r);
              tmem_wait_ld();
              __syncwarp();                                  // the last block has been read out
#pragma unroll
              for (int q = 0; q < 8; ++q)
                sts_v4(stage + lane * 128 + ((q ^ (lane & 7)) << 4),
                       make_uint4(__float_as_uint(__uint_as_float(r[4 * q]) * w), __float_as_uint(__uint_as_float(r[4 * q + 1]) * w),
                                  __float_as_uint(__uint_as_float(r[4 * q + 2]) * w), __float_as_uint(__uint_as_float(r[4 * q + 3]) * w)));
              __syncwarp();
              if (cc + (lane & 7) * 4 < cols) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  const int rl = i * 4 + (lane >> 3);
                  const uint4 v = lds_v4(stage + rl * 128 + (((lane & 7) ^ (rl & 7)) << 4));
                  *reinterpret_cast<uint4*>(to_cols + (size_t)to[i] * (2 * p.D) + cc) = v;
                }
              }
            }
            __syncwarp();
            tc_fence_before();
            if (lane == 0) mbar_arrive(bar(L::kOFree + part));
          }
          if (!ok) break;
        }
      }
    }
    tc_fence_before();
  }

  __syncthreads();
  if (warp == kIssueWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------------------------------------ sums over the entries of a key
// A warp per key; a key with many entries (a sink token that every group selected) is summed by the whole CTA, each warp an equal
// run of its rows.  Both splits depend on the number of entries only.
constexpr int kManyEntries = 64;

template <int C>   // float4 columns per lane
__device__ __forceinline__ void add_rows(const float4* src, int n, int lane, int cols4, float4 (&acc)[C]) {
  constexpr int kUnroll = C == 1 ? 8 : (C == 2 ? 4 : 2);
#pragma unroll 1
  for (int i = 0; i < n; i += kUnroll, src += (size_t)kUnroll * cols4) {
    float4 v[kUnroll][C];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int q = 0; q < C; ++q) {
        v[u][q] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i + u < n && lane + q * 32 < cols4) v[u][q] = __ldcs(src + u * cols4 + lane + q * 32);
      }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int q = 0; q < C; ++q) { acc[q].x += v[u][q].x; acc[q].y += v[u][q].y; acc[q].z += v[u][q].z; acc[q].w += v[u][q].w; }
  }
}

template <int C, bool kFp16>
__global__ void __launch_bounds__(256, 4) attn_bwd_key_sum_kernel(const AttnBwdParams p) {
  __shared__ float4 part[8][C * 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int bh = p.bh0 + blockIdx.y, b = bh / p.H, h = bh % p.H;
  const int cols4 = p.D / 2;                                 // 2 D floats
  const float4* rows = reinterpret_cast<const float4*>(p.parts) + (size_t)blockIdx.y * p.M * p.gather_len * cols4;
  const int32_t* start = p.key_start + (size_t)bh * (p.Sk + 1);
  auto store = [&](int key, const float4 (&acc)[C]) {
#pragma unroll
    for (int q = 0; q < C; ++q) {
      const int col = (lane + q * 32) * 4;
      if (col >= 2 * p.D) continue;
      const bool is_v = col >= p.D;
      const int64_t* st = is_v ? p.dv_stride : p.dk_stride;
      uint8_t* o = reinterpret_cast<uint8_t*>(is_v ? p.dv : p.dk) +
                   2 * ((size_t)b * st[0] + (size_t)key * st[1] + (size_t)h * st[2] + (col - (is_v ? p.D : 0)));
      *reinterpret_cast<uint2*>(o) = make_uint2(pack16<kFp16>(acc[q].x, acc[q].y), pack16<kFp16>(acc[q].z, acc[q].w));
    }
  };
  for (int key0 = blockIdx.x * 8; key0 < p.Sk; key0 += gridDim.x * 8) {
    const int key = key0 + warp;
    int at = 0, n = 0;
    if (key < p.Sk) { at = start[key]; n = start[key + 1] - at; }
    // first every warp's own key, then the keys of this CTA that have many entries, one after the other
#pragma unroll 1
    for (int i = -1; i < 8 && key0 + i < p.Sk; ++i) {
      int r0 = at, m = n <= kManyEntries ? n : 0;
      if (i >= 0) {
        const int a = start[key0 + i], all = start[key0 + i + 1] - a;
        if (all <= kManyEntries) continue;                   // (uniform over the CTA)
        r0 = (int)((long long)all * warp / 8);
        m = (int)((long long)all * (warp + 1) / 8) - r0;
        r0 += a;
      }
      float4 acc[C] = {};
      add_rows<C>(rows + (size_t)r0 * cols4, m, lane, cols4, acc);
      if (i < 0) {
        if (key < p.Sk && n <= kManyEntries) store(key, acc);
        if (!__syncthreads_or(n > kManyEntries)) break;
        continue;
      }
#pragma unroll
      for (int q = 0; q < C; ++q) part[warp][lane + q * 32] = acc[q];
      __syncthreads();
      if (warp == 0) {
        for (int o = 1; o < 8; ++o)
#pragma unroll
          for (int q = 0; q < C; ++q) {
            const float4 v = part[o][lane + q * 32];
            acc[q].x += v.x; acc[q].y += v.y; acc[q].z += v.z; acc[q].w += v.w;
          }
        store(key0 + i, acc);
      }
      __syncthreads();
    }
  }
}

template <int DB, bool kFp16>
int launch_db(AttnBwdParams& p, int heads_per_pass, cudaStream_t stream) {
  auto kern = attn_bwd_gather_dkv_kernel<DB, kFp16>;
  constexpr int kSmem = SmemG<DB>::kDynamic;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess) return -8;
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int bh = p.B * p.H;
  for (p.bh0 = 0; p.bh0 < bh; p.bh0 += heads_per_pass) {
    p.bh_count = bh - p.bh0 < heads_per_pass ? bh - p.bh0 : heads_per_pass;
    const long long items = (long long)p.bh_count * p.M;
    kern<<<(unsigned)(items < sms ? items : sms), kThreadsG, kSmem, stream>>>(p);
    const int per = (p.Sk + 7) / 8;
    attn_bwd_key_sum_kernel<DB, kFp16><<<dim3((unsigned)(per < 4096 ? per : 4096), (unsigned)p.bh_count), 256, 0, stream>>>(p);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -8;
}

}  // namespace

int launch_attn_bwd_gather_rows(const AttnBwdParams& p, int segs, cudaStream_t stream) {
  const int bh = p.B * p.H;
  if (cudaMemsetAsync(p.seg_count, 0, (size_t)bh * segs * p.Sk * 4, stream) != cudaSuccess) return -8;
  const dim3 key_blocks((unsigned)((p.Sk + 1023) / 1024), (unsigned)bh);
  attn_bwd_count_kernel<<<dim3((unsigned)p.M, (unsigned)bh), 256, 0, stream>>>(p, segs);
  attn_bwd_block_sum_kernel<<<key_blocks, 1024, 0, stream>>>(p, segs);
  attn_bwd_scan_kernel<<<key_blocks, 1024, 0, stream>>>(p, segs);
  attn_bwd_rows_kernel<<<dim3((unsigned)segs, (unsigned)bh), 1024, 0, stream>>>(p, segs);
  return cudaGetLastError() == cudaSuccess ? 0 : -8;
}

int launch_attn_bwd_gather_dkv(AttnBwdParams& p, bool fp16, int heads_per_pass, cudaStream_t stream) {
  const int blocks = p.D <= 64 ? 1 : (p.D <= 128 ? 2 : 4);
  if (fp16) return blocks == 1 ? launch_db<1, true>(p, heads_per_pass, stream) : (blocks == 2 ? launch_db<2, true>(p, heads_per_pass, stream) : launch_db<4, true>(p, heads_per_pass, stream));
  return blocks == 1 ? launch_db<1, false>(p, heads_per_pass, stream) : (blocks == 2 ? launch_db<2, false>(p, heads_per_pass, stream) : launch_db<4, false>(p, heads_per_pass, stream));
}

}  // namespace mcs
