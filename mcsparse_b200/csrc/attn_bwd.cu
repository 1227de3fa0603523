// Backward pass of the attention for sm_100a (bf16 / fp16, head dimensions up to 256): row statistics, the kernel of dQ (dense
// and gathered keys), the kernel of dK and dV of the dense call, and the sums of split launches.  The kernel of dK and dV of
// gathered keys is in attn_bwd_gather.cu.
//
// Two launches, one per side, instead of one that forms all five products of a tile pair: dQ sums over keys and dK, dV over
// queries, so a launch that makes them all has to add one side's partial sums in global memory with atomics (order, and with it
// bits, would change from run to run) and needs one operand of dS transposed in shared memory.  Each launch here keeps its own
// side's sums in tensor memory, takes P and dS straight out of tensor memory as the first operand of the next product, and
// writes every result once.  The price is three products more (8 instead of 5): S and dP are computed on either side, and the
// query side carries P K to correct dQ (below).
#include <algorithm>

#include "attn_bwd.cuh"

namespace mcs {

namespace {

using namespace bwd;

constexpr int kMaxSmem = 232448;

// ------------------------------------------------------------------------------------------------ row statistics
// Sixteen lanes per row, four rows at a time: neg_delta = -sum(dout * out) and neg_lse2 of every tile row (memory-bound: dout and out
// are read once, eight 16-byte loads of a thread in flight), and for fp16 the largest norms of rows of dout and of v.  Only rows that take
// part in finite results count for these: rows with an infinity or NaN give no finite dS whatever its scale, and rows of v that no group
// selected (key_start, gathered keys only) may hold anything.  With perm dQ is zeroed on the way: its rows are written through perm, whose
// entries may be out of range.
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
  constexpr int kRows = 4;
  const int bh = blockIdx.y, h = bh % p.H, b = bh / p.H;
  const int l16 = threadIdx.x & 15, sub = threadIdx.x >> 4;
  const int rows = p.stat_rows;
  const int chunks = p.D / 8;
  const uint8_t* gb = reinterpret_cast<const uint8_t*>(p.dout) + 2 * ((size_t)b * p.dout_stride[0] + (size_t)h * p.dout_stride[2]);
  const uint8_t* ob = reinterpret_cast<const uint8_t*>(p.out) + 2 * ((size_t)b * p.out_stride[0] + (size_t)h * p.out_stride[2]);
  uint8_t* qb = reinterpret_cast<uint8_t*>(p.dq) + 2 * ((size_t)b * p.dq_stride[0] + (size_t)h * p.dq_stride[2]);
  float m_do = 0.f, m_v = 0.f;
  // fp16: every second CTA takes rows of v instead
  const int share = kFp16 ? 2 : 1, blk = blockIdx.x / share, step = gridDim.x / share;
  const bool of_v = kFp16 && blockIdx.x % 2 == 1;
  for (int base = blk * (16 * kRows); base < rows && !of_v; base += step * (16 * kRows)) {
    int row[kRows];
    float dot[kRows] = {}, sq[kRows] = {};
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const int i = base + u * 16 + sub, r = i & 127, pos = (i >> 7) * p.group_rows + r;
      row[u] = -1;
      if (i < rows && r < p.group_rows && pos < p.Sq) row[u] = query_row(p, bh, pos);
    }
    if (p.perm != nullptr) {
      // dQ's rows are written through perm: those that no entry of it names have no gradient
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        const int i = base + u * 16 + sub, r = i & 127, pos = (i >> 7) * p.group_rows + r;
        if (i >= rows || r >= p.group_rows || pos >= p.Sq) continue;
        for (int c = l16; c < chunks; c += 16) *reinterpret_cast<uint4*>(qb + 2 * (size_t)pos * p.dq_stride[1] + c * 16) = make_uint4(0, 0, 0, 0);
      }
    }
    for (int c = l16; c < chunks; c += 16) {
      uint4 x[kRows], y[kRows];
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        x[u] = y[u] = make_uint4(0, 0, 0, 0);
        if (row[u] >= 0) {
          x[u] = *reinterpret_cast<const uint4*>(gb + 2 * (size_t)row[u] * p.dout_stride[1] + c * 16);
          y[u] = *reinterpret_cast<const uint4*>(ob + 2 * (size_t)row[u] * p.out_stride[1] + c * 16);
        }
      }
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        dot[u] = dot8<kFp16>(x[u], y[u], dot[u]);
        if constexpr (kFp16) sq[u] = dot8<kFp16>(x[u], x[u], sq[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
#pragma unroll
      for (int off = 8; off >= 1; off >>= 1) {
        dot[u] += __shfl_xor_sync(0xffffffffu, dot[u], off);
        if constexpr (kFp16) sq[u] += __shfl_xor_sync(0xffffffffu, sq[u], off);
      }
      m_do = fmaxf(m_do, sq[u] < INFINITY ? sq[u] : 0.f);
      const int i = base + u * 16 + sub;
      if (l16 == 0 && i < rows) {
        float nl = -INFINITY;                                // rows behind the last one: P = 0
        if (row[u] >= 0) {
          const float l = p.lse[(size_t)bh * p.Sq + row[u]];
          // (a row without keys has lse = -inf and no gradient)
          if (l != -INFINITY) nl = (kFp16 ? kBiasFp16 : 0.f) - l * 1.4426950408889634f;
        }
        p.neg_lse2[(size_t)bh * rows + i] = nl;
        p.neg_delta[(size_t)bh * rows + i] = row[u] >= 0 ? -dot[u] : 0.f;
        if (row[u] < 0) p.neg_delta_kv[(size_t)bh * rows + i] = 0.f;      // (the others are written with dQ)
      }
    }
  }
  if constexpr (kFp16) {
    const uint8_t* vb = reinterpret_cast<const uint8_t*>(p.v) + 2 * ((size_t)b * p.v_stride[0] + (size_t)h * p.v_stride[2]);
    const int32_t* start = p.key_start != nullptr ? p.key_start + (size_t)bh * (p.Sk + 1) : nullptr;
    for (int base = blk * (16 * kRows); base < p.Sk && of_v; base += step * (16 * kRows)) {
      float sq[kRows] = {};
      for (int c = l16; c < chunks; c += 16) {
        uint4 x[kRows];
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
          const int i = base + u * 16 + sub;
          x[u] = i < p.Sk && (start == nullptr || start[i + 1] > start[i]) ? *reinterpret_cast<const uint4*>(vb + 2 * (size_t)i * p.v_stride[1] + c * 16)
                                                                           : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < kRows; ++u) sq[u] = dot8<kFp16>(x[u], x[u], sq[u]);
      }
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
#pragma unroll
        for (int off = 8; off >= 1; off >>= 1) sq[u] += __shfl_xor_sync(0xffffffffu, sq[u], off);
        m_v = fmaxf(m_v, sq[u] < INFINITY ? sq[u] : 0.f);
      }
    }
    __shared__ float2 red[8];
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
      m_do = fmaxf(m_do, __shfl_xor_sync(0xffffffffu, m_do, off));
      m_v = fmaxf(m_v, __shfl_xor_sync(0xffffffffu, m_v, off));
    }
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_float2(m_do, m_v);
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int i = 1; i < 8; ++i) { m_do = fmaxf(m_do, red[i].x); m_v = fmaxf(m_v, red[i].y); }
      p.row_max[(size_t)bh * kMaxBlocks + blockIdx.x] = make_float2(sqrtf(m_do) * 1.0001f, sqrtf(m_v) * 1.0001f);
    }
  }
}

// ------------------------------------------------------------------------------------------------ dQ; dK and dV
// One kernel in three modes.  One CTA per SM walks items (head, tile of 128 resident rows, block of output columns, split of the
// streamed axis).  Two resident tiles A0, A1 stay in shared memory, pairs of tiles T0(t), T1(t) of TN rows come through a ring:
//                    A0   A1   T0   T1     S = A0 T0^T     dP = A1 T1^T    sums over t
//   kDq, kDqGather   Q    dO   K    V      rows: queries                   PK += P K     dQ += dS K
//   kDkv             K    V    Q    dO     rows: keys (S^T, dP^T)          dV += P^T dO  dK += dS^T Q
// Scores lie with the resident row as the tensor-memory lane, so that P and dS are the first operands of the sums where they
// are.  A softmax thread copies its scores to registers, which frees S for the next tile at once, and computes P there; when dP(t) is
// complete it reads it and stores P and dS, 16 bits each, over it.  One warp issues dP(t), sum of P(t), sum of dS(t), dP(t+1), ...:
// products of one thread execute in order, so dP(t+1) may follow the sums that read P(t) and dS(t) without a wait.  Another issues
// S(t+1) behind dP(t).  So the exponentials of t+1 run under the sum of dS(t) and dP(t+1), and S(t+1) covers what the tensor pipe
// could wait for, dP(t) -> P stored.
//
// What bounds it.  Per pair of tiles (128 x 128 x 128) the tensor pipe needs 2,048 cycles, shared memory the same (1,536 for operands
// at 128 bytes a cycle, 512 for the next tiles), the special-function unit 1,024, and the chain dP -> registers -> dS -> sum of dS -> next dP
// about 2,400.  One wave of 148 x 148 tiles of one head: 1.61 us a tile on the key side, 1.64 on the query side (about 3,000
// cycles); D = 64: 1.30 and 1.34; D = 144: 2.35 and 2.45 per 128 rows.  In a loop of calls at 24 heads x 32,760 x 128 the power limit
// lowers the clock: 39.8 ms for 52.8 TFLOP of products (1.33 PFLOP/s, against 1.41 that the library's largest products sustain).
// Steps, same call: P stored over its scores, so that S(t+1) had to follow the sum of P(t): 45.6 ms; scores copied out first: 43.5; two issuing
// warps, and every product issued from one place of the program (with a copy of the issuing code in front of the loop, a tile took 10% to
// 30% longer), 16-bit dS summed by mixed-precision additions: 39.8.  Measured and not kept: two tiles of 64 rows in flight, one for each half of
// the softmax warps (D = 64: 1.56 us against 1.44 then); the sum of dS started at half of a tile (1.68 against 1.65).
//
// PK: the rows of dS sum to zero, but those of its rounded form, with a delta from a rounded out, do not: they sum to r, and
// dQ is off by r times the keys that a row looks at, which does not average out where these keys resemble one another (with
// clusters of neighbouring tokens the error of dQ was 5.6e-3 of its norm in bf16, 1.7e-3 of it the result's own rounding).  The
// kernel therefore sums the rounded dS, and PK = sum_j P_ij K_j beside dQ, and stores dQ - r PK: 2.3e-3.  The fourth product takes
// the tensor pipe as long as the kernel of dK and dV does.  The sum of dS before rounding, too, is taken: it is what delta is off
// by, and the key side, which runs second, gets delta without it (dK: 2.7e-3 -> 2.4e-3 with lists of selected keys).
//
// Short sums, and others on idle SMs (kPaired; see pick_paired): the rounding of P and dS does not average out over a few rows, and
// where these resemble one another (neighbouring tokens) the sums cancel and the rounding does not: 7 queries on 33 keys x 64, bf16: error of dK
// 3.5e-3 of its norm, 1.6e-3 of it the result's own rounding.  A tile then holds TN / 2 rows twice, and the second half of the softmax
// threads stores what the first half's rounding left, so that the sums take P and dS with twice the bits.  Up to TN / 2 rows this fills
// what would be padding.
enum { kDq = 0, kDqGather = 1, kDkv = 2 };

template <int DB, int TN>
struct SmemB {
  using G = Geo<DB, TN>;
  static constexpr int kRing = DB == 4 ? 3 : (DB == 1 ? 8 : 5);
  static constexpr int kA0 = 0, kA1 = G::kResBytes;
  static constexpr int kRingOff = 2 * G::kResBytes;
  static constexpr int kStat = kRingOff + kRing * G::kTileBytes;           // kDkv: TN floats per slot, lse2 with Q, delta with dO; kDq: sums of dS
  static constexpr int kStatBytes = kRing * TN * 4 > 1536 ? kRing * TN * 4 : 1536;
  static constexpr int kBars = kStat + kStatBytes;
  static constexpr int kFull = 0, kEmpty = kRing, kAFull = 2 * kRing, kAEmpty = kAFull + 1, kSFull = kAEmpty + 1, kSFree = kSFull + 1,
                       kDPFull = kSFree + 1, kPReady = kDPFull + 1, kDSReady = kPReady + 1, kOFull = kDSReady + 1, kOFree = kOFull + 1,
                       kRowSum = kOFree + 1, kDrain = kRowSum + 1, kCount = kDrain + 2;
  static constexpr int kSlot = kBars + kCount * 8;
  static constexpr int kDynamic = kSlot + 16;
  static constexpr uint32_t kColS = 0, kColDP = TN, kColA = 2 * TN, kWidth = DB > 2 ? 192 : DB * 64, kColB = kColA + kWidth;
};
template <int DB, int TN>
constexpr bool fits = SmemB<DB, TN>::kDynamic <= kMaxSmem && SmemB<DB, TN>::kColB + SmemB<DB, TN>::kWidth <= 512;
static_assert(fits<1, 128> && fits<2, 128> && fits<3, 64> && fits<4, 64>, "227 KB of shared memory, 512 columns of tensor memory");

// Warps: eight softmax warps, two issuers, then for the dense modes the producers of the resident tiles and of the ring, for gathered keys
// six warps that copy both: 512 threads of 128 registers (about 200 bytes of spills per thread at D <= 128).  24 heads x 256 groups x 2,048 keys
// x 128: 1.39 ms.  With one issuing warp instead of two, three copying warps, which leave 168 registers, took 1.63 ms, four 1.54, seven 1.48.
constexpr int kIssueWarp = 8, kScoreWarp = 9, kLoadWarp0 = 10, kGatherWarps = 6;
constexpr int threads_of(int mode) { return mode == kDqGather ? 32 * (kLoadWarp0 + kGatherWarps) : 384; }

// Blocks of output columns: one, or two of 128 where tensor memory does not hold both sums at full width.
__host__ __device__ constexpr int column_blocks(int D) { return D > 192 ? 2 : 1; }

template <int DB, int TN, bool kFp16, int kMode, bool kPaired>
__global__ void __launch_bounds__(threads_of(kMode), 1) attn_bwd_kernel(const AttnBwdParams p, const __grid_constant__ DenseTileMaps maps,
                                                                const __grid_constant__ DenseTileMaps res) {
  using L = SmemB<DB, TN>;
  using G = Geo<DB, TN>;
  constexpr bool kGather = kMode == kDqGather, kRowsAreKeys = kMode == kDkv;
  constexpr int R = L::kRing, HC = G::kHalf;
  constexpr int TR = kPaired ? HC : TN;                      // different rows of a streamed tile
  static_assert(!kPaired || !kGather, "lists of keys are longer");
  // (no room for a manual alignment: the tiles need 1,024 bytes, which the declaration asks for and the host would be told if it failed)
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t s_base = smem_u32(smem);
  if (s_base & 1023u) {
    if (threadIdx.x == 0) atomicCAS(p.status, 0, 1);
    return;
  }
  auto bar = [&](int i) { return s_base + L::kBars + 8u * i; };
  auto sRing = [&](int slot) { return s_base + L::kRingOff + slot * G::kTileBytes; };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kSlot);
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int nd = (p.D + 15) & ~15, kd = nd / 16;             // columns and k-steps that are not padding
  const int res_tiles = kRowsAreKeys ? (p.Sk + 127) / 128 : p.M;
  const int blocks = DB == 4 ? column_blocks(p.D) : 1;
  const int n_items = p.B * p.H * res_tiles * blocks * p.splits;
  struct Item { int bh, b, h, m, c0, ncol, split, t0, t1; };
  auto decode = [&](int item) {
    Item it;
    it.split = item % p.splits;
    int rest = item / p.splits;
    it.c0 = (rest % blocks) * 128;
    rest /= blocks;
    it.m = rest % res_tiles;
    it.bh = rest / res_tiles;
    it.b = it.bh / p.H;
    it.h = it.bh % p.H;
    it.ncol = blocks == 1 ? nd : min(128, nd - it.c0);
    int T;
    if constexpr (kGather) {
      const int most = p.gather_len / 128;
      T = (p.gl != nullptr ? min(max(p.gl[(size_t)it.bh * p.M + it.m], 1), most) : most) * (128 / TN);
    } else {
      T = ((kRowsAreKeys ? p.Sq : p.Sk) + TR - 1) / TR;
    }
    it.t0 = (int)((long long)T * it.split / p.splits);
    it.t1 = (int)((long long)T * (it.split + 1) / p.splits);
    return it;
  };
  // tensor row behind resident tile row r, or -1
  auto row_of = [&](const Item& it, int r) {
    if constexpr (kRowsAreKeys) {
      const int key = it.m * 128 + r;
      return key < p.Sk ? key : -1;
    } else {
      const int pos = it.m * p.group_rows + r;
      if (r >= p.group_rows || pos >= p.Sq) return -1;
      return query_row(p, it.bh, pos);
    }
  };

  if (tid == 0) {
    for (int i = 0; i < R; ++i) { mbar_init(bar(L::kFull + i), kGather ? TN + kGatherWarps : 1); mbar_init(bar(L::kEmpty + i), 1); }
    mbar_init(bar(L::kAFull), kGather ? 256 : 1);
    mbar_init(bar(L::kAEmpty), 2);
    mbar_init(bar(L::kSFull), 1);
    mbar_init(bar(L::kSFree), kSoftmaxWarps);
    mbar_init(bar(L::kDPFull), 1);
    mbar_init(bar(L::kPReady), kSoftmaxWarps);
    mbar_init(bar(L::kDSReady), kSoftmaxWarps);
    mbar_init(bar(L::kOFull), 1);
    mbar_init(bar(L::kOFree), kSoftmaxWarps);
    mbar_init(bar(L::kRowSum), kSoftmaxWarps);
    for (int i = 0; i < 2; ++i) mbar_init(bar(L::kDrain + i), 1);
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
    // each half of the columns keeps its 16-bit operands inside its own columns of dP: no thread overwrites what another still reads
    const uint32_t tS = tmem + L::kColS + x * HC + lane_addr, tDP = tmem + L::kColDP + x * HC + lane_addr;
    const unsigned long long scale2 = f2_pack(p.scale_log2, p.scale_log2);
    int g = 0, ic = 0;
    bool ok = true;
#pragma unroll 1
    for (int item = blockIdx.x; item < n_items && ok; item += gridDim.x) {
      const Item it = decode(item);
      const float c = ds_scale<kFp16>(p, it.bh);
      const unsigned long long c2 = f2_pack(c, c);
      unsigned long long nl2 = 0, nd2 = 0, es[2] = {0, 0};
      float rs[4] = {0.f, 0.f, 0.f, 0.f};
        // kDq: this row's statistics, sums of its dS rounded and not
      if constexpr (!kRowsAreKeys) {
        const size_t si = (size_t)it.bh * p.stat_rows + it.m * 128 + r_in;
        const float nl = p.neg_lse2[si], ndl = p.neg_delta[si];
        nl2 = f2_pack(nl, nl);
        nd2 = f2_pack(ndl, ndl);
      }
#pragma unroll 1
      for (int t = it.t0; t < it.t1; ++t, ++g) {
        const int n0 = 2 * g, n1 = 2 * g + 1;                // ring loads of T0(t), T1(t)
        const ulonglong2* lse = reinterpret_cast<const ulonglong2*>(smem + L::kStat + (n0 % R) * TN * 4 + x * HC * 4);
        const ulonglong2* dlt = reinterpret_cast<const ulonglong2*>(smem + L::kStat + (n1 % R) * TN * 4 + x * HC * 4);
        ok = mbar_wait(bar(L::kSFull), g & 1, p.status, 130);
        if constexpr (kRowsAreKeys) ok = ok && mbar_wait(bar(L::kFull + n0 % R), (n0 / R) & 1, p.status, 131);
        if (!ok) break;
        tc_fence_after();
        uint32_t sc[HC];
        load_columns<HC>(tS, sc);
        tmem_wait_ld();
        tc_fence_before();
        warp_arrive(bar(L::kSFree));
#pragma unroll
        for (int i = 0; i < HC; i += 4) {
          unsigned long long l0 = nl2, l1 = nl2;
          if constexpr (kRowsAreKeys) {
            const ulonglong2 l = lse[i / 4];
            l0 = l.x;
            l1 = l.y;
          }
          const float2 y0 = f2_unpack(f2_fma(f2_pack(__uint_as_float(sc[i]), __uint_as_float(sc[i + 1])), scale2, l0));
          const float2 y1 = f2_unpack(f2_fma(f2_pack(__uint_as_float(sc[i + 2]), __uint_as_float(sc[i + 3])), scale2, l1));
          sc[i] = __float_as_uint(ex2_approx(y0.x));
          sc[i + 1] = __float_as_uint(ex2_approx(y0.y));
          sc[i + 2] = __float_as_uint(ex2_approx(y1.x));
          sc[i + 3] = __float_as_uint(ex2_approx(y1.y));
        }
        if constexpr (kMode == kDq) {
          // key positions behind the sequence end (zero rows of the last tile): exp2(-lse2) could be anything
          const int rem = p.Sk - t * TR - (kPaired ? 0 : x * HC);
          if (rem < HC) {
#pragma unroll
            for (int i = 0; i < HC; ++i)
              if (i >= rem) sc[i] = 0;
          }
        }
        ok = mbar_wait(bar(L::kDPFull), g & 1, p.status, 132);
        if constexpr (kRowsAreKeys) ok = ok && mbar_wait(bar(L::kFull + n1 % R), (n1 / R) & 1, p.status, 133);
        if (!ok) break;
        tc_fence_after();
        // dP in steps of 32 columns (all 64 at once would spill); P goes over the first half of this thread's columns as soon as
        // those are read, dS over the second half
        constexpr int kStep = 32;
        static_assert(kStep >= HC / 2, "P overwrites columns that have been read");
        uint32_t dp[kStep];
        load_columns<kStep>(tDP, dp);
        tmem_wait_ld();
#pragma unroll
        for (int q = 0; q < HC / 16; ++q) {
          if (kPaired && x == 1) {
            uint32_t rest[16];
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              float a = __uint_as_float(sc[q * 16 + i]), b = __uint_as_float(sc[q * 16 + i + 1]);
              keep_rest<kFp16>(a, b);
              rest[i] = __float_as_uint(a);
              rest[i + 1] = __float_as_uint(b);
            }
            store_packed<kFp16>(tDP + q * 8, rest);
          } else {
            store_packed<kFp16>(tDP + q * 8, &sc[q * 16]);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        warp_arrive(bar(L::kPReady));
#pragma unroll
        for (int s0 = 0; s0 < HC; s0 += kStep) {
          uint32_t pk[kStep / 2];
#pragma unroll
          for (int d = 0; d < kStep; d += 4) {
            const int e = s0 + d;
            unsigned long long e0 = nd2, e1 = nd2;
            if constexpr (kRowsAreKeys) {
              const ulonglong2 l = dlt[e / 4];
              e0 = l.x;
              e1 = l.y;
            }
            unsigned long long d0 = f2_add(f2_pack(__uint_as_float(dp[d]), __uint_as_float(dp[d + 1])), e0);
            unsigned long long d1 = f2_add(f2_pack(__uint_as_float(dp[d + 2]), __uint_as_float(dp[d + 3])), e1);
            if constexpr (kFp16) { d0 = f2_mul(d0, c2); d1 = f2_mul(d1, c2); }
            d0 = f2_mul(f2_pack(__uint_as_float(sc[e]), __uint_as_float(sc[e + 1])), d0);
            d1 = f2_mul(f2_pack(__uint_as_float(sc[e + 2]), __uint_as_float(sc[e + 3])), d1);
            float2 y0 = f2_unpack(d0), y1 = f2_unpack(d1);
            if (kPaired && x == 1) {
              keep_rest<kFp16>(y0.x, y0.y);
              keep_rest<kFp16>(y1.x, y1.y);
            }
            pk[d / 2] = pack16<kFp16>(y0.x, y0.y);
            pk[d / 2 + 1] = pack16<kFp16>(y1.x, y1.y);
            if constexpr (!kRowsAreKeys) {
              if (!kPaired || x == 0) {
                es[0] = f2_add(es[0], d0);
                es[1] = f2_add(es[1], d1);
              }
              add_pair<kFp16>(pk[d / 2], rs[0], rs[1]);
              add_pair<kFp16>(pk[d / 2 + 1], rs[2], rs[3]);
            }
          }
          // (columns from HC / 2 on: those of the second step have been read, or are not there)
          if (s0 + kStep < HC) {
            // ... so the first step's dS waits in registers until the second step's dP has been copied
            uint32_t next[kStep];
            load_columns<kStep>(tDP + s0 + kStep, next);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < kStep; ++i) dp[i] = next[i];
          }
#pragma unroll
          for (int q = 0; q < kStep / 16; ++q) tmem_st8(tDP + HC / 2 + s0 / 2 + q * 8, *reinterpret_cast<const uint32_t(*)[8]>(&pk[q * 8]));
        }
        tmem_wait_st();
        tc_fence_before();
        warp_arrive(bar(L::kDSReady));
      }
      if (!ok) break;
      const float unbias = kFp16 ? 6.103515625e-05f : 1.f;                     // 2^-14
      float fix = 0.f, off = 0.f;
      if constexpr (!kRowsAreKeys) {
        // The row's sums of dS from its two threads.  A thread arrives at kOFree behind its reads of the other's, and none writes here before
        // all have arrived there for the item before: an item of one tile gets this far on S and dP, for which nobody waits for kOFree.
        if (ic > 0) ok = mbar_wait(bar(L::kOFree), (ic - 1) & 1, p.status, 146);
        if (!ok) break;
        float* sums = reinterpret_cast<float*>(smem + L::kStat);
        const float2 a2 = f2_unpack(es[0]), b2 = f2_unpack(es[1]);
        sums[x * 128 + r_in] = (rs[0] + rs[1]) + (rs[2] + rs[3]);
        off = (a2.x + a2.y) + (b2.x + b2.y);
        if (x == 1) sums[256 + r_in] = off;
        warp_arrive(bar(L::kRowSum));
        ok = mbar_wait(bar(L::kRowSum), ic & 1, p.status, 134);
        if (!ok) break;
        fix = sums[r_in] + sums[128 + r_in];
        off = (off + sums[256 + r_in]) * unbias / c;         // (used by the first half only)
        if (p.splits == 1 && x == 0 && it.c0 == 0) {
          const size_t si = (size_t)it.bh * p.stat_rows + it.m * 128 + r_in;
          p.neg_delta_kv[si] = p.neg_delta[si] - off;
        }
      }
      ok = mbar_wait(bar(L::kOFull), ic & 1, p.status, 135);
      if (!ok) break;
      tc_fence_after();
      const int row = row_of(it, r_in);
      const size_t safe = row < 0 ? 0 : row;
      // kDkv: the first half of the warps stores dV, the second dK; kDq: each half stores its half of the columns of dQ
      const bool second = kRowsAreKeys && x == 1;
      const float w = kRowsAreKeys && x == 0 ? unbias : p.out_scale / c * unbias;
      const int64_t* st = kRowsAreKeys ? (second ? p.dk_stride : p.dv_stride) : p.dq_stride;
      void* dst = kRowsAreKeys ? (second ? p.dk : p.dv) : p.dq;
      uint8_t* optr = reinterpret_cast<uint8_t*>(dst) + 2 * ((size_t)it.b * st[0] + safe * st[1] + (size_t)it.h * st[2]);
      // (32-byte stores where every row starts on a 32-byte boundary)
      const bool wide = ((reinterpret_cast<uintptr_t>(dst) | (uintptr_t)(2 * (st[0] | st[1] | st[2]))) & 31) == 0;
      const int S = kRowsAreKeys ? p.Sk : p.Sq;
      // a row of partial sums: dK | dV, or dQ | PK | the sums of dS (padded to 8 floats)
      const int pitch = kRowsAreKeys ? 2 * p.D : 2 * p.D + 8;
      float* part = p.parts + (((size_t)it.split * p.B * p.H + it.bh) * S + safe) * pitch;
      const int mid = ((it.ncol / 16 + 1) / 2) * 16;
      const int b0 = kRowsAreKeys || x == 0 ? 0 : mid, b1 = kRowsAreKeys || x == 1 ? it.ncol : mid;
      const uint32_t tA = tmem + L::kColA + lane_addr, tB = tmem + L::kColB + lane_addr;
#pragma unroll 1
      for (int cc = b0; cc < b1; cc += 16) {
        uint32_t ra[16], rb[16];
        if (!kRowsAreKeys || x == 0) tmem_ld16(tA + cc, ra);
        if (!kRowsAreKeys || x == 1) tmem_ld16(tB + cc, rb);
        tmem_wait_ld();
        float f[16], e[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if constexpr (kRowsAreKeys) {
            f[i] = __uint_as_float(x == 0 ? ra[i] : rb[i]) * w;
          } else if (p.splits > 1) {
            f[i] = __uint_as_float(rb[i]) * w;
            e[i] = __uint_as_float(ra[i]) * unbias;
          } else {
            f[i] = fmaf(-fix * unbias, __uint_as_float(ra[i]), __uint_as_float(rb[i])) * w;
          }
        }
        const int col = it.c0 + cc;
        if (row >= 0 && p.splits > 1) {
#pragma unroll
          for (int q = 0; q < 16; q += 8) {
            if (col + q >= p.D) break;
            store8(part + (kRowsAreKeys && x == 0 ? p.D : 0) + col + q, f + q);
            if constexpr (!kRowsAreKeys) store8(part + p.D + col + q, e + q);
          }
        } else if (row >= 0) {
          float o[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] = __uint_as_float(pack16<kFp16>(f[2 * i], f[2 * i + 1]));
          if (wide && col + 16 <= p.D) {
            store8(reinterpret_cast<float*>(optr + 2 * col), o);
          } else {
            *reinterpret_cast<float4*>(optr + 2 * col) = make_float4(o[0], o[1], o[2], o[3]);
            if (col + 16 <= p.D) *reinterpret_cast<float4*>(optr + 2 * col + 16) = make_float4(o[4], o[5], o[6], o[7]);
          }
        }
        __syncwarp();
      }
      if (!kRowsAreKeys && p.splits > 1 && x == 0 && row >= 0 && it.c0 == 0) {
        part[2 * p.D] = fix * w;
        part[2 * p.D + 1] = off;
      }
      tc_fence_before();
      warp_arrive(bar(L::kOFree));
      ++ic;
    }
    tc_fence_before();
  } else if (warp == kIssueWarp || warp == kScoreWarp) {
    // ---- issuers of the products: S by one warp, dP and the sums, whose order matters, by the other.  Issuing a product's eight steps takes
    // a warp about as long as they take the tensor pipe; one warp for all four had the pipe wait for it.
    constexpr uint32_t kFmt = kFp16 ? 0u : 1u;
    constexpr uint32_t idesc_s = mma_idesc(kFmt, kFmt, 0, 0, 128, TN);
    const bool leader = elect_one();
    bool ok = true;
    int g = 0, ic = 0;
    auto wait_full = [&](int load) {
      ok = ok && mbar_wait(bar(L::kFull + load % R), (load / R) & 1, p.status, 136);
      if (!ok) return;
      if constexpr (kGather) fence_proxy_async_smem();
      tc_fence_after();
    };
    // (unrolled, the k-steps of padding predicated off: with a rolled loop of kd steps one of the products had its last step
    // accumulated nine times; why is not known)
    auto scores = [&](uint32_t d, uint32_t a_tile, int load) {
      const uint32_t alo = lo_kmajor(a_tile), blo = lo_kmajor(sRing(load % R));
      auto step = [&](int j) {
        const uint32_t in = (j & 3) * 2;
        if (leader) mma_f16_ss(d, desc_lo(alo + (j >> 2) * (16384 >> 4) + in), desc_lo(blo + (j >> 2) * (TN * 128 >> 4) + in), idesc_s, j > 0);
      };
      if (kd == DB * 4) {
#pragma unroll
        for (int j = 0; j < DB * 4; ++j) step(j);
      } else {
#pragma unroll
        for (int j = 0; j < DB * 4; ++j)
          if (j < kd) step(j);
      }
    };
    // sum over a tile of T rows; the operands of the two halves of the columns lie HC columns apart
    auto sum = [&](uint32_t d, uint32_t a, int load, const Item& it, uint32_t idesc, bool first) {
      const uint32_t blo = lo_mnmajor(sRing(load % R) + (it.c0 >> 6) * TN * 128, TN * 128);
#pragma unroll
      for (int j = 0; j < TN / 16; ++j)
        if (leader) mma_f16_ts(d, a + (j / (HC / 16)) * HC + (j % (HC / 16)) * 8, desc_lo(blo + j * (2048 >> 4)), idesc, !first || j > 0);
    };
    auto wait_resident = [&]() {
      ok = mbar_wait(bar(L::kAFull), ic & 1, p.status, 137);
      if (!ok) return;
      if constexpr (kGather) fence_proxy_async_smem();
      tc_fence_after();
    };
    // (tiles of 64 rows, whose products are short, do better in any order: 18,944 x 144 takes 385 us a side against 460)
    constexpr bool kOrdered = TN == 128;
    if (warp == kScoreWarp) {
#pragma unroll 1
      for (int item = blockIdx.x; item < n_items && ok; item += gridDim.x, ++ic) {
        const Item it = decode(item);
        wait_resident();
#pragma unroll 1
        for (int t = it.t0; t < it.t1 && ok; ++t, ++g) {
          // Its columns are free once the tile before has been copied out.  That tile's dP goes first: the softmax waits for it longer.
          // (dP of tile g in turn is issued behind a wait for this product, so neither barrier can run two phases ahead of its waits.)
          wait_full(2 * g);
          if (ok && kOrdered && t > it.t0) ok = mbar_wait(bar(L::kDPFull), (g - 1) & 1, p.status, 144);
          if (ok && g > 0) ok = mbar_wait(bar(L::kSFree), (g - 1) & 1, p.status, 143);
          if (!ok) break;
          tc_fence_after();
          scores(tmem + L::kColS, s_base + L::kA0, 2 * g);
          if (leader) {
            tc_commit(bar(L::kSFull));
            if (t == it.t1 - 1) tc_commit(bar(L::kAEmpty));
          }
        }
      }
    } else {
#pragma unroll 1
      for (int item = blockIdx.x; item < n_items && ok; item += gridDim.x, ++ic) {
        const Item it = decode(item);
        const uint32_t idesc_o = mma_idesc(kFmt, kFmt, 0, 1, 128, it.ncol);
        wait_resident();
        if (!ok) break;
#pragma unroll 1
        for (int t = it.t0; t < it.t1; ++t, ++g) {
          const bool first = t == it.t0, last = t == it.t1 - 1;
          const int n = 2 * g;
          if (kOrdered && !first) ok = mbar_wait(bar(L::kSFull), g & 1, p.status, 145);
          wait_full(n + 1);
          if (!ok) break;
          scores(tmem + L::kColDP, s_base + L::kA1, n + 1);
          if (leader) {
            tc_commit(bar(L::kDPFull));
            if (!kRowsAreKeys) tc_commit(bar(L::kEmpty + (n + 1) % R));
            if (last) tc_commit(bar(L::kAEmpty));
          }
          ok = mbar_wait(bar(L::kPReady), g & 1, p.status, 138);
          if (ok && first && ic > 0) ok = mbar_wait(bar(L::kOFree), (ic - 1) & 1, p.status, 139);
          if (!ok) break;
          tc_fence_after();
          sum(tmem + L::kColA, tmem + L::kColDP, kRowsAreKeys ? n + 1 : n, it, idesc_o, first);
          if (kRowsAreKeys && leader) tc_commit(bar(L::kEmpty + (n + 1) % R));
          ok = mbar_wait(bar(L::kDSReady), g & 1, p.status, 140);
          if (!ok) break;
          tc_fence_after();
          sum(tmem + L::kColB, tmem + L::kColDP + HC / 2, n, it, idesc_o, first);
          if (leader) {
            tc_commit(bar(L::kEmpty + n % R));
            if (last) tc_commit(bar(L::kOFull));
          }
        }
      }
    }
    if (!ok) {
      // error path: let outstanding products retire before tensor memory is released
      if (leader) tc_commit(bar(L::kDrain + (warp == kScoreWarp ? 1 : 0)));
      mbar_wait_quiet(bar(L::kDrain + (warp == kScoreWarp ? 1 : 0)), 0, 1 << 20);
    }
    __syncwarp();
    tc_fence_before();
  } else if (kGather) {
    // ---- gathered keys: the warps take batches of 32 rows in turn.  The resident tiles of an item follow its first pair of T tiles,
    // which do not have to wait for the item before to be done with A0 and A1.
    constexpr int kBatches = TN / 32, kWarps = kGatherWarps;
    const int w = warp - kLoadWarp0;
    int n = 0, ic = 0, batch = 0;
    bool ok = true;
    // indices of the tile that is copied, and of the next one of the item, in flight meanwhile
    int key[kBatches], next[kBatches];
    auto fetch = [&](const int32_t* gi, int t, int (&dst)[kBatches]) {
#pragma unroll
      for (int q = 0; q < kBatches; ++q) dst[q] = __ldg(gi + (size_t)t * TN + q * 32 + lane);
    };
#pragma unroll 1
    for (int item = blockIdx.x; item < n_items && ok; item += gridDim.x, ++ic) {
      const Item it = decode(item);
      const int32_t* gi = p.gi + ((size_t)it.bh * p.M + it.m) * p.gather_len;
      const uint8_t* kb = reinterpret_cast<const uint8_t*>(p.k) + 2 * ((size_t)it.b * p.k_stride[0] + (size_t)it.h * p.k_stride[2]);
      const uint8_t* vb = reinterpret_cast<const uint8_t*>(p.v) + 2 * ((size_t)it.b * p.v_stride[0] + (size_t)it.h * p.v_stride[2]);
      fetch(gi, it.t0, key);
#pragma unroll 1
      for (int t = it.t0; t < it.t1 && ok; ++t) {
        if (t + 1 < it.t1) fetch(gi, t + 1, next);
#pragma unroll 1
        for (int is_t1 = 0; is_t1 < 2; ++is_t1, ++n) {
          const int slot = n % R;
          if (n >= R) ok = mbar_wait(bar(L::kEmpty + slot), (n / R - 1) & 1, p.status, 142);
          if (!ok) break;
#pragma unroll
          for (int q = 0; q < kBatches; ++q) {
            if (batch == w) {
              warp_copy_rows<DB>(sRing(slot), TN, q * 32, min(max(key[q], 0), p.Sk - 1), p.D, is_t1 ? vb : kb,
                                 2 * (size_t)(is_t1 ? p.v_stride[1] : p.k_stride[1]), p.k);
              cp_async_arrive_noinc(bar(L::kFull + slot));
            }
            batch = batch == kWarps - 1 ? 0 : batch + 1;
          }
          // Every warp has a part in every load, with rows of it or without: a load that could be consumed without this warp might free its
          // slot again before the wait above has seen the phase that it waits for, whose parity would then never come back.
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(L::kFull + slot));
        }
        if (!ok) break;
        if (t == it.t0) {
          if (ic > 0) ok = mbar_wait(bar(L::kAEmpty), (ic - 1) & 1, p.status, 141);
          if (!ok) break;
#pragma unroll 1
          for (int q = 0; q < 8; ++q) {
            if (batch == w) {
              const bool a1 = q >= 4;
              const int64_t* ast = a1 ? p.dout_stride : p.q_stride;
              const uint8_t* src = reinterpret_cast<const uint8_t*>(a1 ? p.dout : p.q) + 2 * ((size_t)it.b * ast[0] + (size_t)it.h * ast[2]);
              warp_copy_rows<DB>(s_base + (a1 ? L::kA1 : L::kA0), 128, (q & 3) * 32, row_of(it, (q & 3) * 32 + lane), p.D, src, 2 * (size_t)ast[1], p.q);
              cp_async_arrive_noinc(bar(L::kAFull));
            }
            batch = batch == kWarps - 1 ? 0 : batch + 1;
          }
        }
#pragma unroll
        for (int q = 0; q < kBatches; ++q) key[q] = next[q];
      }
    }
    cp_async_wait_all();
    tc_fence_before();
  } else if (warp == kLoadWarp0) {
    // ---- the resident tiles of an item, by TMA
    const bool leader = elect_one();
    int ic = 0;
    bool ok = true;
#pragma unroll 1
    for (int item = blockIdx.x; item < n_items && ok; item += gridDim.x, ++ic) {
      const Item it = decode(item);
      if (ic > 0) ok = mbar_wait(bar(L::kAEmpty), (ic - 1) & 1, p.status, 141);
      if (!ok) break;
      if (leader) {
        mbar_arrive_expect_tx(bar(L::kAFull), 2 * G::kResBytes);
        int c0[4] = {0, 0, 0, 0}, c1[4] = {0, 0, 0, 0};
        c0[res.k_pos_h] = it.h; c0[res.k_pos_b] = it.b; c0[res.k_pos_row] = it.m * 128;
        c1[res.v_pos_h] = it.h; c1[res.v_pos_b] = it.b; c1[res.v_pos_row] = it.m * 128;
#pragma unroll
        for (int cb = 0; cb < DB; ++cb) {
          tma_load_4d(s_base + L::kA0 + cb * 16384, res.k, cb * 64, c0[1], c0[2], c0[3], bar(L::kAFull));
          tma_load_4d(s_base + L::kA1 + cb * 16384, res.v, cb * 64, c1[1], c1[2], c1[3], bar(L::kAFull));
        }
      }
    }
    if (!ok && ic > 0) mbar_wait_quiet(bar(L::kAFull), (ic - 1) & 1, 1 << 16);   // copies in flight
    tc_fence_before();
  } else if (warp == kLoadWarp0 + 1) {
    // ---- the ring: T0(0), T1(0), T0(1), ... by TMA
    const bool leader = elect_one();
    int n = 0;
    bool ok = true;
#pragma unroll 1
    for (int item = blockIdx.x; item < n_items && ok; item += gridDim.x) {
      const Item it = decode(item);
      int c0[4] = {0, 0, 0, 0}, c1[4] = {0, 0, 0, 0};
      c0[maps.k_pos_h] = it.h; c0[maps.k_pos_b] = it.b;
      c1[maps.v_pos_h] = it.h; c1[maps.v_pos_b] = it.b;
#pragma unroll 1
      for (int e = 2 * it.t0; e < 2 * it.t1 && ok; ++e, ++n) {
        const bool is_t1 = e & 1;
        const int slot = n % R;
        if (n >= R) ok = mbar_wait(bar(L::kEmpty + slot), (n / R - 1) & 1, p.status, 142);
        if (!ok) break;
        if (leader) {
          mbar_arrive_expect_tx(bar(L::kFull + slot), G::kTileBytes + (kRowsAreKeys ? TN * 4 : 0));
          const void* map = is_t1 ? static_cast<const void*>(maps.v) : static_cast<const void*>(maps.k);
          int co[4] = {0, is_t1 ? c1[1] : c0[1], is_t1 ? c1[2] : c0[2], is_t1 ? c1[3] : c0[3]};
          co[is_t1 ? maps.v_pos_row : maps.k_pos_row] = (e >> 1) * TR;
#pragma unroll
          for (int half = 0; half < TN / TR; ++half) {       // (boxes of TR rows)
#pragma unroll
            for (int cb = 0; cb < DB; ++cb)
              tma_load_4d(sRing(slot) + (cb * TN + half * TR) * 128, map, cb * 64, co[1], co[2], co[3], bar(L::kFull + slot));
            if constexpr (kRowsAreKeys)
              bulk_load(s_base + L::kStat + (slot * TN + half * TR) * 4,
                        (is_t1 ? p.neg_delta_kv : p.neg_lse2) + (size_t)it.bh * p.stat_rows + (size_t)(e >> 1) * TR, TR * 4, bar(L::kFull + slot));
          }
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
// kFix (dQ): minus the row's sum of rounded dS (at 2 D) times its PK (at D), each summed over the splits first; the sum of dS before
// rounding (at 2 D + 1) corrects the row's delta for the key side.
template <bool kFp16, bool kFix>
__global__ void __launch_bounds__(256) attn_bwd_sum_kernel(const float* parts, int splits, long long split_pitch, int pitch, int col0, int D, int H, int S,
                                                           long long rows, void* out, long long sb, long long ss, long long sh,
                                                           const float* neg_delta, float* neg_delta_kv, int stat_rows) {
  const int chunks = D / 8;
  const long long n = rows * chunks;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const long long row = i / chunks;
    const int c = (int)(i - row * chunks) * 8;
    const float* base = parts + row * pitch;
    auto total = [&](int at, float (&f)[8]) {
      const float* src = base + at;
      for (int s = 0; s < splits; ++s, src += split_pitch) {
        const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
        f[0] += a.x; f[1] += a.y; f[2] += a.z; f[3] += a.w;
        f[4] += b.x; f[5] += b.y; f[6] += b.z; f[7] += b.w;
      }
    };
    float f[8] = {};
    total(col0 + c, f);
    if constexpr (kFix) {
      float pk[8] = {}, r = 0.f;
      total(D + c, pk);
      for (int s = 0; s < splits; ++s) r += base[2 * D + s * split_pitch];
      if (c == 0) {
        float off = 0.f;
        for (int s = 0; s < splits; ++s) off += base[2 * D + 1 + s * split_pitch];
        const long long bh = row / S, si = bh * stat_rows + (row - bh * S);
        neg_delta_kv[si] = neg_delta[si] - off;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = fmaf(-r, pk[j], f[j]);
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

// Splits of the summed axis (T tiles) for `items` items without splits, whose partial sums are `part_bytes` per split.  Measured
// at 1.9 GHz: a tile takes tile_us; an item besides 3.5 us to fill, drain and store (5.5 us with fp32 partial sums); the kernel that
// adds the partial sums reads them at 4.3 TB/s and takes 5.5 us besides (2 heads x 257 x 64: dQ's 5.3, dK's and dV's together 5.9).
int pick_splits(long long items, int T, double tile_us, double part_bytes) {
  // (for the B200's 148 SMs, whatever the current device: the workspace must not depend on the device that asks)
  constexpr int kSms = 148;
  double best = 0;
  int pick = 1;
  for (int s = 1; s <= T && s <= 32; ++s) {
    const double waves = (double)((items * s + kSms - 1) / kSms);
    const double us = waves * ((T + s - 1) / s * tile_us + (s > 1 ? 5.5 : 3.5)) + (s > 1 ? 5.5 + s * part_bytes / 4.3e6 : 0.0);
    if (s == 1 || us < best) { best = us; pick = s; }
  }
  return pick;
}

// Most bytes of one pass's contributions in the gather call (a single head's may be more).  24 heads x 256 groups x 2,048 keys x 128, whole call:
// 7.41 ms in passes of 4 GiB, 7.44 in 2, 7.73 in 1 (more launches with a partly filled last wave).
constexpr size_t kPartsBytes = 4ull << 30;

struct Plan { bool pair_k, pair_q; int stat_rows, dq_splits, kv_splits, segs, heads_per_pass; size_t stats, row_max, entries, starts, counts, blocks, parts, total; };

constexpr size_t kAlign = 256;
size_t up(size_t n) { return (n + kAlign - 1) / kAlign * kAlign; }

// Whether tiles of a streamed axis of S rows hold their rows twice: up to 64 rows, where that fills padding (D <= 128), and where the tiles of
// all items, now twice as many, are no more than the SMs, most of which would be idle: there accuracy takes time from nobody else.  Errors
// relative to those of a 32-bit computation that rounds its results once, 1 to 8 heads, 130 to 2,000 rows on 7 to 2,000, D 64 to 144: single
// parts about 1.4 whatever the length, up to 1.9 where few rows carry the sum, and 88 of 1,632 calls above 1.5; with this rule 1.0 where it takes
// two parts, and 2 calls above 1.5 (1.52).  Time of a captured call in bf16, D = 128: 128 x 128 17.9 -> 21.6 us, 2 heads x 300 x 300
// 26.7 -> 34.5, 4 heads x 512 x 512 29.0 -> 37.0, 1,000 x 1,000 37.0 -> 39.3, 2,000 x 300 34.9 -> 44.4.
bool pick_paired(long long items, int S, int TN) { return S <= 64 || items * ((S + TN / 2 - 1) / (TN / 2)) <= 148; }

// Rows of a streamed tile: as many as tensor memory holds beside both sums, and shared memory beside the resident tiles.  (96 rows up to
// D = 160 would fit, with a ring of three tiles instead of five: 18,944 x 144 took 488 us a side against 455.)
int tile_rows(int D) { return D <= 128 ? 128 : 64; }

int padded_blocks(int D) { return D <= 64 ? 1 : (D <= 128 ? 2 : (D <= 192 ? 3 : 4)); }

Plan make_plan(const AttnBwdParams& p, bool gather) {
  constexpr int kSms = 148;
  Plan w{};
  const int TN = tile_rows(p.D);
  const long long bh = (long long)p.B * p.H;
  const int blocks = column_blocks(p.D);
  if (gather) {
    w.dq_splits = w.kv_splits = 1;
  } else {
    const double tile_us = p.D <= 64 ? 1.3 : (p.D <= 128 ? 1.6 : 1.2);
    const long long q_items = bh * p.M * blocks, k_items = bh * ((p.Sk + 127) / 128) * blocks;
    w.pair_k = pick_paired(q_items, p.Sk, TN);
    w.pair_q = pick_paired(k_items, p.Sq, TN);
    const int tk = w.pair_k ? TN / 2 : TN, tq = w.pair_q ? TN / 2 : TN;
    w.dq_splits = pick_splits(q_items, (p.Sk + tk - 1) / tk, tile_us, (double)bh * p.Sq * (2 * p.D + 8) * 4);
    w.kv_splits = pick_splits(k_items, (p.Sq + tq - 1) / tq, tile_us, (double)bh * p.Sk * 2 * p.D * 4);
  }
  w.stat_rows = p.M * 128;
  w.stats = up((size_t)bh * w.stat_rows * 4);
  w.row_max = up((size_t)bh * kMaxBlocks * 8);
  size_t a = w.dq_splits > 1 ? (size_t)w.dq_splits * bh * p.Sq * (2 * p.D + 8) * 4 : 0, b = w.kv_splits > 1 ? (size_t)w.kv_splits * bh * p.Sk * 2 * p.D * 4 : 0;
  w.parts = up(a > b ? a : b);
  if (gather) {
    // segments of groups: enough CTAs for the counting sort without counts that outgrow the indices
    const long long want = (4 * kSms + bh - 1) / bh;
    w.segs = (int)(want < 16 ? want : 16);
    if (w.segs > p.M) w.segs = p.M;
    w.entries = up((size_t)bh * p.M * p.gather_len * 4);
    w.starts = up((size_t)bh * (p.Sk + 1) * 4);
    w.counts = up((size_t)bh * w.segs * p.Sk * 4);
    w.blocks = up((size_t)bh * ((p.Sk + 1023) / 1024) * 4);
    // the contributions of as many heads at a time as fit kPartsBytes, at least one
    const size_t head = (size_t)p.M * p.gather_len * 2 * p.D * 4;
    const long long fit = (long long)(kPartsBytes / head);
    w.heads_per_pass = (int)(fit < 1 ? 1 : (fit > bh ? bh : fit));
    const int passes = (int)((bh + w.heads_per_pass - 1) / w.heads_per_pass);
    w.heads_per_pass = (int)((bh + passes - 1) / passes);
    w.parts = up(w.heads_per_pass * head);
  }
  w.total = 3 * w.stats + w.row_max + w.entries + w.starts + w.counts + w.blocks + w.parts;
  return w;
}

template <typename K>
int set_smem(K kern, int bytes) {
  return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess ? 0 : -8;
}

template <int DB, int TN, bool kFp16>
int launch_dense(AttnBwdParams& p, const Plan& w, cudaStream_t stream) {
  // boxes of TN rows (paired: half as many, twice) for streamed tiles, of 128 for resident ones
  const int rows_k = w.pair_k ? TN / 2 : TN, rows_q = w.pair_q ? TN / 2 : TN;
  auto maps = [&](DenseTileMaps& m, const void* a, const int64_t* as, const void* b, const int64_t* bs, int S, int rows) {
    return encode_tile_map(a, as, p.B, S, p.H, p.D, m.k, m.k_pos_h, m.k_pos_row, m.k_pos_b, rows) &&
           encode_tile_map(b, bs, p.B, S, p.H, p.D, m.v, m.v_pos_h, m.v_pos_row, m.v_pos_b, rows);
  };
  DenseTileMaps kv, qd, res_kv, res_qd;
  if (!maps(kv, p.k, p.k_stride, p.v, p.v_stride, p.Sk, rows_k) || !maps(qd, p.q, p.q_stride, p.dout, p.dout_stride, p.Sq, rows_q)) return -9;
  res_kv = kv;
  res_qd = qd;
  if (rows_k != 128 && !maps(res_kv, p.k, p.k_stride, p.v, p.v_stride, p.Sk, 128)) return -9;
  if (rows_q != 128 && !maps(res_qd, p.q, p.q_stride, p.dout, p.dout_stride, p.Sq, 128)) return -9;
  const int sms = sm_count();
  const long long bh = (long long)p.B * p.H;
  auto dq = w.pair_k ? attn_bwd_kernel<DB, TN, kFp16, kDq, true> : attn_bwd_kernel<DB, TN, kFp16, kDq, false>;
  auto dkv = w.pair_q ? attn_bwd_kernel<DB, TN, kFp16, kDkv, true> : attn_bwd_kernel<DB, TN, kFp16, kDkv, false>;
  constexpr int kSmem = SmemB<DB, TN>::kDynamic;
  if (set_smem(dq, kSmem) || set_smem(dkv, kSmem)) return -8;
  const int blocks = column_blocks(p.D);
  auto grid_of = [](long long n) { return (unsigned)(n / 256 + 1 < 148 * 8 ? n / 256 + 1 : 148 * 8); };
  p.splits = w.dq_splits;
  long long items = bh * p.M * blocks * p.splits;
  dq<<<(unsigned)(items < sms ? items : sms), 384, kSmem, stream>>>(p, kv, res_qd);
  if (p.splits > 1)
    attn_bwd_sum_kernel<kFp16, true><<<grid_of(bh * p.Sq * (p.D / 8)), 256, 0, stream>>>(
        p.parts, p.splits, bh * p.Sq * (2 * p.D + 8), 2 * p.D + 8, 0, p.D, p.H, p.Sq, bh * p.Sq, p.dq, p.dq_stride[0], p.dq_stride[1], p.dq_stride[2],
        p.neg_delta, p.neg_delta_kv, p.stat_rows);
  p.splits = w.kv_splits;
  items = bh * ((p.Sk + 127) / 128) * blocks * p.splits;
  dkv<<<(unsigned)(items < sms ? items : sms), 384, kSmem, stream>>>(p, qd, res_kv);
  if (p.splits > 1) {
    const unsigned grid = grid_of(bh * p.Sk * (p.D / 8));
    attn_bwd_sum_kernel<kFp16, false><<<grid, 256, 0, stream>>>(p.parts, p.splits, bh * p.Sk * 2 * p.D, 2 * p.D, 0, p.D, p.H, p.Sk, bh * p.Sk, p.dk,
                                                                p.dk_stride[0], p.dk_stride[1], p.dk_stride[2], nullptr, nullptr, 0);
    attn_bwd_sum_kernel<kFp16, false><<<grid, 256, 0, stream>>>(p.parts, p.splits, bh * p.Sk * 2 * p.D, 2 * p.D, p.D, p.D, p.H, p.Sk, bh * p.Sk, p.dv,
                                                                p.dv_stride[0], p.dv_stride[1], p.dv_stride[2], nullptr, nullptr, 0);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -8;
}

template <int DB, int TN, bool kFp16>
int launch_gather_dq(AttnBwdParams& p, cudaStream_t stream) {
  auto dq = attn_bwd_kernel<DB, TN, kFp16, kDqGather, false>;
  constexpr int kSmem = SmemB<DB, TN>::kDynamic;
  if (set_smem(dq, kSmem)) return -8;
  const int sms = sm_count();
  p.splits = 1;
  const long long items = (long long)p.B * p.H * p.M * column_blocks(p.D);
  dq<<<(unsigned)(items < sms ? items : sms), threads_of(kDqGather), kSmem, stream>>>(p, DenseTileMaps{}, DenseTileMaps{});
  return cudaGetLastError() == cudaSuccess ? 0 : -8;
}

template <bool kFp16>
int launch_type(AttnBwdParams& p, const Plan& w, bool gather, cudaStream_t stream) {
  // (fp16: at most kMaxBlocks CTAs per head, whose maxima are kept apart)
  const int bh = p.B * p.H, per = (std::max(p.stat_rows, kFp16 ? p.Sk : 0) + 63) / 64;
  p.max_blocks = kFp16 ? 2 * std::min(per, kMaxBlocks / 2) : std::min(per, std::max(1, 148 * 8 * 4 / bh));
  // (before the statistics, which ask which keys have entries)
  if (gather) {
    const int rc = launch_attn_bwd_gather_rows(p, w.segs, stream);
    if (rc != 0) return rc;
  }
  attn_bwd_stats_kernel<kFp16><<<dim3((unsigned)p.max_blocks, (unsigned)bh), 256, 0, stream>>>(p);
  if (gather) {
    const int db = padded_blocks(p.D);
    const int rc = db == 1   ? launch_gather_dq<1, 128, kFp16>(p, stream)
                   : db == 2 ? launch_gather_dq<2, 128, kFp16>(p, stream)
                   : db == 3 ? launch_gather_dq<3, 64, kFp16>(p, stream)
                             : launch_gather_dq<4, 64, kFp16>(p, stream);
    return rc != 0 ? rc : launch_attn_bwd_gather_dkv(p, kFp16, w.heads_per_pass, stream);
  }
  switch (padded_blocks(p.D)) {
    case 1: return launch_dense<1, 128, kFp16>(p, w, stream);
    case 2: return launch_dense<2, 128, kFp16>(p, w, stream);
    case 3: return launch_dense<3, 64, kFp16>(p, w, stream);
    default: return launch_dense<4, 64, kFp16>(p, w, stream);
  }
}

}  // namespace

int64_t attn_bwd_workspace_bytes(const AttnBwdParams& p, bool gather) { return (int64_t)make_plan(p, gather).total; }

int launch_attn_bwd(AttnBwdParams& p, bool gather, bool fp16, void* workspace, cudaStream_t stream) {
  const Plan w = make_plan(p, gather);
  p.stat_rows = w.stat_rows;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.neg_lse2 = reinterpret_cast<float*>(ws);
  p.neg_delta = reinterpret_cast<float*>(ws + w.stats);
  p.neg_delta_kv = reinterpret_cast<float*>(ws + 2 * w.stats);
  p.row_max = reinterpret_cast<float2*>(ws + 3 * w.stats);
  ws += 3 * w.stats + w.row_max;
  p.entry_row = reinterpret_cast<int32_t*>(ws);
  p.key_start = gather ? reinterpret_cast<int32_t*>(ws + w.entries) : nullptr;
  p.seg_count = reinterpret_cast<int32_t*>(ws + w.entries + w.starts);
  p.block_sum = reinterpret_cast<int32_t*>(ws + w.entries + w.starts + w.counts);
  p.parts = reinterpret_cast<float*>(ws + w.entries + w.starts + w.counts + w.blocks);
  return fp16 ? launch_type<true>(p, w, gather, stream) : launch_type<false>(p, w, gather, stream);
}

}  // namespace mcs
