// w4_linear.cu -- products of a few tokens with a packed 4-bit matrix: out[t, n] = sum over k of x[t, k] q[n, k] s[n, k / G],
// x and out bf16 or f16, sums in fp32, one rounding.
//
// tiles_kernel (few tokens and small matrices): one CTA per 16-row tile and block of up to 8 NT tokens; its eight warps take
// the tiles along K in turn and their partial sums are added in warp order through shared memory.  Bound by latency.
//
// rows_kernel: 128 rows of the matrix are the M of a tcgen05 product, up to 64 tokens its N.  Per K position (128 columns)
// two tensor copies bring the eight row tiles' values and scales and two bring x; four warps decode, a thread per row, to
// exact 16-bit floats q in tensor memory, the product's A operand; the tensor core sums each scale group into columns of its
// own (x and q exact, sums fp32), and eight warps, a thread per row and half of the tokens, add s times that sum to totals in
// registers.  So no weight is rounded and the matrix is read once for all tokens.  A cluster of S CTAs splits K where there
// are fewer blocks of rows than half the SMs; their totals are added in rank order through shared memory.
//
// N = 18432, K = 7168, G = 128 on a B200: 22.5 us for 9 to 16 tokens, 24.1 for 32, 27.6 for 64 (reading alone 10.5 to 10.9),
// tiles_kernel 30 to 99; G = 32: 26.1, 29.1, 41.9.  What it cost on the way, at 64 tokens: 50 us with the decoded tile in
// shared memory (32 KB written and 32 KB read per position: 1350 cycles), 44 with it in tensor memory, 32.5 with two issuing
// threads, one commit per position and two groups of decoders, 31.2 with lanes chosen by elect.sync, 28.4 with two groups of
// totals (in turns by position in place of by tokens: 32.9), 27.3 with the values swizzled by the copy in place of exchanged
// in registers.  Bound by instructions (60 to 64% of the issue slots, the decoding above all) and by the roles' waits on one
// another, 0.35 to 0.43 us a position.  Before that last step, without the decoding's arithmetic 21.6 us at 16 tokens and 25.8
// at 64, without the totals' sums 23.1 and 25.2, without either, the stores and most products 16.8 and 17.9, of which the
// reading is less than 1.  More places, four groups of decoders or two CTAs per SM are no faster.
#include <type_traits>
#include "fbmoe.h"
#include "fbmoe_launch.h"
#include "w4_common.cuh"

namespace fbmoe {
namespace w4 {
namespace {

constexpr int kWarps = 8;

// STREAM: the values take no place in the L1 cache, so that x stays there.  Volatile: not before pdl_wait, the kernel before
// may have written them.
template <bool STREAM>
__device__ __forceinline__ uint4 load_values(const uint8_t* p) {
  if (!STREAM) return __ldg(reinterpret_cast<const uint4*>(p));
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

template <typename A, int G, int NT, bool STREAM>
__global__ void __launch_bounds__(kWarps * 32) tiles_kernel(const typename A::Raw* __restrict__ x, long ldx, int T,
                                                             const uint8_t* __restrict__ packed, int N, int K,
                                                             typename A::Raw* __restrict__ out, long ldo) {
  __shared__ float part[kWarps][NT * 128];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int kt_n = K / kTileK, t0 = blockIdx.y * (8 * NT);
  pdl_wait();
  pdl_trigger();
  float acc[NT][4] = {};
  for (int kt = warp; kt < kt_n; kt += kWarps) {
    const uint8_t* tile = packed + ((size_t)blockIdx.x * kt_n + kt) * tile_bytes(G);
    const uint4 qlo = load_values<STREAM>(tile + 16 * lane);
    const uint4 qhi = load_values<STREAM>(tile + 512 + 16 * lane);
    uint32_t sw[128 / G];
#pragma unroll
    for (int gr = 0; gr < 128 / G; ++gr)
      sw[gr] = __ldg(reinterpret_cast<const uint32_t*>(tile + kTileQ + 32 * gr + 4 * g));
    uint4 xv[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int row = t0 + 8 * n + g;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        xv[n][j] = row < T ? __ldg(reinterpret_cast<const uint4*>(x + (size_t)row * ldx + kt * kTileK + 32 * j + 8 * t))
                           : make_uint4(0, 0, 0, 0);
    }
    tile_product<A, G, NT>(qlo, qhi, sw, xv, magic_register<A>(), acc);
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[warp][(8 * n + 2 * t + (i & 1)) * 16 + g + 8 * (i >> 1)] = acc[n][i];
  __syncthreads();
  for (int i = threadIdx.x; i < NT * 128; i += kWarps * 32) {
    const int row = t0 + i / 16, n = blockIdx.x * kTileN + i % 16;
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sum += part[w][i];
    if (row < T && n < N) out[(size_t)row * ldo + n] = A::of(sum);
  }
}

// ---------------------------------------------------------------- rows_kernel
constexpr int kM = 128;  // rows of the matrix per CTA
// Groups of four warps that decode, taking turns at K positions; that add up, half of the tokens each; and threads that issue
// products, taking turns at batches (below).
constexpr int kDecoders = 2, kTotals = 2, kIssuers = 2;
// Places in shared and tensor memory.  What is used in turns has a number of places that is a multiple of the users': a place
// then always has the same one, whose phases follow one another.
constexpr int kRawStages = 6, kXStages = 4;
constexpr int kScaleSlots = 16;  // more than the decoders can be ahead of the totals (kDecoded + kSums, 12 at most)
constexpr int kFirstTotals = 4, kFirstDecoder = kFirstTotals + 4 * kTotals;  // warps; 0 and 3 copy, 1 and 2 issue products
constexpr int kRowsThreads = 32 * (kFirstDecoder + 4 * kDecoders);
constexpr uint64_t kWaitBudgetNs = 4000000000ull;

template <int G, int NP>
struct RowsSmem {
  static constexpr int kTile = tile_bytes(G), kScaleBytes = kTile - kTileQ, kRawTx = 8 * kTile;
  static constexpr int kRaw = 9 * 1024;  // values, then scales
  static constexpr int kX = NP * kTileK * 2;
  static constexpr int kGroups = kTileK / G;
  // Tensor memory: the first half holds group sums, the other decoded tiles of 64 columns (six of those were no faster).
  static constexpr int kDecodedAt = 256, kDecoded = (512 - kDecodedAt) / 64;
  static constexpr int kSumCols = NP < 32 ? 32 : NP, kSums = kDecodedAt / kSumCols;
  // group sums per commit: a commit costs its thread 90 ns (measured), so as many as leave two places of that many
  static constexpr int kBatch = kGroups < kSums / 2 ? kGroups : kSums / 2, kBatches = kGroups / kBatch;  // per K position
  static constexpr int kPlaces = kSums / kBatch;
  static_assert(kPlaces % kIssuers == 0 && kXStages % kIssuers == 0 && kDecoded % kIssuers == 0 && kDecoded % kDecoders == 0 &&
                    kRawStages % kDecoders == 0 && kScaleSlots % kDecoders == 0 && kScaleSlots > kDecoded + kSums,
                "see kRawStages");
  static constexpr int x_at = 0;
  static constexpr int raw_at = x_at + kXStages * kX;
  static constexpr int scale_at = raw_at + kRawStages * kRaw;
  static constexpr int bar_at = scale_at + kScaleSlots * kGroups * kM * 4;
  static constexpr int used = bar_at + 640 + 1024;  // and the alignment of the first
  // More than half of an SM's, so that no two share one: each takes all of its tensor memory, and CTAs of two clusters that
  // waited for each other's would wait for good.
  static constexpr int total = used > 116 * 1024 ? used : 116 * 1024;
};

// One lane of a warp that has not diverged.  The compiler then keeps what is the same in all lanes in uniform registers, as
// copies and products take it; a branch on the lane's number made the whole 1 to 2 us slower.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float load_cluster(uint32_t smem_addr, uint32_t rank) {
  uint32_t at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

// tmem_ld16_pairs of eight columns.
__device__ __forceinline__ void tmem_ld8_pairs(uint32_t taddr, uint64_t (&v)[4]) {
  uint32_t r[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 4; ++i) asm("mov.b64 %0, {%1, %2};" : "=l"(v[i]) : "r"(r[2 * i]), "r"(r[2 * i + 1]));
}
// Box (0, 0, k, row tile) of a map of one matrix.
__device__ __forceinline__ void load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int k, int tile, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint "
      "[%0], [%1, {%3, %3, %4, %5}], [%2], %6;" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(0), "r"(k), "r"(tile), "l"(policy)
      : "memory");
}

template <typename A, int G, int NP>
__global__ void __launch_bounds__(kRowsThreads, 1)
    rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_s,
                const __grid_constant__ CUtensorMap map_x, int T, int N, int kt_n,
                int splits, typename A::Raw* __restrict__ out, long ldo, uint64_t wait_ns, bool expire, uint32_t* sink) {
  using S = RowsSmem<G, NP>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *xs = smem + S::x_at, *raw = smem + S::raw_at;
  float* scale = reinterpret_cast<float*>(smem + S::scale_at);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::bar_at);
  uint64_t *raw_full = bars, *raw_empty = raw_full + kRawStages, *x_full = raw_empty + kRawStages,
           *x_empty = x_full + kXStages, *dec_full = x_empty + kXStages, *dec_empty = dec_full + S::kDecoded,
           *sum_full = dec_empty + S::kDecoded, *sum_empty = sum_full + 8, *scale_full = sum_empty + 8,
           *drain = scale_full + kScaleSlots;
  uint64_t* never = drain + kIssuers;  // test hook: nothing arrives there
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(never + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_at + 1);
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = splits > 1 ? (int)cluster_rank() : 0, unit = blockIdx.x / splits;
  const int k0 = kt_n * rank / splits, steps = kt_n * (rank + 1) / splits - k0;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kRawStages; ++i) mbar_init(&raw_full[i], 1), mbar_init(&raw_empty[i], 4);
    for (int i = 0; i < kXStages; ++i) mbar_init(&x_full[i], 1), mbar_init(&x_empty[i], 4 * kTotals);
    for (int i = 0; i < S::kDecoded; ++i) mbar_init(&dec_full[i], 4), mbar_init(&dec_empty[i], 4 * kTotals);
    for (int i = 0; i < 8; ++i) mbar_init(&sum_full[i], 1), mbar_init(&sum_empty[i], 4 * kTotals);
    for (int i = 0; i < kScaleSlots; ++i) mbar_init(&scale_full[i], 4);
    for (int i = 0; i < kIssuers; ++i) mbar_init(&drain[i], 1);
    mbar_init(never, 1);
    *abort = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_at, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();  // every thread: a role's limit counts from here, however long the predecessor takes
  pdl_trigger();
  const uint32_t tmem = *tmem_at;
  // A wait that gives up raises `abort`, and every role ends; the CTA's outputs are then NaN, and the sink tells.
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (mbar_wait(bar, parity, abort, wait_ns)) return true;
    *abort = 1;
    return false;
  };
  auto wait_warp = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)); };

  constexpr int kMine = NP / kTotals;  // tokens of a totals warp
  const bool totals = warp >= kFirstTotals && warp < kFirstDecoder;
  const int t_first = totals ? (warp - kFirstTotals) / 4 * kMine : 0;
  uint64_t acc[kMine / 2];  // totals of row 32 q + lane, two tokens each
#pragma unroll
  for (int i = 0; i < kMine / 2; ++i) acc[i] = 0;

  if (warp == 0 || warp == 3) {  // copies of the matrix; of x
    fence_proxy_async_global();
    const uint64_t policy = l2_policy_evict_first();
    // One after the other through `stages` places.
    auto copies = [&](auto stages, uint64_t* full, uint64_t* empty, auto copy) {
      constexpr int n = decltype(stages)::value;
      int at = 0, issued = 0;
      uint32_t phase = 0;
      for (; issued < steps; ++issued) {
        if (!wait_warp(&empty[at], phase ^ 1)) break;
        if (elect_one()) copy(&full[at], at, k0 + issued);
        __syncwarp();
        if (++at == n) at = 0, phase ^= 1;
      }
      // no copy may be under way when the CTA ends
      for (int i = issued > n ? issued - n : 0; i < issued; ++i) mbar_wait_drain(&full[i % n], i / n & 1, kWaitBudgetNs);
    };
    if (warp == 0) {
      copies(std::integral_constant<int, kRawStages>(), raw_full, raw_empty, [&](uint64_t* bar, int at, int k) {
        mbar_arrive_expect_tx(bar, S::kRawTx);
        load_4d(raw + at * S::kRaw, &map_w, bar, k, unit * 8, policy);
        load_4d(raw + at * S::kRaw + 8 * kTileQ, &map_s, bar, k, unit * 8, policy);
      });
    } else {
      copies(std::integral_constant<int, kXStages>(), x_full, x_empty, [&](uint64_t* bar, int at, int k) {
        mbar_arrive_expect_tx(bar, S::kX);
        tma_load_2d_nohint(xs + at * S::kX, &map_x, bar, k * kTileK, 0);
        tma_load_2d_nohint(xs + at * S::kX + S::kX / 2, &map_x, bar, k * kTileK + 64, 0);
      });
    }
    __syncwarp();
  } else if (warp <= kIssuers) {
    constexpr uint32_t idesc = umma_idesc(sizeof(typename A::Raw) == 2 && A::kMagic == Bf16::kMagic ? 1u : 0u, kM, NP);
    bool any = false;
    for (int batch = warp - 1; batch < steps * S::kBatches; batch += kIssuers) {
      const int i = batch / S::kBatches, g0 = batch % S::kBatches * S::kBatch;  // K position, first group
      const int xi = i % kXStages, di = i % S::kDecoded, bi = batch % S::kPlaces;
      if (!wait_warp(&x_full[xi], i / kXStages & 1) || !wait_warp(&dec_full[di], i / S::kDecoded & 1) ||
          !wait_warp(&sum_empty[bi], (batch / S::kPlaces & 1) ^ 1))
        break;
      tc_fence_after();
      any = true;
      if (elect_one()) {
        const uint64_t b0 = umma_desc_sw128(smem_u32(xs + xi * S::kX));
        const uint32_t a0 = tmem + S::kDecodedAt + di * 64, d0 = tmem + bi * S::kBatch * S::kSumCols;
#pragma unroll
        for (int gr = 0; gr < S::kBatch; ++gr)
#pragma unroll
          for (int k = 0; k < G / 16; ++k) {
            const int at = (g0 + gr) * G + 16 * k;  // column; x has 64 of them per swizzled half
            mma_f16_tmem_a(d0 + gr * S::kSumCols, a0 + at / 2, b0 + (at / 64 * (S::kX / 2 / 16) + at % 64 / 8), idesc,
                           k ? 1u : 0u);
          }
        tc_commit(&sum_full[bi]);
      }
      __syncwarp();
    }
    if (any) {
      if (elect_one()) tc_commit(&drain[warp - 1]);
      __syncwarp();
      mbar_wait_drain(&drain[warp - 1], 0, kWaitBudgetNs);
    }
    __syncwarp();
  } else if (totals) {
    const int q = warp & 3, row = 32 * q + lane;
    const uint32_t from = tmem + ((uint32_t)(32 * q) << 16) + t_first;
    bool ok = !expire || wait_warp(never, 0);
    for (int i = 0; i < steps && ok; ++i) {
      const int ci = i % kScaleSlots;
      ok = wait(&scale_full[ci], i / kScaleSlots & 1);
#pragma unroll
      for (int g0 = 0; g0 < S::kGroups; g0 += S::kBatch) {
        const int batch = i * S::kBatches + g0 / S::kBatch, bi = batch % S::kPlaces;
        ok = ok && wait(&sum_full[bi], batch / S::kPlaces & 1);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (g0 + S::kBatch == S::kGroups && lane == 0) {  // these products, and with them all of the K position's, are done
          mbar_arrive(&dec_empty[i % S::kDecoded]);
          mbar_arrive(&x_empty[i % kXStages]);
        }
#pragma unroll
        for (int gr = g0; gr < g0 + S::kBatch; ++gr) {
          const float s = scale[(ci * S::kGroups + gr) * kM + row];
          const uint64_t s2 = f32x2_pack(s, s);
          uint64_t v[kMine / 2];
          const uint32_t at = from + (bi * S::kBatch + gr - g0) * S::kSumCols;
          if constexpr (kMine == 8) {
            tmem_ld8_pairs(at, v);
          } else {
#pragma unroll
            for (int n = 0; n < kMine; n += 16) tmem_ld16_pairs(at + n, *reinterpret_cast<uint64_t(*)[8]>(v + n / 2));
          }
          tmem_wait_ld();
#pragma unroll
          for (int n = 0; n < kMine / 2; ++n) f32x2_fma(acc[n], v[n], s2);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sum_empty[bi]);
      }
    }
  } else {
    // row 32 q + lane of the group's K positions
    const int q = warp & 3, row = 32 * q + lane, tile = row / kTileN, h = row / 8 % 2, g = row % 8;
    const uint32_t magic = magic_register<A>();
    for (int i = (warp - kFirstDecoder) / 4; i < steps; i += kDecoders) {
      const int ri = i % kRawStages, di = i % S::kDecoded, ci = i % kScaleSlots;
      const bool ok = wait(&raw_full[ri], i / kRawStages & 1) && wait(&dec_empty[di], (i / S::kDecoded & 1) ^ 1);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      const uint8_t *from = raw + ri * S::kRaw, *sc = from + 8 * kTileQ + tile * S::kScaleBytes;
      uint4 w[4];  // pieces t of the row's 64 bytes, swizzled by the row's bits 1 and 2
#pragma unroll
      for (int t = 0; t < 4; ++t) w[t] = *reinterpret_cast<const uint4*>(from + row * 64 + ((t ^ (row >> 1 & 3)) << 4));
#pragma unroll
      for (int gr = 0; gr < S::kGroups; ++gr) {
        const uint16_t b = *reinterpret_cast<const uint16_t*>(sc + 32 * gr + 4 * g + 2 * h);
        scale[(ci * S::kGroups + gr) * kM + row] = __uint_as_float((uint32_t)b << 16);
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {  // words 2 half, 2 half + 1 of each piece: columns 64 half .. + 63
        uint32_t p[32];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          uint32_t v[4];
          decode_word<A>(half ? w[t].z : w[t].x, magic, v);
#pragma unroll
          for (int k = 0; k < 4; ++k) p[4 * t + k] = v[k];
          decode_word<A>(half ? w[t].w : w[t].y, magic, v);
#pragma unroll
          for (int k = 0; k < 4; ++k) p[16 + 4 * t + k] = v[k];
        }
        tmem_st32(tmem + S::kDecodedAt + di * 64 + 32 * half + ((uint32_t)(32 * q) << 16), p);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&raw_empty[ri]);
        mbar_arrive(&scale_full[ci]);
        mbar_arrive(&dec_full[di]);
      }
    }
  }
  __syncwarp();
  const float bad = __uint_as_float(0x7FC00000u);
  const int row = 32 * (warp & 3) + lane, n = unit * kM + row;
  // x and the tiles have been used: with more splits than one their place takes the totals, [token][row]
  float* part = reinterpret_cast<float*>(smem);
  if (splits > 1) __syncthreads();
  if (totals) {
    const bool failed = *abort;
#pragma unroll
    for (int t = 0; t < kMine; ++t) {
      float v[2];
      f32x2_unpack(acc[t / 2], v[0], v[1]);
      const int token = t_first + t;
      const float total = failed ? bad : v[t % 2];
      if (token >= T) continue;
      if (splits > 1)
        part[token * kM + row] = total;
      else if (n < N)
        out[(size_t)token * ldo + n] = A::of(total);
    }
  }
  if (splits > 1) {
    __syncthreads();
    cluster_sync();
    for (int i = rank * kRowsThreads + threadIdx.x; i < T * kM; i += splits * kRowsThreads) {
      float sum = 0.0f;
      for (int k = 0; k < splits; ++k) sum += load_cluster(smem_u32(part + i), k);
      const int m = unit * kM + i % kM;
      if (m < N) out[(size_t)(i / kM) * ldo + m] = A::of(sum);
    }
    cluster_sync();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (threadIdx.x == 0 && sink && *abort) {
    *reinterpret_cast<volatile uint32_t*>(sink) = kStatusTimeoutEpilogue;
    __threadfence_system();
  }
}

template <typename A, int G, int NP>
cudaError_t run_rows(const void* x, long ldx, int T, const void* packed, int N, int K, void* out, long ldo,
                     uint32_t* sink, cudaStream_t stream) {
  using S = RowsSmem<G, NP>;
  static DeviceFlags smem_set;
  cudaError_t e = set_max_dynamic_smem(rows_kernel<A, G, NP>, S::total, smem_set);
  if (e != cudaSuccess) return e;
  const int kt = K / kTileK, units = (N - 1) / kM + 1, sms = num_sms_of_current_device();
  int splits = 1;
  while (splits < 8 && units * splits * 2 <= sms && kt >= 8 * splits) splits *= 2;
  CUtensorMap map_w, map_s, map_x;
  const uint64_t tb = S::kTile, row_tiles = (N - 1) / kTileN + 1;
  const uint64_t dims_q[4] = {8, kTileN, (uint64_t)kt, row_tiles}, strides[3] = {64, tb, kt * tb};
  const uint64_t dims_s[4] = {(uint64_t)S::kScaleBytes / 8, 1, (uint64_t)kt, row_tiles};
  const uint32_t box_q[4] = {8, kTileN, 1, 8}, box_s[4] = {S::kScaleBytes / 8, 1, 1, 8};
  if (encode_4d_words(&map_w, packed, dims_q, strides, box_q, CU_TENSOR_MAP_SWIZZLE_64B) != FBMOE_OK ||
      encode_4d_words(&map_s, reinterpret_cast<const uint8_t*>(packed) + kTileQ, dims_s, strides, box_s,
                      CU_TENSOR_MAP_SWIZZLE_NONE) != FBMOE_OK ||
      encode_strided_2d(&map_x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, x, K, T, (uint64_t)ldx * 2, 64, NP,
                        CU_TENSOR_MAP_SWIZZLE_128B) != FBMOE_OK)
    return cudaErrorUnknown;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(units * splits);
  cfg.blockDim = dim3(kRowsThreads);
  cfg.dynamicSmemBytes = S::total;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = splits;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = splits > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, rows_kernel<A, G, NP>, map_w, map_s, map_x, T, N, kt, splits,
                            reinterpret_cast<typename A::Raw*>(out), ldo, test_short_waits() ? kTestGridWaitNs : kWaitBudgetNs,
                            test_expire_grid_wait(), sink);
}

// Which kernel, by how much there is to spread over the SMs.  tiles_kernel reads the matrix once per 16 tokens and starts and
// ends at once; rows_kernel reads it once, and costs 4 us before its first and after its last product.  Measured, tiles /
// rows, in us (G = 128; 32 moves the same way):
//   N x K          tiles to read    T = 8          T = 16         T = 64
//   1024 x 4096    2048             3.2 / 5.5      4.0 / 5.6      6.1 / 7.0
//   7168 x 2048    7168             4.6 / 7.2      7.0 / 7.5      18.0 / 9.9
//   4096 x 7168    14336            7.8 / 9.9      11.4 / 10.0    32.3 / 12.4
//   18432 x 7168   64512            19.3 / 22.4    31.8 / 22.5    98.6 / 27.6
//   32001 x 7168   112056           28.5 / 43.8    49.6 / 43.9    170.7 / 52.6
//   256 x 14336    1792             8.0 / 8.4      9.9 / 8.5      16.1 / 10.7
// So rows_kernel takes more than 8 tokens if tiles_kernel would read more than 8192 tiles, or if K is so long that each of
// its warps has twelve or more in a row.
constexpr long kMany = 8192;
long tiles_to_read(int T, int N, int K) { return ((long)(N - 1) / kTileN + 1) * (K / kTileK) * ((T + 15) / 16); }
bool rows_pay(int T, int N, int K) {
  const long kt = K / kTileK, tiles = tiles_to_read(T, N, K);
  return T > 8 && (tiles > kMany || kt >= 12 * kWarps);
}

template <typename A, int G>
cudaError_t run_linear(const void* x, long ldx, int T, const void* packed, int N, int K, void* out, long ldo,
                       uint32_t* sink, cudaStream_t stream) {
  using Raw = typename A::Raw;
  const unsigned nt = (unsigned)((N - 1) / kTileN + 1);
  const Raw* xp = reinterpret_cast<const Raw*>(x);
  const uint8_t* wp = reinterpret_cast<const uint8_t*>(packed);
  Raw* op = reinterpret_cast<Raw*>(out);
  if (rows_pay(T, N, K)) {
    if (T <= 16) return run_rows<A, G, 16>(x, ldx, T, packed, N, K, out, ldo, sink, stream);
    if (T <= 32) return run_rows<A, G, 32>(x, ldx, T, packed, N, K, out, ldo, sink, stream);
    return run_rows<A, G, 64>(x, ldx, T, packed, N, K, out, ldo, sink, stream);
  }
  const dim3 grid(nt, (unsigned)((T + 15) / 16)), block(kWarps * 32);
  if (T > 8) return launch_pdl(tiles_kernel<A, G, 2, false>, grid, block, 0, stream, xp, ldx, T, wp, N, K, op, ldo);
  // Streamed, large matrices gain (4096 x 7168, 8 tokens: 10.6 us, 7.8; 18432 x 7168: 24.6, 19.6) and small ones lose (1024 x
  // 4096, G = 32: 4.5, 5.2).  One token's x takes little of the cache, and its matrix may still lie in L2, from where
  // streaming is slower (4096 x 7168, G = 32: up to 8.7 us, 9.7; from HBM 12.3, 9.9), so only a matrix of four times that
  // size, 32 MB or more, is streamed for it (18432 x 7168, G = 32: 23.9, 20.6).
  if (tiles_to_read(T, N, K) > (T == 1 ? 4 * kMany : kMany))
    return launch_pdl(tiles_kernel<A, G, 1, true>, grid, block, 0, stream, xp, ldx, T, wp, N, K, op, ldo);
  return launch_pdl(tiles_kernel<A, G, 1, false>, grid, block, 0, stream, xp, ldx, T, wp, N, K, op, ldo);
}
template <typename A>
cudaError_t pick_linear(int group, const void* x, long ldx, int T, const void* packed, int N, int K, void* out,
                        long ldo, uint32_t* sink, cudaStream_t stream) {
  if (group == 32) return run_linear<A, 32>(x, ldx, T, packed, N, K, out, ldo, sink, stream);
  if (group == 64) return run_linear<A, 64>(x, ldx, T, packed, N, K, out, ldo, sink, stream);
  return run_linear<A, 128>(x, ldx, T, packed, N, K, out, ldo, sink, stream);
}

}  // namespace
}  // namespace w4
}  // namespace fbmoe

using namespace fbmoe;

extern "C" FBMOE_API int fbmoe_linear_w4(const void* x, int64_t x_stride, int type, int T, const void* packed, int N,
                                         int K, int group, void* out, int64_t out_stride, void* stream) {
  return fbmoe_linear_w4_status(x, x_stride, type, T, packed, N, K, group, out, out_stride, nullptr, stream);
}

extern "C" FBMOE_API int fbmoe_linear_w4_status(const void* x, int64_t x_stride, int type, int T, const void* packed,
                                                int N, int K, int group, void* out, int64_t out_stride,
                                                uint32_t* status_sink, void* stream_) {
  if (T < 0 || T > w4::kMaxTokens || N < 1 || K < 128 || K % 128 != 0 || !w4::valid_group(group) ||
      (type != FBMOE_BF16 && type != FBMOE_F16) || x_stride < K || out_stride < N)
    return FBMOE_ERR_INVALID_ARG;
  if (T == 0) return FBMOE_OK;
  if (!x || !packed || !out) return FBMOE_ERR_NULL_POINTER;
  if (((uintptr_t)x & 15) || (x_stride & 7) || ((uintptr_t)packed & 15) || ((uintptr_t)out & 1) ||
      ((uintptr_t)status_sink & 3))
    return FBMOE_ERR_MISALIGNED;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  const cudaError_t e =
      type == FBMOE_BF16
          ? w4::pick_linear<w4::Bf16>(group, x, x_stride, T, packed, N, K, out, out_stride, status_sink, stream)
          : w4::pick_linear<w4::F16>(group, x, x_stride, T, packed, N, K, out, out_stride, status_sink, stream);
  return e == cudaSuccess ? FBMOE_OK : (int)e;
}
