// w4_stream.cuh -- the 4-bit products at the speed of the weights: a warp's ring of tiles, and the tile's product.
//
// These products read every weight once and do little else.  Two things count.
//
// Bytes in flight.  At 6.5 TB/s one SM takes 44 GB/s, and 1 to 2 us of latency under load ask for about 100 KB under way
// per SM.  A ring belongs to one warp, which fills it itself: no producer warp, no empty barrier (a warp-wide sync orders
// a slot's last read before its next copy).  A step is four tiles in one tensor copy, a ring two steps: 135 KB per SM, 147
// for G = 32.  Plain streaming of such copies took 6.8 TB/s with 100 KB per SM under way, 6.5 with 134, 5.6 with 200.
//
// Instructions.  86 cycles per two tiles and SM at that rate are 344 issue slots; the logic pipe takes two instructions a
// cycle.  Decoding to pairs of 16-bit floats takes 7 logic instructions and 4 subtractions per word of eight weights, 242
// instructions per two tiles in all: 84 to 90 cycles (measured, 16 warps, weights in shared memory).  So the decoding is the
// limit: T = 64 on a quarter of the experts takes 195 us, 177 without the subtractions and 151 with no decoding (both wrong,
// to time the rest).  Twice as many sums under way, x loaded a step ahead, fewer registers, and shifts as products on the
// other pipe are no faster (196, 204, 195, 248).
//
// Activations: x as it is, bf16 or f16.  The layer's intermediate h is held as two bf16 numbers, the nearest and the
// nearest to what that one lost, in two columns of one product: within 2^-16 of h whatever stands beside it, a 32nd of
// what rounding the outputs to f16 loses.  (x and h as 16-bit integers with a power of two per block of columns decode in
// half the instructions, 147 us for those 195, but lose 2^-16 of the block's largest value, which is no small part of the
// other terms' sum where one channel is large: with 2048 beside values of 0.05 at which weights look, and none at the 2048,
// outputs were off by 860 times what fp32 sums leave.)
#pragma once

#include "w4_common.cuh"

namespace fbmoe {
namespace w4 {

constexpr int kStreamWarps = 16;                    // warps of a CTA, each with its own ring
constexpr int kDepth = 2;                           // steps of a ring: what an SM's memory holds
constexpr int kStepTiles = 4;                       // tiles of a step
constexpr uint64_t kWaitBudgetNs = 4000000000ull;   // any wait's limit

__host__ __device__ constexpr int step_bytes(int group) { return kStepTiles * tile_bytes(group); }

// ---------------------------------------------------------------- ring ------
// One warp's ring.  Steps are issued and consumed in order.  Slots and barriers are shared-memory addresses.  Its waits
// are for its own copies, which land by themselves; if one gives up all the same, the warp ends its role with the unit
// unfinished, and the caller reports the call as failed.
template <int SLOT>
struct Ring {
  uint32_t slots, bars;
  int put, got;  // steps issued, steps consumed

  __device__ __forceinline__ void init(uint32_t slots_, uint32_t barriers) {
    slots = slots_;
    bars = barriers;
    put = got = 0;
  }
  __device__ __forceinline__ bool full() const { return put - got >= kDepth; }
  // The slot of the next step to be consumed.
  __device__ __forceinline__ uint32_t slot() const { return slots + got % kDepth * SLOT; }
  // Issue one step: the box of `map` at (x, row, 0, matrix), `bytes` in all.
  __device__ __forceinline__ void issue(const CUtensorMap* map, int x, int row, int matrix, uint32_t bytes) {
    if ((threadIdx.x & 31) == 0) {
      const uint32_t at = put % kDepth, bar = bars + at * 8;
      asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n\t}" ::"r"(bar), "r"(bytes)
                   : "memory");
      asm volatile(
          "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint "
          "[%0], [%1, {%3, %4, %5, %6}], [%2], %7;" ::"r"(slots + at * SLOT),
          "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(row), "r"(0), "r"(matrix), "l"(l2_policy_evict_first())
          : "memory");
    }
    ++put;
  }
  static __device__ __forceinline__ bool test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
  }
  // Wait for the next step's tiles; false, for all lanes, when the limit runs out.
  __device__ __forceinline__ bool wait() const {
    const uint32_t bar = bars + got % kDepth * 8, parity = got / kDepth & 1;
    return __all_sync(0xffffffffu, test(bar, parity)) || __all_sync(0xffffffffu, wait_slow(bar, parity));
  }
  static __device__ __noinline__ bool wait_slow(uint32_t bar, uint32_t parity) {
    const uint64_t t0 = globaltimer_ns();
    for (uint32_t it = 1;; ++it) {
      if (test(bar, parity)) return true;
      if ((it & 15u) == 0 && globaltimer_ns() - t0 > kWaitBudgetNs) return false;
    }
  }
  // The slot has been read by every lane: it may be filled again.
  __device__ __forceinline__ void release() {
    __syncwarp();
    ++got;
  }
  // Before the CTA ends no copy may be under way: those issued and not consumed are waited for (none after a complete
  // call).  False when the limit runs out.
  __device__ __forceinline__ bool drain() {
    bool ok = true;
    for (; got < put; ++got) ok &= wait_slow(bars + got % kDepth * 8, got / kDepth & 1);
    return ok;
  }
};

// ---------------------------------------------------------------- product ---
// Shared loads at a register and a constant.
template <int AT>
__device__ __forceinline__ uint4 lds128(uint32_t base) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4+%5];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(base), "n"(AT));
  return v;
}
template <int AT>
__device__ __forceinline__ uint32_t lds32(uint32_t base) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1+%2];" : "=r"(v) : "r"(base), "n"(AT));
  return v;
}

// One K position's activations in a lane (lane l = 4g + t): 32j + 8t .. + 7 of column 8n + g of the product.
template <int NT>
struct Columns {
  uint4 v[NT][4];
};

// The tile at shared address words + AT (words = slot + 16 * lane, scales = slot + 4 * g) times the columns, into
// acc[n][i], row g + 8 i of the tile.  !PAIR: x holds 8 rows, row 4n + t in column 2t + n, NT of the two n used.  PAIR: NT
// times four rows as two columns each, row 4n + t in columns 2t and 2t + 1 of the n-th product.  q is exact in 16 bits, the
// tensor core sums a scale group in fp32, and the sum is multiplied by the group's scale.  reload(j) is called once the
// columns' words j have been used.
template <typename A, int G, int NT, bool PAIR, int AT, typename Reload>
__device__ __forceinline__ void tile_product(uint32_t words, uint32_t scales, const Columns<PAIR ? NT : 1>& x,
                                             uint32_t magic, float (&acc)[NT][2], const Reload& reload) {
  constexpr int NC = PAIR ? NT : 1;
  const uint4 lo = lds128<AT>(words), hi = lds128<AT + 512>(words);
  const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
  uint32_t sw[4];
  sw[0] = lds32<AT + kTileQ>(scales);
  if constexpr (G <= 64) sw[1] = lds32<AT + kTileQ + 32>(scales);
  if constexpr (G <= 32) {
    sw[2] = lds32<AT + kTileQ + 64>(scales);
    sw[3] = lds32<AT + kTileQ + 96>(scales);
  }
  float c[NC][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (j * 32 % G == 0) {
#pragma unroll
      for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) c[n][i] = 0.0f;
    }
    uint32_t pl[4], ph[4];
    decode_word<A>(wl[j], magic, pl);
    decode_word<A>(wh[j], magic, ph);
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      mma_16816<A>(c[n], pl[0], ph[0], pl[1], ph[1], x.v[n][j].x, x.v[n][j].y);
      mma_16816<A>(c[n], pl[2], ph[2], pl[3], ph[3], x.v[n][j].z, x.v[n][j].w);
    }
    reload(j);
    if ((j + 1) * 32 % G == 0) {
      const uint32_t s = sw[j * 32 / G];
      const float s0 = __uint_as_float(s << 16), s1 = __uint_as_float(s & 0xFFFF0000u);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        acc[n][0] = fmaf(s0, PAIR ? c[n % NC][0] + c[n % NC][1] : c[0][n], acc[n][0]);
        acc[n][1] = fmaf(s1, PAIR ? c[n % NC][2] + c[n % NC][3] : c[0][2 + n], acc[n][1]);
      }
    }
  }
}

}  // namespace w4
}  // namespace fbmoe
