// w4_stream.cuh -- the 4-bit products at the speed of the weights: a warp's ring of tiles, and the integer product.
//
// These products read every weight once and do little else.  Two things count.
//
// Bytes in flight.  At 6.5 TB/s one SM takes 44 GB/s, and 1 to 2 us of latency under load ask for about 100 KB under way
// per SM.  A ring belongs to one warp, which fills it itself: no producer warp, no empty barrier (a warp-wide sync orders
// a slot's last read before its next copy).  A step is four tiles in one tensor copy.  More under way is slower (plain
// streaming of 1056-byte copies on a B200: 6.8 TB/s with 100 KB per SM, 6.5 with 134, 5.6 with 200).
//
// Instructions.  86 cycles per two tiles and SM at that rate are 344 issue slots; the logic pipe takes two instructions a
// cycle.  Decoding to pairs of 16-bit floats takes 7 logic instructions and 4 subtractions per word of eight weights, 242
// instructions per two tiles in all: 84 to 90 cycles (measured, 16 warps, weights in shared memory), so the decoding
// would be the limit.  As 8-bit integers a word takes 4: (w & 0xF0F0F0F0) ^ 0x80808080 of the word rotated to either side
// gives four bytes 16 q in two's complement.  The activations are two 8-bit planes of a 16-bit integer, x = s (256 hi + lo),
// in two columns of one product; their sums are exact in 32 bits, which leaves half the slots free.
//
// Activations: s is a power of two per token and 128 columns (32 for the layer's intermediate), so that the largest
// |x / s| lies in [2^14, 2^15): a bf16 value within 2^-7 of the largest, an f16 value within 2^-4, is exact, a smaller
// one is rounded to 2^-15 to 2^-16 of the largest.  That is below 1e-4 of the outputs, which are rounded to 2^-9 or 2^-11.
// A NaN or an infinity makes s NaN, and with it the token's outputs.
#pragma once

#include "w4_common.cuh"

namespace fbmoe {
namespace w4 {

constexpr int kStreamWarps = 16;                    // warps of a CTA, each with its own ring
constexpr int kMaxDepth = 4;                        // steps of a ring at most
constexpr int kStepTiles = 4;                       // tiles of a step
constexpr uint64_t kWaitBudgetNs = 4000000000ull;   // any wait's limit

__host__ __device__ constexpr int step_bytes(int group) { return kStepTiles * tile_bytes(group); }

// ---------------------------------------------------------------- ring ------
// One warp's ring.  Steps are issued and consumed in order.  Slots and barriers are shared-memory addresses.  Its waits
// are for its own copies, which land by themselves; one that gives up all the same raises `abort` and closes the ring:
// nothing more is issued, and the warp goes on over whatever the slots hold until it meets one of the waits that look at
// `abort`.  The caller reports the call as failed.
struct Ring {
  uint32_t begin, end, bars, put, put_bar, got, got_bar, parity;
  int slot_bytes, free;  // free: steps that may be issued (far below 0: closed)

  __device__ __forceinline__ void init(uint32_t slots, uint32_t barriers, int bytes, int depth) {
    begin = put = got = slots;
    bars = put_bar = got_bar = barriers;
    slot_bytes = bytes;
    free = depth;
    end = slots + depth * bytes;
    parity = 0;
  }
  // Issue one step: the box of `map` at (x, row, half, matrix), `bytes` in all.
  __device__ __forceinline__ void issue(const CUtensorMap* map, int x, int row, int half, int matrix, uint32_t bytes, uint64_t policy) {
    if ((threadIdx.x & 31) == 0) {
      asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n\t}" ::"r"(put_bar),
                   "r"(bytes)
                   : "memory");
      asm volatile(
          "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint "
          "[%0], [%1, {%3, %4, %5, %6}], [%2], %7;" ::"r"(put),
          "l"(reinterpret_cast<uint64_t>(map)), "r"(put_bar), "r"(x), "r"(row), "r"(half), "r"(matrix), "l"(policy)
          : "memory");
    }
    --free;
    put += slot_bytes;
    put_bar += 8;
    if (put == end) {
      put = begin;
      put_bar = bars;
    }
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
  // Wait for the next step's tiles.
  __device__ __forceinline__ void wait(volatile int* abort) {
    if (test(got_bar, parity)) return;
    if (free >= 0 && !wait_slow(got_bar, parity)) {
      *abort = 1;
      free = -(1 << 30);
    }
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
    ++free;
    got += slot_bytes;
    got_bar += 8;
    if (got == end) {
      got = begin;
      got_bar = bars;
      parity ^= 1;
    }
  }
  // Before the CTA ends no copy may be under way: those issued and not consumed are waited for (none after a complete
  // call).  False when the limit runs out.
  __device__ __forceinline__ bool drain(int depth) {
    if (free < 0) return wait_slow(got_bar, parity);
    bool ok = true;
    while (free < depth) {
      ok &= wait_slow(got_bar, parity);
      release();
    }
    return ok;
  }
};

// ---------------------------------------------------------------- planes ----
// Activations of a row as planes: 256 bytes per K position (128 columns): [plane hi, lo][t 4][j 4][8], the eight columns
// 32j + 8t .. + 7 in the order 0 4 1 5 2 6 3 7 that the weights' bytes have.
constexpr int kPlaneTile = 256;

// The power of two s for a largest magnitude m: m / s in [2^14, 2^15 * 127.5 / 128).  Its exponent e; NaN inputs aside.
__device__ __forceinline__ int plane_exponent(float m) {
  // m (1 + 2^-7): a value that would round past 127 * 256 + 127 gets the next power
  const float v = fmaf(m, 0.0078125f, m);
  return (int)(__float_as_uint(v) >> 23) - 127 - 14;
}
__device__ __forceinline__ float exp2_int(int e) {  // 2^e for e in [-149, 127]
  return e >= -126 ? __uint_as_float((uint32_t)(e + 127) << 23) : __uint_as_float(1u << (e + 149));
}
// rint(v / 2^e) for |v / 2^e| < 2^15 and e in [-149, 113].
__device__ __forceinline__ int plane_int(float v, int e) {
  const int a = -e / 2;
  return __float2int_rn(v * exp2_int(a) * exp2_int(-e - a));
}

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

// (v & 0xF0F0F0F0) ^ flip in one instruction; flip = 0x80808080 in a register (see and_or).
__device__ __forceinline__ uint32_t and_xor(uint32_t v, uint32_t flip) {
  uint32_t r;
  asm("lop3.b32 %0, %1, 0xF0F0F0F0, %2, 0x6A;" : "=r"(r) : "r"(v), "r"(flip));
  return r;
}
__device__ __forceinline__ uint32_t flip_register() {
  uint32_t r;
  asm volatile("mov.b32 %0, 0x80808080;" : "=r"(r));
  return r;
}

// d (16 x 8, s32) = a (16 x 32, s8) * b (32 x 8, s8) + c.
__device__ __forceinline__ void mma_16832(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1, int c0, int c1, int c2, int c3) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %11, %12, %13};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c0), "r"(c1), "r"(c2), "r"(c3));
}

// One K position's activations of 4 NT tokens: b[n][j] the lane's two words of column 8n + g (plane g & 1 of token
// 4n + g / 2), s[n] the scales of token 4n + t (one, or one per 32 columns), times 2^-4.
template <int NT, bool FINE>
struct Columns {
  uint2 b[NT][4];
  float s[NT][FINE ? 4 : 1];
};

// acc[n][i] (row g + 8 i of a tile, token 4n + t) += the tile at shared address words + AT (words = slot + 16 * lane,
// scales = slot + 4 * g) times the columns.  reload(j) is called once the columns' words 2j, 2j + 1 have been used.
template <int G, int NT, bool FINE, int AT, typename Reload>
__device__ __forceinline__ void tile_product(uint32_t words, uint32_t scales, const Columns<NT, FINE>& x, uint32_t flip,
                                             float (&acc)[NT][2], const Reload& reload) {
  const uint4 lo = lds128<AT>(words), hi = lds128<AT + 512>(words);
  const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
  uint32_t sw[4];
  sw[0] = lds32<AT + kTileQ>(scales);
  if constexpr (G <= 64) sw[1] = lds32<AT + kTileQ + 32>(scales);
  if constexpr (G <= 32) {
    sw[2] = lds32<AT + kTileQ + 64>(scales);
    sw[3] = lds32<AT + kTileQ + 96>(scales);
  }
  int c[NT][4];
  float part[NT][2];  // FINE: a weight group's sum
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool first = j * 32 % G == 0, last = (j + 1) * 32 % G == 0;  // of the weight group
    const uint32_t el = and_xor(__funnelshift_l(wl[j], wl[j], 1), flip), eh = and_xor(__funnelshift_l(wh[j], wh[j], 1), flip);
    const uint32_t ol = and_xor(__funnelshift_r(wl[j], wl[j], 3), flip), oh = and_xor(__funnelshift_r(wh[j], wh[j], 3), flip);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (FINE || first)
        mma_16832(c[n], el, eh, ol, oh, x.b[n][j].x, x.b[n][j].y, 0, 0, 0, 0);
      else
        mma_16832(c[n], el, eh, ol, oh, x.b[n][j].x, x.b[n][j].y, c[n][0], c[n][1], c[n][2], c[n][3]);
    }
    if (j % 2 == 1) reload(j / 2);
    if (FINE) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float v = (float)(c[n][2 * i] * 256 + c[n][2 * i + 1]);
          part[n][i] = first ? x.s[n][j] * v : fmaf(x.s[n][j], v, part[n][i]);
        }
    }
    if (last) {
      const uint32_t s = sw[j * 32 / G];
      const float s0 = __uint_as_float(s << 16), s1 = __uint_as_float(s & 0xFFFF0000u);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if (FINE) {
          acc[n][0] = fmaf(s0, part[n][0], acc[n][0]);
          acc[n][1] = fmaf(s1, part[n][1], acc[n][1]);
        } else {
          acc[n][0] = fmaf(s0 * x.s[n][0], (float)(c[n][0] * 256 + c[n][1]), acc[n][0]);
          acc[n][1] = fmaf(s1 * x.s[n][0], (float)(c[n][2] * 256 + c[n][3]), acc[n][1]);
        }
      }
    }
  }
}

}  // namespace w4
}  // namespace fbmoe
