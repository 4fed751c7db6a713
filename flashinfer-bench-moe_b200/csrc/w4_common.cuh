// w4_common.cuh -- the packed 4-bit weight format and its tile product.
//
// A matrix [N, K] (K a multiple of 128) is cut into tiles of 16 rows by 128 columns, stored
// [ceil(N / 16)][K / 128][tile]; rows past N hold zeros.  A tile is contiguous: 1024 bytes of 4-bit values, then its
// bf16 scales, 16 rows x 128 / G groups (4096 / G bytes).
//
// Values: u = q + 8 with q in [-8, 7].  The 256 words of 32 bits are ordered [h 2][g 8][t 4][j 4]: word (h, g, t, j)
// holds row 8h + g, columns 32j + 8t .. + 7.  So lane l = 4g + t of a warp reads its four words of a half h as 16
// contiguous bytes (a half is 512 bytes, one conflict-free 128-bit load), and all columns that the warp multiplies
// from words j lie in [32j, 32j + 32), inside one scale group for every G.
//
// Bits: word = rotl32(sum over i < 4 of u[2i] << 4i | u[2i + 1] << (16 + 4i), 3).  Rotated right by 4i it holds the
// pair (2i, 2i + 1) at bits 3..6 of its halves, where one AND-OR makes two 16-bit floats of it: 16 + u in bf16
// (0x4180 | u << 3) and 128 + u in f16 (0x5800 | u << 3), both exact.
//
// Scales: [group][g 8][h 2], so that a lane reads those of its rows g and g + 8 as one word.
#pragma once

#include "fbmoe_common.cuh"

namespace fbmoe {
namespace w4 {

constexpr int kTileN = 16;   // rows of a tile
constexpr int kTileK = 128;  // columns of a tile
constexpr int kTileQ = 1024;  // bytes of a tile's 4-bit values
constexpr int kMaxTokens = 64;  // the most tokens the products take

__host__ __device__ constexpr int tile_bytes(int group) { return kTileQ + 4096 / group; }

inline bool valid_group(int group) { return group == 32 || group == 64 || group == 128; }

// Pairs of 16-bit values of the two activation types.
struct Bf16 {
  using Raw = __nv_bfloat16;
  static constexpr uint32_t kMagic = 0x41804180u;  // 16 + u
  static __device__ __forceinline__ uint32_t minus_bias(uint32_t v) {  // - 24: q
    const __nv_bfloat162 b = __halves2bfloat162(__float2bfloat16_rn(24.0f), __float2bfloat16_rn(24.0f));
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), b);
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ Raw of(float v) { return __float2bfloat16_rn(v); }
};
struct F16 {
  using Raw = __half;
  static constexpr uint32_t kMagic = 0x58005800u;  // 128 + u
  static __device__ __forceinline__ uint32_t minus_bias(uint32_t v) {  // - 136: q
    const __half2 b = __float2half2_rn(136.0f);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&v), b);
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ Raw of(float v) { return __float2half_rn(v); }
};

// (v & mask) | magic in one instruction: an instruction holds one 32-bit constant, so the other one has to be in a
// register, where the compiler does not put it by itself (it makes two instructions of the expression).
__device__ __forceinline__ uint32_t and_or(uint32_t v, uint32_t magic) {
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x00780078, %2, 0xEA;" : "=r"(r) : "r"(v), "r"(magic));
  return r;
}
template <typename A>
__device__ __forceinline__ uint32_t magic_register() {
  uint32_t r;
  asm volatile("mov.b32 %0, %1;" : "=r"(r) : "n"(A::kMagic));
  return r;
}

// The word's four pairs (q[2i], q[2i + 1]) as exact 16-bit floats.
template <typename A>
__device__ __forceinline__ void decode_word(uint32_t w, uint32_t magic, uint32_t (&p)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = A::minus_bias(and_or(i ? __funnelshift_r(w, w, 4 * i) : w, magic));
}

// c (16 x 8, fp32) += a (16 x 16) * b (16 x 8).
template <typename A>
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<Bf16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<F16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// acc (16 tile rows x 8 NT columns) += tile * x.  qlo, qhi: the lane's words of rows g and g + 8 (lane l = 4g + t);
// scales: the tile's scale words [group][g]; x[n][j]: the lane's 8 activations 32j + 8t .. + 7 of column 8n + g.  Each
// group's products are summed exactly scaled: q is exact in 16 bits, the tensor core adds in fp32, and the group's
// sum is multiplied by its fp32 scale.  acc[n][0..1] are row g, columns 8n + 2t, + 1; acc[n][2..3] row g + 8.
template <typename A, int G, int NT>
__device__ __forceinline__ void tile_product(const uint4& qlo, const uint4& qhi, const uint32_t (&scales)[128 / G],
                                             const uint4 (&x)[NT][4], uint32_t magic, float (&acc)[NT][4]) {
  const uint32_t wl[4] = {qlo.x, qlo.y, qlo.z, qlo.w}, wh[4] = {qhi.x, qhi.y, qhi.z, qhi.w};
#pragma unroll
  for (int gr = 0; gr < 128 / G; ++gr) {
    float c[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) c[n][i] = 0.0f;
#pragma unroll
    for (int j = gr * (G / 32); j < (gr + 1) * (G / 32); ++j) {
      uint32_t pl[4], ph[4];
      decode_word<A>(wl[j], magic, pl);
      decode_word<A>(wh[j], magic, ph);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mma_16816<A>(c[n], pl[0], ph[0], pl[1], ph[1], x[n][j].x, x[n][j].y);
        mma_16816<A>(c[n], pl[2], ph[2], pl[3], ph[3], x[n][j].z, x[n][j].w);
      }
    }
    const float slo = __uint_as_float(scales[gr] << 16), shi = __uint_as_float(scales[gr] & 0xFFFF0000u);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      acc[n][0] = fmaf(slo, c[n][0], acc[n][0]);
      acc[n][1] = fmaf(slo, c[n][1], acc[n][1]);
      acc[n][2] = fmaf(shi, c[n][2], acc[n][2]);
      acc[n][3] = fmaf(shi, c[n][3], acc[n][3]);
    }
  }
}

}  // namespace w4
}  // namespace fbmoe
