// w4_quant.cu -- weights to and from the packed 4-bit format of w4_common.cuh.
//
// Quantiser: per row and group of G columns s = bf16(max |w| / 7) (IEEE fp32 division, then round to nearest; 0 when
// that is below the smallest normal number), or the caller's s; q = clamp(rint(w / s), -8, 7) with w / s the IEEE
// fp32 quotient, 0 where s is not positive.  A group that holds a NaN or an infinity gets the scale NaN.
// Reader: v = q * s, exact in fp32 (4 bits times 8), rounded once to the output type.
//
// The reader is bound by HBM (4096 x 7168 to bf16: 12.2 us, 6.0 TB/s; 8 x 7168 x 2048, G = 32, to fp32: 5.6 TB/s), the
// quantiser by its arithmetic: about 16 instructions per weight and lane, 60 to 72% of the issue slots (4096 x 7168 bf16: 20
// us, of which reading and writing alone would take 11).  One warp per tile: lane l = 4g + t owns rows g and g + 8, columns
// 32j + 8t .. + 7, which are its packed words, so values go from the loads to the packed stores without shared memory: a
// quad reads 32 contiguous columns of a row, a half tile is stored as one coalesced 512-byte row of 16-byte words, and a
// group's maximum is at most two shuffles over the quad.
#include <limits.h>
#include "fbmoe.h"
#include "fbmoe_launch.h"
#include "w4_common.cuh"

namespace fbmoe {
namespace w4 {
namespace {

constexpr int kWarps = 8;
constexpr float kMinNormal = 1.17549435e-38f;

enum Type { kBf16 = FBMOE_BF16, kF16 = FBMOE_F16, kF32 = FBMOE_F32, kE4m3 = FBMOE_E4M3 };

// Eight consecutive weights as they are held, and as fp32.
template <int TYPE>
struct Raw8 {
  uint4 a, b;  // b: fp32 only
  __device__ __forceinline__ void load(const void* base, size_t at) {
    if constexpr (TYPE == kE4m3) {
      const uint2 r = __ldg(reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(base) + at));
      a.x = r.x;
      a.y = r.y;
    } else if constexpr (TYPE == kF32) {
      const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(base) + at);
      a = __ldg(p);
      b = __ldg(p + 1);
    } else {
      a = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(base) + at));
    }
  }
  __device__ __forceinline__ void zero() { a = b = make_uint4(0, 0, 0, 0); }
  // bs: the scale of an e4m3 block
  __device__ __forceinline__ void widen(float (&v)[8], float bs) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
    if constexpr (TYPE == kBf16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      }
    } else if constexpr (TYPE == kF16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    } else if constexpr (TYPE == kF32) {
      const uint32_t u[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = __uint_as_float(w[i]);
        v[4 + i] = __uint_as_float(u[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i >> 1] >> (16 * (i & 1))), __NV_E4M3);
        const float2 f = __half22float2(__half2(h));
        v[2 * i] = __fmul_rn(f.x, bs);
        v[2 * i + 1] = __fmul_rn(f.y, bs);
      }
    }
  }
};

// max(m, |v|), NaN if either is.
__device__ __forceinline__ float max_abs_nan(float m, float v) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(v)));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// The word of eight weights v, s their scale, r = 1 / s: u = clamp(rint(v / s), -8, 7) + 8 with the IEEE quotient.
// y = v * r is within 3 ulps of it, so only a y next to a half integer needs the division; y + 1.5 * 2^23 + 8 holds u in its
// low bits.  CLAMP: the scale was given (one made from the largest |v| leaves |y| < 7.04).
template <bool CLAMP>
__device__ __forceinline__ uint32_t quantize8(const float (&v)[8], float s, float r) {
  constexpr float kMagic = 12582912.0f;
  const uint64_t rr = f32x2_pack(r, r), up = f32x2_pack(kMagic, kMagic), down = f32x2_pack(-kMagic, -kMagic),
                 eight = f32x2_pack(8.0f, 8.0f), minus = f32x2_pack(-1.0f, -1.0f);
  float off = 0.0f;  // largest distance of a y from its integer
  uint32_t b[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint64_t y = f32x2_mul(f32x2_pack(v[2 * i], v[2 * i + 1]), rr);
    if (CLAMP) {
      float p, q;
      f32x2_unpack(y, p, q);
      y = f32x2_pack(fminf(fmaxf(p, -9.0f), 8.0f), fminf(fmaxf(q, -9.0f), 8.0f));
    }
    const uint64_t m = add2(y, up), n = add2(m, down);  // n = rint(y)
    uint64_t d = y;
    f32x2_fma(d, n, minus);
    float p, q;
    f32x2_unpack(d, p, q);
    off = fmaxf(off, fmaxf(fabsf(p), fabsf(q)));
    float lo, hi;
    f32x2_unpack(add2(m, eight), lo, hi);
    if (CLAMP) {
      lo = fminf(fmaxf(lo, kMagic), kMagic + 15.0f);
      hi = fminf(fmaxf(hi, kMagic), kMagic + 15.0f);
    }
    b[2 * i] = __float_as_uint(lo);
    b[2 * i + 1] = __float_as_uint(hi);
  }
  if (off > 0.499995f) {  // rare, but common for ties of short weights
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float n = rintf(__fdiv_rn(v[i], s));
      b[i] = __float_as_uint(fminf(fmaxf(n, -8.0f), 7.0f) + (kMagic + 8.0f));
    }
  }
  // bytes of elements (0, 4, 1, 5) and (2, 6, 3, 7): the even and the odd nibbles
  const uint32_t even = __byte_perm(__byte_perm(b[0], b[4], 0x0040), __byte_perm(b[1], b[5], 0x0040), 0x5410);
  const uint32_t odd = __byte_perm(__byte_perm(b[2], b[6], 0x0040), __byte_perm(b[3], b[7], 0x0040), 0x5410);
  const uint32_t u = (even & 0x0F0F0F0Fu) | ((odd & 0x0F0F0F0Fu) << 4);
  return __funnelshift_l(u, u, 3);
}
// bf16(m / 7) with the IEEE quotient: m * RN(1 / 7) is within 2 ulps of it, which matters only next to the middle between
// two bf16 numbers.
__device__ __forceinline__ uint32_t scale_bits(float m) {
  float q = m * (1.0f / 7.0f);
  if ((__float_as_uint(q) & 0xFFFFu) - 0x7FFCu <= 8u) q = __fdiv_rn(m, 7.0f);
  const uint32_t sb = __bfloat16_as_ushort(__float2bfloat16_rn(q));
  return sb < 0x0080u ? 0u : sb;  // below the smallest normal number
}
constexpr uint32_t kZeroWord = 0x44444444u;  // rotl32(0x88888888, 3): q = 0

template <int TYPE, int G, bool GIVEN>
__global__ void __launch_bounds__(kWarps * 32, TYPE == kF32 ? 2 : 4) quantize_kernel(const void* __restrict__ w,
                                                               const float* __restrict__ block_scale,
                                                               const uint16_t* __restrict__ given, uint32_t tiles, int N,
                                                               int K, uint8_t* __restrict__ packed) {
  constexpr int kGroups = 128 / G, kPer = G / 32;  // groups of a tile; words of a lane per group
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t kt_n = K / kTileK, nt_n = ((uint32_t)N + kTileN - 1) / kTileN;
  pdl_wait();
  pdl_trigger();
  const uint32_t tile = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (tile >= tiles) return;
  const uint32_t row_tile = tile / kt_n, kt = tile - row_tile * kt_n, b = row_tile / nt_n, nt = row_tile - b * nt_n;
  uint8_t* out = packed + (size_t)tile * tile_bytes(G);
  uint32_t scale_word[kGroups] = {};
  Raw8<TYPE> raw[2][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row = nt * kTileN + 8 * h + g;
    const size_t at = ((size_t)b * N + row) * K + (size_t)kt * kTileK + 8 * t;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (row < N) raw[h][j].load(w, at + 32 * j);
      else raw[h][j].zero();
    }
  }
  // a tile lies inside one 128 x 128 block
  const float bs = TYPE == kE4m3 ? __ldg(block_scale + ((size_t)b * (((uint32_t)N + 127) / 128) + nt / 8) * kt_n + kt) : 1.0f;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row = nt * kTileN + 8 * h + g;
    uint32_t word[4];
#pragma unroll
    for (int gr = 0; gr < kGroups; ++gr) {
      float v[kPer][8], m = 0.0f;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        raw[h][gr * kPer + j].widen(v[j], bs);
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max_abs_nan(m, v[j][i]);
      }
      m = max_abs_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = max_abs_nan(m, __shfl_xor_sync(0xffffffffu, m, 2));
      uint32_t sb;
      if (GIVEN)
        sb = row < N ? given[((size_t)b * N + row) * (K / G) + (size_t)kt * kGroups + gr] : 0u;
      else
        sb = scale_bits(m);
      if (!(m <= 3.402823466e38f)) sb = 0x7FC0u;  // an infinity or a NaN among them
      const float s = __uint_as_float(sb << 16);
      float r;
      asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(s));
      const bool use = s >= kMinNormal && s <= 3.402823466e38f;
#pragma unroll
      for (int j = 0; j < kPer; ++j) word[gr * kPer + j] = use ? quantize8<GIVEN>(v[j], s, r) : kZeroWord;
      scale_word[gr] |= sb << (16 * h);
    }
    *reinterpret_cast<uint4*>(out + 512 * h + 16 * lane) = make_uint4(word[0], word[1], word[2], word[3]);
  }
#pragma unroll
  for (int gr = 0; gr < kGroups; ++gr)
    if (t == 0) *reinterpret_cast<uint32_t*>(out + kTileQ + 32 * gr + 4 * g) = scale_word[gr];
}

// Eight consecutive values in the output type, stored where `there`; called by all lanes of a warp.
template <int TYPE>
__device__ __forceinline__ void store8(void* base, size_t at, const float (&v)[8], bool there) {
  if constexpr (TYPE == kF32) {
    // Two lanes of a quad swap halves, so that a store writes whole 32-byte sectors: first the even lane's, then the odd's.
    const bool odd = threadIdx.x & 1;
    float o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __shfl_xor_sync(0xffffffffu, odd ? v[i] : v[4 + i], 1);
    if (!there) return;
    float* p = reinterpret_cast<float*>(base) + at - (odd ? 4 : 0);
    *reinterpret_cast<float4*>(p) = odd ? make_float4(o[0], o[1], o[2], o[3]) : make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 8) = odd ? make_float4(v[4], v[5], v[6], v[7]) : make_float4(o[0], o[1], o[2], o[3]);
  } else {
    if (!there) return;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (TYPE == kBf16) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&p);
      } else {
        const __half2 p = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&p);
      }
    }
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(base) + at) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <int TYPE, int G>
__global__ void __launch_bounds__(kWarps * 32) dequantize_kernel(const uint8_t* __restrict__ packed, uint32_t tiles, int N,
                                                                 int K, void* __restrict__ out) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t kt_n = K / kTileK, nt_n = ((uint32_t)N + kTileN - 1) / kTileN;
  pdl_wait();
  pdl_trigger();
  for (uint32_t tile = blockIdx.x * kWarps + (threadIdx.x >> 5); tile < tiles; tile += gridDim.x * kWarps) {
  const uint32_t row_tile = tile / kt_n, kt = tile - row_tile * kt_n, b = row_tile / nt_n, nt = row_tile - b * nt_n;
  const uint8_t* in = packed + (size_t)tile * tile_bytes(G);
  const uint4 q[2] = {__ldg(reinterpret_cast<const uint4*>(in + 16 * lane)),
                      __ldg(reinterpret_cast<const uint4*>(in + 512 + 16 * lane))};
  const uint32_t magic = magic_register<Bf16>();
  uint32_t sw[128 / G];
#pragma unroll
  for (int gr = 0; gr < 128 / G; ++gr) sw[gr] = __ldg(reinterpret_cast<const uint32_t*>(in + kTileQ + 32 * gr + 4 * g));
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row = nt * kTileN + 8 * h + g;
    const size_t at = ((size_t)b * N + row) * K + (size_t)kt * kTileK + 8 * t;
    const uint32_t w[4] = {q[h].x, q[h].y, q[h].z, q[h].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t s2 = sw[j * 32 / G];
      const float s = h == 0 ? __uint_as_float(s2 << 16) : __uint_as_float(s2 & 0xFFFF0000u);
      uint32_t p[4];
      decode_word<Bf16>(w[j], magic, p);
      float v[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(p[i] << 16) * s;
        v[2 * i + 1] = __uint_as_float(p[i] & 0xFFFF0000u) * s;
      }
      store8<TYPE>(out, at + 32 * j, v, row < N);
    }
  }
  }
}

// CTAs for a warp per tile, `most` at most.  The quantiser takes all of them and the reader, whose warps walk their tiles, 32
// per SM: with eight per SM, quantising and reading took 165 in place of 146 us (8 x 7168 x 2048, e4m3 to fp32) and reading
// 13.0 in place of 12.2 (4096 x 7168, bf16).  A reader without the loop is slower (5 x 2045 x 1408, f16: 6.6 us, 5.75).
unsigned grid_for(long tiles, long most) {
  const long n = (tiles + kWarps - 1) / kWarps;
  return (unsigned)(n < most ? n : most);
}

template <int TYPE, int G>
cudaError_t run_quantize(const void* w, const float* bs, const void* given, long tiles, int N, int K, void* packed,
                         cudaStream_t stream) {
  return launch_pdl(given ? quantize_kernel<TYPE, G, true> : quantize_kernel<TYPE, G, false>, dim3(grid_for(tiles, LONG_MAX)),
                    dim3(kWarps * 32), 0, stream, w, bs, reinterpret_cast<const uint16_t*>(given), (uint32_t)tiles, N, K,
                    reinterpret_cast<uint8_t*>(packed));
}
template <int TYPE>
cudaError_t pick_quantize(int group, const void* w, const float* bs, const void* given, long tiles, int N, int K,
                          void* packed, cudaStream_t stream) {
  if (group == 32) return run_quantize<TYPE, 32>(w, bs, given, tiles, N, K, packed, stream);
  if (group == 64) return run_quantize<TYPE, 64>(w, bs, given, tiles, N, K, packed, stream);
  return run_quantize<TYPE, 128>(w, bs, given, tiles, N, K, packed, stream);
}
template <int TYPE, int G>
cudaError_t run_dequantize(const void* packed, long tiles, int N, int K, void* out, cudaStream_t stream) {
  return launch_pdl(dequantize_kernel<TYPE, G>, dim3(grid_for(tiles, 32L * num_sms_of_current_device())), dim3(kWarps * 32), 0, stream,
                    reinterpret_cast<const uint8_t*>(packed), (uint32_t)tiles, N, K, out);
}
template <int TYPE>
cudaError_t pick_dequantize(int group, const void* packed, long tiles, int N, int K, void* out, cudaStream_t stream) {
  if (group == 32) return run_dequantize<TYPE, 32>(packed, tiles, N, K, out, stream);
  if (group == 64) return run_dequantize<TYPE, 64>(packed, tiles, N, K, out, stream);
  return run_dequantize<TYPE, 128>(packed, tiles, N, K, out, stream);
}

bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

}  // namespace
}  // namespace w4
}  // namespace fbmoe

using namespace fbmoe;

extern "C" FBMOE_API size_t fbmoe_w4_bytes(int64_t batch, int N, int K, int group) {
  if (batch < 0 || N < 1 || K < 128 || K % 128 != 0 || !w4::valid_group(group)) return 0;
  return (size_t)batch * (((size_t)N + 15) / 16) * (K / 128) * w4::tile_bytes(group);
}

extern "C" FBMOE_API int fbmoe_quantize_w4(const void* w, int w_type, const float* block_scale, const void* scale_bf16,
                                           int64_t batch, int N, int K, int group, void* packed, void* stream_) {
  if (batch < 0 || N < 1 || K < 128 || K % 128 != 0 || !w4::valid_group(group)) return FBMOE_ERR_INVALID_ARG;
  if (w_type < FBMOE_BF16 || w_type > FBMOE_E4M3) return FBMOE_ERR_INVALID_ARG;
  if (batch == 0) return FBMOE_OK;
  if (!w || !packed || (w_type == FBMOE_E4M3 && !block_scale)) return FBMOE_ERR_NULL_POINTER;
  if (w4::misaligned(w) || w4::misaligned(packed) || ((uintptr_t)block_scale & 3) || ((uintptr_t)scale_bf16 & 1))
    return FBMOE_ERR_MISALIGNED;
  if (batch > INT64_C(0x7fffffff) / ((N - 1) / 16 + 1) / (K / 128)) return FBMOE_ERR_INVALID_ARG;  // 4e12 weights
  const long tiles = (long)batch * ((N - 1) / 16 + 1) * (K / 128);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  cudaError_t e;
  switch (w_type) {
    case FBMOE_BF16: e = w4::pick_quantize<w4::kBf16>(group, w, block_scale, scale_bf16, tiles, N, K, packed, stream); break;
    case FBMOE_F16: e = w4::pick_quantize<w4::kF16>(group, w, block_scale, scale_bf16, tiles, N, K, packed, stream); break;
    case FBMOE_F32: e = w4::pick_quantize<w4::kF32>(group, w, block_scale, scale_bf16, tiles, N, K, packed, stream); break;
    default: e = w4::pick_quantize<w4::kE4m3>(group, w, block_scale, scale_bf16, tiles, N, K, packed, stream); break;
  }
  return e == cudaSuccess ? FBMOE_OK : (int)e;
}

extern "C" FBMOE_API int fbmoe_dequantize_w4(const void* packed, int64_t batch, int N, int K, int group, int out_type,
                                             void* out, void* stream_) {
  if (batch < 0 || N < 1 || K < 128 || K % 128 != 0 || !w4::valid_group(group)) return FBMOE_ERR_INVALID_ARG;
  if (out_type < FBMOE_BF16 || out_type > FBMOE_F32) return FBMOE_ERR_INVALID_ARG;
  if (batch == 0) return FBMOE_OK;
  if (!packed || !out) return FBMOE_ERR_NULL_POINTER;
  if (w4::misaligned(packed) || w4::misaligned(out)) return FBMOE_ERR_MISALIGNED;
  if (batch > INT64_C(0x7fffffff) / ((N - 1) / 16 + 1) / (K / 128)) return FBMOE_ERR_INVALID_ARG;  // 4e12 weights
  const long tiles = (long)batch * ((N - 1) / 16 + 1) * (K / 128);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  cudaError_t e;
  switch (out_type) {
    case FBMOE_BF16: e = w4::pick_dequantize<w4::kBf16>(group, packed, tiles, N, K, out, stream); break;
    case FBMOE_F16: e = w4::pick_dequantize<w4::kF16>(group, packed, tiles, N, K, out, stream); break;
    default: e = w4::pick_dequantize<w4::kF32>(group, packed, tiles, N, K, out, stream); break;
  }
  return e == cudaSuccess ? FBMOE_OK : (int)e;
}
