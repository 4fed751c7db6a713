// w4_quant.cu -- weights to and from the packed 4-bit format of w4_common.cuh.
//
// Quantiser: per row and group of G columns s = bf16(max |w| / 7) (IEEE fp32 division, then round to nearest; 0 when
// that is below the smallest normal number), or the caller's s; q = clamp(rint(w / s), -8, 7) with w / s the IEEE
// fp32 quotient, 0 where s is not positive.  A group that holds a NaN or an infinity gets the scale NaN.
// Reader: v = q * s, exact in fp32 (4 bits times 8), rounded once to the output type.
//
// Both are bound by HBM.  One warp per tile: lane l = 4g + t owns rows g and g + 8, columns 32j + 8t .. + 7, which are
// its packed words, so values go from the loads to the packed stores without shared memory: a quad reads 32
// contiguous columns of a row, a half tile is stored as one coalesced 512-byte row of 16-byte words, and a group's
// maximum is at most two shuffles over the quad.
#include "fbmoe.h"
#include "fbmoe_launch.h"
#include "w4_common.cuh"

namespace fbmoe {
namespace w4 {
namespace {

constexpr int kWarps = 8;
constexpr float kMinNormal = 1.17549435e-38f;

enum Type { kBf16 = FBMOE_BF16, kF16 = FBMOE_F16, kF32 = FBMOE_F32, kE4m3 = FBMOE_E4M3 };

// Eight consecutive weights as fp32.
template <int TYPE>
__device__ __forceinline__ void load8(const void* base, size_t at, float (&v)[8]) {
  if constexpr (TYPE == kBf16) {
    const uint4 r = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(base) + at));
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  } else if constexpr (TYPE == kF16) {
    const uint4 r = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(base) + at));
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  } else if constexpr (TYPE == kF32) {
    const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + at);
    const float4 a = __ldg(p), b = __ldg(p + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint2 r = __ldg(reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(base) + at));
    const uint32_t w[2] = {r.x, r.y};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i >> 1] >> (16 * (i & 1))), __NV_E4M3);
      const float2 f = __half22float2(__half2(h));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}

// rint(w / s) with the IEEE quotient, r = 1 / s: y = w * r is within 2 ulps of it, so only a y next to a half integer
// needs the division itself.
__device__ __forceinline__ int quotient(float w, float s, float r) {
  const float y = w * r;
  float n = rintf(y);
  if (fabsf(y - n) > 0.499995f) n = rintf(__fdiv_rn(w, s));
  return (int)fminf(fmaxf(n, -8.0f), 7.0f);
}

template <int TYPE, int G>
__global__ void __launch_bounds__(kWarps * 32) quantize_kernel(const void* __restrict__ w,
                                                               const float* __restrict__ block_scale,
                                                               const uint16_t* __restrict__ given, long tiles, int N,
                                                               int K, uint8_t* __restrict__ packed) {
  constexpr int kGroups = 128 / G, kPer = G / 32;  // groups of a tile; words of a lane per group
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int kt_n = K / kTileK, nt_n = (N + kTileN - 1) / kTileN;
  pdl_wait();
  pdl_trigger();
  for (long tile = (long)blockIdx.x * kWarps + (threadIdx.x >> 5); tile < tiles; tile += (long)gridDim.x * kWarps) {
    const int kt = (int)(tile % kt_n);
    const long b = tile / kt_n / nt_n;
    const int nt = (int)(tile / kt_n % nt_n);
    uint8_t* out = packed + (size_t)tile * tile_bytes(G);
    uint32_t scale_word[kGroups] = {};
    float v[2][4][8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = nt * kTileN + 8 * h + g;
      const size_t at = ((size_t)b * N + row) * K + (size_t)kt * kTileK + 8 * t;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (row < N) {
          load8<TYPE>(w, at + 32 * j, v[h][j]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[h][j][i] = 0.0f;
        }
      }
    }
    if (TYPE == kE4m3) {  // a tile lies inside one 128 x 128 block
      const float bs = __ldg(block_scale + ((size_t)b * ((N + 127) / 128) + nt / 8) * kt_n + kt);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) v[h][j][i] = __fmul_rn(v[h][j][i], bs);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = nt * kTileN + 8 * h + g;
      uint32_t word[4];
#pragma unroll
      for (int gr = 0; gr < kGroups; ++gr) {
        float m = 0.0f;
        bool bad = false;  // a NaN or an infinity
#pragma unroll
        for (int j = gr * kPer; j < (gr + 1) * kPer; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            m = fmaxf(m, fabsf(v[h][j][i]));
            bad |= !(fabsf(v[h][j][i]) <= 3.402823466e38f);
          }
        m = bad ? INFINITY : m;
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        uint32_t sb;
        if (given != nullptr) {
          sb = row < N ? given[((size_t)b * N + row) * (K / G) + (size_t)kt * kGroups + gr] : 0u;
        } else {
          sb = __bfloat16_as_ushort(__float2bfloat16_rn(__fdiv_rn(m, 7.0f)));
          if (__uint_as_float(sb << 16) < kMinNormal) sb = 0u;
        }
        if (m == INFINITY) sb = 0x7FC0u;
        const float s = __uint_as_float(sb << 16), r = __frcp_rn(s);
        const bool use = s >= kMinNormal && s <= 3.402823466e38f;
#pragma unroll
        for (int j = gr * kPer; j < (gr + 1) * kPer; ++j) {
          uint32_t u = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            u |= (uint32_t)((use ? quotient(v[h][j][i], s, r) : 0) + 8) << (4 * (i >> 1) + 16 * (i & 1));
          word[j] = __funnelshift_l(u, u, 3);
        }
        scale_word[gr] |= sb << (16 * h);
      }
      *reinterpret_cast<uint4*>(out + 512 * h + 16 * lane) = make_uint4(word[0], word[1], word[2], word[3]);
    }
#pragma unroll
    for (int gr = 0; gr < kGroups; ++gr)
      if (t == 0) *reinterpret_cast<uint32_t*>(out + kTileQ + 32 * gr + 4 * g) = scale_word[gr];
  }
}

// Eight consecutive values in the output type.
template <int TYPE>
__device__ __forceinline__ void store8(void* base, size_t at, const float (&v)[8]) {
  if constexpr (TYPE == kF32) {
    float4* p = reinterpret_cast<float4*>(reinterpret_cast<float*>(base) + at);
    p[0] = make_float4(v[0], v[1], v[2], v[3]);
    p[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
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
__global__ void __launch_bounds__(kWarps * 32) dequantize_kernel(const uint8_t* __restrict__ packed, long tiles, int N,
                                                                 int K, void* __restrict__ out) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int kt_n = K / kTileK, nt_n = (N + kTileN - 1) / kTileN;
  pdl_wait();
  pdl_trigger();
  for (long tile = (long)blockIdx.x * kWarps + (threadIdx.x >> 5); tile < tiles; tile += (long)gridDim.x * kWarps) {
    const int kt = (int)(tile % kt_n);
    const long b = tile / kt_n / nt_n;
    const int nt = (int)(tile / kt_n % nt_n);
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
      if (row >= N) continue;
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
        store8<TYPE>(out, at + 32 * j, v);
      }
    }
  }
}

// One wave of resident CTAs at most: a warp walks its tiles.
unsigned grid_for(long tiles) {
  const long blocks = (tiles + kWarps - 1) / kWarps;
  return (unsigned)(blocks < 148L * 8 ? blocks : 148L * 8);
}

template <int TYPE, int G>
cudaError_t run_quantize(const void* w, const float* bs, const void* given, long tiles, int N, int K, void* packed,
                         cudaStream_t stream) {
  return launch_pdl(quantize_kernel<TYPE, G>, dim3(grid_for(tiles)), dim3(kWarps * 32), 0, stream, w, bs,
                    reinterpret_cast<const uint16_t*>(given), tiles, N, K, reinterpret_cast<uint8_t*>(packed));
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
  return launch_pdl(dequantize_kernel<TYPE, G>, dim3(grid_for(tiles)), dim3(kWarps * 32), 0, stream,
                    reinterpret_cast<const uint8_t*>(packed), tiles, N, K, out);
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
