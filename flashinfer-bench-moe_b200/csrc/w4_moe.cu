// w4_moe.cu -- the whole MoE layer for a few tokens (T <= 64) on packed 4-bit weights.
//
//   route as fbmoe_route; h = silu(x Wg^T) * (x Wu^T) for every (token, local expert) pair; out = sum over a token's
//   pairs, in slot order, of weight * (h W2^T).
//
// W1's rows [0, I) are the linear half and [I, 2I) the silu half, as in fbmoe_forward.  h keeps fp32's leading 16 bits
// as two bf16 planes, hi = bf16(h) and lo = bf16(h - hi), which ride as two columns of one bf16 product: no range to
// clamp, relative error 2^-17.
#include "fbmoe.h"
#include "fbmoe_launch.h"
#include "w4_common.cuh"

namespace fbmoe {
namespace w4 {
namespace {

constexpr int kWarps = 8;

struct MoeLayout {
  size_t topk_idx, topk_w, h, pair_out, total;
};
MoeLayout moe_layout(int T, int H, int I) {
  MoeLayout L;
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t o = off;
    off = (off + bytes + 255) / 256 * 256;
    return o;
  };
  take(256);
  L.topk_idx = take((size_t)T * kTopK * 4);
  L.topk_w = take((size_t)T * kTopK * 4);
  L.h = take((size_t)T * kTopK * 2 * I * 2);       // [pair][hi, lo][I] bf16
  L.pair_out = take((size_t)T * kTopK * H * 4);    // [pair][H] fp32
  L.total = off;
  return L;
}

// The pairs (token * 8 + slot) of one expert in token order, into pairs[]; returns how many.  Needs a CTA of at least
// 64 threads and synchronises it.
__device__ __forceinline__ int expert_pairs(const int32_t* __restrict__ topk_idx, int T, int expert, int* pairs) {
  __shared__ unsigned long long mask;
  if (threadIdx.x == 0) mask = 0;
  __syncthreads();
  int slot = -1;
  const int t = threadIdx.x;
  if (t < T)
    for (int s = 0; s < kTopK; ++s)
      if (topk_idx[t * kTopK + s] == expert) slot = s;
  if (slot >= 0) atomicOr(&mask, 1ull << t);
  __syncthreads();
  const unsigned long long m = mask;
  if (slot >= 0) pairs[__popcll(m & ((1ull << t) - 1))] = t * kTopK + slot;
  __syncthreads();
  return __popcll(m);
}

// One 16-row tile times up to 8 columns over all K: the CTA's warps take the K tiles in turn and leave their partial
// sums in part[warp][column * 16 + row].  column_at: the lane's column's activations, or null.
template <typename A, int G>
__device__ __forceinline__ void tile_row_product(const uint8_t* __restrict__ tiles, int kt_n,
                                                 const typename A::Raw* column_at, float (*part)[128]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  float acc[1][4] = {};
  for (int kt = warp; kt < kt_n; kt += kWarps) {
    const uint8_t* tile = tiles + (size_t)kt * tile_bytes(G);
    const uint4 qlo = __ldg(reinterpret_cast<const uint4*>(tile + 16 * lane));
    const uint4 qhi = __ldg(reinterpret_cast<const uint4*>(tile + 512 + 16 * lane));
    uint32_t sw[128 / G];
#pragma unroll
    for (int gr = 0; gr < 128 / G; ++gr)
      sw[gr] = __ldg(reinterpret_cast<const uint32_t*>(tile + kTileQ + 32 * gr + 4 * g));
    uint4 xv[1][4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      xv[0][j] = column_at ? *reinterpret_cast<const uint4*>(column_at + kt * kTileK + 32 * j + 8 * t)
                           : make_uint4(0, 0, 0, 0);
    tile_product<A, G, 1>(qlo, qhi, sw, xv, acc);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) part[warp][(2 * t + (i & 1)) * 16 + g + 8 * (i >> 1)] = acc[0][i];
}
__device__ __forceinline__ float sum_parts(const float (*part)[128], int at) {
  float sum = 0.0f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) sum += part[w][at];
  return sum;
}

template <typename A, int G>
__global__ void __launch_bounds__(kWarps * 32) up_kernel(const typename A::Raw* __restrict__ x, int T,
                                                         const uint8_t* __restrict__ w1, int H, int I, int offset,
                                                         const int32_t* __restrict__ topk_idx,
                                                         __nv_bfloat16* __restrict__ h) {
  __shared__ float up[kWarps][128], gate[kWarps][128];
  __shared__ int pairs[kMaxTokens];
  pdl_wait();
  pdl_trigger();
  const int rows = expert_pairs(topk_idx, T, offset + blockIdx.y, pairs);
  const int g = (threadIdx.x & 31) >> 2, kt_n = H / kTileK;
  const uint8_t* tiles = w1 + ((size_t)blockIdx.y * (2 * I / kTileN) + blockIdx.x) * kt_n * tile_bytes(G);
  for (int r0 = 0; r0 < rows; r0 += 8) {
    const typename A::Raw* col = r0 + g < rows ? x + (size_t)(pairs[r0 + g] / kTopK) * H : nullptr;
    tile_row_product<A, G>(tiles, kt_n, col, up);
    tile_row_product<A, G>(tiles + (size_t)(I / kTileN) * kt_n * tile_bytes(G), kt_n, col, gate);
    __syncthreads();
    if (threadIdx.x < 128 && r0 + threadIdx.x / 16 < rows) {
      const float a = sum_parts(gate, threadIdx.x);
      const float v = a / (1.0f + expf(-a)) * sum_parts(up, threadIdx.x);
      const __nv_bfloat16 hi = __float2bfloat16_rn(v);
      const float rest = v - __bfloat162float(hi);
      __nv_bfloat16* at = h + (size_t)pairs[r0 + threadIdx.x / 16] * 2 * I + blockIdx.x * kTileN + threadIdx.x % 16;
      at[0] = hi;
      at[I] = __float2bfloat16_rn(isfinite(rest) ? rest : 0.0f);
    }
    __syncthreads();
  }
}

template <int G>
__global__ void __launch_bounds__(kWarps * 32) down_kernel(const __nv_bfloat16* __restrict__ h, int T,
                                                           const uint8_t* __restrict__ w2, int H, int I, int offset,
                                                           const int32_t* __restrict__ topk_idx,
                                                           const float* __restrict__ topk_w,
                                                           float* __restrict__ pair_out) {
  __shared__ float part[kWarps][128];
  __shared__ int pairs[kMaxTokens];
  pdl_wait();
  pdl_trigger();
  const int rows = expert_pairs(topk_idx, T, offset + blockIdx.y, pairs);
  const int g = (threadIdx.x & 31) >> 2, kt_n = I / kTileK;
  const uint8_t* tiles = w2 + ((size_t)blockIdx.y * (H / kTileN) + blockIdx.x) * kt_n * tile_bytes(G);
  for (int r0 = 0; r0 < rows; r0 += 4) {
    const __nv_bfloat16* col = r0 + (g >> 1) < rows ? h + ((size_t)pairs[r0 + (g >> 1)] * 2 + (g & 1)) * I : nullptr;
    tile_row_product<Bf16, G>(tiles, kt_n, col, part);
    __syncthreads();
    if (threadIdx.x < 64 && r0 + threadIdx.x / 16 < rows) {
      const int pair = pairs[r0 + threadIdx.x / 16], at = threadIdx.x / 16 * 32 + threadIdx.x % 16;
      pair_out[(size_t)pair * H + blockIdx.x * kTileN + threadIdx.x % 16] =
          (sum_parts(part, at) + sum_parts(part, at + 16)) * topk_w[pair];
    }
    __syncthreads();
  }
}

template <typename A>
__global__ void __launch_bounds__(256) combine_kernel(const float* __restrict__ pair_out, int E, int offset, int H,
                                                      const int32_t* __restrict__ topk_idx,
                                                      typename A::Raw* __restrict__ out) {
  pdl_wait();
  pdl_trigger();
  const int t = blockIdx.y, n = blockIdx.x * 256 + threadIdx.x;
  if (n >= H) return;
  float sum = 0.0f;
#pragma unroll
  for (int s = 0; s < kTopK; ++s) {
    const int e = topk_idx[t * kTopK + s] - offset;
    if (e >= 0 && e < E) sum += pair_out[((size_t)t * kTopK + s) * H + n];
  }
  out[(size_t)t * H + n] = A::of(sum);
}

struct MoeArgs {
  const float* logits;
  const void* bias;
  const void* x;
  const uint8_t *w1, *w2;
  int group1, group2, T, H, I, E, offset;
  float scale;
  void* out;
  uint8_t* ws;
  cudaStream_t stream;
};

template <typename A, int G>
cudaError_t run_up(const MoeArgs& a, const MoeLayout& L) {
  return launch_pdl(up_kernel<A, G>, dim3(a.I / kTileN, a.E), dim3(kWarps * 32), 0, a.stream,
                    reinterpret_cast<const typename A::Raw*>(a.x), a.T, a.w1, a.H, a.I, a.offset,
                    reinterpret_cast<const int32_t*>(a.ws + L.topk_idx), reinterpret_cast<__nv_bfloat16*>(a.ws + L.h));
}
template <int G>
cudaError_t run_down(const MoeArgs& a, const MoeLayout& L) {
  return launch_pdl(down_kernel<G>, dim3(a.H / kTileN, a.E), dim3(kWarps * 32), 0, a.stream,
                    reinterpret_cast<const __nv_bfloat16*>(a.ws + L.h), a.T, a.w2, a.H, a.I, a.offset,
                    reinterpret_cast<const int32_t*>(a.ws + L.topk_idx), reinterpret_cast<const float*>(a.ws + L.topk_w),
                    reinterpret_cast<float*>(a.ws + L.pair_out));
}
template <typename A>
cudaError_t run_moe(const MoeArgs& a) {
  const MoeLayout L = moe_layout(a.T, a.H, a.I);
  cudaError_t e = launch_route(a.logits, a.bias, a.T, a.scale, reinterpret_cast<int32_t*>(a.ws + L.topk_idx),
                               reinterpret_cast<float*>(a.ws + L.topk_w), nullptr, a.stream);
  if (e != cudaSuccess) return e;
  e = a.group1 == 32 ? run_up<A, 32>(a, L) : a.group1 == 64 ? run_up<A, 64>(a, L) : run_up<A, 128>(a, L);
  if (e != cudaSuccess) return e;
  e = a.group2 == 32 ? run_down<32>(a, L) : a.group2 == 64 ? run_down<64>(a, L) : run_down<128>(a, L);
  if (e != cudaSuccess) return e;
  return launch_pdl(combine_kernel<A>, dim3((a.H + 255) / 256, a.T), dim3(256), 0, a.stream,
                    reinterpret_cast<const float*>(a.ws + L.pair_out), a.E, a.offset, a.H,
                    reinterpret_cast<const int32_t*>(a.ws + L.topk_idx), reinterpret_cast<typename A::Raw*>(a.out));
}

bool bad_sizes(int T, int H, int I) {
  return T < 0 || T > kMaxTokens || H < 128 || H % 128 != 0 || I < 128 || I % 128 != 0 || H > (1 << 20) || I > (1 << 20);
}

}  // namespace
}  // namespace w4
}  // namespace fbmoe

using namespace fbmoe;

extern "C" FBMOE_API size_t fbmoe_w4_workspace_size(int T, int H, int I) {
  return w4::bad_sizes(T, H, I) ? 0 : w4::moe_layout(T, H, I).total;
}

extern "C" FBMOE_API int fbmoe_forward_w4(const float* routing_logits, const void* routing_bias,
                                          const void* hidden_states, int type, const void* gemm1_weights, int group1,
                                          const void* gemm2_weights, int group2, int T, int H, int I, int E_local,
                                          int local_expert_offset, float routed_scaling_factor, void* out,
                                          void* workspace, size_t workspace_bytes, void* stream) {
  if (w4::bad_sizes(T, H, I) || E_local < 1 || E_local > kExperts || local_expert_offset < 0 ||
      local_expert_offset >= kExperts || !w4::valid_group(group1) || !w4::valid_group(group2) ||
      (type != FBMOE_BF16 && type != FBMOE_F16))
    return FBMOE_ERR_INVALID_ARG;
  if (T == 0) return FBMOE_OK;
  if (!routing_logits || !routing_bias || !hidden_states || !gemm1_weights || !gemm2_weights || !out || !workspace)
    return FBMOE_ERR_NULL_POINTER;
  for (const void* p : {(const void*)routing_logits, routing_bias, hidden_states, gemm1_weights, gemm2_weights,
                        (const void*)out})
    if ((uintptr_t)p & 15) return FBMOE_ERR_MISALIGNED;
  if ((uintptr_t)workspace & 255) return FBMOE_ERR_MISALIGNED;
  if (workspace_bytes < w4::moe_layout(T, H, I).total) return FBMOE_ERR_WORKSPACE_TOO_SMALL;
  const w4::MoeArgs a = {routing_logits, routing_bias, hidden_states,
                         reinterpret_cast<const uint8_t*>(gemm1_weights), reinterpret_cast<const uint8_t*>(gemm2_weights),
                         group1, group2, T, H, I, E_local, local_expert_offset, routed_scaling_factor, out,
                         reinterpret_cast<uint8_t*>(workspace), reinterpret_cast<cudaStream_t>(stream)};
  const cudaError_t e = type == FBMOE_BF16 ? w4::run_moe<w4::Bf16>(a) : w4::run_moe<w4::F16>(a);
  return e == cudaSuccess ? FBMOE_OK : (int)e;
}
