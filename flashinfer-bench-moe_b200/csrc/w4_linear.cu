// w4_linear.cu -- products of a few tokens with a packed 4-bit matrix: out[t, n] = sum over k of x[t, k] q[n, k] s[n, k / G],
// x and out bf16 or f16, sums in fp32, one rounding.
//
// One CTA per 16-row tile and block of up to 8 NT tokens; its eight warps take the tiles along K in turn and their
// partial sums are added in warp order through shared memory.
#include "fbmoe.h"
#include "fbmoe_launch.h"
#include "w4_common.cuh"

namespace fbmoe {
namespace w4 {
namespace {

constexpr int kWarps = 8;

template <typename A, int G, int NT>
__global__ void __launch_bounds__(kWarps * 32) linear_kernel(const typename A::Raw* __restrict__ x, long ldx, int T,
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
    const uint4 qlo = __ldg(reinterpret_cast<const uint4*>(tile + 16 * lane));
    const uint4 qhi = __ldg(reinterpret_cast<const uint4*>(tile + 512 + 16 * lane));
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

template <typename A, int G>
cudaError_t run_linear(const void* x, long ldx, int T, const void* packed, int N, int K, void* out, long ldo,
                       cudaStream_t stream) {
  using Raw = typename A::Raw;
  const unsigned nt = (unsigned)((N - 1) / kTileN + 1);
  const Raw* xp = reinterpret_cast<const Raw*>(x);
  const uint8_t* wp = reinterpret_cast<const uint8_t*>(packed);
  Raw* op = reinterpret_cast<Raw*>(out);
  if (T <= 8)
    return launch_pdl(linear_kernel<A, G, 1>, dim3(nt), dim3(kWarps * 32), 0, stream, xp, ldx, T, wp, N, K, op, ldo);
  return launch_pdl(linear_kernel<A, G, 2>, dim3(nt, (unsigned)((T + 15) / 16)), dim3(kWarps * 32), 0, stream, xp, ldx,
                    T, wp, N, K, op, ldo);
}
template <typename A>
cudaError_t pick_linear(int group, const void* x, long ldx, int T, const void* packed, int N, int K, void* out,
                        long ldo, cudaStream_t stream) {
  if (group == 32) return run_linear<A, 32>(x, ldx, T, packed, N, K, out, ldo, stream);
  if (group == 64) return run_linear<A, 64>(x, ldx, T, packed, N, K, out, ldo, stream);
  return run_linear<A, 128>(x, ldx, T, packed, N, K, out, ldo, stream);
}

}  // namespace
}  // namespace w4
}  // namespace fbmoe

using namespace fbmoe;

extern "C" FBMOE_API int fbmoe_linear_w4(const void* x, int64_t x_stride, int type, int T, const void* packed, int N,
                                         int K, int group, void* out, int64_t out_stride, void* stream_) {
  if (T < 0 || T > w4::kMaxTokens || N < 1 || K < 128 || K % 128 != 0 || !w4::valid_group(group) ||
      (type != FBMOE_BF16 && type != FBMOE_F16) || x_stride < K || out_stride < N)
    return FBMOE_ERR_INVALID_ARG;
  if (T == 0) return FBMOE_OK;
  if (!x || !packed || !out) return FBMOE_ERR_NULL_POINTER;
  if (((uintptr_t)x & 15) || (x_stride & 7) || ((uintptr_t)packed & 15) || ((uintptr_t)out & 1))
    return FBMOE_ERR_MISALIGNED;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  const cudaError_t e =
      type == FBMOE_BF16
          ? w4::pick_linear<w4::Bf16>(group, x, x_stride, T, packed, N, K, out, out_stride, stream)
          : w4::pick_linear<w4::F16>(group, x, x_stride, T, packed, N, K, out, out_stride, stream);
  return e == cudaSuccess ? FBMOE_OK : (int)e;
}
