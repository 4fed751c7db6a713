// w4_moe.cu -- the whole MoE layer for a few tokens (T <= 64) on packed 4-bit weights, in two kernels.
//
//   route as fbmoe_route; h = silu(x Wg^T) * (x Wu^T) for every (token, local expert) pair; out = sum over a token's
//   pairs, in slot order, of weight * (h W2^T).
//
// W1's rows [0, I) are the linear half and [I, 2I) the silu half, as in fbmoe_forward.  x enters its product as it is, h
// as two bf16 numbers (w4_stream.cuh).
//
// route_kernel: a warp per token; also zeroes the layer kernel's counters.
//
// layer_kernel: one CTA per SM, working on units handed out by a ticket counter in the order
//   up: (up to 8 rows of an expert; 32 MW pairs of W1 rows, two linear and two silu tiles side by side),
//   down: (up to 8 rows of an expert; 64 MW rows of W2),
//   combine: 2048 outputs.
// A down unit needs its expert's up units, a combine unit all down units.  Tickets are taken in order, so whatever a unit
// waits for has been taken by a CTA that is running already and that waits for less: no co-residency is assumed, and two
// calls may share the GPU.
//
// The scheduler warp takes tickets ahead and waits for what a unit needs; 16 consumer warps, KW along K times MW along
// the rows, stream the unit's tiles through their rings (w4_stream.cuh) and on into the next unit's; two finisher warps
// add their partial sums in a fixed order, apply SwiGLU or the routing weight, store and report.  A unit takes an SM 4 to
// 8 us at H = 7168, so phases and the end of the call are balanced to that; with a unit per warp or group of warps they were
// not, and T = 64 took a fifth longer.  Every order of summation depends on the sizes and the routing alone.
#include "fbmoe.h"
#include "fbmoe_launch.h"
#include "moe_route.cuh"
#include "w4_stream.cuh"

namespace fbmoe {
namespace w4 {
namespace {

constexpr int kRows = 8;                    // token rows of a unit
constexpr int kUpSpan = 32, kDownSpan = 64;   // columns of h, rows of W2 of a consumer warp (four tiles)
constexpr int kFinishers = 2;
constexpr int kThreads = (kStreamWarps + 4) * 32;  // consumers; finishers, scheduler, one idle
// Registers: five warps per quarter of an SM are launched with 96 each; the fifth gives up 32, the consumers take 8.
constexpr int kConsumerRegs = 104, kHelperRegs = 64;
constexpr int kCombine = 4 * 32 * kStreamWarps;  // outputs of a combine unit
constexpr int kQueue = 2;                   // units known: the one worked on, and the one whose tiles are under way
constexpr int kMaxBlocks = kMaxTokens * kTopK / kRows + kExperts;  // row blocks of all experts
constexpr int kPart = 512;                  // floats of a consumer warp's partial sums: [4 tokens][half][lane][4]

// counters in the workspace, zeroed by route_kernel
struct Counters {
  uint32_t status, ticket, done, pad;
  uint32_t ready[kExperts];  // finished (up unit, finisher) pairs of each local expert
};

struct MoeLayout {
  size_t counters, topk_idx, topk_w, h, pair_out, total;
};
MoeLayout moe_layout(int T, int H, int I) {
  MoeLayout L;
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t o = off;
    off = (off + bytes + 255) / 256 * 256;
    return o;
  };
  L.counters = take(sizeof(Counters));
  L.topk_idx = take((size_t)T * kTopK * 4);
  L.topk_w = take((size_t)T * kTopK * 4);
  L.h = take((size_t)T * kTopK * I * 4);         // [pair][two bf16 numbers][I]
  L.pair_out = take((size_t)T * kTopK * H * 4);    // [pair][H] fp32
  L.total = off;
  return L;
}

__global__ void __launch_bounds__(32) route_kernel(const float* __restrict__ logits, const __nv_bfloat16* __restrict__ bias,
                                                   float scale, int32_t* __restrict__ topk_idx, float* __restrict__ topk_w,
                                                   Counters* __restrict__ counters) {
  __shared__ float wv[kExperts], ws[kExperts];
  __shared__ int wi[kExperts], sel[kTopK];
  const int t = blockIdx.x;
  pdl_wait();
  pdl_trigger();
  for (int i = t * 32 + threadIdx.x; i < (int)(sizeof(Counters) / 4); i += gridDim.x * 32)
    reinterpret_cast<uint32_t*>(counters)[i] = 0;
  float l[8], b[8];
  route_dev::load_logits8(logits, t, l);
  route_dev::load_bias8(bias, b);
  route_dev::route_token(l, t, b, scale, topk_idx, topk_w, wv, wi, ws, sel);
}

struct LayerArgs {
  CUtensorMap map1, map2;  // W1, W2
  int T, H, I, E, offset;
  int kw1[2], kw2[2];    // consumer warps along K of an up / down unit: for small calls, for large ones
  const int32_t* topk_idx;
  const float* topk_w;
  const void* x;
  __nv_bfloat16* h;
  float* pair_out;
  Counters* counters;
  void* out;
  uint32_t* sink;
  uint64_t wait_ns;      // limit of a wait for other CTAs' units
  uint32_t extra;        // arrivals that never come (test hook)
};

// A row block: local expert, its first pair's place in the pair list, its rows.
__device__ __forceinline__ uint32_t block_word(int e, int pos, int rows) { return e | pos << 8 | rows << 20; }
__device__ __forceinline__ int block_expert(uint32_t w) { return w & 0xff; }
__device__ __forceinline__ int block_pos(uint32_t w) { return w >> 8 & 0xfff; }
__device__ __forceinline__ int block_rows_of(uint32_t w) { return w >> 20 & 0xff; }

enum Kind { kStop = 0, kUp = 1, kDown = 2, kSum = 3 };
// A unit: its row block, its place along the rows (or, to be summed, along the outputs).
struct __align__(8) Unit {
  uint32_t block;  // and the kind in bits 28, 29
  uint32_t row;
};
__device__ __forceinline__ int kind_of(const Unit& u) { return u.block >> 28; }

struct Shared {
  unsigned long long mask[kExperts];  // tokens of each local expert
  uint64_t ring_full[kStreamWarps][kDepth];
  uint64_t known[kQueue], go[kQueue], done[kQueue];  // a queue slot's unit is there; may be begun; is finished
  uint64_t part_full[2], part_empty[2];
  Unit unit[kQueue];
  uint32_t block[kMaxBlocks];
  uint32_t warp_sum[8];
  uint16_t pair_at[kExperts];          // first place of an expert's pairs
  uint16_t pairs[kMaxTokens * kTopK];  // token * 8 + slot, by expert, tokens ascending
  float pair_w[kMaxTokens * kTopK];    // their weights
  int n_blocks;                        // row blocks
  int kw1, kw2;                        // the call's choice
  int abort;
};

__device__ __forceinline__ uint32_t load_acquire(const uint32_t* p) {
  uint32_t v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void add_release(uint32_t* p, uint32_t v) {
  asm volatile("red.release.gpu.global.add.u32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}
// The row lists of all local experts, from the routing.
__device__ __forceinline__ void build_lists(const LayerArgs& a, Shared& s) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < kExperts) s.mask[tid] = 0;
  __syncthreads();
  int e = -1;
  if (tid < a.T * kTopK) {
    e = a.topk_idx[tid] - a.offset;
    if (e < 0 || e >= a.E) e = -1;
    if (e >= 0) atomicOr(&s.mask[e], 1ull << (tid / kTopK));
  }
  __syncthreads();
  uint32_t mine = 0, sum = 0;  // pairs and row blocks, 16 bits each
  int rows = 0;
  if (tid < kExperts) {
    rows = __popcll(s.mask[tid]);
    mine = rows | (uint32_t)((rows + kRows - 1) / kRows) << 16;
    sum = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const uint32_t o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    if (lane == 31) s.warp_sum[warp] = sum;
  }
  __syncthreads();
  if (tid < kExperts) {
    for (int w = 0; w < warp; ++w) sum += s.warp_sum[w];
    if (tid == kExperts - 1) s.n_blocks = sum >> 16;
    sum -= mine;
    const int pos = sum & 0xffff, block = sum >> 16;
    s.pair_at[tid] = (uint16_t)pos;
    for (int r = 0; r < rows; r += kRows) s.block[block + r / kRows] = block_word(tid, pos + r, min(kRows, rows - r));
  }
  __syncthreads();
  if (e >= 0) {
    const int at = s.pair_at[e] + __popcll(s.mask[e] & ((1ull << (tid / kTopK)) - 1));
    s.pairs[at] = (uint16_t)tid;
    s.pair_w[at] = a.topk_w[tid];
  }
  __syncthreads();
}

constexpr float kMaxBf16 = 3.38953139e38f;  // an h beyond it would round to infinity
__device__ __forceinline__ float swiglu(float gate, float up) { return gate / (1.0f + expf(-gate)) * up; }

// What a consumer warp has of a unit: K positions [k0, k0 + steps) of four row tiles.
struct Span {
  int k0, steps;
};
__device__ __forceinline__ Span span_of(const LayerArgs& a, const Shared& s, bool up) {
  Span w;
  const int kw = up ? s.kw1 : s.kw2, kt = (up ? a.H : a.I) / kTileK, kg = threadIdx.x / 32 & (kw - 1);
  w.k0 = kt * kg / kw;
  w.steps = kt * (kg + 1) / kw - w.k0;
  return w;
}
// The warp's row group (32 columns of h, or 64 rows of W2) of a unit; it may lie past the last one.
__device__ __forceinline__ uint32_t row_group(const Shared& s, const Unit& u, int warp) {
  const int kw = kind_of(u) == kUp ? s.kw1 : s.kw2;
  return u.row * (kStreamWarps / kw) + warp / kw;
}
__device__ __forceinline__ uint32_t row_groups(const LayerArgs& a, const Unit& u) {
  return kind_of(u) == kUp ? a.I / kUpSpan : a.H / kDownSpan;
}

// A consumer warp's stream: the copies of its tiles, ahead of what it works on.  A step is one K position of four row
// tiles, one tensor copy: a tile's bytes are kTileWords 8-byte elements, W1 maps as [expert][half][row tile][K position x
// element] with boxes of two row tiles of both halves, W2 the same with one half and boxes of four.
constexpr int tile_words(int group) { return tile_bytes(group) / 8; }
template <int G1, int G2>
struct Stream {
  Ring<step_bytes(G1 < G2 ? G1 : G2)> ring;
  int x, row;
  uint32_t unit;  // the local expert, and whether it is an up unit in bit 8
  int left;       // steps of the unit being issued that are still to be issued
  uint32_t seq;   // units begun; kNoMore: there are none left
  static constexpr uint32_t kNoMore = 1u << 31;

  __device__ __forceinline__ void step(const LayerArgs& a) {
    const bool up = unit >> 8;
    const int words = up ? tile_words(G1) : tile_words(G2);
    ring.issue(up ? &a.map1 : &a.map2, x, row, unit & 0xff, words * 32);
    x += words;
    --left;
  }
  // Issue steps while the ring has room.
  __device__ __forceinline__ void fill(const LayerArgs& a, Shared& s) {
    while (!ring.full()) {
      if (left > 0) {
        step(a);
        continue;
      }
      // the next unit, if it is known
      if (seq >= kNoMore || !__all_sync(0xffffffffu, ring.test(smem_u32(&s.known[seq % kQueue]), seq / kQueue & 1))) return;
      const Unit u = s.unit[seq % kQueue];
      ++seq;
      const int kind = kind_of(u);
      if (kind != kUp && kind != kDown) {
        seq |= kNoMore;
        return;
      }
      const uint32_t group = row_group(s, u, threadIdx.x / 32);
      if (group >= row_groups(a, u)) continue;
      const Span w = span_of(a, s, kind == kUp);
      x = w.k0 * (kind == kUp ? tile_words(G1) : tile_words(G2));
      row = kind == kUp ? 2 * group : 4 * group;
      unit = block_expert(u.block) | (kind == kUp) << 8;
      left = w.steps;
    }
  }
};

// The lane's places in the activations of a task's rows from K position k0 on, columns as tile_product takes them (rows
// that are not there read the first one's: their sums are not used).  The loads are plain ones: x may be the call's output,
// which is written once no unit reads it any more, and h is written while the kernel runs.
template <int NT, bool PAIR>
struct Places {
  static constexpr int NC = PAIR ? NT : 1;
  const uint8_t* p[NC];

  __device__ __forceinline__ void at(const void* base, int width, int k0, const Shared& s, uint32_t block) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int pos = block_pos(block), rows = block_rows_of(block);
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int r = PAIR ? 4 * n + (g >> 1) : 4 * (g & 1) + (g >> 1);
      const int pair = s.pairs[pos + (r < rows ? r : 0)];
      const size_t row = PAIR ? 2 * pair + (g & 1) : pair / kTopK;
      p[n] = reinterpret_cast<const uint8_t*>(base) + (row * width + (size_t)k0 * kTileK + 8 * t) * 2;
    }
  }
  // The current K position's words j.
  __device__ __forceinline__ void load(Columns<NC>& c, int j) const {
#pragma unroll
    for (int n = 0; n < NC; ++n) c.v[n][j] = *reinterpret_cast<const uint4*>(p[n] + 64 * j);
  }
  __device__ __forceinline__ void advance() {
#pragma unroll
    for (int n = 0; n < NC; ++n) p[n] += kTileK * 2;
  }
};

// A consumer warp's part of a unit of up to 4 NT rows, its sums left in `part` ([n][tiles 0 1, tiles 2 3][lane][tile, 8 i]:
// row 8 i + g of the tile, token 4n + t).
template <typename A, int G, int NT, bool UP, typename S, typename Wait>
__device__ __forceinline__ bool consume(const LayerArgs& a, Shared& s, S& st, const Unit& u, const Span& w, float* part,
                                        const Wait& free_part) {
  const int lane = threadIdx.x & 31, g = lane >> 2;
  const uint32_t magic = magic_register<A>();
  float acc[4][NT][2] = {};
  if (row_group(s, u, threadIdx.x / 32) < row_groups(a, u)) {
    Places<NT, !UP> at;
    at.at(UP ? a.x : a.h, UP ? a.H : a.I, w.k0, s, u.block);
    Columns<UP ? 1 : NT> x;
#pragma unroll
    for (int j = 0; j < 4; ++j) at.load(x, j);
    auto keep = [](int) {};
    // the last tile's product is followed word by word by the loads of the next K position's columns: no registers of
    // their own, and their latency passes under the next wait and the first tile
    auto reload = [&](int j) { at.load(x, j); };
#pragma unroll 1
    for (int left = w.steps; left > 0; --left) {
      if (left > 1) at.advance();  // the last one is read twice
      if (!st.ring.wait()) {
        s.abort = 1;
        return false;
      }
      const uint32_t slot = st.ring.slot(), words = slot + 16 * lane, scales = slot + 4 * g;
      tile_product<A, G, NT, !UP, 0>(words, scales, x, magic, acc[0], keep);
      tile_product<A, G, NT, !UP, tile_bytes(G)>(words, scales, x, magic, acc[1], keep);
      tile_product<A, G, NT, !UP, 2 * tile_bytes(G)>(words, scales, x, magic, acc[2], keep);
      tile_product<A, G, NT, !UP, 3 * tile_bytes(G)>(words, scales, x, magic, acc[3], reload);
      st.ring.release();
      st.fill(a, s);
    }
  }
  if (!free_part()) return false;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float4* p = reinterpret_cast<float4*>(part + n * 256 + lane * 4);
    p[0] = make_float4(acc[0][n][0], acc[0][n][1], acc[1][n][0], acc[1][n][1]);
    p[32] = make_float4(acc[2][n][0], acc[2][n][1], acc[3][n][0], acc[3][n][1]);
  }
  return true;
}

// The finishers: 8 values of a lane for token row 4n + t of row group `group`, summed over the K groups in order.
__device__ __forceinline__ void sum_parts(const float* part, int kw, int n, float (&v)[8]) {
  const float4* p = reinterpret_cast<const float4*>(part + n * 256 + (threadIdx.x & 31) * 4);
  float4 lo = p[0], hi = p[32];
#pragma unroll 4
  for (int k = 1; k < kw; ++k) {
    const float4 l = p[k * (kPart / 4)], h = p[k * (kPart / 4) + 32];
    lo = make_float4(lo.x + l.x, lo.y + l.y, lo.z + l.z, lo.w + l.w);
    hi = make_float4(hi.x + h.x, hi.y + h.y, hi.z + h.z, hi.w + h.w);
  }
  v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w;
  v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
}

// 32 columns of h: v holds the linear tiles, then the silu tiles.
__device__ __forceinline__ void finish_up(const LayerArgs& a, const Shared& s, uint32_t block, int n, uint32_t group,
                                          const float (&v)[8]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, r = 4 * n + t;
  if (r >= block_rows_of(block)) return;
  __nv_bfloat16* dst = a.h + (size_t)s.pairs[block_pos(block) + r] * 2 * a.I + group * kUpSpan + g;
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // columns 8 i + g
    const float h = swiglu(v[4 + i], v[i]);
    const bool finite = fabsf(h) <= FLT_MAX;
    const __nv_bfloat16 hi = __float2bfloat16_rn(finite ? fminf(fmaxf(h, -kMaxBf16), kMaxBf16) : h);
    dst[8 * i] = hi;
    dst[8 * i + a.I] = __float2bfloat16_rn(finite ? h - __bfloat162float(hi) : 0.0f);
  }
}

// 64 outputs of each pair, weighted.
__device__ __forceinline__ void finish_down(const LayerArgs& a, const Shared& s, uint32_t block, int n, uint32_t group,
                                            const float (&v)[8]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, r = 4 * n + t;
  if (r >= block_rows_of(block)) return;
  const int at = block_pos(block) + r;
  const float w = s.pair_w[at];
  float* dst = a.pair_out + (size_t)s.pairs[at] * a.H + group * kDownSpan + g;
#pragma unroll
  for (int i = 0; i < 8; ++i) dst[8 * i] = v[i] * w;
}

// Four outputs per thread: the sum of a token's local pairs in slot order.
template <typename A>
__device__ __forceinline__ void combine(const LayerArgs& a, uint32_t unit) {
  const long at = (long)unit * kCombine + 4 * threadIdx.x;
  if (at >= (long)a.T * a.H) return;
  const int t = (int)(at / a.H), n = (int)(at % a.H);
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
  for (int k = 0; k < kTopK; ++k) {
    const int e = a.topk_idx[t * kTopK + k] - a.offset;
    if (e >= 0 && e < a.E) {
      const float4 q = __ldcg(reinterpret_cast<const float4*>(a.pair_out + (size_t)(t * kTopK + k) * a.H + n));
      v = make_float4(v.x + q.x, v.y + q.y, v.z + q.z, v.w + q.w);
    }
  }
  typename A::Raw r[4] = {A::of(v.x), A::of(v.y), A::of(v.z), A::of(v.w)};
  *reinterpret_cast<uint2*>(reinterpret_cast<typename A::Raw*>(a.out) + at) = *reinterpret_cast<const uint2*>(r);
}

constexpr size_t kFixedSmem = (sizeof(Shared) + 127) / 128 * 128;

template <typename A, int G1, int G2>
__global__ void __launch_bounds__(kThreads, 1) layer_kernel(const __grid_constant__ LayerArgs a) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int kSlot = step_bytes(G1 < G2 ? G1 : G2);
  Shared& s = *reinterpret_cast<Shared*>(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x < kStreamWarps * kDepth) mbar_init(&s.ring_full[0][0] + threadIdx.x, 1);
  if (threadIdx.x == 0) {
    for (int i = 0; i < kQueue; ++i) {
      mbar_init(&s.known[i], 1);
      mbar_init(&s.go[i], 1);
      mbar_init(&s.done[i], kStreamWarps + kFinishers);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.part_full[i], kStreamWarps);
      mbar_init(&s.part_empty[i], kFinishers);
    }
    s.abort = 0;
  }
  fence_barrier_init();
  pdl_wait();
  fence_proxy_async_global();  // the weights, read by tensor copies, may be a kernel's of this stream
  pdl_trigger();
  build_lists(a, s);  // synchronises the CTA
  if (threadIdx.x < 2) {
    // Longer runs along K per warp where that still leaves four units per SM (T = 64, a quarter of the experts: 207 us with
    // the shorter ones, 195 with the longer), shorter ones otherwise (T = 33, H 2048, I 768: 61 us, 65.5 with the longer).
    const int* kw = threadIdx.x ? a.kw2 : a.kw1;
    const int groups = threadIdx.x ? a.H / kDownSpan : a.I / kUpSpan, mw = kStreamWarps / kw[1];
    (threadIdx.x ? s.kw2 : s.kw1) = s.n_blocks * ((groups + mw - 1) / mw) >= 4 * (int)gridDim.x ? kw[1] : kw[0];
  }
  __syncthreads();
  float* parts = reinterpret_cast<float*>(smem + kFixedSmem);
  constexpr int kParts = kStreamWarps * kPart;  // floats of a unit's partial sums
  volatile int* abort = &s.abort;
  // a wait that gives up, its own limit run out or another's, ends the role; the call is reported as failed
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    const bool ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, kWaitBudgetNs));
    if (!ok) *abort = 1;
    return ok;
  };

  if (warp >= kStreamWarps)
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kHelperRegs));
  else
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kConsumerRegs));
  if (warp >= kStreamWarps + kFinishers) {
    if (warp == kStreamWarps + kFinishers && lane == 0) {
      const uint32_t mw1 = kStreamWarps / s.kw1, mw2 = kStreamWarps / s.kw2;
      const uint32_t per_up = (a.I / kUpSpan + mw1 - 1) / mw1, per_down = (a.H / kDownSpan + mw2 - 1) / mw2;
      const uint32_t n_up = s.n_blocks * per_up, n_down = s.n_blocks * per_down;
      const uint32_t n_all = n_up + n_down + (uint32_t)(((long)a.T * a.H + kCombine - 1) / kCombine);
      auto wait_for = [&](const uint32_t* c, uint32_t need) {  // *c >= need: other CTAs' finishers bring it about
        const uint64_t t0 = globaltimer_ns();
        for (uint32_t it = 1; load_acquire(c) < need; ++it) {
          if (*abort) break;
          if ((it & 15u) == 0 && globaltimer_ns() - t0 > a.wait_ns) {
            *abort = 1;
            break;
          }
        }
      };
      int ready = -1;
      bool all_done = false;
      uint32_t next = atomicAdd(&a.counters->ticket, 1u);
      for (uint32_t seq = 0;; ++seq) {
        const uint32_t ticket = next;
        if (ticket < n_all) next = atomicAdd(&a.counters->ticket, 1u);  // under way while this one is queued
        const int slot = seq % kQueue;
        Unit u = {0, 0};
        if (ticket < n_up + n_down) {
          const bool up = ticket < n_up;
          const uint32_t at = up ? ticket : ticket - n_up, per = up ? per_up : per_down, b = at / per;
          const uint32_t block = s.block[b];
          u.block = block | (up ? kUp : kDown) << 28;
          u.row = at - b * per;
        } else if (ticket < n_all) {
          u.block = kSum << 28;
          u.row = ticket - n_up - n_down;
        }
        if (!mbar_wait(&s.done[slot], (seq / kQueue & 1) ^ 1, abort, kWaitBudgetNs)) {
          *abort = 1;
          break;
        }
        s.unit[slot] = u;
        mbar_arrive(&s.known[slot]);
        const int kind = kind_of(u), e = block_expert(u.block);
        if (kind == kDown && e != ready) {
          wait_for(&a.counters->ready[e], (uint32_t)((__popcll(s.mask[e]) + kRows - 1) / kRows) * per_up * kFinishers + a.extra);
          ready = e;
        }
        if (kind == kSum && !all_done) {
          wait_for(&a.counters->done, n_down * kFinishers + a.extra);
          all_done = true;
        }
        if (*abort) break;
        mbar_arrive(&s.go[slot]);
        if (kind == kStop) break;
      }
    }
  } else if (warp >= kStreamWarps) {
    uint32_t n = 0, downs = 0;  // units with sums so far; down units finished and not reported
    for (uint32_t seq = 0;; ++seq) {
      const int slot = seq % kQueue;
      if (!wait(&s.known[slot], seq / kQueue & 1)) break;
      const Unit u = s.unit[slot];
      const int kind = kind_of(u);
      if (kind == kUp || kind == kDown) {
        const int b = n & 1, kw = kind == kUp ? s.kw1 : s.kw2;
        const int tokens = block_rows_of(u.block) <= 4 ? 1 : 2, works = kStreamWarps / kw * tokens;
        if (!wait(&s.part_full[b], n / 2 & 1)) break;
        for (int i = warp - kStreamWarps; i < works; i += kFinishers) {
          const int mg = i / tokens, k = i % tokens;
          const uint32_t group = u.row * (kStreamWarps / kw) + mg;
          if (group >= row_groups(a, u)) break;
          float v[8];
          sum_parts(parts + b * kParts + mg * kw * kPart, kw, k, v);
          if (kind == kUp) finish_up(a, s, u.block, k, group, v);
          else finish_down(a, s, u.block, k, group, v);
        }
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&s.part_empty[b]);
          if (kind == kUp) add_release(&a.counters->ready[block_expert(u.block)], 1u);
        }
        downs += kind == kDown;
        ++n;
      } else if (downs > 0) {  // only now: each report waits for the stores before it
        if (lane == 0) add_release(&a.counters->done, downs);
        downs = 0;
      }
      if (kind == kStop) break;
      if (lane == 0) mbar_arrive(&s.done[slot]);
    }
  } else {
    const Span up = span_of(a, s, true), down = span_of(a, s, false);
    Stream<G1, G2> st;
    st.ring.init(smem_u32(parts + 2 * kParts) + warp * kDepth * kSlot, smem_u32(s.ring_full[warp]));
    st.left = 0;
    st.seq = 0;
    uint32_t n = 0;
    for (uint32_t seq = 0;; ++seq) {
      const int slot = seq % kQueue;
      if (!wait(&s.known[slot], seq / kQueue & 1)) break;
      st.fill(a, s);
      if (!wait(&s.go[slot], seq / kQueue & 1)) break;
      const Unit u = s.unit[slot];
      const int kind = kind_of(u);
      if (kind == kStop) break;
      if (kind == kSum) {
        combine<A>(a, u.row);
      } else {
        const int b = n & 1;
        const uint32_t parity = (n / 2 & 1) ^ 1;
        float* part = parts + b * kParts + warp * kPart;
        auto free_part = [&] { return wait(&s.part_empty[b], parity); };
        bool ok;
        if (kind == kUp) {
          if (block_rows_of(u.block) <= 4) ok = consume<A, G1, 1, true>(a, s, st, u, up, part, free_part);
          else ok = consume<A, G1, 2, true>(a, s, st, u, up, part, free_part);
        } else {
          if (block_rows_of(u.block) <= 4) ok = consume<Bf16, G2, 1, false>(a, s, st, u, down, part, free_part);
          else ok = consume<Bf16, G2, 2, false>(a, s, st, u, down, part, free_part);
        }
        if (!ok) break;
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.part_full[b]);
        ++n;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.done[slot]);
    }
    if (!st.ring.drain() && lane == 0) {
      s.abort = 1;
      atomicOr(&a.counters->status, kStatusTimeoutDrain);
    }
  }
  __syncthreads();
  if (s.abort) {
    if (threadIdx.x == 0) atomicOr(&a.counters->status, kStatusTimeoutEpilogue);
    // All outputs become NaN.  A CTA that combines after this found all units finished, and writes right values over it.
    typename A::Raw* out = reinterpret_cast<typename A::Raw*>(a.out);
    for (long i = threadIdx.x; i < (long)a.T * a.H; i += kThreads) out[i] = A::of(__uint_as_float(0x7FC00000u));
  }
  __syncthreads();
  if (threadIdx.x == 0) forward_status_to_sink(&a.counters->status, a.sink);
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
  uint32_t* sink;
  cudaStream_t stream;
};

constexpr int kSmemMax = 227 * 1024;

// Consumer warps along K: the largest power of two that leaves each `least` steps and whose rounds over K waste no more
// than one step in eight.
int k_groups(int k_tiles, int least) {
  for (int kw = kStreamWarps; kw > 1; kw /= 2)
    if (k_tiles >= least * kw && 8 * kw * ((k_tiles + kw - 1) / kw) <= 9 * k_tiles + 4) return kw;
  return 1;
}

// Packed matrices as a tensor [matrices][halves][row tiles][K positions x words], boxes [1][halves][rows][words].
bool map_weights(CUtensorMap* map, const uint8_t* base, int k_tiles, int words, int row_tiles, int halves, int matrices,
                 int rows) {
  const uint64_t row = (uint64_t)k_tiles * words * 8;
  const uint64_t dims[4] = {(uint64_t)k_tiles * words, (uint64_t)row_tiles, (uint64_t)halves, (uint64_t)matrices};
  const uint64_t strides[3] = {row, row * row_tiles, row * row_tiles * halves};
  const uint32_t box[4] = {(uint32_t)words, (uint32_t)rows, (uint32_t)halves, 1};
  return encode_4d_words(map, base, dims, strides, box) == FBMOE_OK;
}

template <typename A, int G1, int G2>
cudaError_t run_layer(const MoeArgs& m, const MoeLayout& L, int sms) {
  static DeviceFlags smem_set;
  constexpr int kSmem = (int)kFixedSmem + 2 * kStreamWarps * kPart * 4 + kStreamWarps * kDepth * step_bytes(G1 < G2 ? G1 : G2);
  static_assert(kSmem <= kSmemMax, "shared memory over the per-CTA limit");
  cudaError_t e = set_max_dynamic_smem(layer_kernel<A, G1, G2>, kSmem, smem_set);
  if (e != cudaSuccess) return e;
  alignas(64) LayerArgs a;
  if (!map_weights(&a.map1, m.w1, m.H / kTileK, tile_words(G1), m.I / kTileN, 2, m.E, 2) ||
      !map_weights(&a.map2, m.w2, m.I / kTileK, tile_words(G2), m.H / kTileN, 1, m.E, 4))
    return cudaErrorUnknown;
  a.T = m.T;
  a.H = m.H;
  a.I = m.I;
  a.E = m.E;
  a.offset = m.offset;
  for (int i = 0; i < 2; ++i) {
    a.kw1[i] = k_groups(m.H / kTileK, 2 + 2 * i);
    a.kw2[i] = k_groups(m.I / kTileK, 2 + 2 * i);
  }
  a.topk_idx = reinterpret_cast<const int32_t*>(m.ws + L.topk_idx);
  a.topk_w = reinterpret_cast<const float*>(m.ws + L.topk_w);
  a.x = m.x;
  a.h = reinterpret_cast<__nv_bfloat16*>(m.ws + L.h);
  a.pair_out = reinterpret_cast<float*>(m.ws + L.pair_out);
  a.counters = reinterpret_cast<Counters*>(m.ws + L.counters);
  a.out = m.out;
  a.sink = m.sink;
  const bool expire = test_expire_grid_wait();
  a.wait_ns = expire ? kTestGridWaitNs : kWaitBudgetNs;
  a.extra = expire ? 1u : 0u;
  return launch_pdl(layer_kernel<A, G1, G2>, dim3(sms), dim3(kThreads), kSmem, m.stream, a);
}
template <typename A, int G1>
cudaError_t pick_layer(const MoeArgs& m, const MoeLayout& L, int sms) {
  if (m.group2 == 32) return run_layer<A, G1, 32>(m, L, sms);
  if (m.group2 == 64) return run_layer<A, G1, 64>(m, L, sms);
  return run_layer<A, G1, 128>(m, L, sms);
}
template <typename A>
cudaError_t run_moe(const MoeArgs& m) {
  const MoeLayout L = moe_layout(m.T, m.H, m.I);
  cudaError_t e = launch_pdl(route_kernel, dim3(m.T), dim3(32), 0, m.stream, m.logits,
                             reinterpret_cast<const __nv_bfloat16*>(m.bias), m.scale,
                             reinterpret_cast<int32_t*>(m.ws + L.topk_idx), reinterpret_cast<float*>(m.ws + L.topk_w),
                             reinterpret_cast<Counters*>(m.ws + L.counters));
  if (e != cudaSuccess) return e;
  const int sms = num_sms_of_current_device();
  if (m.group1 == 32) return pick_layer<A, 32>(m, L, sms);
  if (m.group1 == 64) return pick_layer<A, 64>(m, L, sms);
  return pick_layer<A, 128>(m, L, sms);
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
                                          void* workspace, size_t workspace_bytes, uint32_t* status_sink, void* stream) {
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
  if (((uintptr_t)workspace & 255) || ((uintptr_t)status_sink & 3)) return FBMOE_ERR_MISALIGNED;
  if (workspace_bytes < w4::moe_layout(T, H, I).total) return FBMOE_ERR_WORKSPACE_TOO_SMALL;
  const w4::MoeArgs a = {routing_logits, routing_bias, hidden_states,
                         reinterpret_cast<const uint8_t*>(gemm1_weights), reinterpret_cast<const uint8_t*>(gemm2_weights),
                         group1, group2, T, H, I, E_local, local_expert_offset, routed_scaling_factor, out,
                         reinterpret_cast<uint8_t*>(workspace), status_sink, reinterpret_cast<cudaStream_t>(stream)};
  const cudaError_t e = type == FBMOE_BF16 ? w4::run_moe<w4::Bf16>(a) : w4::run_moe<w4::F16>(a);
  return e == cudaSuccess ? FBMOE_OK : (int)e;
}
