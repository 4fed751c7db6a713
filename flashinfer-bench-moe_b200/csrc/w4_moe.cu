// w4_moe.cu -- the whole MoE layer for a few tokens (T <= 64) on packed 4-bit weights, in two kernels.
//
//   route as fbmoe_route; h = silu(x Wg^T) * (x Wu^T) for every (token, local expert) pair; out = sum over a token's
//   pairs, in slot order, of weight * (h W2^T).
//
// W1's rows [0, I) are the linear half and [I, 2I) the silu half, as in fbmoe_forward.  x and h enter the products as
// 16-bit integers with a power-of-two scale per 128 (x) or 32 (h) columns (w4_stream.cuh).
//
// route_kernel: one CTA per token; a warp routes it, all make its planes; also zeroes the layer kernel's counters.
//
// layer_kernel: one CTA of 16 warps per SM.  Groups of P warps, P chosen so that there are about as many groups as
// tasks, work alone on tasks handed out by a ticket counter in the order
//   up: (up to 8 rows of an expert; 32 pairs of W1 rows, two linear and two silu tiles side by side),
//   down: (up to 8 rows of an expert; 32 rows of W2),
//   combine: 128 P outputs.
// A group's warps split K and join their partial sums in shared memory.  Each warp streams its part's tiles through its
// ring, and a group knows its tickets ahead of what it works on, so the stream does not stop between tasks or phases.  A
// down task needs its expert's up tasks, a combine task all down tasks.  Tickets are taken in order, so whatever a task
// waits for has been taken by a group that is running already and that waits for less: no co-residency is assumed, and
// two calls may share the GPU.  Every order of summation depends on the sizes and the numbers of row blocks alone.
#include "fbmoe.h"
#include "fbmoe_launch.h"
#include "moe_route.cuh"
#include "w4_stream.cuh"

namespace fbmoe {
namespace w4 {
namespace {

constexpr int kRows = 8;                    // token rows of a task
constexpr int kSpan = 2 * kTileN;           // rows of h that an up task makes, and of W2 that a down task takes
constexpr int kThreads = kStreamWarps * 32;
constexpr int kCombine = 128;               // outputs of a combine task
constexpr int kMaxBlocks = kMaxTokens * kTopK / kRows + kExperts;  // row blocks of all experts
constexpr int kPart = 256;                  // floats of a warp's partial sums that are joined at a time

// counters in the workspace, zeroed by route_kernel
struct Counters {
  uint32_t status, ticket, done, pad;
  uint32_t ready[kExperts];  // finished up tasks of each local expert
};

struct MoeLayout {
  size_t counters, topk_idx, topk_w, xq, xs, hq, hs, pair_out, total;
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
  L.xq = take((size_t)T * H * 2);                // planes of x
  L.xs = take((size_t)T * (H / kTileK) * 4);     // their scales / 16
  L.hq = take((size_t)T * kTopK * I * 2);        // planes of h, by pair
  L.hs = take((size_t)T * kTopK * (I / 32) * 4);
  L.pair_out = take((size_t)T * kTopK * H * 4);    // [pair][H] fp32
  L.total = off;
  return L;
}

constexpr int kRouteThreads = 256;

template <typename A>
__device__ __forceinline__ float widen(typename A::Raw v) {
  if constexpr (sizeof(A) == sizeof(Bf16) && A::kMagic == Bf16::kMagic) return __bfloat162float(v);
  else return __half2float(v);
}

// Four consecutive values of a lane, 128 of a warp: their planes at the K position `dst`, their scale / 16 returned.
__device__ __forceinline__ float make_planes(const float (&v)[4], uint8_t* dst) {
  const int lane = threadIdx.x & 31;
  float m = 0.0f;
  bool bad = false;  // a NaN or an infinity
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m = fmaxf(m, fabsf(v[i]));
    bad |= !(fabsf(v[i]) <= 3.402823466e38f);
  }
  if (bad) m = INFINITY;
#pragma unroll
  for (int d = 16; d >= 1; d /= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  const bool finite = m <= 3.402823466e38f;
  const int e = plane_exponent(m);
  uint32_t hi = 0, lo = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int k = finite ? plane_int(v[i], e) : 0;
    hi |= (uint32_t)((k + 128) >> 8 & 0xff) << (8 * i);
    lo |= (uint32_t)(k & 0xff) << (8 * i);
  }
  // an even lane holds elements 0..3 of an eight, the odd one next to it 4..7: bytes 0 4 1 5 | 2 6 3 7
  const uint32_t ohi = __shfl_xor_sync(0xffffffffu, hi, 1), olo = __shfl_xor_sync(0xffffffffu, lo, 1);
  const uint32_t order = lane & 1 ? 0x3726u : 0x5140u;
  uint8_t* at = dst + (lane / 2 % 4) * 32 + (lane / 8) * 8 + (lane & 1) * 4;
  *reinterpret_cast<uint32_t*>(at) = __byte_perm(hi, ohi, order);
  *reinterpret_cast<uint32_t*>(at + 128) = __byte_perm(lo, olo, order);
  return finite ? exp2_int(e) * 0.0625f : NAN;
}

template <typename A>
__global__ void __launch_bounds__(kRouteThreads) route_kernel(const float* __restrict__ logits,
                                                              const __nv_bfloat16* __restrict__ bias, float scale,
                                                              const typename A::Raw* __restrict__ x, int H,
                                                              int32_t* __restrict__ topk_idx, float* __restrict__ topk_w,
                                                              uint8_t* __restrict__ xq, float* __restrict__ xs,
                                                              Counters* __restrict__ counters) {
  __shared__ float wv[kExperts], ws[kExperts];
  __shared__ int wi[kExperts], sel[kTopK];
  const int t = blockIdx.x, warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_trigger();
  for (int i = t * kRouteThreads + threadIdx.x; i < (int)(sizeof(Counters) / 4); i += gridDim.x * kRouteThreads)
    reinterpret_cast<uint32_t*>(counters)[i] = 0;
  if (warp == 0) {
    float l[8], b[8];
    route_dev::load_logits8(logits, t, l);
    route_dev::load_bias8(bias, b);
    route_dev::route_token(l, t, b, scale, topk_idx, topk_w, wv, wi, ws, sel);
    return;
  }
  const int kt_n = H / kTileK;
  for (int kt = warp - 1; kt < kt_n; kt += kRouteThreads / 32 - 1) {
    const uint2 r = *reinterpret_cast<const uint2*>(x + (size_t)t * H + kt * kTileK + 4 * lane);
    const typename A::Raw* p = reinterpret_cast<const typename A::Raw*>(&r);
    const float v[4] = {widen<A>(p[0]), widen<A>(p[1]), widen<A>(p[2]), widen<A>(p[3])};
    const float sc = make_planes(v, xq + ((size_t)t * kt_n + kt) * kPlaneTile);
    if (lane == 0) xs[(size_t)t * kt_n + kt] = sc;
  }
}

struct LayerArgs {
  const uint8_t *w1, *w2;
  int T, H, I, E, offset;
  int depth;             // steps of a ring
  const int32_t* topk_idx;
  const float* topk_w;
  const uint8_t* xq;
  const float* xs;
  uint8_t* hq;
  float *hs, *pair_out;
  Counters* counters;
  void* out;
  uint32_t* sink;
  uint64_t wait_ns;      // limit of a wait for other warps' tasks
  uint32_t extra;        // arrivals that never come (test hook)
};

// A row block: local expert, its first pair's place in the pair list, its rows.
__device__ __forceinline__ uint32_t block_word(int e, int pos, int rows) { return e | pos << 8 | rows << 20; }
__device__ __forceinline__ int block_expert(uint32_t w) { return w & 0xff; }
__device__ __forceinline__ int block_pos(uint32_t w) { return w >> 8 & 0xfff; }
__device__ __forceinline__ int block_rows_of(uint32_t w) { return w >> 20; }

// The tasks of a call.
struct Plan {
  int log_p;               // log2 of the warps of a group
  uint32_t up_rows, n_up;  // row positions per row block, tasks
  uint32_t down_rows, n_down;
  uint32_t n_all;
};

struct Shared {
  unsigned long long mask[kExperts];  // tokens of each local expert
  uint64_t ring_full[kStreamWarps][kMaxDepth];
  uint32_t tickets[kStreamWarps][4];   // a group's tasks: the one it works on, the next, and the one after that
  float part[kStreamWarps][kPart];
  uint32_t block[kMaxBlocks];
  uint32_t warp_sum[8];
  uint16_t pair_at[kExperts];          // first place of an expert's pairs
  uint16_t pairs[kMaxTokens * kTopK];  // token * 8 + slot, by expert, tokens ascending
  int n_blocks;                        // row blocks
  Plan plan;
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
  if (e >= 0) s.pairs[s.pair_at[e] + __popcll(s.mask[e] & ((1ull << (tid / kTopK)) - 1))] = (uint16_t)tid;
  __syncthreads();
}

// P doubles while that leaves no more groups than tasks of the smaller phase, and every warp a K position.
__device__ __forceinline__ Plan make_plan(const LayerArgs& a, const Shared& s) {
  Plan p;
  p.up_rows = a.I / kSpan;
  p.n_up = s.n_blocks * p.up_rows;
  p.down_rows = a.H / kSpan;
  p.n_down = s.n_blocks * p.down_rows;
  const uint32_t tasks = min(p.n_up, p.n_down), warps = gridDim.x * kStreamWarps;
  const int k_tiles = min(a.H, a.I) / kTileK;
  p.log_p = 0;
  while (p.log_p < 4 && tasks << (p.log_p + 1) <= warps && k_tiles >> (p.log_p + 1) > 0) ++p.log_p;
  p.n_all = p.n_up + p.n_down + (uint32_t)(((long)a.T * a.H + (kCombine << p.log_p) - 1) / (kCombine << p.log_p));
  return p;
}

// A warp's part of a task.
struct Task {
  uint32_t block;    // row block
  int row, k0, tiles;
  const uint8_t* tile;
};
template <int G1, int G2>
__device__ __noinline__ Task decode_task(const LayerArgs& a, const Shared& s, uint32_t ticket) {
  const Plan& p = s.plan;
  Task t;
  const bool up = ticket < p.n_up;
  const uint32_t rows = up ? p.up_rows : p.down_rows, at = up ? ticket : ticket - p.n_up, b = at / rows;
  t.row = at - b * rows;
  t.block = s.block[b];
  const int kt = (up ? a.H : a.I) / kTileK, part = threadIdx.x / 32 & ((1 << p.log_p) - 1);
  t.k0 = kt * part >> p.log_p;
  t.tiles = (kt * (part + 1) >> p.log_p) - t.k0;
  const size_t e = block_expert(t.block);
  const size_t first = e * ((up ? 2 * a.I : a.H) / kTileN) + 2 * t.row;  // row tile
  t.tile = (up ? a.w1 : a.w2) + (first * kt + t.k0) * (up ? tile_bytes(G1) : tile_bytes(G2));
  return t;
}

// A warp's stream: the copies of its tasks' tiles, ahead of what it works on.  An up step is one K position of four row
// tiles, a down step two K positions of two; lane i < copies holds the place of copy i.
template <int G1, int G2>
struct Stream {
  Ring ring;
  const uint8_t* src;
  int left;              // steps of the task being issued that are still to be issued
  int copies;
  uint32_t bytes, last;  // of a copy, and of the task's last step
  uint32_t task, known;  // tasks begun, and tasks whose tickets are known

  // Issue the next steps while the ring has room.
  __device__ __forceinline__ void fill(const LayerArgs& a, Shared& s) {
    if (left > 1 && ring.free == 1) {  // the usual case: the step just released
      ring.issue(src, copies, bytes, bytes);
      src += bytes;
      --left;
      return;
    }
    fill_slow(a, s);
  }
  __device__ __forceinline__ void fill_slow(const LayerArgs& a, Shared& s) {
    while (ring.free > 0) {
      if (left == 0) {
        if (task == known) return;
        const uint32_t t = s.tickets[threadIdx.x / 32 >> s.plan.log_p][task % 4];
        if (t >= s.plan.n_up + s.plan.n_down) return;  // no tiles from here on
        ++task;
        const Task k = decode_task<G1, G2>(a, s, t);
        const int lane = threadIdx.x & 31;
        if (t < s.plan.n_up) {
          const size_t row = (size_t)(a.H / kTileK) * tile_bytes(G1);  // bytes of a row tile
          src = k.tile + (lane & 1) * row + (lane >> 1 & 1) * (a.I / kTileN) * row;
          copies = 4;
          left = k.tiles;
          bytes = last = tile_bytes(G1);
        } else {
          src = k.tile + (lane & 1) * (size_t)(a.I / kTileK) * tile_bytes(G2);
          copies = 2;
          left = (k.tiles + 1) / 2;
          bytes = 2 * tile_bytes(G2);
          last = k.tiles & 1 ? tile_bytes(G2) : bytes;
        }
      }
      ring.issue(src, copies, left == 1 ? last : bytes, bytes);
      src += bytes;
      --left;
    }
  }
};

__device__ __forceinline__ void group_sync(int log_p) {
  if (log_p == 0)
    __syncwarp();
  else
    named_barrier_sync(1 + (threadIdx.x / 32 >> log_p), 32 << log_p);
}

__device__ __forceinline__ float swiglu(float gate, float up) { return gate / (1.0f + expf(-gate)) * up; }

// The sums of a group's partial values, in order, for its first warp (true).
__device__ __forceinline__ bool join(Shared& s, int log_p, float (&v)[8]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  if (log_p == 0) return true;
  group_sync(log_p);  // the first warp has read what the last call left
#pragma unroll
  for (int i = 0; i < 8; ++i) s.part[warp][32 * i + lane] = v[i];
  group_sync(log_p);
  if (warp & ((1 << log_p) - 1)) return false;
  for (int w = 1; w < 1 << log_p; ++w)
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += s.part[warp + w][32 * i + lane];
  return true;
}

// The lane's places in the planes and scales of up to 4 NT tokens of a task (rows that are not there read the first
// one's: their sums are not used), from K position k0 on.
template <int NT, bool FINE>
struct Places {
  const uint8_t* q[NT];
  const float* s[NT];

  __device__ __forceinline__ void at(const uint8_t* planes, const float* scales, int kt_n, int k0, const Shared& s_,
                                     uint32_t block, bool by_pair) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int pos = block_pos(block), rows = block_rows_of(block);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int rq = 4 * n + (g >> 1), rs = 4 * n + t;
      int pq = s_.pairs[pos + (rq < rows ? rq : 0)], ps = s_.pairs[pos + (rs < rows ? rs : 0)];
      if (!by_pair) {
        pq /= kTopK;
        ps /= kTopK;
      }
      q[n] = planes + ((size_t)pq * kt_n + k0) * kPlaneTile + (g & 1) * 128 + t * 32;
      s[n] = scales + ((size_t)ps * kt_n + k0) * (FINE ? 4 : 1);
    }
  }
  // The columns of the current K position.  x is constant while the kernel runs, h is not.
  __device__ __forceinline__ void load(Columns<NT, FINE>& c) const {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const uint4* p = reinterpret_cast<const uint4*>(q[n]);
      const uint4 u = FINE ? p[0] : __ldg(p), v = FINE ? p[1] : __ldg(p + 1);
      c.b[n][0] = make_uint2(u.x, u.y);
      c.b[n][1] = make_uint2(u.z, u.w);
      c.b[n][2] = make_uint2(v.x, v.y);
      c.b[n][3] = make_uint2(v.z, v.w);
      if constexpr (FINE) {
        const float4 f = *reinterpret_cast<const float4*>(s[n]);
        c.s[n][0] = f.x;
        c.s[n][1] = f.y;
        c.s[n][2] = f.z;
        c.s[n][3] = f.w;
      } else {
        c.s[n][0] = __ldg(s[n]);
      }
    }
  }
  __device__ __forceinline__ void advance() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      q[n] += kPlaneTile;
      s[n] += FINE ? 4 : 1;
    }
  }
};

// An up task of up to 4 NT rows: 32 columns of h and their planes.
template <int G, int NT, typename S>
__device__ __forceinline__ void up_task(const LayerArgs& a, Shared& s, S& st, const Task& k) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, log_p = s.plan.log_p;
  const uint32_t flip = flip_register();
  Places<NT, false> at;
  at.at(a.xq, a.xs, a.H / kTileK, k.k0, s, k.block, false);
  Columns<NT, false> x, ahead;  // one K position ahead: from the L2 they take longer than a step's products
  at.load(ahead);
  float acc[4][NT][2] = {};
#pragma unroll 1
  for (int left = k.tiles; left > 0; --left) {
    x = ahead;
    if (left > 1) at.advance();  // the last one is read twice
    at.load(ahead);
    st.ring.wait(&s.abort);
    const uint32_t words = st.ring.got + 16 * lane, scales = st.ring.got + 4 * g;
    tile_product<G, NT, false, 0>(words, scales, x, flip, acc[0]);
    tile_product<G, NT, false, tile_bytes(G)>(words, scales, x, flip, acc[1]);
    tile_product<G, NT, false, 2 * tile_bytes(G)>(words, scales, x, flip, acc[2]);
    tile_product<G, NT, false, 3 * tile_bytes(G)>(words, scales, x, flip, acc[3]);
    st.ring.release();
    st.fill(a, s);
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    // linear tiles, silu tiles: [tile][8 i + g] of token 4n + t
    float v[8] = {acc[0][n][0], acc[0][n][1], acc[1][n][0], acc[1][n][1],
                  acc[2][n][0], acc[2][n][1], acc[3][n][0], acc[3][n][1]};
    if (!join(s, log_p, v)) continue;
    float h[4], m = 0.0f;  // columns 8 i + g of the task's 32
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      h[i] = swiglu(v[4 + i], v[i]);
      m = fmaxf(m, fabsf(h[i]));
      bad |= !(fabsf(h[i]) <= 3.402823466e38f);
    }
    if (bad) m = INFINITY;
#pragma unroll
    for (int d = 16; d >= 4; d /= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    const bool finite = m <= 3.402823466e38f;
    const int e = plane_exponent(m), r = 4 * n + t;
    if (r < block_rows_of(k.block)) {
      const size_t pair = s.pairs[block_pos(k.block) + r];
      // column 8 i + g of these 32: eight i, element g, which is byte g / 4 + g % 4 * 2 of its eight
      uint8_t* dst = a.hq + (pair * (a.I / kTileK) + k.row / 4) * kPlaneTile + k.row % 4 * 8 + (g >> 2) + (g & 3) * 2;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int q = finite ? plane_int(h[i], e) : 0;
        dst[32 * i] = (uint8_t)((q + 128) >> 8);
        dst[32 * i + 128] = (uint8_t)q;
      }
      if (g == 0) a.hs[pair * (a.I / 32) + k.row] = finite ? exp2_int(e) * 0.0625f : NAN;
    }
  }
}

// A down task of up to 4 NT rows: 32 outputs of each pair, weighted.
template <int G, int NT, typename S>
__device__ __forceinline__ void down_task(const LayerArgs& a, Shared& s, S& st, const Task& k) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, log_p = s.plan.log_p;
  const uint32_t flip = flip_register();
  Places<NT, true> at;
  at.at(a.hq, a.hs, a.I / kTileK, k.k0, s, k.block, true);
  Columns<NT, true> x, ahead;
  at.load(ahead);
  float acc[2][NT][2] = {};
  uint32_t slot = 0;
#pragma unroll 1
  for (int i = 0; i < k.tiles; ++i) {
    x = ahead;
    if (i + 1 < k.tiles) at.advance();
    at.load(ahead);
    if (i % 2 == 0) {
      st.ring.wait(&s.abort);
      slot = st.ring.got;
    } else {
      slot += tile_bytes(G);
    }
    const uint32_t words = slot + 16 * lane, scales = slot + 4 * g;
    tile_product<G, NT, true, 0>(words, scales, x, flip, acc[0]);
    tile_product<G, NT, true, 2 * tile_bytes(G)>(words, scales, x, flip, acc[1]);
    if (i % 2 == 1 || i + 1 == k.tiles) {
      st.ring.release();
      st.fill(a, s);
    }
  }
  // [tile][8 i + g] of tokens 4n + t
  float v[8] = {acc[0][0][0], acc[0][0][1], acc[1][0][0], acc[1][0][1],
                acc[0][NT - 1][0], acc[0][NT - 1][1], acc[1][NT - 1][0], acc[1][NT - 1][1]};
  if (!join(s, log_p, v)) return;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = 4 * n + t;
    if (r < block_rows_of(k.block)) {
      const int pair = s.pairs[block_pos(k.block) + r];
      const float w = a.topk_w[pair];
      float* dst = a.pair_out + (size_t)pair * a.H + k.row * kSpan + g;
#pragma unroll
      for (int i = 0; i < 4; ++i) dst[8 * i] = v[4 * n + i] * w;
    }
  }
}

// Four outputs per lane: the sum of a token's local pairs in slot order.
template <typename A>
__device__ __forceinline__ void combine(const LayerArgs& a, uint32_t task) {
  const long at = (long)task * kCombine + 4 * (threadIdx.x & 31);
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
  if (threadIdx.x < kStreamWarps * kMaxDepth) mbar_init(&s.ring_full[0][0] + threadIdx.x, 1);
  if (threadIdx.x == 0) s.abort = 0;
  fence_barrier_init();
  pdl_wait();
  pdl_trigger();
  build_lists(a, s);  // synchronises the CTA
  if (threadIdx.x == 0) {
    const Plan p = make_plan(a, s);
    s.plan = p;
    const int groups = kStreamWarps >> p.log_p;
    const uint32_t base = atomicAdd(&a.counters->ticket, (uint32_t)groups);
    for (int i = 0; i < groups; ++i) s.tickets[i][0] = base + i;
  }
  __syncthreads();
  const int log_p = s.plan.log_p, group = warp >> log_p;
  const bool leads = (warp & ((1 << log_p) - 1)) == 0 && lane == 0;  // takes the group's tickets, reports its work
  Stream<G1, G2> st;
  st.ring.init(smem_u32(smem + kFixedSmem) + warp * a.depth * kSlot, smem_u32(s.ring_full[warp]), kSlot, a.depth);
  st.left = 0;
  st.task = 0;
  st.known = 1;
  st.fill_slow(a, s);
  if (threadIdx.x == 0) {  // the groups' second tickets, while the first tiles are on their way
    const int groups = kStreamWarps >> log_p;
    const uint32_t base = atomicAdd(&a.counters->ticket, (uint32_t)groups);
    for (int i = 0; i < groups; ++i) s.tickets[i][1] = base + i;
  }
  __syncthreads();
  st.known = 2;
  st.fill_slow(a, s);
  int ready = -1;
  bool all_done = false;
  // lane 0 waits for *c >= need, the warp follows
  auto wait_for = [&](const uint32_t* c, uint32_t need) {
    if (lane == 0 && load_acquire(c) < need) {
      const uint64_t t0 = globaltimer_ns();
      for (uint32_t it = 1; load_acquire(c) < need; ++it) {
        if (*(volatile int*)&s.abort) break;
        if ((it & 15u) == 0 && globaltimer_ns() - t0 > a.wait_ns) {
          *(volatile int*)&s.abort = 1;
          break;
        }
      }
    }
    __syncwarp();
  };
  for (uint32_t n = 0;; ++n) {
    const uint32_t ticket = s.tickets[group][n % 4];
    if (ticket >= s.plan.n_all) break;
    uint32_t next = 0;
    if (leads) next = atomicAdd(&a.counters->ticket, 1u);  // under way while the task runs
    uint32_t* report = nullptr;
    if (ticket < s.plan.n_up) {
      const Task k = decode_task<G1, G2>(a, s, ticket);
      report = &a.counters->ready[block_expert(k.block)];
      if (block_rows_of(k.block) <= 4) up_task<G1, 1>(a, s, st, k);
      else up_task<G1, 2>(a, s, st, k);
    } else if (ticket < s.plan.n_up + s.plan.n_down) {
      const Task k = decode_task<G1, G2>(a, s, ticket);
      const int e = block_expert(k.block);
      if (e != ready)
        wait_for(&a.counters->ready[e], (uint32_t)((__popcll(s.mask[e]) + kRows - 1) / kRows) * s.plan.up_rows + a.extra);
      ready = e;
      report = &a.counters->done;
      if (block_rows_of(k.block) <= 4) down_task<G2, 1>(a, s, st, k);
      else down_task<G2, 2>(a, s, st, k);
    } else {
      if (!all_done) wait_for(&a.counters->done, s.plan.n_down + a.extra);
      all_done = true;
      combine<A>(a, ((ticket - s.plan.n_up - s.plan.n_down) << log_p) + (warp & ((1 << log_p) - 1)));
    }
    if (leads) s.tickets[group][(n + 2) % 4] = next;
    group_sync(log_p);
    st.known = n + 3;
    if (leads && report) add_release(report, 1u);  // the first warp's stores are all the task's
    st.fill_slow(a, s);
  }
  const bool drained = st.ring.drain();
  __syncthreads();
  if (lane == 0 && !drained) atomicOr(&a.counters->status, kStatusTimeoutDrain);
  if (threadIdx.x == 0 && s.abort) atomicOr(&a.counters->status, kStatusTimeoutEpilogue);
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

template <typename A, int G1, int G2>
cudaError_t run_layer(const MoeArgs& m, const MoeLayout& L, int sms) {
  static DeviceFlags smem_set;
  cudaError_t e = set_max_dynamic_smem(layer_kernel<A, G1, G2>, kSmemMax, smem_set);
  if (e != cudaSuccess) return e;
  LayerArgs a;
  a.w1 = m.w1;
  a.w2 = m.w2;
  a.T = m.T;
  a.H = m.H;
  a.I = m.I;
  a.E = m.E;
  a.offset = m.offset;
  constexpr int kSlot = step_bytes(G1 < G2 ? G1 : G2);
  a.depth = (kSmemMax - (int)kFixedSmem) / (kStreamWarps * kSlot);
  if (a.depth > kMaxDepth) a.depth = kMaxDepth;
  a.topk_idx = reinterpret_cast<const int32_t*>(m.ws + L.topk_idx);
  a.topk_w = reinterpret_cast<const float*>(m.ws + L.topk_w);
  a.xq = m.ws + L.xq;
  a.xs = reinterpret_cast<const float*>(m.ws + L.xs);
  a.hq = m.ws + L.hq;
  a.hs = reinterpret_cast<float*>(m.ws + L.hs);
  a.pair_out = reinterpret_cast<float*>(m.ws + L.pair_out);
  a.counters = reinterpret_cast<Counters*>(m.ws + L.counters);
  a.out = m.out;
  a.sink = m.sink;
  const bool expire = test_expire_grid_wait();
  a.wait_ns = expire ? kTestGridWaitNs : kWaitBudgetNs;
  a.extra = expire ? 1u : 0u;
  return launch_pdl(layer_kernel<A, G1, G2>, dim3(sms), dim3(kThreads), kFixedSmem + (size_t)a.depth * kStreamWarps * kSlot,
                    m.stream, a);
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
  cudaError_t e = launch_pdl(route_kernel<A>, dim3(m.T), dim3(kRouteThreads), 0, m.stream, m.logits,
                             reinterpret_cast<const __nv_bfloat16*>(m.bias), m.scale,
                             reinterpret_cast<const typename A::Raw*>(m.x), m.H,
                             reinterpret_cast<int32_t*>(m.ws + L.topk_idx), reinterpret_cast<float*>(m.ws + L.topk_w), m.ws + L.xq,
                             reinterpret_cast<float*>(m.ws + L.xs), reinterpret_cast<Counters*>(m.ws + L.counters));
  if (e != cudaSuccess) return e;
  int dev = 0, sms = 0;
  e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return e;
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
