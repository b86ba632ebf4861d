// The mixture-of-experts block that runs between the attention layers
// (qwen36_chat_batch.py:127-178 `batched_moe_step`, qwen36_router.py:96 `route`).
//
//   moe_route_kernel    router logits -> each token's experts and weights
//   moe_plan_kernel     (token, slot) pairs sorted by expert, cut into tiles
//   x8_tile_kernel      an expert's gate and up rows with SwiGLU, its down rows
//   moe_combine_kernel  the sum over a token's slots
//
//     (g | u) = W13[e] Q(x_t)      Q: e4m3, a power-of-two scale per 128 values
//     y_t     = sum_j w[t, j] W2[e_j] Q(SiLU(g) u)
#include <algorithm>

#include "x8_tile.h"

namespace ria {

// ----------------------------------------------------------------------------- routing
constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxK = 32;
constexpr int kRouteMaxGroups = 64;
constexpr int kRouteWaves = 4;

struct RouteArgs {
  const void* logits;
  int64_t stride;
  int tokens, experts, top_k;
  const float* bias;
  int sigmoid, groups, top_groups, top2, renorm, shared;
  float scale;
  float* weights;
  int64_t w_stride;
  int32_t* ids;
  int64_t id_stride;
};

// Integers in the order of doubles: -inf lowest, NaN above every number.
__device__ __forceinline__ int64_t order_key(double v) {
  if (v != v) return INT64_MAX;
  const int64_t b = __double_as_longlong(v == 0.0 ? 0.0 : v);  // -0 ranks as 0
  return b >= 0 ? b : INT64_MIN + 1 + ~b;
}

__device__ __forceinline__ int64_t shfl_xor64(int64_t v, int m) {
  const int lo = __shfl_xor(static_cast<int>(v), m), hi = __shfl_xor(static_cast<int>(v >> 32), m);
  return (static_cast<int64_t>(hi) << 32) | static_cast<uint32_t>(lo);
}
__device__ __forceinline__ double shfl_xor_f64(double v, int m) {
  return __longlong_as_double(shfl_xor64(__double_as_longlong(v), m));
}

// One wave per token, lane l holding experts l, l + 64, ..  Choices are compared
// in 64 bits: a bias brings scores of unlike experts within a rounding of each
// other, and the ids have to be the formula's.  Without a bias (and without
// groups ranked by sums) the logits themselves are compared: scores grow with them.
template <int XT, int V>
__global__ __launch_bounds__(64 * kRouteWaves) void moe_route_kernel(const RouteArgs a) {
  __shared__ double choice_s[kRouteWaves][64 * V];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t t = (int64_t)blockIdx.x * kRouteWaves + wave;
  if (t >= a.tokens) return;
  const int e = a.experts;
  const double ninf = -__builtin_inf();
  double x[V], c[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int i = v * 64 + lane;
    x[v] = i < e ? static_cast<double>(load_act<XT>(a.logits, t * a.stride + i)) : ninf;
  }
  double top = ninf, total = 0.0;
  if (!a.sigmoid) {  // the softmax's largest logit and normaliser
#pragma unroll
    for (int v = 0; v < V; ++v) top = x[v] > top || x[v] != x[v] ? x[v] : top;
#pragma unroll
    for (int m = 32; m; m >>= 1) {
      const double o = shfl_xor_f64(top, m);
      top = o > top || o != o ? o : top;
    }
    const double base = top == ninf ? 0.0 : top;
    top = base;
#pragma unroll
    for (int v = 0; v < V; ++v) total += exp(x[v] - base);
#pragma unroll
    for (int m = 32; m; m >>= 1) total += shfl_xor_f64(total, m);
    if (total == 0.0) total = 1.0;
  }
  auto score = [&](double l) { return a.sigmoid ? 1.0 / (1.0 + exp(-l)) : exp(l - top) / total; };
  const bool by_score = a.bias || (a.groups > 1 && a.top2);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int i = v * 64 + lane;
    c[v] = x[v];
    if (by_score && i < e && x[v] != ninf) c[v] = score(x[v]) + (a.bias ? static_cast<double>(a.bias[i]) : 0.0);
  }
  if (a.groups > 1) {
    double* s = choice_s[wave];
#pragma unroll
    for (int v = 0; v < V; ++v) s[v * 64 + lane] = c[v];
    __builtin_amdgcn_wave_barrier();
    const int per = e / a.groups;
    int64_t g = INT64_MIN;
    if (lane < a.groups) {
      double b0 = ninf, b1 = ninf;  // the group's best two
      for (int i = 0; i < per; ++i) {
        const double v = s[lane * per + i];
        if (order_key(v) > order_key(b0)) {
          b1 = b0;
          b0 = v;
        } else if (order_key(v) > order_key(b1)) {
          b1 = v;
        }
      }
      g = order_key(a.top2 && per > 1 ? b0 + b1 : b0);
    }
    int better = 0;  // groups that come before this one
    for (int j = 0; j < a.groups; ++j) {
      const int lo = __shfl(static_cast<int>(g), j), hi = __shfl(static_cast<int>(g >> 32), j);
      const int64_t o = (static_cast<int64_t>(hi) << 32) | static_cast<uint32_t>(lo);
      better += o > g || (o == g && j < lane);
    }
    const uint64_t open = __ballot(lane < a.groups && better < a.top_groups);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int i = v * 64 + lane;
      if (i < e && !(open >> (i / per) & 1)) c[v] = ninf;
    }
  }
  // top_k times the best that is left; ties go to the lowest index
  int64_t key[V];
#pragma unroll
  for (int v = 0; v < V; ++v) key[v] = v * 64 + lane < e ? order_key(c[v]) : INT64_MIN;
  const int64_t none = order_key(ninf);
  int my_id = -1;
  double my_x = ninf;
  for (int j = 0; j < a.top_k; ++j) {
    int64_t best = INT64_MIN;
    int at = 0x7fffffff;
    double bx = ninf;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (key[v] > best) {  // lower indexes first
        best = key[v];
        at = v * 64 + lane;
        bx = x[v];
      }
#pragma unroll
    for (int m = 32; m; m >>= 1) {
      const int64_t o = shfl_xor64(best, m);
      const int oi = __shfl_xor(at, m);
      const double ox = shfl_xor_f64(bx, m);
      if (o > best || (o == best && oi < at)) {
        best = o;
        at = oi;
        bx = ox;
      }
    }
    if (lane == j && best > none) {
      my_id = at;
      my_x = bx;
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v * 64 + lane == at) key[v] = INT64_MIN;
  }
  // weights of the chosen (lanes 0 .. top_k - 1)
  double w = 0.0;
  if (my_id >= 0) w = score(my_x);
  if (a.renorm) {
    // softmax: about the largest chosen logit, so that the weights hold where the row's largest was not chosen
    if (!a.sigmoid) {
      double m0 = my_x;
#pragma unroll
      for (int m = 32; m; m >>= 1) {
        const double o = shfl_xor_f64(m0, m);
        m0 = o > m0 || o != o ? o : m0;
      }
      if (my_id >= 0) w = exp(my_x - m0) * (total != total ? total : 1.0);
    }
    double sum = w;
#pragma unroll
    for (int m = 32; m; m >>= 1) sum += shfl_xor_f64(sum, m);
    if (sum != 0.0) w /= sum;
  }
  if (lane < a.top_k) {
    a.weights[t * a.w_stride + lane] = static_cast<float>(w * static_cast<double>(a.scale));
    a.ids[t * a.id_stride + lane] = my_id;
  }
  if (a.shared && lane == 0) {
    const double l = static_cast<double>(load_act<XT>(a.logits, t * a.stride + e));
    a.weights[t * a.w_stride + a.top_k] = static_cast<float>(1.0 / (1.0 + exp(-l)));
    a.ids[t * a.id_stride + a.top_k] = l == ninf ? -1 : e;
  }
}

template <int XT>
static void launch_route(const RouteArgs& a, hipStream_t st) {
  const dim3 grid((a.tokens + kRouteWaves - 1) / kRouteWaves), block(64 * kRouteWaves);
  const int v = (a.experts + 63) / 64;
  if (v <= 1)
    hipLaunchKernelGGL((moe_route_kernel<XT, 1>), grid, block, 0, st, a);
  else if (v <= 4)
    hipLaunchKernelGGL((moe_route_kernel<XT, 4>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((moe_route_kernel<XT, 16>), grid, block, 0, st, a);
}

// ----------------------------------------------------------------------------- experts
constexpr int kMoeMaxExperts = 1024;
constexpr int kPlanPairs = 4096;  // pairs a planning workgroup takes
constexpr int kPlanPer = kPlanPairs / 256;

struct PlanArgs {
  const int32_t* ids;
  int64_t id_stride;
  int pairs, top_k, experts;
  int blocks;      // planning workgroups: ceil(pairs / kPlanPairs)
  int tile;        // pairs of one expert in a tile
  int32_t* counts; // [blocks, experts] (more than one workgroup)
  int32_t* order;
  X8Tile* tiles;
  int32_t* ntiles;
};

struct PlanShared {
  int count[kMoeMaxExperts];  // pairs of the expert; then the next free position
  int part[2][4];
};

// The experts of this thread's pairs (-1: none) and, in LDS, the workgroup's histogram.
__device__ __forceinline__ void plan_count(const PlanArgs& a, int block, PlanShared& s, int (&e)[kPlanPer]) {
  const int tid = threadIdx.x;
  for (int i = tid; i < a.experts; i += 256) s.count[i] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPlanPer; ++i) {
    const int p = block * kPlanPairs + i * 256 + tid;
    e[i] = -1;
    if (p < a.pairs) e[i] = a.ids[(int64_t)(p / a.top_k) * a.id_stride + p % a.top_k];
    if (e[i] >= a.experts) e[i] = -1;
  }
#pragma unroll
  for (int i = 0; i < kPlanPer; ++i)
    if (e[i] >= 0) atomicAdd(&s.count[e[i]], 1);
  __syncthreads();
}

// Running sums of the experts' pairs and tiles (thread t: experts 4 t .. 4 t +
// 3), this workgroup's first position of each expert, and its pairs' places.
// Which of an expert's positions a pair gets does not change its results.
__device__ __forceinline__ void plan_place(const PlanArgs& a, int block, PlanShared& s, const int (&e)[kPlanPer]) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int total[4], before[4], sum = 0, tiles = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int x = 4 * tid + j;
    total[j] = before[j] = 0;
    if (x < a.experts) {
      if (a.blocks == 1) {
        total[j] = s.count[x];
      } else {
        for (int b = 0; b < a.blocks; ++b) {
          const int c = a.counts[b * a.experts + x];
          before[j] += b < block ? c : 0;
          total[j] += c;
        }
      }
    }
    sum += total[j];
    tiles += (total[j] + a.tile - 1) / a.tile;
  }
  int run = sum, trun = tiles;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int u = __shfl_up(run, d), v = __shfl_up(trun, d);
    if (lane >= d) {
      run += u;
      trun += v;
    }
  }
  if (lane == 63) {
    s.part[0][wave] = run;
    s.part[1][wave] = trun;
  }
  __syncthreads();
  run -= sum;
  trun -= tiles;
  for (int w = 0; w < wave; ++w) {
    run += s.part[0][w];
    trun += s.part[1][w];
  }
  if (block == 0 && tid == 255) *a.ntiles = trun + tiles;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int x = 4 * tid + j;
    if (x < a.experts) {
      s.count[x] = run + before[j];
      if (block == 0)
        for (int i = 0; i < total[j]; i += a.tile)
          a.tiles[trun++] = X8Tile{x, run + i, min(a.tile, total[j] - i), 0};
      run += total[j];
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPlanPer; ++i)
    if (e[i] >= 0) a.order[atomicAdd(&s.count[e[i]], 1)] = block * kPlanPairs + i * 256 + tid;
}

// First launch: workgroups 0 .. blocks - 1 count their pairs' experts (a lone
// one places them too), the others quantise x.
template <int XT>
__global__ __launch_bounds__(256) void moe_prepare_kernel(const PlanArgs a, const QuantArgs q) {
  __shared__ PlanShared s;
  if (static_cast<int>(blockIdx.x) >= a.blocks) {
    quant_unit<XT>(q, (int64_t)(blockIdx.x - a.blocks) * 256 + threadIdx.x);
    return;
  }
  const int block = blockIdx.x;
  int e[kPlanPer];
  plan_count(a, block, s, e);
  if (a.blocks == 1) {
    plan_place(a, 0, s, e);
  } else {
    for (int i = threadIdx.x; i < a.experts; i += 256) a.counts[block * a.experts + i] = s.count[i];
  }
}

__global__ __launch_bounds__(256) void moe_place_kernel(const PlanArgs a) {
  __shared__ PlanShared s;
  int e[kPlanPer];
  plan_count(a, blockIdx.x, s, e);
  plan_place(a, blockIdx.x, s, e);
}

// ---- few tokens: the weights stream through registers
//
// A decode batch leaves an expert a handful of tokens, so the time is the
// weights' way from HBM: each is read once, straight into MFMA operands (16
// rows x 128 bytes of K per product, widened to fp16), by many small
// workgroups with all of their loads in flight.  A tile is up to 16 tokens of
// one expert, the 16 columns of a product.
constexpr int kFewTile = 16;
constexpr int kFewAhead = 4;      // blocks of K a wave loads at once
constexpr int kFewChunk = 2048;   // hidden values quantised into LDS at a time

struct FewArgs {
  const int32_t* order;           // tiles of the plan, or (pairs mode) each pair its own tile
  const X8Tile* tiles;
  const int32_t* ntiles;
  const int32_t* ids;
  int64_t id_stride;
  const void* x;                  // pairs mode: x itself
  int64_t x_stride;
  const uint8_t* x8;
  const float* xs;
  const float* pair_w;
  int64_t pair_w_stride;
  int tokens, top_k, experts, hidden, inter;
  const uint8_t* w13;
  const float* s13;
  const uint8_t* w2;
  const float* s2;
  float* act;                     // [positions or pairs, inter]: SiLU(g) u
  void* slots;
  int slot_dtype;
  void* out;                      // pairs mode: the sums
  int64_t out_stride;
  int out_dtype, add;
};

// act = SiLU(g) u of one tile and 16 CG features, NW waves sharing K, each with
// AH blocks of K in flight.  PAIRS: the tile is one (token, slot) pair, and x is
// quantised here.
template <int XT, bool PAIRS, int CG, int NW, int AH>
__global__ __launch_bounds__(64 * NW) void moe_up_few_kernel(const FewArgs a) {
  static_assert(64 * NW == 256 * CG, "a thread for each result of 16 rows");
  extern __shared__ __attribute__((aligned(16))) uint8_t xq_s[];  // PAIRS: hidden e4m3 values, then their scales
  __shared__ f32x4 red[NW][2 * CG][64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int groups = a.inter / (16 * CG);
  const int tile = blockIdx.x / groups, c0 = blockIdx.x % groups * 16 * CG;
  int expert, first, rows = 1;
  if constexpr (PAIRS) {
    first = tile;
    expert = a.ids[(int64_t)(tile / a.top_k) * a.id_stride + tile % a.top_k];
    if (expert < 0 || expert >= a.experts) return;
  } else {
    const X8Tile t = a.tiles[tile];  // in step with the count: entries past it are allocated, and not used
    if (tile >= *a.ntiles) return;
    expert = t.expert;
    first = t.first;
    rows = t.rows;
  }
  expert = __builtin_amdgcn_readfirstlane(expert);
  const int k = a.hidden, kblocks = k / kX8Block;
  const uint8_t* wg = a.w13 + ((int64_t)expert * 2 * a.inter + c0) * k;
  const uint8_t* wu = wg + (int64_t)a.inter * k;
  const float* sg = a.s13 + ((int64_t)expert * 2 * (a.inter / kX8Block) + c0 / kX8Block) * kblocks;
  const float* su = sg + (int64_t)(a.inter / kX8Block) * kblocks;
  const int at = first + min(lane & 15, rows - 1);
  const int64_t token = PAIRS ? tile / a.top_k : a.order[at] / a.top_k;
  const uint8_t* x8 = a.x8 + token * k;
  const float* xs = a.xs + token * kblocks;

  // a wave's blocks kb0 .. kb0 + AH - 1: weights first, so that no wait for them comes early
  u32x4 w[AH][2 * CG][2], b[AH][2];
  float fg[AH], fu[AH], fx[AH];
  auto load = [&](int kb0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < AH; ++i) {
      const int kb = min(kb0 + i, kblocks - 1);
#pragma unroll
      for (int c = 0; c < CG; ++c) {
        load_rows16(wg + (int64_t)16 * c * k, k, kb, lane, w[i][c]);
        load_rows16(wu + (int64_t)16 * c * k, k, kb, lane, w[i][CG + c]);
      }
    }
#pragma unroll
    for (int i = 0; i < AH; ++i) {
      const int kb = min(kb0 + i, kblocks - 1);
      fg[i] = sg[kb];
      fu[i] = su[kb];
      if constexpr (!PAIRS) {
        load_chunks(x8 + kb * kX8Block, lane, b[i]);
        fx[i] = xs[kb];
      }
    }
    __builtin_amdgcn_sched_barrier(0);  // all of them in flight before the first product
  };
  load(wave * AH);
  if constexpr (PAIRS) {
    uint8_t* q = xq_s;
    float* qs = reinterpret_cast<float*>(xq_s + k);
    const int64_t x0 = token * a.x_stride;
    for (int c = 8 * tid; c < k; c += 8 * 64 * NW) {
      float v[8];
      load_act8<XT>(a.x, x0 + c, v);
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, finite_abs(v[i]));
      const uint32_t e = x8_scale_exp(row16_max(top));
      const float inv = x8_inverse(e);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = x8_value(v[i], inv);
      *reinterpret_cast<u32x2*>(q + c) = u32x2{pack_x8(v[0], v[1], v[2], v[3]), pack_x8(v[4], v[5], v[6], v[7])};
      if ((c & (kX8Block - 1)) == 0) qs[c / kX8Block] = x8_scale(e);
    }
    lds_barrier();
  }
  f32x4 acc[2 * CG];
#pragma unroll
  for (int c = 0; c < 2 * CG; ++c) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int kb0 = wave * AH; kb0 < kblocks; kb0 += NW * AH) {
#pragma unroll
    for (int i = 0; i < AH; ++i) {
      const int kb = kb0 + i;
      if (kb >= kblocks) break;
      if constexpr (PAIRS) {
        load_chunks(xq_s + kb * kX8Block, lane, b[i]);
        fx[i] = reinterpret_cast<const float*>(xq_s + k)[kb];
      }
      const float s0 = fx[i] * fg[i], s1 = fx[i] * fu[i];
#pragma unroll
      for (int c = 0; c < 2 * CG; ++c) {
        const f32x4 part = mfma_x8_16(w[i][c], b[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[c][j] = fmaf(part[j], c < CG ? s0 : s1, acc[c][j]);
      }
    }
    if (kb0 + NW * AH < kblocks) load(kb0 + NW * AH);
  }
#pragma unroll
  for (int c = 0; c < 2 * CG; ++c) red[wave][c][lane] = acc[c];
  __syncthreads();
  // thread (row, feature): result (feature, row) of a product is value feature % 4 of lane row + 16 (feature / 4)
  const int row = tid / (16 * CG), f = tid % 16, c = tid / 16 % CG;
  if (row >= rows) return;
  float gate = 0.f, up = 0.f;
#pragma unroll
  for (int v = 0; v < NW; ++v) {
    gate += red[v][c][row + 16 * (f >> 2)][f & 3];
    up += red[v][CG + c][row + 16 * (f >> 2)][f & 3];
  }
  a.act[(int64_t)(first + row) * a.inter + c0 + 16 * c + f] = x8_swiglu(gate, up);
}

// 8 values of act to e4m3 at d, their block's scale to s (16 lanes a block).
__device__ __forceinline__ void quant_act8(const float* p, uint8_t* d, float* s, int lane) {
  const f32x4 v0 = *reinterpret_cast<const f32x4*>(p), v1 = *reinterpret_cast<const f32x4*>(p + 4);
  float v[8] = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = fmaxf(top, finite_abs(v[i]));
  const uint32_t e = x8_scale_exp(row16_max(top));
  const float inv = x8_inverse(e);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = x8_value(v[i], inv);
  *reinterpret_cast<u32x2*>(d) = u32x2{pack_x8(v[0], v[1], v[2], v[3]), pack_x8(v[4], v[5], v[6], v[7])};
  if ((lane & 15) == 0) *s = x8_scale(e);
}

// One tile's rows of 32 NW features of the output (a wave: 32 of them), to the
// pairs' slots.
template <int NW>
__global__ __launch_bounds__(64 * NW) void moe_down_few_kernel(const FewArgs a) {
  constexpr int kPitch = kFewChunk + 16;  // 16 rows' reads meet all banks
  __shared__ __attribute__((aligned(16))) uint8_t h_s[kFewTile * kPitch];
  __shared__ float hs_s[kFewTile][kFewChunk / kX8Block];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int groups = (a.hidden + 32 * NW - 1) / (32 * NW);
  const int tile = blockIdx.x / groups;
  const X8Tile t = a.tiles[tile];
  if (tile >= *a.ntiles) return;
  const int expert = __builtin_amdgcn_readfirstlane(t.expert), rows = __builtin_amdgcn_readfirstlane(t.rows);
  const int n0 = min(blockIdx.x % groups * 32 * NW + wave * 32, a.hidden - 32);  // waves past the last feature repeat its group
  const int k = a.inter, kblocks = k / kX8Block;
  const uint8_t* w = a.w2 + ((int64_t)expert * a.hidden + n0) * k;
  const float* s2 = a.s2 + ((int64_t)expert * (a.hidden / kX8Block) + n0 / kX8Block) * kblocks;
  u32x4 v[2][kFewAhead][2];
  auto load = [&](int kb0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kFewAhead; ++i) {
      const int kb = min(kb0 + i, kblocks - 1);
      load_rows16(w, k, kb, lane, v[0][i]);
      load_rows16(w + (int64_t)16 * k, k, kb, lane, v[1][i]);
    }
  };
  load(0);
  const int row = min(lane & 15, rows - 1);
  const int pair = a.order[t.first + row];  // ahead of the end, where its wait would show
  const float pw = a.pair_w[(int64_t)(pair / a.top_k) * a.pair_w_stride + pair % a.top_k];
  f32x4 acc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
  for (int c0 = 0; c0 < k; c0 += kFewChunk) {
    const int cols = min(kFewChunk, k - c0), units = cols / 8;
    if (c0) __syncthreads();
    for (int u = tid; u < rows * units; u += 64 * NW) {
      const int r = u / units, c = (u - r * units) * 8;
      quant_act8(a.act + (int64_t)(t.first + r) * k + c0 + c, h_s + r * kPitch + c, &hs_s[r][c / kX8Block], tid);
    }
    lds_barrier();
    for (int b0 = 0; b0 < cols / kX8Block; b0 += kFewAhead) {
#pragma unroll
      for (int i = 0; i < kFewAhead; ++i) {
        const int kb = b0 + i;  // of the chunk
        if (kb >= cols / kX8Block) break;
        u32x4 b[2];
        load_chunks(h_s + row * kPitch + kb * kX8Block, lane, b);
        const float s = hs_s[row][kb] * s2[c0 / kX8Block + kb];
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          const f32x4 part = mfma_x8_16(v[f][i], b);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[f][j] = fmaf(part[j], s, acc[f][j]);
        }
      }
      const int next = c0 / kX8Block + b0 + kFewAhead;
      if (next < kblocks) load(next);
    }
  }
  if ((lane & 15) >= rows) return;
#pragma unroll
  for (int f = 0; f < 2; ++f) {
    const int64_t o = (int64_t)pair * a.hidden + n0 + 16 * f + 4 * (lane >> 4);
    float r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = pw * acc[f][j];
    if (a.slot_dtype == RIA_DT_F32)
      store_act4<RIA_DT_F32>(a.slots, o, r);
    else if (a.slot_dtype == RIA_DT_F16)
      store_act4<RIA_DT_F16>(a.slots, o, r);
    else
      store_act4<RIA_DT_BF16>(a.slots, o, r);
  }
}

// Pairs mode: 16 features of one token's sum, a wave for each slot (in turns of
// kSumWaves); the terms meet in LDS and are added in slot order.
constexpr int kSumWaves = 8;
template <int DT>
__global__ __launch_bounds__(64 * kSumWaves) void moe_down_pairs_kernel(const FewArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t h_s[kSumWaves][kFewChunk];
  __shared__ float hs_s[kSumWaves][kFewChunk / kX8Block];
  __shared__ float term[kSumWaves][16];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int groups = a.hidden / 16;
  const int t = blockIdx.x / groups, n0 = blockIdx.x % groups * 16;
  const int k = a.inter, kblocks = k / kX8Block;
  float sum = 0.f;  // thread f < 16: feature n0 + f
  for (int j0 = 0; j0 < a.top_k; j0 += kSumWaves) {
    const int j = j0 + wave;
    int expert = j < a.top_k ? a.ids[(int64_t)t * a.id_stride + j] : -1;
    expert = __builtin_amdgcn_readfirstlane(expert);
    const bool some = expert >= 0 && expert < a.experts;
    f32x4 acc{0.f, 0.f, 0.f, 0.f};
    if (some) {
      const uint8_t* w = a.w2 + ((int64_t)expert * a.hidden + n0) * k;
      const float* s2 = a.s2 + ((int64_t)expert * (a.hidden / kX8Block) + n0 / kX8Block) * kblocks;
      const float* act = a.act + ((int64_t)t * a.top_k + j) * k;
      for (int c0 = 0; c0 < k; c0 += kFewChunk) {
        const int cols = min(kFewChunk, k - c0);
        for (int b0 = 0; b0 < cols / kX8Block; b0 += kFewAhead) {
          u32x4 v[kFewAhead][2];
#pragma unroll
          for (int i = 0; i < kFewAhead; ++i) load_rows16(w, k, min(c0 / kX8Block + b0 + i, kblocks - 1), lane, v[i]);
          if (b0 == 0)  // 64 lanes: four blocks at a time (whole groups of 16 lanes)
            for (int c = 8 * lane; c < cols; c += 8 * 64)
              quant_act8(act + c0 + c, h_s[wave] + c, &hs_s[wave][c / kX8Block], lane);
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int i = 0; i < kFewAhead; ++i) {
            const int kb = b0 + i;
            if (kb >= cols / kX8Block) break;
            u32x4 b[2];
            load_chunks(h_s[wave] + kb * kX8Block, lane, b);
            const float s = hs_s[wave][kb] * s2[c0 / kX8Block + kb];
            const f32x4 part = mfma_x8_16(v[i], b);
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[q] = fmaf(part[q], s, acc[q]);
          }
          __builtin_amdgcn_wave_barrier();
        }
      }
    }
    if ((lane & 15) == 0) {  // column 0: every column is the pair's
      const float pw = some ? a.pair_w[(int64_t)t * a.pair_w_stride + j] : 0.f;
#pragma unroll
      for (int q = 0; q < 4; ++q) term[wave][4 * (lane >> 4) + q] = some ? through_dtype<DT>(pw * acc[q]) : 0.f;
    }
    __syncthreads();
    if (tid < 16)
      for (int w = 0; w < min(kSumWaves, a.top_k - j0); ++w) sum = add_rn(sum, term[w][tid]);
    __syncthreads();
  }
  if (tid < 16) {
    const int64_t o = (int64_t)t * a.out_stride + n0 + tid;
    if constexpr (DT == RIA_DT_F32) {
      if (a.add) sum = add_rn(static_cast<const float*>(a.out)[o], sum);
    }
    store_act<DT>(a.out, o, sum);
  }
}

struct CombineArgs {
  const void* slots;  // [tokens * top_k, hidden], in out's dtype
  const int32_t* ids;
  int64_t id_stride;
  int tokens, top_k, experts, hidden;
  void* out;
  int64_t out_stride;
  int add, vec;
};
constexpr int kCombineAhead = 4;  // slots loaded ahead of their sums

// out[t] (+)= the sum of the token's slots in slot order, in fp32; slots of no
// expert were never written and are left out.
template <int DT>
__global__ __launch_bounds__(256) void moe_combine_kernel(const CombineArgs a) {
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int per = a.hidden / 8;
  const int64_t t = u / per;
  if (t >= a.tokens) return;
  const int c = static_cast<int>(u - t * per) * 8;
  float s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = 0.f;
  for (int j0 = 0; j0 < a.top_k; j0 += kCombineAhead) {
    float v[kCombineAhead][8];
#pragma unroll
    for (int j = 0; j < kCombineAhead; ++j) {
      const int e = j0 + j < a.top_k ? a.ids[t * a.id_stride + j0 + j] : -1;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] = 0.f;
      if (e >= 0 && e < a.experts) load_act8<DT>(a.slots, (t * a.top_k + j0 + j) * a.hidden + c, v[j]);
    }
#pragma unroll
    for (int j = 0; j < kCombineAhead; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = add_rn(s[i], v[j][i]);
  }
  X8Args o{};
  o.y = a.out;
  o.y_dtype = DT;
  o.y_add = a.add;
  o.vec = a.vec;
  store_eight(o, t * a.out_stride + c, s);
}

static int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

// Most tiles of any routing: an expert's last tile may be partly filled.
static int64_t moe_tiles(int64_t pairs, int experts, int tile) {
  return std::min<int64_t>(pairs, pairs / tile + std::min<int64_t>(experts, pairs));
}

// How a call is run, by its pairs: each pair by itself, tiles of 16 pairs whose
// weights stream through registers, or tiles of 64 or 256 pairs in LDS.
enum class MoeKind { kPairs, kFew, kTiles };
static MoeKind moe_kind(int64_t pairs, int experts) {
  if (pairs <= 32) return MoeKind::kPairs;
  return pairs <= (int64_t)experts * 8 ? MoeKind::kFew : MoeKind::kTiles;
}

// Pairs of one expert that a tile takes.
static int moe_tile(int64_t pairs, int experts, int out_dtype) {
  if (moe_kind(pairs, experts) != MoeKind::kTiles) return kFewTile;
  return out_dtype != RIA_DT_F32 && pairs >= (int64_t)experts * 128 ? 256 : 64;
}

struct MoeLayout {
  int64_t x8, xs, counts, order, tiles, ntiles, act, h8, hs, slots, bytes;
};
static MoeLayout moe_layout(int64_t tokens, int top_k, int experts, int hidden, int inter, int out_dtype) {
  MoeLayout l{};
  const int64_t pairs = tokens * top_k;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += align256(bytes);
    return here;
  };
  l.x8 = take(tokens * hidden);
  l.xs = take(tokens * (hidden / kX8Block) * 4);
  l.counts = take((pairs + kPlanPairs - 1) / kPlanPairs * experts * 4);
  l.order = take(pairs * 4);
  l.tiles = take(moe_tiles(pairs, experts, moe_tile(pairs, experts, out_dtype)) * static_cast<int64_t>(sizeof(X8Tile)));
  l.ntiles = take(4);
  const bool tiled = moe_kind(pairs, experts) == MoeKind::kTiles;
  l.act = take(tiled ? 0 : pairs * inter * 4);
  l.h8 = take(tiled ? pairs * inter : 0);
  l.hs = take(tiled ? pairs * (inter / kX8Block) * 4 : 0);
  l.slots = take(pairs * hidden * (out_dtype == RIA_DT_F32 ? 4 : 2));
  l.bytes = at;
  return l;
}

// The tiled kernels: gate and up rows, then down rows, of `most` tiles at the most.
static void launch_moe_tiles(const ria_moe_experts_desc& d, const MoeLayout& l, int64_t most, int tile, hipStream_t st) {
  char* ws = static_cast<char*>(d.workspace);
  auto at = [&](int64_t o) { return static_cast<void*>(ws + o); };
  X8Args up{};
  up.x = static_cast<const uint8_t*>(at(l.x8));
  up.x_stride = d.hidden;
  up.xs = static_cast<const float*>(at(l.xs));
  up.xs_stride = d.hidden / kX8Block;
  up.w = static_cast<const uint8_t*>(d.w13);
  up.ws = d.w13_scale_inv;
  up.n = 2 * d.inter;
  up.k = d.hidden;
  up.order = static_cast<const int32_t*>(at(l.order));
  up.tiles = static_cast<const X8Tile*>(at(l.tiles));
  up.ntiles = static_cast<const int32_t*>(at(l.ntiles));
  up.top_k = d.top_k;
  up.h8 = static_cast<uint8_t*>(at(l.h8));
  up.hs = static_cast<float*>(at(l.hs));
  up.m = d.tokens;
  const bool wide = d.out_dtype == RIA_DT_F32;
  auto grid_of = [&](int feature_tiles) { return dim3(static_cast<unsigned>((most * feature_tiles + 7) / 8 * 8)); };
  if (wide)
    hipLaunchKernelGGL((x8_tile_kernel<kX8Up, 2, 2, 4, 1, true>), grid_of(d.inter / 128), dim3(256), 0, st, up);
  else if (tile == 256)
    hipLaunchKernelGGL((x8_tile_kernel<kX8Up, 4, 2, 2, 4, false>), grid_of(d.inter / 128), dim3(512), 0, st, up);
  else
    hipLaunchKernelGGL((x8_tile_kernel<kX8Up, 2, 2, 4, 1, false>), grid_of(d.inter / 128), dim3(256), 0, st, up);
  X8Args dn = up;
  dn.x = up.h8;
  dn.x_stride = d.inter;
  dn.xs = up.hs;
  dn.xs_stride = d.inter / kX8Block;
  dn.w = static_cast<const uint8_t*>(d.w2);
  dn.ws = d.w2_scale_inv;
  dn.n = d.hidden;
  dn.k = d.inter;
  dn.y = at(l.slots);
  dn.y_stride = d.hidden;
  dn.y_dtype = d.out_dtype;
  dn.vec = 1;
  dn.pair_w = d.weights;
  dn.pair_w_stride = d.weights_row_stride;
  if (wide)
    hipLaunchKernelGGL((x8_tile_kernel<kX8Down, 2, 1, 2, 2, true>), grid_of(d.hidden / 128), dim3(256), 0, st, dn);
  else if (tile == 256)
    hipLaunchKernelGGL((x8_tile_kernel<kX8Down, 4, 2, 2, 4, false>), grid_of((d.hidden + 255) / 256), dim3(512), 0, st, dn);
  else
    hipLaunchKernelGGL((x8_tile_kernel<kX8Down, 2, 1, 2, 2, false>), grid_of(d.hidden / 128), dim3(256), 0, st, dn);
}

static const char* moe_sizes_error(int64_t tokens, int top_k, int experts, int hidden, int inter) {
  if (tokens < 0 || top_k < 1 || experts < 1 || experts > kMoeMaxExperts) return "bad sizes (1 to 1024 experts)";
  if (hidden <= 0 || hidden % kX8Block || hidden > 32768) return "hidden must be a multiple of 128 up to 32768";
  if (inter <= 0 || inter % kX8Block || inter > 32768) return "inter must be a multiple of 128 up to 32768";
  if (tokens * top_k >= (int64_t(1) << 30)) return "too many (token, slot) pairs";
  if (tokens * hidden >= (int64_t(1) << 32)) return "too many tokens (their e4m3 copy takes 4 GiB or more)";
  return nullptr;
}

}  // namespace ria

using namespace ria;

extern "C" int ria_moe_route(int tokens, int experts, int top_k, const void* logits, int logits_dtype,
                             int64_t logits_row_stride, int scoring, const float* bias, int num_groups, int top_groups,
                             int group_score, int renormalize, float scale, int shared_expert, float* weights,
                             int64_t weights_row_stride, int32_t* ids, int64_t ids_row_stride, void* stream) {
  const char* who = "ria_moe_route";
  if (tokens < 0 || experts < 1 || experts > kRouteMaxExperts)
    return set_error(RIA_ERR_INVALID, "%s: 1 to %d experts (got %d)", who, kRouteMaxExperts, experts);
  if (scoring != RIA_ROUTE_SOFTMAX && scoring != RIA_ROUTE_SIGMOID) return set_error(RIA_ERR_INVALID, "%s: unknown scoring", who);
  if (group_score != RIA_ROUTE_GROUP_MAX && group_score != RIA_ROUTE_GROUP_TOP2)
    return set_error(RIA_ERR_INVALID, "%s: unknown group score", who);
  if (num_groups < 1 || num_groups > kRouteMaxGroups || experts % num_groups)
    return set_error(RIA_ERR_INVALID, "%s: the experts must split into 1 to %d equal groups", who, kRouteMaxGroups);
  if (top_groups < 1 || top_groups > num_groups) return set_error(RIA_ERR_INVALID, "%s: top_groups must be 1 to %d", who, num_groups);
  const int open = experts / num_groups * top_groups;
  if (top_k < 1 || top_k > kRouteMaxK || top_k > open)
    return set_error(RIA_ERR_INVALID, "%s: top_k must be 1 to %d (got %d)", who, std::min(kRouteMaxK, open), top_k);
  if (!x8_dtype_ok(logits_dtype)) return set_error(RIA_ERR_INVALID, "%s: unknown dtype code", who);
  if (tokens == 0) return RIA_OK;
  if (!logits || !weights || !ids) return set_error(RIA_ERR_INVALID, "%s: null pointer", who);
  const int s = shared_expert ? 1 : 0;
  if (logits_row_stride < experts + s || weights_row_stride < top_k + s || ids_row_stride < top_k + s)
    return set_error(RIA_ERR_INVALID, "%s: row stride too small", who);
  const RouteArgs a{logits, logits_row_stride, tokens, experts, top_k, bias, scoring == RIA_ROUTE_SIGMOID, num_groups,
                    top_groups, group_score == RIA_ROUTE_GROUP_TOP2, renormalize != 0, s, scale, weights,
                    weights_row_stride, ids, ids_row_stride};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (logits_dtype == RIA_DT_BF16)
    launch_route<RIA_DT_BF16>(a, st);
  else if (logits_dtype == RIA_DT_F16)
    launch_route<RIA_DT_F16>(a, st);
  else
    launch_route<RIA_DT_F32>(a, st);
  return check_launch(who);
}

extern "C" int64_t ria_moe_experts_workspace_bytes(int tokens, int top_k, int experts, int hidden, int inter,
                                                   int out_dtype) {
  if (moe_sizes_error(tokens, top_k, experts, hidden, inter) || !x8_dtype_ok(out_dtype)) return -1;
  return moe_layout(tokens, top_k, experts, hidden, inter, out_dtype).bytes;
}

extern "C" int ria_moe_experts(const ria_moe_experts_desc* d, void* stream) {
  const char* who = "ria_moe_experts";
  if (!d) return set_error(RIA_ERR_INVALID, "%s: null descriptor", who);
  if (const char* e = moe_sizes_error(d->tokens, d->top_k, d->experts, d->hidden, d->inter))
    return set_error(RIA_ERR_INVALID, "%s: %s", who, e);
  if (!x8_dtype_ok(d->x_dtype) || !x8_dtype_ok(d->out_dtype)) return set_error(RIA_ERR_INVALID, "%s: unknown dtype code", who);
  if (d->accumulate && d->out_dtype != RIA_DT_F32) return set_error(RIA_ERR_INVALID, "%s: accumulating needs an fp32 out", who);
  if (d->tokens == 0) return RIA_OK;
  if (!d->x || !d->ids || !d->weights || !d->w13 || !d->w13_scale_inv || !d->w2 || !d->w2_scale_inv || !d->out || !d->workspace)
    return set_error(RIA_ERR_INVALID, "%s: null pointer", who);
  if (d->x_row_stride < d->hidden || d->x_row_stride % 8 || reinterpret_cast<uintptr_t>(d->x) % 16)
    return set_error(RIA_ERR_INVALID, "%s: x must be 16-byte aligned with a row stride of at least hidden, a multiple of 8", who);
  if (d->ids_row_stride < d->top_k || d->weights_row_stride < d->top_k || d->out_row_stride < d->hidden)
    return set_error(RIA_ERR_INVALID, "%s: row stride too small", who);
  if ((reinterpret_cast<uintptr_t>(d->w13) | reinterpret_cast<uintptr_t>(d->w2)) % 16)
    return set_error(RIA_ERR_INVALID, "%s: the weights must be 16-byte aligned", who);
  if (reinterpret_cast<uintptr_t>(d->workspace) % 256) return set_error(RIA_ERR_INVALID, "%s: workspace must be 256-byte aligned", who);
  const MoeLayout l = moe_layout(d->tokens, d->top_k, d->experts, d->hidden, d->inter, d->out_dtype);
  if (d->workspace_bytes < l.bytes)
    return set_error(RIA_ERR_WORKSPACE, "%s: workspace of %lld bytes, %lld needed", who, (long long)d->workspace_bytes,
                     (long long)l.bytes);
  hipStream_t st = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(d->workspace);
  auto at = [&](int64_t o) { return static_cast<void*>(ws + o); };
  int32_t* order = static_cast<int32_t*>(at(l.order));
  X8Tile* tiles = static_cast<X8Tile*>(at(l.tiles));
  int32_t* ntiles = static_cast<int32_t*>(at(l.ntiles));
  const int64_t pairs = (int64_t)d->tokens * d->top_k;
  const MoeKind kind = moe_kind(pairs, d->experts);
  const int tile = moe_tile(pairs, d->experts, d->out_dtype);
  const int64_t most = moe_tiles(pairs, d->experts, tile);
  if (std::max(most, pairs) * (std::max(d->hidden, d->inter) / 16) > 0x7ffffff0)
    return set_error(RIA_ERR_INVALID, "%s: too many (token, slot) pairs", who);
  FewArgs few{order, tiles, ntiles, d->ids, d->ids_row_stride, d->x, d->x_row_stride,
              static_cast<const uint8_t*>(at(l.x8)), static_cast<const float*>(at(l.xs)), d->weights,
              d->weights_row_stride, d->tokens, d->top_k, d->experts, d->hidden, d->inter,
              static_cast<const uint8_t*>(d->w13), d->w13_scale_inv, static_cast<const uint8_t*>(d->w2),
              d->w2_scale_inv, static_cast<float*>(at(l.act)), at(l.slots), d->out_dtype, d->out, d->out_row_stride,
              d->out_dtype, d->accumulate != 0};
  if (kind == MoeKind::kPairs) {
    const dim3 ugrid(static_cast<unsigned>(pairs * (d->inter / 16)));
    const dim3 dgrid(static_cast<unsigned>((int64_t)d->tokens * (d->hidden / 16)));
    const size_t lds = d->hidden + d->hidden / kX8Block * 4;
    if (d->x_dtype == RIA_DT_BF16)
      hipLaunchKernelGGL((moe_up_few_kernel<RIA_DT_BF16, true, 1, 4, 4>), ugrid, dim3(256), lds, st, few);
    else if (d->x_dtype == RIA_DT_F16)
      hipLaunchKernelGGL((moe_up_few_kernel<RIA_DT_F16, true, 1, 4, 4>), ugrid, dim3(256), lds, st, few);
    else
      hipLaunchKernelGGL((moe_up_few_kernel<RIA_DT_F32, true, 1, 4, 4>), ugrid, dim3(256), lds, st, few);
    if (d->out_dtype == RIA_DT_BF16)
      hipLaunchKernelGGL((moe_down_pairs_kernel<RIA_DT_BF16>), dgrid, dim3(64 * kSumWaves), 0, st, few);
    else if (d->out_dtype == RIA_DT_F16)
      hipLaunchKernelGGL((moe_down_pairs_kernel<RIA_DT_F16>), dgrid, dim3(64 * kSumWaves), 0, st, few);
    else
      hipLaunchKernelGGL((moe_down_pairs_kernel<RIA_DT_F32>), dgrid, dim3(64 * kSumWaves), 0, st, few);
    return check_launch(who);
  }
  const PlanArgs plan{d->ids, d->ids_row_stride, static_cast<int>(pairs), d->top_k, d->experts,
                      static_cast<int>((pairs + kPlanPairs - 1) / kPlanPairs), tile, static_cast<int32_t*>(at(l.counts)),
                      order, tiles, ntiles};
  const QuantArgs quant{d->tokens * (int64_t)(d->hidden / 8), d->hidden / 8, d->x, d->x_row_stride,
                        static_cast<uint8_t*>(at(l.x8)), static_cast<float*>(at(l.xs))};
  const dim3 pgrid(static_cast<unsigned>(plan.blocks + (quant.units + 255) / 256));
  if (d->x_dtype == RIA_DT_BF16)
    hipLaunchKernelGGL((moe_prepare_kernel<RIA_DT_BF16>), pgrid, dim3(256), 0, st, plan, quant);
  else if (d->x_dtype == RIA_DT_F16)
    hipLaunchKernelGGL((moe_prepare_kernel<RIA_DT_F16>), pgrid, dim3(256), 0, st, plan, quant);
  else
    hipLaunchKernelGGL((moe_prepare_kernel<RIA_DT_F32>), pgrid, dim3(256), 0, st, plan, quant);
  if (plan.blocks > 1) hipLaunchKernelGGL(moe_place_kernel, dim3(plan.blocks), dim3(256), 0, st, plan);
  if (kind == MoeKind::kFew) {
    hipLaunchKernelGGL((moe_up_few_kernel<RIA_DT_F32, false, 2, 8, 2>), dim3(static_cast<unsigned>(most * (d->inter / 32))),
                       dim3(512), 0, st, few);
    hipLaunchKernelGGL((moe_down_few_kernel<4>), dim3(static_cast<unsigned>(most * (d->hidden / 128))), dim3(256), 0, st, few);
  } else {
    launch_moe_tiles(*d, l, most, tile, st);
  }
  const CombineArgs c{at(l.slots), d->ids, d->ids_row_stride, d->tokens, d->top_k, d->experts, d->hidden, d->out,
                      d->out_row_stride, d->accumulate != 0,
                      reinterpret_cast<uintptr_t>(d->out) % 16 == 0 && d->out_row_stride % 8 == 0};
  const dim3 grid(static_cast<unsigned>(((int64_t)d->tokens * (d->hidden / 8) + 255) / 256));
  if (d->out_dtype == RIA_DT_BF16)
    hipLaunchKernelGGL((moe_combine_kernel<RIA_DT_BF16>), grid, dim3(256), 0, st, c);
  else if (d->out_dtype == RIA_DT_F16)
    hipLaunchKernelGGL((moe_combine_kernel<RIA_DT_F16>), grid, dim3(256), 0, st, c);
  else
    hipLaunchKernelGGL((moe_combine_kernel<RIA_DT_F32>), grid, dim3(256), 0, st, c);
  return check_launch(who);
}
