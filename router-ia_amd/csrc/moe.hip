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

struct CombineArgs {
  const void* slots;  // [tokens * top_k, hidden], in out's dtype
  const int32_t* ids;
  int64_t id_stride;
  int tokens, top_k, experts, hidden;
  void* out;
  int64_t out_stride;
  int add;
};

// out[t] (+)= the sum of the token's slots in slot order, in fp32; slots of no
// expert were never written and are left out.
template <int DT>
__global__ __launch_bounds__(256) void moe_combine_kernel(const CombineArgs a) {
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int per = a.hidden / 4;
  const int64_t t = u / per;
  if (t >= a.tokens) return;
  const int c = static_cast<int>(u - t * per) * 4;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j < a.top_k; ++j) {
    const int e = a.ids[t * a.id_stride + j];
    if (e < 0 || e >= a.experts) continue;
    float v[4];
    load_act4<DT>(a.slots, (t * a.top_k + j) * a.hidden + c, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = add_rn(s[i], v[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t o = t * a.out_stride + c + i;
    if constexpr (DT == RIA_DT_F32) {
      if (a.add) s[i] = add_rn(static_cast<const float*>(a.out)[o], s[i]);
    }
    store_act<DT>(a.out, o, s[i]);
  }
}

static int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

// Most tiles of any routing: an expert's last tile may be partly filled.
static int64_t moe_tiles(int64_t pairs, int experts, int tile) {
  return std::min<int64_t>(pairs, pairs / tile + std::min<int64_t>(experts, pairs));
}

// Pairs of one expert that a tile takes.
static int moe_tile(int64_t pairs, int experts, int out_dtype) {
  return out_dtype != RIA_DT_F32 && pairs >= (int64_t)experts * 128 ? 256 : 64;
}

struct MoeLayout {
  int64_t x8, xs, counts, order, tiles, ntiles, h8, hs, slots, bytes;
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
  l.h8 = take(pairs * inter);
  l.hs = take(pairs * (inter / kX8Block) * 4);
  l.slots = take(pairs * hidden * (out_dtype == RIA_DT_F32 ? 4 : 2));
  l.bytes = at;
  return l;
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
  const int tile = moe_tile(pairs, d->experts, d->out_dtype);
  const int64_t most = moe_tiles(pairs, d->experts, tile);
  if (most * (std::max(d->hidden, d->inter) / 128) > 0x7ffffff0)
    return set_error(RIA_ERR_INVALID, "%s: too many (token, slot) pairs", who);
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
  X8Args up{};
  up.x = static_cast<const uint8_t*>(at(l.x8));
  up.x_stride = d->hidden;
  up.xs = static_cast<const float*>(at(l.xs));
  up.xs_stride = d->hidden / kX8Block;
  up.w = static_cast<const uint8_t*>(d->w13);
  up.ws = d->w13_scale_inv;
  up.n = 2 * d->inter;
  up.k = d->hidden;
  up.order = order;
  up.tiles = tiles;
  up.ntiles = ntiles;
  up.top_k = d->top_k;
  up.h8 = static_cast<uint8_t*>(at(l.h8));
  up.hs = static_cast<float*>(at(l.hs));
  up.m = d->tokens;
  const bool wide = d->out_dtype == RIA_DT_F32;
  auto grid_of = [&](int feature_tiles) { return dim3(static_cast<unsigned>((most * feature_tiles + 7) / 8 * 8)); };
  if (wide)
    hipLaunchKernelGGL((x8_tile_kernel<kX8Up, 2, 2, 4, 1, true>), grid_of(d->inter / 128), dim3(256), 0, st, up);
  else if (tile == 256)
    hipLaunchKernelGGL((x8_tile_kernel<kX8Up, 4, 2, 2, 4, false>), grid_of(d->inter / 128), dim3(512), 0, st, up);
  else
    hipLaunchKernelGGL((x8_tile_kernel<kX8Up, 2, 2, 4, 1, false>), grid_of(d->inter / 128), dim3(256), 0, st, up);
  X8Args dn = up;
  dn.x = up.h8;
  dn.x_stride = d->inter;
  dn.xs = up.hs;
  dn.xs_stride = d->inter / kX8Block;
  dn.w = static_cast<const uint8_t*>(d->w2);
  dn.ws = d->w2_scale_inv;
  dn.n = d->hidden;
  dn.k = d->inter;
  dn.y = at(l.slots);
  dn.y_stride = d->hidden;
  dn.y_dtype = d->out_dtype;
  dn.vec = 1;
  dn.pair_w = d->weights;
  dn.pair_w_stride = d->weights_row_stride;
  if (wide)
    hipLaunchKernelGGL((x8_tile_kernel<kX8Down, 2, 1, 2, 2, true>), grid_of(d->hidden / 128), dim3(256), 0, st, dn);
  else if (tile == 256)
    hipLaunchKernelGGL((x8_tile_kernel<kX8Down, 4, 2, 2, 4, false>), grid_of((d->hidden + 255) / 256), dim3(512), 0, st, dn);
  else
    hipLaunchKernelGGL((x8_tile_kernel<kX8Down, 2, 1, 2, 2, false>), grid_of(d->hidden / 128), dim3(256), 0, st, dn);
  const CombineArgs c{at(l.slots), d->ids, d->ids_row_stride, d->tokens, d->top_k, d->experts, d->hidden, d->out,
                      d->out_row_stride, d->accumulate};
  const dim3 grid(static_cast<unsigned>(((int64_t)d->tokens * (d->hidden / 4) + 255) / 256));
  if (d->out_dtype == RIA_DT_BF16)
    hipLaunchKernelGGL((moe_combine_kernel<RIA_DT_BF16>), grid, dim3(256), 0, st, c);
  else if (d->out_dtype == RIA_DT_F16)
    hipLaunchKernelGGL((moe_combine_kernel<RIA_DT_F16>), grid, dim3(256), 0, st, c);
  else
    hipLaunchKernelGGL((moe_combine_kernel<RIA_DT_F32>), grid, dim3(256), 0, st, c);
  return check_launch(who);
}
