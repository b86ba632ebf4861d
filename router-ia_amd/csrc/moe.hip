// The mixture-of-experts block that runs between the attention layers
// (qwen36_chat_batch.py:127-178 `batched_moe_step`, qwen36_router.py:96 `route`).
//
//   moe_route_rows_kernel,   router logits -> each token's experts and weights
//   moe_route_kernel
//   moe_prepare_kernel,      x to e4m3; (token, slot) pairs sorted by expert and
//   moe_place_kernel         cut into tiles
//   x8_tile_kernel           an expert's gate and up rows with SwiGLU, its down rows
//   moe_combine_kernel       the sum over a token's slots
//   moe_up_pairs_kernel,     the same for a few tokens, each pair by itself
//   moe_down_pairs_kernel
//
//     (g | u) = W13[e] Q(x_t)      Q: e4m3, a power-of-two scale per 128 values
//     y_t     = sum_j w[t, j] W2[e_j] Q(SiLU(g) u)
#include <algorithm>
#include <cmath>
#include <type_traits>

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
  int vec;   // rows and their groups of four logits are aligned for whole loads
  int wide;  // scores are compared in 64 bits at once (a wave per token)
  int lanes; // lanes of a group, a power of two, where groups are whole lanes (a wave per token), else 0
};

// Unsigned integers in the order of floating values: 0 for a taken or absent
// expert, -inf above it, NaN above every number; -0 ranks as 0.
__device__ __forceinline__ uint32_t order_key(float v) {
  const int32_t b = __float_as_int(v == 0.f ? 0.f : v);
  const uint32_t o = static_cast<uint32_t>(b ^ (b >> 31 | static_cast<int32_t>(0x80000000u)));
  return v != v ? 0xffffffffu : o;
}
__device__ __forceinline__ uint64_t order_key(double v) {
  const int64_t b = __double_as_longlong(v == 0.0 ? 0.0 : v);
  const uint64_t o = static_cast<uint64_t>(b ^ (b >> 63 | INT64_MIN));
  return v != v ? ~uint64_t(0) : o;
}

// V consecutive logits of a token from expert i0 on, -inf past the last.  No
// load is in a branch (each would be waited for at its join): past the last
// expert the last ones are loaded again.
template <int XT, int V>
__device__ __forceinline__ void load_logits(const RouteArgs& a, int64_t t, int i0, float (&x)[V]) {
  const float ninf = -__builtin_inff();
  if (V % 4 == 0 && a.vec) {  // whole groups of four, aligned
#pragma unroll
    for (int v = 0; v < V; v += 4) {
      float f[4];
      load_act4<XT>(a.logits, t * a.stride + min(i0 + v, a.experts - 4), f);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[(v + i) % V] = f[i];
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = load_act<XT>(a.logits, t * a.stride + min(i0 + v, a.experts - 1));
  }
#pragma unroll
  for (int v = 0; v < V; ++v) x[v] = i0 + v < a.experts ? x[v] : ninf;
}

// The value behind an fp32 key.
__device__ __forceinline__ float key_value(uint32_t k) {
  return k == 0xffffffffu ? __builtin_nanf("") : __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint64_t uniform(uint64_t v) {
  return static_cast<uint64_t>(uniform(static_cast<uint32_t>(v >> 32))) << 32 | uniform(static_cast<uint32_t>(v));
}

// A value of lane ^ OFF, in lane exchanges of a few cycles (after the xor 8 step
// of a reduction a rotation by 4 serves as xor 4).
template <int OFF>
__device__ __forceinline__ uint32_t lane_xor(uint32_t u) {
  if constexpr (OFF == 32 || OFF == 16) {
    const auto r = OFF == 32 ? __builtin_amdgcn_permlane32_swap(u, u, false, false)
                             : __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return (threadIdx.x & OFF) ? r[0] : r[1];
  } else {
    constexpr int kCtrl = OFF == 8 ? 0x128 : OFF == 4 ? 0x124 : OFF == 2 ? 0x4E : 0xB1;
    return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(u), kCtrl, 0xf, 0xf, true));
  }
}
template <int OFF>
__device__ __forceinline__ uint64_t lane_xor(uint64_t u) {
  return static_cast<uint64_t>(lane_xor<OFF>(static_cast<uint32_t>(u >> 32))) << 32 | lane_xor<OFF>(static_cast<uint32_t>(u));
}
template <typename T>
__device__ __forceinline__ T wave_max(T v) {
  v = max(v, lane_xor<32>(v));
  v = max(v, lane_xor<16>(v));
  v = max(v, lane_xor<8>(v));
  v = max(v, lane_xor<4>(v));
  v = max(v, lane_xor<2>(v));
  return max(v, lane_xor<1>(v));
}
template <>
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto r = i == 0 ? __builtin_amdgcn_permlane32_swap(v, v, false, false)
                          : __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(r[0], r[1]);
  }
  v = max(v, lane_xor<8>(v));
  v = max(v, lane_xor<4>(v));
  v = max(v, lane_xor<2>(v));
  return max(v, lane_xor<1>(v));
}
// Sum over the wave in 64 bits.
__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v += __longlong_as_double(__shfl_xor(__double_as_longlong(v), m));
  return v;
}

// exp(a - b) in fp32 from fp32 a and b: what the difference loses to rounding is
// put back, so far-apart logits keep their relative accuracy.
__device__ __forceinline__ float exp_diff(float a, float b) {
  const float d = a - b;
  const float lost = static_cast<float>((static_cast<double>(a) - static_cast<double>(b)) - static_cast<double>(d));
  return expf(d) * (1.f + (lost == lost ? lost : 0.f));
}

// sigmoid(x) exp(-min(m0, 0)), m0 the largest chosen logit: a common factor that
// renormalising takes out again, and that keeps the scores of very negative
// logits from vanishing.
__device__ __forceinline__ float sigmoid_from(float x, float m0) {
  const float c = m0 < 0.f ? m0 : 0.f;
  return x > 0.f ? 1.f / (1.f + expf(-x)) : exp_diff(x, c) / (1.f + expf(x));
}

// The slot of the expert that every token visits.
template <int XT>
__device__ __forceinline__ void route_shared(const RouteArgs& a, int64_t t) {
  const float l = load_act<XT>(a.logits, t * a.stride + a.experts);
  a.weights[t * a.w_stride + a.top_k] = 1.f / (1.f + expf(-l));
  a.ids[t * a.id_stride + a.top_k] = l == -__builtin_inff() ? -1 : a.experts;
}

// A value of lane 7 - l of each 8.
__device__ __forceinline__ uint32_t half_mirror(uint32_t u) {
  return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(u), 0x141, 0xf, 0xf, true));
}
__device__ __forceinline__ uint64_t half_mirror(uint64_t u) {
  return static_cast<uint64_t>(half_mirror(static_cast<uint32_t>(u >> 32))) << 32 | half_mirror(static_cast<uint32_t>(u));
}

// Largest over each row of 16 lanes.
template <typename T>
__device__ __forceinline__ T row_max(T v) {
  v = max(v, lane_xor<8>(v));
  v = max(v, lane_xor<4>(v));
  v = max(v, lane_xor<2>(v));
  return max(v, lane_xor<1>(v));
}

// Whether two fp32 choices lie too near for their order to be sure: scores are
// within 2^-20.5 of the formula's (exp to 3 ulps, a sum of up to 1024 terms), a
// sum of two and the compared other add up to 2^-18.5, roundings of the choices
// themselves to 2^-22 of them.
__device__ __forceinline__ bool unsure(uint32_t a, uint32_t b) {
  const float x = key_value(a), y = key_value(b);
  return !(fabsf(x - y) > 0x1p-18f * (1.f + fabsf(x)));
}
__device__ __forceinline__ bool unsure(uint64_t, uint64_t) { return false; }
__device__ __forceinline__ float key_sum(uint32_t a, uint32_t b) { return key_value(a) + key_value(b); }
__device__ __forceinline__ double key_sum(uint64_t a, uint64_t b) {
  auto value = [](uint64_t k) {
    const double v = __longlong_as_double(static_cast<int64_t>(k ^ (k >> 63 ? uint64_t(1) << 63 : ~uint64_t(0))));
    return k == ~uint64_t(0) ? __builtin_nan("") : v;
  };
  return value(a) + value(b);
}

// One token's groups and top_k from the keys of its choices, lane l holding
// experts V l .. V l + V - 1, so that of equal choices the lowest lane has the
// lowest index.  Lane j gets the j-th expert and its logit.  GUARD (fp32 keys of
// scores): false where the outcome hangs on choices that are too near.
template <typename Key, int V, bool GUARD>
__device__ __forceinline__ bool route_select(const RouteArgs& a, int lane, Key (&key)[V], const float (&x)[V], Key* s,
                                             int& my_id, float& my_x) {
  const int e = a.experts;
  const Key none = static_cast<Key>(order_key(std::conditional_t<sizeof(Key) == 8, double, float>(-__builtin_inff())));
  bool sure = true;
  // which groups stay open, from each group's rank in lanes step g (and their neighbours, if they hold it too)
  auto open_groups = [&](Key rank, int g, int step) -> uint64_t {
    rank = g < a.groups ? rank : 0;
    int better = 0;  // groups that come before this one
    for (int j = 0; j < a.groups; ++j) {
      Key o;
      if constexpr (sizeof(Key) == 8)
        o = static_cast<Key>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(rank >> 32), j * step))) << 32 |
            static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(rank), j * step));
      else
        o = static_cast<Key>(__builtin_amdgcn_readlane(static_cast<int>(rank), j * step));
      better += o > rank || (o == rank && j < g);
    }
    const bool in = g < a.groups && better < a.top_groups;
    if constexpr (GUARD) {
      const Key best_out = uniform(wave_max(in ? Key(0) : rank)), worst_in = uniform(~wave_max(in ? ~rank : Key(0)));
      if (best_out > none && unsure(worst_in, best_out)) sure = false;
    }
    return __ballot(in);
  };
  auto rank_of = [&](Key b0, Key b1) { return a.top2 && e > a.groups ? static_cast<Key>(order_key(key_sum(b0, b1))) : b0; };
  if (a.groups > 1 && !a.lanes) {  // groups of no whole lanes: lane g reads group g's choices
    const int per = e / a.groups;
#pragma unroll
    for (int v = 0; v < V; ++v) s[lane * V + v] = key[v];
    __builtin_amdgcn_wave_barrier();
    Key b0 = 0, b1 = 0;  // the group's best two
    const int base = min(lane, a.groups - 1) * per;
    for (int i = 0; i < per; i += 4) {
      Key c[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) c[q] = s[base + min(i + q, per - 1)];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const Key k = i + q < per ? c[q] : 0;
        b1 = max(b1, min(b0, k));
        b0 = max(b0, k);
      }
    }
    const uint64_t open = open_groups(rank_of(b0, b1), lane, 1);
    const float inv = 1.f / static_cast<float>(per);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int g = static_cast<int>((static_cast<float>(lane * V + v) + 0.5f) * inv);  // (lane V + v) / per: both below 2^11
      key[v] = open >> min(g, 63) & 1 ? key[v] : 0;
    }
  }
  // each lane's experts, the best first (an odd-even merge network; the lower index of equal ones)
  int at[V];
#pragma unroll
  for (int v = 0; v < V; ++v) at[v] = v;
#pragma unroll
  for (int p = 1; p < V; p *= 2)
#pragma unroll
    for (int k = p; k >= 1; k /= 2)
#pragma unroll
      for (int j = k % p; j + k < V; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; ++i)
          if (i + j + k < V && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
            const int u = i + j, v = i + j + k;
            const Key ku = key[u], kv = key[v];
            const int au = at[u], av = at[v];
            const bool swap = kv > ku || (kv == ku && av < au);
            key[u] = swap ? kv : ku;
            key[v] = swap ? ku : kv;
            at[u] = swap ? av : au;
            at[v] = swap ? au : av;
          }
  if (a.groups > 1 && a.lanes) {  // a group is a.lanes whole lanes: their best two meet by exchanges
    Key b0 = key[0], b1 = V > 1 ? key[V > 1] : 0;
    auto meet = [&](Key o0, Key o1) {
      b1 = max(min(b0, o0), max(b1, o1));
      b0 = max(b0, o0);
    };
    if (a.lanes >= 2) meet(lane_xor<1>(b0), lane_xor<1>(b1));
    if (a.lanes >= 4) meet(lane_xor<2>(b0), lane_xor<2>(b1));
    if (a.lanes >= 8) meet(half_mirror(b0), half_mirror(b1));
    if (a.lanes >= 16) meet(lane_xor<8>(b0), lane_xor<8>(b1));
    if (a.lanes >= 32) meet(lane_xor<16>(b0), lane_xor<16>(b1));
    const bool in = open_groups(rank_of(b0, b1), lane / a.lanes, a.lanes) >> lane & 1;
#pragma unroll
    for (int v = 0; v < V; ++v) key[v] = in ? key[v] : 0;
  }
  // top_k times the best that is left; who holds it is scalar work, beside the other waves' vector work
  my_id = -1;
  Key last = 0;
  for (int j = 0; j < a.top_k + (GUARD ? 1 : 0); ++j) {
    const Key best = uniform(wave_max(key[0]));
    if (best <= none) break;  // the slots left over keep id -1
    if (GUARD && j > 0 && unsure(last, best)) sure = false;
    if (GUARD && j == a.top_k) break;  // looked at only
    last = best;
    const int from = __builtin_ctzll(__ballot(key[0] == best));  // the lowest lane
    const int id = from * V + __builtin_amdgcn_readlane(at[0], from);
    const bool taken = lane == from;
#pragma unroll
    for (int v = 0; v + 1 < V; ++v) {  // (values, not elements, to choose from: no index of the lane's own)
      const Key here = key[v], next = key[v + 1];
      const int at_here = at[v], at_next = at[v + 1];
      key[v] = taken ? next : here;
      at[v] = taken ? at_next : at_here;
    }
    key[V - 1] = taken ? 0 : key[V - 1];
    my_id = lane == j ? id : my_id;
  }
  my_x = -__builtin_inff();
  const int held = max(my_id, 0);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float there = __shfl(x[v], held / V);
    my_x = my_id >= 0 && held % V == v ? there : my_x;
  }
  return sure;
}

// The same from scores in 64 bits, where the fp32 ones did not decide.  top: the
// softmax's largest logit.
template <int V>
__device__ void route_select_wide(const RouteArgs& a, int lane, const float (&x)[V], float top, uint64_t* s, int& my_id,
                                  float& my_x) {
  const float ninf = -__builtin_inff();
  double total = 1.0;
  if (!a.sigmoid) {
    double sum = 0.0;
#pragma unroll
    for (int v = 0; v < V; ++v) sum += exp(static_cast<double>(x[v]) - static_cast<double>(top));
    total = wave_sum64(sum);
    if (total == 0.0) total = 1.0;
  }
  uint64_t key[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int i = lane * V + v;
    const double l = x[v];
    const double p = a.sigmoid ? 1.0 / (1.0 + exp(-l)) : exp(l - static_cast<double>(top)) / total;
    const double c = x[v] == ninf ? static_cast<double>(ninf) : p + (a.bias ? static_cast<double>(a.bias[min(i, a.experts - 1)]) : 0.0);
    key[v] = i < a.experts ? order_key(c) : 0;
  }
  __builtin_amdgcn_wave_barrier();
  route_select<uint64_t, V, false>(a, lane, key, x, s, my_id, my_x);
}

// An fp32 score's choice.  top, total: the softmax's largest logit and sum.
__device__ __forceinline__ float route_choice(const RouteArgs& a, float x, float bias, float top, float total) {
  const float p = a.sigmoid ? 1.f / (1.f + expf(-x)) : exp_diff(x, top) / total;
  return x == -__builtin_inff() ? x : p + bias;
}

// Lanes of a group, where groups are whole lanes of v experts, a power of two of
// them; else 0.
static int route_group_lanes(const RouteArgs& a, int v) {
  const int per = a.experts / a.groups, lanes = per / v;
  return per % v == 0 && (lanes & (lanes - 1)) == 0 ? lanes : 0;
}

// Up to 256 experts and 16 of them chosen: four tokens a wave, 16 lanes each,
// lane l holding experts V l .. V l + V - 1 of its token.  A key is a choice's
// order with the expert's complement below it (32 bits where choices are 16-bit
// logits, else 64), so no two are equal and the lowest index wins ties by
// itself.  Each lane sorts its keys (an odd-even merge network: no branches),
// and the token's best is then the largest of 16 heads, top_k times.  SCORED:
// choices are scores (with a bias, or ranked by sums), compared in fp32; a token
// whose order is not sure, which takes choices within some 2^-18 of each other,
// is chosen again by the whole wave with scores in 64 bits, so that the ids are
// the formula's.
//
// Bound by instructions and, at few tokens, by their latencies.  Against one
// wave per token and the best of all keys each time, which waits on its lane
// exchanges: 16384 tokens, 8 of 256, 15.1 us in the kernel, now 6.8 (the logits'
// 8.4 MB take 1.6).
template <int XT, int V, int KM, bool SCORED>
__global__ __launch_bounds__(64 * kRouteWaves) void moe_route_rows_kernel(const RouteArgs a) {
  constexpr bool kNarrow = XT != RIA_DT_F32 && !SCORED;
  constexpr int kLow = !kNarrow ? 32 : XT == RIA_DT_BF16 ? 16 : 13;  // bits of a key below the choice's
  constexpr int kList = KM + (SCORED ? 1 : 0) < V ? KM + (SCORED ? 1 : 0) : V;  // a lane's keys that are looked at
  constexpr int kWide = V / 4;                                       // experts a lane takes with a wave to a token
  using Key = std::conditional_t<kNarrow, uint32_t, uint64_t>;
  constexpr Key kMask = (Key(1) << kLow) - 1;
  __shared__ float logits_s[SCORED ? kRouteWaves : 1][SCORED ? 4 * 16 * V : 1];
  __shared__ uint64_t wide_s[SCORED ? kRouteWaves : 1][SCORED ? 64 * kWide : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15;
  const int64_t row = ((int64_t)blockIdx.x * kRouteWaves + wave) * 4 + (lane >> 4);
  const int64_t t = min(row, (int64_t)a.tokens - 1);  // rows past the last repeat it, and store nothing
  const int e = a.experts;
  const float ninf = -__builtin_inff();
  auto row_sum = [](float v) {
    v = add_xor<8>(v);
    v = add_rn(v, __uint_as_float(lane_xor<4>(__float_as_uint(v))));
    return add_xor<1>(add_xor<2>(v));
  };
  float x[V];
  load_logits<XT, V>(a, t, l16 * V, x);
  auto top_bits = [](uint32_t o) { return kNarrow ? static_cast<Key>(o >> kLow % 32 << kLow % 32) : static_cast<Key>(o) << kLow % 64; };
  auto order_of = [](Key k) {  // the order key of a key's choice
    uint32_t o = static_cast<uint32_t>(kNarrow ? k >> kLow % 32 << kLow % 32 : k >> kLow % 64);
    if (kNarrow && !(o >> 31)) o |= static_cast<uint32_t>(kMask);  // a negative one's zeros are ones in its order
    return o;
  };
  float top = 0.f, total = 1.f;  // of the softmax: its largest logit (NaN if there is one) and its sum
  Key key[V];
  if constexpr (SCORED) {
    float bias[V];
#pragma unroll
    for (int v = 0; v < V; ++v) bias[v] = a.bias ? a.bias[min(l16 * V + v, e - 1)] : 0.f;
#pragma unroll
    for (int v = 0; v < V; v += 4)
      *reinterpret_cast<f32x4*>(&logits_s[wave][lane * V + v]) = f32x4{x[v], x[v + 1], x[v + 2], x[v + 3]};
    if (!a.sigmoid) {
      uint32_t m = 0;
#pragma unroll
      for (int v = 0; v < V; ++v) m = max(m, order_key(x[v]));
      top = key_value(row_max(m));
      if (top == ninf) top = 0.f;
      float s = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v) s += exp_diff(x[v], top);
      total = row_sum(s);
      if (total == 0.f) total = 1.f;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int i = l16 * V + v;
      const Key k = top_bits(order_key(route_choice(a, x[v], bias[v], top, total))) | (kMask - static_cast<Key>(i));
      key[v] = i < e ? k : 0;
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int i = l16 * V + v;
      const Key k = top_bits(order_key(x[v])) | (kMask - static_cast<Key>(i));
      key[v] = i < e ? k : 0;
    }
  }
#pragma unroll
  for (int p = 1; p < V; p *= 2)
#pragma unroll
    for (int k = p; k >= 1; k /= 2)
#pragma unroll
      for (int j = k % p; j + k < V; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; ++i)
          if (i + j + k < V && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
            const Key lo = min(key[i + j], key[i + j + k]);
            key[i + j] = max(key[i + j], key[i + j + k]);
            key[i + j + k] = lo;
          }
  const uint32_t none32 = order_key(ninf);
  bool sure = true;
  if (a.groups > 1) {  // a group is 1, 2, 4 or 8 whole lanes
    const int lanes = e / a.groups / V, g = l16 / lanes;
    Key b0 = key[0], b1 = key[1];  // the group's best two
    auto meet = [&](Key o0, Key o1) {
      b1 = max(min(b0, o0), max(b1, o1));
      b0 = max(b0, o0);
    };
    if (lanes >= 2) meet(lane_xor<1>(b0), lane_xor<1>(b1));
    if (lanes >= 4) meet(lane_xor<2>(b0), lane_xor<2>(b1));
    if (lanes >= 8) meet(half_mirror(b0), half_mirror(b1));
    uint32_t rank = SCORED && a.top2 ? order_key(key_sum(order_of(b0), order_of(b1))) : order_of(b0);
    rank = g < a.groups ? rank : 0;
    int better = 0;  // groups that come before this one
    for (int j = 0; j < a.groups; ++j) {
      const uint32_t o = static_cast<uint32_t>(__shfl(static_cast<int>(rank), (lane & 48) + j * lanes));
      better += o > rank || (o == rank && j < g);
    }
    const bool in = g < a.groups && better < a.top_groups;
    if constexpr (SCORED) {
      const uint32_t best_out = row_max(in ? 0u : rank), worst_in = ~row_max(in ? ~rank : 0u);
      if (best_out > none32 && unsure(worst_in, best_out)) sure = false;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) key[v] = in ? key[v] : 0;
  }
  Key mine = 0, first = 0, last = 0;
  for (int j = 0; j < a.top_k + (SCORED ? 1 : 0); ++j) {
    const Key best = row_max(key[0]);
    if constexpr (SCORED) {
      if (j > 0 && order_of(best) > none32 && unsure(order_of(last), order_of(best))) sure = false;
      if (j == a.top_k) break;  // looked at only
      last = best;
    }
    const bool taken = key[0] == best;
#pragma unroll
    for (int v = 0; v + 1 < kList; ++v) {  // (values, not elements, to choose from: no index of the lane's own)
      const Key here = key[v], next = key[v + 1];
      key[v] = taken ? next : here;
    }
    key[kList - 1] = taken ? 0 : key[kList - 1];
    if (j == 0) first = best;
    if (l16 == j) mine = best;
  }
  bool chosen = order_of(mine) > none32;
  int my_id = chosen ? static_cast<int>(kMask - (mine & kMask)) : -1;
  float my_x = ninf, m0 = 0.f;  // this lane's logit; the largest of the chosen ones, NaN if there is one
  if constexpr (SCORED) {
    __builtin_amdgcn_wave_barrier();
    if (chosen) my_x = logits_s[wave][(lane & 48) * V + my_id];
    uint64_t again = __ballot(!sure);
    while (again) {  // (the wave's: a token at a time)
      const int from = __builtin_ctzll(again) & 48;
      again &= ~(uint64_t(0xffff) << from);
      float wx[kWide];
#pragma unroll
      for (int v = 0; v < kWide; ++v) wx[v] = logits_s[wave][from * V + lane * kWide + v];
      const float its_top = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(top), from));
      int id;
      float idx;
      route_select_wide<kWide>(a, lane, wx, its_top, wide_s[wave], id, idx);
      id = __shfl(id, l16);
      idx = __shfl(idx, l16);
      if ((lane & 48) == from) {
        my_id = id;
        my_x = idx;
      }
    }
    chosen = my_id >= 0;
    const uint32_t m = row_max(chosen ? order_key(my_x) : 0u);
    if (m) m0 = key_value(m);
  } else {
    if (chosen) my_x = key_value(order_of(mine));
    if (order_of(first) > none32) m0 = key_value(order_of(first));
  }
  float w = 0.f;
  if (a.renorm) {  // about the largest chosen logit: the weights hold where every score underflows
    if (chosen) w = a.sigmoid ? sigmoid_from(my_x, m0) : exp_diff(my_x, m0);
    if (SCORED && !a.sigmoid && total != total) w = __builtin_nanf("");  // a NaN logit that was not chosen
    const float sum = row_sum(w);
    if (sum != 0.f) w = w / sum;
  } else if (a.sigmoid) {
    if (chosen) w = 1.f / (1.f + expf(-my_x));
  } else {
    if constexpr (!SCORED) {
      top = m0;  // (the largest logit's group is always open)
      float s = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v) s += exp_diff(x[v], top);
      total = row_sum(s);
    }
    if (chosen) w = exp_diff(my_x, top) / total;
  }
  if (row >= a.tokens) return;
  if (l16 < a.top_k) {
    a.weights[t * a.w_stride + l16] = w * a.scale;
    a.ids[t * a.id_stride + l16] = my_id;
  }
  if (a.shared && l16 == 15) route_shared<XT>(a, t);
}

// One wave per token: scores of few tokens, many experts, groups of no whole
// lanes.  SCORED as above, or with a.wide in 64 bits at once.  Bound by each
// choice's chain of exchanges: 4099 tokens, 8 of 256 in 4 of 8 groups with a bias
// and a shared expert, 12.6 us; 16.2 with the choices unsorted in their lanes and
// the groups' best read back from LDS.
template <int XT, int V, bool SCORED>
__global__ __launch_bounds__(64 * kRouteWaves) void moe_route_kernel(const RouteArgs a) {
  __shared__ uint64_t group_s[kRouteWaves][64 * V];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t t = (int64_t)blockIdx.x * kRouteWaves + wave;
  if (t >= a.tokens) return;
  const int e = a.experts;
  const float ninf = -__builtin_inff();
  float x[V];
  load_logits<XT, V>(a, t, lane * V, x);
  // the softmax's largest logit (NaN if there is one) and normaliser
  float top = 0.f, total = 1.f;
  if (!a.sigmoid && (SCORED || !a.renorm)) {
    uint32_t m = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) m = max(m, order_key(x[v]));
    top = key_value(wave_max(m));
    if (top == ninf) top = 0.f;
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) s += exp_diff(x[v], top);
    total = wave_sum(s);
    if (total == 0.f) total = 1.f;
  }
  int my_id;
  float my_x;
  if constexpr (SCORED) {
    bool sure = false;
    if (!a.wide) {
      float bias[V];
#pragma unroll
      for (int v = 0; v < V; ++v) bias[v] = a.bias ? a.bias[min(lane * V + v, e - 1)] : 0.f;
      uint32_t key[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const uint32_t k = order_key(route_choice(a, x[v], bias[v], top, total));
        key[v] = lane * V + v < e ? k : 0;
      }
      sure = route_select<uint32_t, V, true>(a, lane, key, x, reinterpret_cast<uint32_t*>(group_s[wave]), my_id, my_x);
    }
    if (!sure) route_select_wide<V>(a, lane, x, top, group_s[wave], my_id, my_x);
  } else {
    uint32_t key[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const uint32_t k = order_key(x[v]);
      key[v] = lane * V + v < e ? k : 0;
    }
    route_select<uint32_t, V, false>(a, lane, key, x, reinterpret_cast<uint32_t*>(group_s[wave]), my_id, my_x);
  }
  // the chosen scores (lanes 0 .. top_k - 1)
  float w = 0.f;
  if (a.renorm) {
    // about the largest chosen logit: the weights hold where every score underflows
    const uint32_t m = wave_max(my_id >= 0 ? order_key(my_x) : 0u);
    const float m0 = m == 0 ? 0.f : key_value(m);
    if (my_id >= 0) w = a.sigmoid ? sigmoid_from(my_x, m0) : exp_diff(my_x, m0);
    if (SCORED && !a.sigmoid && total != total) w = __builtin_nanf("");  // a NaN logit that was not chosen
    const float sum = wave_sum(w);
    if (sum != 0.f) w = w / sum;
  } else if (my_id >= 0) {
    w = a.sigmoid ? 1.f / (1.f + expf(-my_x)) : exp_diff(my_x, top) / total;
  }
  if (lane < a.top_k) {
    a.weights[t * a.w_stride + lane] = w * a.scale;
    a.ids[t * a.id_stride + lane] = my_id;
  }
  if (a.shared && lane == 63) route_shared<XT>(a, t);
}

// Scores of fewer tokens are chosen by a wave each: its chain of instructions is
// shorter.  256 experts, a wave for four tokens / for one: with 8 groups and a bias
// 4099 tokens 15.0 / 12.1 us, 16384 tokens 24.4 / 23.8, 65536 tokens 61 / 74; with
// a bias alone 15.7 / 9.9, 21.6 / 19.5, 55 / 59; a softmax with a bias 15.0 / 11.6,
// 27.2 / 24.4, 65 / 75.
constexpr int kRouteRowsTokens = 32768;

// Where some token is likely to be chosen again (one in fifty is) and the card has
// room, all of them are chosen in 64 bits at once: the end of a launch is then
// one choice's chain, not two.  256 experts, at once / fp32 first, with 8 groups
// and a bias: 16 tokens 7.0 / 6.6 us or, with one chosen again, 8.4; 512 tokens
// 7.1 / 9.2, 2048 tokens 8.2 / 10.1, 4099 tokens 11.9 / 12.0, 8192 tokens 17.0 /
// 15.9; with a bias alone 512 tokens 7.0 / 7.6, 2048 tokens 7.2 / 8.7, 4099 tokens
// 10.1 / 9.9, 8192 tokens 14.5 / 12.8.
constexpr int kRouteWideFrom = 32, kRouteWideTo = 3200;

template <int XT, bool SCORED>
static void launch_route(RouteArgs a, hipStream_t st) {
  const bool few = a.top_k <= 8;
  const int per_lane = a.experts <= 64 ? 4 : a.experts <= 128 && few ? 8 : 16;
  if (a.experts <= 256 && a.top_k <= 16 && (a.groups == 1 || route_group_lanes(a, per_lane)) &&
      (!SCORED || a.tokens >= kRouteRowsTokens)) {
    a.lanes = route_group_lanes(a, per_lane / 4);  // of a token that the whole wave chooses again
    const dim3 grid((a.tokens + 4 * kRouteWaves - 1) / (4 * kRouteWaves)), block(64 * kRouteWaves);
    if (per_lane == 4)
      hipLaunchKernelGGL((moe_route_rows_kernel<XT, 4, 16, SCORED>), grid, block, 0, st, a);
    else if (per_lane == 8)
      hipLaunchKernelGGL((moe_route_rows_kernel<XT, 8, 8, SCORED>), grid, block, 0, st, a);
    else if (few)
      hipLaunchKernelGGL((moe_route_rows_kernel<XT, 16, 8, SCORED>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((moe_route_rows_kernel<XT, 16, 16, SCORED>), grid, block, 0, st, a);
    return;
  }
  const dim3 grid((a.tokens + kRouteWaves - 1) / kRouteWaves), block(64 * kRouteWaves);
  const int v = a.experts <= 64 ? 1 : a.experts <= 256 ? 4 : a.experts <= 512 ? 8 : 16;
  a.lanes = route_group_lanes(a, v);
  if (v == 1)
    hipLaunchKernelGGL((moe_route_kernel<XT, 1, SCORED>), grid, block, 0, st, a);
  else if (v == 4)
    hipLaunchKernelGGL((moe_route_kernel<XT, 4, SCORED>), grid, block, 0, st, a);
  else if (v == 8)
    hipLaunchKernelGGL((moe_route_kernel<XT, 8, SCORED>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((moe_route_kernel<XT, 16, SCORED>), grid, block, 0, st, a);
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
  int32_t* order;  // the pair at each position of the sorted ones
  int32_t* where;  // the position of each pair of an expert
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

// Running sums of the experts' pairs and tiles (thread t: experts per t .. per t
// + per - 1), this workgroup's first position of each expert, and its pairs' places.
// Which of an expert's positions a pair gets does not change its results.  Terms
// are kept in the order of the positions, so that a tile's stores are neighbours:
// 16384 tokens' down rows 362 us, 385 with the terms at their pairs' places.
__device__ __forceinline__ void plan_place(const PlanArgs& a, int block, PlanShared& s, const int (&e)[kPlanPer]) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per = (a.experts + 255) / 256;
  int total[4], before[4], sum = 0, tiles = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int x = per * tid + j;
    total[j] = before[j] = 0;
    if (j < per && x < a.experts) {
      if (a.blocks == 1) {
        total[j] = s.count[x];
      } else {
#pragma unroll 16
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
    const int x = per * tid + j;
    if (j < per && x < a.experts) {
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
    if (e[i] >= 0) {
      const int pair = block * kPlanPairs + i * 256 + tid, at = atomicAdd(&s.count[e[i]], 1);
      a.order[at] = pair;
      a.where[pair] = at;
    }
}

// First launch: workgroups 0 .. blocks - 1 count their pairs' experts (a lone
// one places them too), the others quantise x.  16384 tokens of 2048 values in
// bf16, 8 of 256 experts: 20.5 us (102 MB at 5 TB/s), the placing launch 16 (its
// chain of loads: ids, the other workgroups' counts).
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

// ---- a few tokens: each (token, slot) pair by itself
//
// The time is the weights' way from HBM: they go straight into MFMA operands (16
// rows x 128 bytes of K per product, widened to fp16), by many small workgroups
// with all of their loads in flight, and nothing is planned or sorted first.
constexpr int kFewAhead = 4;      // blocks of K a wave loads at once
constexpr int kFewChunk = 2048;   // hidden values quantised into LDS at a time

struct PairsArgs {
  const int32_t* ids;
  int64_t id_stride;
  const void* x;
  int64_t x_stride;
  const float* pair_w;
  int64_t pair_w_stride;
  int tokens, top_k, experts, hidden, inter;
  const uint8_t* w13;
  const float* s13;
  const uint8_t* w2;
  const float* s2;
  float* act;                     // [pairs, inter]: SiLU(g) u
  void* out;
  int out_dtype;
  int64_t out_stride;
  int add;
};

// act = SiLU(g) u of one pair and 16 features, four waves sharing K; x is
// quantised here.  Column 0 of the products is the pair's (all 16 are).
template <int XT>
__global__ __launch_bounds__(256) void moe_up_pairs_kernel(const PairsArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t xq_s[];  // hidden e4m3 values, then their scales
  __shared__ float red[4][2][16];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int groups = a.inter / 16;
  const int pair = blockIdx.x / groups, c0 = blockIdx.x % groups * 16;
  const int token = pair / a.top_k;
  const int expert = __builtin_amdgcn_readfirstlane(a.ids[(int64_t)token * a.id_stride + pair % a.top_k]);
  if (expert < 0 || expert >= a.experts) return;
  const int k = a.hidden, kblocks = k / kX8Block;
  const uint8_t* wg = a.w13 + ((int64_t)expert * 2 * a.inter + c0) * k;
  const uint8_t* wu = wg + (int64_t)a.inter * k;
  const float* sg = a.s13 + ((int64_t)expert * 2 * (a.inter / kX8Block) + c0 / kX8Block) * kblocks;
  const float* su = sg + (int64_t)(a.inter / kX8Block) * kblocks;
  u32x4 g[kFewAhead][2], u[kFewAhead][2];
  float fg[kFewAhead], fu[kFewAhead];
  auto load = [&](int kb0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kFewAhead; ++i) {
      const int kb = min(kb0 + i, kblocks - 1);
      load_rows16(wg, k, kb, lane, g[i]);
      load_rows16(wu, k, kb, lane, u[i]);
    }
#pragma unroll
    for (int i = 0; i < kFewAhead; ++i) {
      const int kb = min(kb0 + i, kblocks - 1);
      fg[i] = sg[kb];
      fu[i] = su[kb];
    }
    __builtin_amdgcn_sched_barrier(0);  // all of them in flight before the first product
  };
  load(wave * kFewAhead);
  float* qs = reinterpret_cast<float*>(xq_s + k);
  for (int c = 8 * tid; c < k; c += 8 * 256) {
    float v[8];
    load_act8<XT>(a.x, token * a.x_stride + c, v);
    quant_eight(v, xq_s + c, qs + c / kX8Block, tid);
  }
  lds_barrier();
  f32x4 ag{0.f, 0.f, 0.f, 0.f}, au = ag;
  for (int kb0 = wave * kFewAhead; kb0 < kblocks; kb0 += 4 * kFewAhead) {
#pragma unroll
    for (int i = 0; i < kFewAhead; ++i) {
      const int kb = kb0 + i;
      if (kb >= kblocks) break;
      u32x4 b[2];
      load_chunks(xq_s + kb * kX8Block, lane, b);
      const f32x4 pg = mfma_x8_16(g[i], b), pu = mfma_x8_16(u[i], b);
      const float s0 = qs[kb] * fg[i], s1 = qs[kb] * fu[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        ag[j] = fmaf(pg[j], s0, ag[j]);
        au[j] = fmaf(pu[j], s1, au[j]);
      }
    }
    if (kb0 + 4 * kFewAhead < kblocks) load(kb0 + 4 * kFewAhead);
  }
  if ((lane & 15) == 0) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      red[wave][0][4 * (lane >> 4) + j] = ag[j];
      red[wave][1][4 * (lane >> 4) + j] = au[j];
    }
  }
  __syncthreads();
  if (tid < 16) {
    const float gate = (red[0][0][tid] + red[1][0][tid]) + (red[2][0][tid] + red[3][0][tid]);
    const float up = (red[0][1][tid] + red[1][1][tid]) + (red[2][1][tid] + red[3][1][tid]);
    a.act[(int64_t)pair * a.inter + c0 + tid] = x8_swiglu(gate, up);
  }
}

// 16 features of one token's sum, a wave for each slot (in turns of
// kSumWaves); the terms meet in LDS and are added in slot order.
constexpr int kSumWaves = 8;
__global__ __launch_bounds__(64 * kSumWaves) void moe_down_pairs_kernel(const PairsArgs a) {
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
            for (int c = 8 * lane; c < cols; c += 8 * 64) {
              float h[8];
              load_act8<RIA_DT_F32>(act, c0 + c, h);
              quant_eight(h, h_s[wave] + c, &hs_s[wave][c / kX8Block], lane);
            }
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
      for (int q = 0; q < 4; ++q) term[wave][4 * (lane >> 4) + q] = some ? pw * acc[q] : 0.f;
    }
    __syncthreads();
    if (tid < 16)
      for (int w = 0; w < min(kSumWaves, a.top_k - j0); ++w) sum = add_rn(sum, term[w][tid]);
    __syncthreads();
  }
  if (tid < 16) {
    const int64_t o = (int64_t)t * a.out_stride + n0 + tid;
    if (a.add) sum = add_rn(static_cast<const float*>(a.out)[o], sum);
    store_act_dt(a.out, o, sum, a.out_dtype);
  }
}

struct CombineArgs {
  const void* slots;      // [positions, hidden]: fp32, or fp16 times 2^(e - 127)
  const uint8_t* slot_e;  // e [positions, hidden / 64]
  const int32_t* where;   // the position of each pair of an expert
  const int32_t* ids;
  int64_t id_stride;
  int tokens, top_k, experts, hidden;
  void* out;
  int out_dtype;
  int64_t out_stride;
  int add, vec;
};
constexpr int kCombineAhead = 4;  // slots loaded ahead of their sums

// out[t] (+)= the sum of the token's slots in slot order, in fp32; slots of no
// expert are left out (position 0 is loaded for them, and not used).
// Bound by the slots' way from HBM.  STREAM: past the caches, where the slots
// outgrow them: 16384 tokens, 8 slots of 2048 values, 609 MB in 104 us (5.9 TB/s),
// some 18 more through the caches; 33 MB of slots take the same either way.
template <int DT, bool STREAM>
__global__ __launch_bounds__(256) void moe_combine_kernel(const CombineArgs a) {
  constexpr int kRaw = DT == RIA_DT_F32 ? 2 : 1;  // 16-byte loads of a slot
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int per = a.hidden / 8;
  const int64_t t = u / per;
  if (t >= a.tokens) return;
  const int c = static_cast<int>(u - t * per) * 8;
  float s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = 0.f;
  for (int j0 = 0; j0 < a.top_k; j0 += kCombineAhead) {
    u32x4 raw[kCombineAhead][kRaw];
    bool on[kCombineAhead];
    int64_t pos[kCombineAhead];
    uint32_t e[kCombineAhead];
#pragma unroll
    for (int j = 0; j < kCombineAhead; ++j) {
      const int at = min(j0 + j, a.top_k - 1);
      const int id = a.ids[t * a.id_stride + at], p = a.where[t * a.top_k + at];
      on[j] = j0 + j < a.top_k && id >= 0 && id < a.experts;
      pos[j] = on[j] ? p : 0;
    }
#pragma unroll
    for (int j = 0; j < kCombineAhead; ++j) {
      if constexpr (DT != RIA_DT_F32) e[j] = a.slot_e[pos[j] * (a.hidden / 64) + c / 64];
      const u32x4* p = static_cast<const u32x4*>(a.slots) + (pos[j] * a.hidden + c) / 8 * kRaw;
#pragma unroll
      for (int i = 0; i < kRaw; ++i) raw[j][i] = STREAM ? __builtin_nontemporal_load(p + i) : p[i];
    }
#pragma unroll
    for (int j = 0; j < kCombineAhead; ++j) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float v;
        if constexpr (DT == RIA_DT_F32)
          v = __uint_as_float(raw[j][i / 4][i % 4]);
        else
          v = f16_bits_to_f32(static_cast<uint16_t>(raw[j][0][i / 2] >> (16 * (i % 2)))) * x8_scale(e[j]);
        s[i] = add_rn(s[i], on[j] ? v : 0.f);
      }
    }
  }
  X8Args o{};
  o.y = a.out;
  o.y_dtype = a.out_dtype;
  o.y_add = a.add;
  o.vec = a.vec;
  store_eight(o, t * a.out_stride + c, s);
}

static int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

// Most tiles of any routing: an expert's last tile may be partly filled.
static int64_t moe_tiles(int64_t pairs, int experts, int tile) {
  return std::min<int64_t>(pairs, pairs / tile + std::min<int64_t>(experts, pairs));
}

// Whether each pair is run by itself.  That reads an expert's weights again for
// each further pair of it, but saves the planning and combining launches, some
// 10 us: with the pairs spread evenly, up to 40 MB of repeated weights.
// Measured by pairs / in tiles of 64 (experts, top_k, hidden, inter): (256, 8,
// 2048, 512) 8 tokens 39 / 49 us, 16 tokens 67 / 75, 32 tokens 118 / 113; (16, 2,
// 2048, 1024) 8 tokens 25 / 33, 16 tokens 38 / 34; (60, 4, 1024, 768) 8 tokens
// 24 / 27, 16 tokens 40 / 30.
static bool moe_by_pairs(int64_t pairs, int experts, int hidden, int inter) {
  if (pairs > 512) return false;
  const double met = experts * (1.0 - std::pow(1.0 - 1.0 / experts, static_cast<double>(pairs)));
  return (pairs - met) * 3.0 * hidden * inter <= 40e6;
}

// Whether most experts' pairs fill one tile: the time is the weights' then.  They
// are read once and kept in no cache (a pure read of 512 MB: 5.8 TB/s, 6.5 past
// the caches), and widened for the products, which costs next to nothing beside
// the reading: (256, 8, 2048, 512) 128 tokens 140 us, 144 in e4m3 products, 158
// through the caches; 1024 tokens 189, 182 and 204.
static bool moe_once(int64_t pairs, int experts) { return pairs <= (int64_t)experts * 32; }

// Gate and up tiles of 64 pairs, with an expert's last one half full.
static int64_t moe_tiles64(int64_t pairs, int experts, int inter) {
  return static_cast<int64_t>(static_cast<double>(pairs) / 64 + 0.5 * experts) * (inter / 128);
}

// Pairs of one expert that a tile takes.  32 or 64 for the weights' way from HBM:
// (256, 8, 2048, 512) tiles of 32 / 64: 128 tokens 140 / 157 us, 512 tokens 159 /
// 169, 768 tokens 184 / 182.  64 or 256 by rounds of the gate and up tiles over
// the card, with the pairs spread evenly and an expert's last tile half full: two
// tiles of 64 to a CU, one of 256, whose round takes 1.5 times as long.  Measured
// on both sides, 64 / 256: (256, 8, 2048, 512) 2048 tokens 241 / 285 us, 4096
// tokens 322 / 340, 6000 tokens 408 / 375, 16384 tokens 963 / 836; (16, 2, 4096,
// 2048) 512 tokens 134 / 130, 1024 tokens 178 / 150, 3000 tokens 364 / 258; (16,
// 2, 2048, 1024) 1024 tokens 56 / 68; (60, 4, 1024, 768) 4096 tokens 103 / 122,
// 6000 tokens 134 / 132; (64, 6, 1024, 512) 1024 tokens 54 / 58, 2048 tokens 74 /
// 69.  (Only a bf16 x has kernels of 256: widened operands' registers do not fit.)
static int moe_tile(int64_t pairs, int experts, int inter, int x_dtype) {
  if (pairs <= (int64_t)experts * 16) return 32;
  if (x_dtype != RIA_DT_BF16 || moe_once(pairs, experts)) return 64;
  const int64_t cus = device_cus(), across = inter / 128;
  const double each = static_cast<double>(pairs) / experts;
  const int64_t n64 = moe_tiles64(pairs, experts, inter);
  const int64_t n256 = static_cast<int64_t>(experts * (each <= 224 ? 1.0 : each / 256 + 0.5)) * across;
  const int64_t rounds64 = (n64 + 2 * cus - 1) / (2 * cus), rounds256 = (n256 + cus - 1) / cus;
  return 3 * rounds256 < 2 * rounds64 ? 256 : 64;
}

struct MoeLayout {
  int64_t x8, xs, counts, order, where, tiles, ntiles, act, h8, hs, slots, slot_e, bytes;
};
static MoeLayout moe_layout(int64_t tokens, int top_k, int experts, int hidden, int inter, int x_dtype) {
  MoeLayout l{};
  const int64_t pairs = tokens * top_k;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += align256(bytes);
    return here;
  };
  if (moe_by_pairs(pairs, experts, hidden, inter)) {
    l.act = take(pairs * inter * 4);
  } else {
    l.x8 = take(tokens * hidden);
    l.xs = take(tokens * (hidden / kX8Block) * 4);
    l.counts = take((pairs + kPlanPairs - 1) / kPlanPairs * experts * 4);
    l.order = take(pairs * 4);
    l.where = take(pairs * 4);
    l.tiles = take(moe_tiles(pairs, experts, moe_tile(pairs, experts, inter, x_dtype)) * static_cast<int64_t>(sizeof(X8Tile)));
    l.ntiles = take(4);
    l.h8 = take(pairs * inter);
    l.hs = take(pairs * (inter / kX8Block) * 4);
    l.slots = take(pairs * hidden * (x_dtype == RIA_DT_F32 ? 4 : 2));
    l.slot_e = take(x_dtype == RIA_DT_F32 ? 0 : pairs * (hidden / 64));
  }
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
  const int64_t pairs = (int64_t)d.tokens * d.top_k;
  const bool wide = d.x_dtype == RIA_DT_F32, once = moe_once(pairs, d.experts);
  // tiles of 64 in e4m3 products: one LDS buffer where there are more than two for a CU.  (256, 8, 2048, 512) 4096 tokens
  // 311 us, 322 with two buffers, (60, 4, 1024, 768) 4096 tokens 100 and 104; (8, 2, 4096, 1024) 512 tokens 72 and 60
  const bool many = moe_tiles64(pairs, d.experts, d.inter) > 2 * (int64_t)device_cus();
  auto grid_of = [&](int feature_tiles) { return dim3(static_cast<unsigned>((most * feature_tiles + 7) / 8 * 8)); };
  // Where the e4m3 products' 3e-5 carry a hidden value over a rounding border of e4m3, it moves by up to 2^-3: results
  // are 1e-3 off (2-norm) by that, four times an fp16 rounding, half a bf16 one.  So only a bf16 x takes them here; an
  // fp16 one's gate and up rows are summed from widened operands, as an fp32 one's are (16384 tokens, 8 of 256 experts
  // of 2048 x 512: 1121 us, 840 without; 2048 tokens 249 and 240).
  const bool wide_up = d.x_dtype != RIA_DT_BF16;
  if (tile == 32)
    hipLaunchKernelGGL((x8_tile_kernel<kX8Up, 2, 1, 4, 1, true, true>), grid_of(d.inter / 128), dim3(256), 0, st, up);
  else if (once)
    hipLaunchKernelGGL((x8_tile_kernel<kX8Up, 2, 2, 4, 1, true, true>), grid_of(d.inter / 128), dim3(256), 0, st, up);
  else if (tile == 256)
    hipLaunchKernelGGL((x8_tile_kernel<kX8Up, 4, 2, 2, 4, false>), grid_of(d.inter / 128), dim3(512), 0, st, up);
  else if (wide_up)
    hipLaunchKernelGGL((x8_tile_kernel<kX8Up, 2, 2, 4, 1, true>), grid_of(d.inter / 128), dim3(256), 0, st, up);
  else if (many)
    hipLaunchKernelGGL((x8_tile_kernel<kX8Up, 2, 2, 4, 1, false, false, 3>), grid_of(d.inter / 128), dim3(256), 0, st, up);
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
  dn.y_dtype = wide ? RIA_DT_F32 : RIA_DT_F16;
  dn.ye = static_cast<uint8_t*>(at(l.slot_e));
  dn.ye_stride = d.hidden / 64;
  dn.vec = 1;
  dn.pair_w = d.weights;
  dn.pair_w_stride = d.weights_row_stride;
  if (tile == 32)
    hipLaunchKernelGGL((x8_tile_kernel<kX8Down, 2, 1, 2, 1, true, true>), grid_of(d.hidden / 128), dim3(128), 0, st, dn);
  else if (once)
    hipLaunchKernelGGL((x8_tile_kernel<kX8Down, 2, 1, 2, 2, true, true>), grid_of(d.hidden / 128), dim3(256), 0, st, dn);
  else if (wide)
    hipLaunchKernelGGL((x8_tile_kernel<kX8Down, 2, 1, 2, 2, true>), grid_of(d.hidden / 128), dim3(256), 0, st, dn);
  else if (tile == 256)
    hipLaunchKernelGGL((x8_tile_kernel<kX8Down, 4, 2, 2, 4, false>), grid_of((d.hidden + 255) / 256), dim3(512), 0, st, dn);
  else if (many)
    hipLaunchKernelGGL((x8_tile_kernel<kX8Down, 2, 1, 2, 2, false, false, 4>), grid_of(d.hidden / 128), dim3(256), 0, st, dn);
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
  const int size = logits_dtype == RIA_DT_F32 ? 4 : 2;
  const bool vec = experts % 4 == 0 && logits_row_stride % 4 == 0 && reinterpret_cast<uintptr_t>(logits) % (4 * size) == 0;
  const RouteArgs a{logits, logits_row_stride, tokens, experts, top_k, bias, scoring == RIA_ROUTE_SIGMOID, num_groups,
                    top_groups, group_score == RIA_ROUTE_GROUP_TOP2, renormalize != 0, s, scale, weights,
                    weights_row_stride, ids, ids_row_stride, vec, tokens >= kRouteWideFrom && tokens < kRouteWideTo, 0};
  // scores need comparing where a bias or a sum of two stands between them and the logits
  const bool scored = bias || (num_groups > 1 && group_score == RIA_ROUTE_GROUP_TOP2);
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto launch = [&](auto dt) {
    constexpr int XT = decltype(dt)::value;
    if (scored)
      launch_route<XT, true>(a, st);
    else
      launch_route<XT, false>(a, st);
  };
  if (logits_dtype == RIA_DT_BF16)
    launch(std::integral_constant<int, RIA_DT_BF16>{});
  else if (logits_dtype == RIA_DT_F16)
    launch(std::integral_constant<int, RIA_DT_F16>{});
  else
    launch(std::integral_constant<int, RIA_DT_F32>{});
  return check_launch(who);
}

extern "C" int64_t ria_moe_experts_workspace_bytes(int tokens, int top_k, int experts, int hidden, int inter,
                                                   int x_dtype) {
  if (moe_sizes_error(tokens, top_k, experts, hidden, inter) || !x8_dtype_ok(x_dtype)) return -1;
  return moe_layout(tokens, top_k, experts, hidden, inter, x_dtype).bytes;
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
  const MoeLayout l = moe_layout(d->tokens, d->top_k, d->experts, d->hidden, d->inter, d->x_dtype);
  if (d->workspace_bytes < l.bytes)
    return set_error(RIA_ERR_WORKSPACE, "%s: workspace of %lld bytes, %lld needed", who, (long long)d->workspace_bytes,
                     (long long)l.bytes);
  hipStream_t st = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(d->workspace);
  auto at = [&](int64_t o) { return static_cast<void*>(ws + o); };
  const int64_t pairs = (int64_t)d->tokens * d->top_k;
  if (moe_by_pairs(pairs, d->experts, d->hidden, d->inter)) {
    const PairsArgs p{d->ids, d->ids_row_stride, d->x, d->x_row_stride, d->weights, d->weights_row_stride, d->tokens,
                      d->top_k, d->experts, d->hidden, d->inter, static_cast<const uint8_t*>(d->w13), d->w13_scale_inv,
                      static_cast<const uint8_t*>(d->w2), d->w2_scale_inv, static_cast<float*>(at(l.act)), d->out,
                      d->out_dtype, d->out_row_stride, d->accumulate != 0};
    const dim3 ugrid(static_cast<unsigned>(pairs * (d->inter / 16)));
    const dim3 dgrid(static_cast<unsigned>((int64_t)d->tokens * (d->hidden / 16)));
    const size_t lds = d->hidden + d->hidden / kX8Block * 4;
    if (d->x_dtype == RIA_DT_BF16)
      hipLaunchKernelGGL((moe_up_pairs_kernel<RIA_DT_BF16>), ugrid, dim3(256), lds, st, p);
    else if (d->x_dtype == RIA_DT_F16)
      hipLaunchKernelGGL((moe_up_pairs_kernel<RIA_DT_F16>), ugrid, dim3(256), lds, st, p);
    else
      hipLaunchKernelGGL((moe_up_pairs_kernel<RIA_DT_F32>), ugrid, dim3(256), lds, st, p);
    hipLaunchKernelGGL(moe_down_pairs_kernel, dgrid, dim3(64 * kSumWaves), 0, st, p);
    return check_launch(who);
  }
  const int tile = moe_tile(pairs, d->experts, d->inter, d->x_dtype);
  const int64_t most = moe_tiles(pairs, d->experts, tile);
  if (most * (std::max(d->hidden, d->inter) / 128) > 0x7ffffff0)
    return set_error(RIA_ERR_INVALID, "%s: too many (token, slot) pairs", who);
  const PlanArgs plan{d->ids, d->ids_row_stride, static_cast<int>(pairs), d->top_k, d->experts,
                      static_cast<int>((pairs + kPlanPairs - 1) / kPlanPairs), tile, static_cast<int32_t*>(at(l.counts)),
                      static_cast<int32_t*>(at(l.order)), static_cast<int32_t*>(at(l.where)),
                      static_cast<X8Tile*>(at(l.tiles)), static_cast<int32_t*>(at(l.ntiles))};
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
  launch_moe_tiles(*d, l, most, tile, st);
  const CombineArgs c{at(l.slots), static_cast<const uint8_t*>(at(l.slot_e)),
                      static_cast<const int32_t*>(at(l.where)), d->ids, d->ids_row_stride, d->tokens,
                      d->top_k, d->experts, d->hidden, d->out, d->out_dtype, d->out_row_stride, d->accumulate != 0,
                      reinterpret_cast<uintptr_t>(d->out) % 16 == 0 && d->out_row_stride % 8 == 0};
  const dim3 grid(static_cast<unsigned>(((int64_t)d->tokens * (d->hidden / 8) + 255) / 256));
  if (d->x_dtype == RIA_DT_F32)
    hipLaunchKernelGGL((moe_combine_kernel<RIA_DT_F32, false>), grid, dim3(256), 0, st, c);
  else if (pairs * d->hidden * 2 >= int64_t(32) << 20)
    hipLaunchKernelGGL((moe_combine_kernel<RIA_DT_F16, true>), grid, dim3(256), 0, st, c);
  else
    hipLaunchKernelGGL((moe_combine_kernel<RIA_DT_F16, false>), grid, dim3(256), 0, st, c);
  return check_launch(who);
}
