// Products of e4m3 activations with block-FP8 weights, shared by the dense
// product (linear_x8.hip) and the experts (moe.hip).
//
// Both operands are float8_e4m3fn with scales of their own: one fp32 per 128
// values of an activation row, one per 128 x 128 block of a weight, as block-FP8
// checkpoints store them.  With kb running over the blocks of K,
//
//     y[m, n] = sum_kb xs[m, kb] ws[n / 128, kb] (sum_{k in kb} x8[m, k] w8[n, k])
//
// The inner sum is the matrix cores', the outer one an fp32 FMA per result and
// block.
#pragma once

#include "ria_common.h"

namespace ria {

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kX8Block = 128;  // values per scale

// The matrix cores' e4m3 products: each group of 16 is aligned to its largest
// and cut 13 bits below it (measured on single pairs: 2^14 + 2^1 is exact, of
// 2^14 + 2^0 the second is lost), which leaves results 3e-5 of their size off
// (2-norm, normal inputs): 1/16 of a rounding to fp16.  Where a result stays in
// fp32, and in the streaming kernels, which wait for memory anyway, both
// operands are widened to fp16 instead (exact: e4m3 fits) and summed in fp32.

// Two e4m3 bytes of w (low or high pair) as fp16.
template <bool HIGH>
__device__ __forceinline__ uint32_t x8_to_f16x2(int w) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HIGH));
}
__device__ __forceinline__ u32x4 x8_to_f16x8(int w0, int w1) {
  return u32x4{x8_to_f16x2<false>(w0), x8_to_f16x2<true>(w0), x8_to_f16x2<false>(w1), x8_to_f16x2<true>(w1)};
}

// 32x32 (K 64) and 16x16 (K 128) products of e4m3 operands, 32 bytes a lane: a
// lane's bytes are one row's (l % 32 or l % 16), its K part l / 32 or l / 16.
// Which K a byte stands for does not matter as long as both operands agree.
template <bool WIDE>
__device__ __forceinline__ f32x16 mfma_x8_32(i32x8 a, i32x8 b, f32x16 c) {
  if constexpr (WIDE) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      c = Kv16<RIA_DT_F16>::mfma32(x8_to_f16x8(a[2 * i], a[2 * i + 1]), x8_to_f16x8(b[2 * i], b[2 * i + 1]), c);
    return c;
  } else {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
  }
}

__device__ __forceinline__ i32x8 join_x8(u32x4 lo, u32x4 hi) {
  return i32x8{static_cast<int>(lo[0]), static_cast<int>(lo[1]), static_cast<int>(lo[2]), static_cast<int>(lo[3]),
               static_cast<int>(hi[0]), static_cast<int>(hi[1]), static_cast<int>(hi[2]), static_cast<int>(hi[3])};
}

// ---- quantisation: x8 = e4m3(x / s), s the smallest power of two with |x| / s <= 448
// for every finite x of the block (1 for a block of zeros, 2^-126 at the least).
// A power of two makes x / s exact, so the only rounding is the one to e4m3 and
// every arithmetic finds the same bits; e4m3 is a floating type, so values
// but the smallest (below 2^-15 of the largest) lose nothing against amax / 448.

// |x| with infinities and NaN as 0: they do not set the block's scale.
__device__ __forceinline__ float finite_abs(float x) {
  const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
  return u < 0x7f800000u ? __uint_as_float(u) : 0.f;
}

// Biased exponent of the scale of a block whose largest finite |x| is top (448 = 1.75 2^8).
__device__ __forceinline__ uint32_t x8_scale_exp(float top) {
  const uint32_t u = __float_as_uint(top);
  if (u == 0) return 127;
  const int e = static_cast<int>(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return static_cast<uint32_t>(max(e, 1));
}
__device__ __forceinline__ float x8_scale(uint32_t e) { return __uint_as_float(e << 23); }
__device__ __forceinline__ float x8_inverse(uint32_t e) { return __uint_as_float((254u - e) << 23); }

// Infinities become NaN (e4m3fn has no infinity).
__device__ __forceinline__ float x8_value(float x, float inv) {
  const float v = x * inv;
  return (__float_as_uint(x) & 0x7fffffffu) < 0x7f800000u ? v : __uint_as_float(0x7fc00000u);
}

__device__ __forceinline__ uint32_t pack_x8(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
}

// Largest over each group of 16 lanes.
__device__ __forceinline__ float row16_max(float v) {
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x128, 0xf, 0xf, true)));  // row_ror:8
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x124, 0xf, 0xf, true)));  // row_ror:4
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x4E, 0xf, 0xf, true)));   // quad_perm
  return fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0xB1, 0xf, 0xf, true)));
}

// ---- the tiled product
enum X8Mode {
  kX8Dense = 0,  // y [m, n]
  kX8Up = 1,     // an expert's gate and up rows of its tokens, SwiGLU, quantised
  kX8Down = 2    // an expert's down rows of its pairs, times the router's weight, to the pair's slot
};

struct X8Tile {  // rows of one expert that a workgroup takes: positions first .. first + rows - 1
  int32_t expert, first, rows, pad;
};

struct X8Args {
  const uint8_t* x;  // e4m3 rows
  int64_t x_stride;
  const float* xs;   // their scales
  int64_t xs_stride;
  const uint8_t* w;  // [n, k] e4m3, of each expert in turn
  const float* ws;   // [ceil(n / 128), k / 128]
  int m, n, k;
  void* y;
  int64_t y_stride;
  int y_dtype, y_add;
  int vec;           // y and its rows are 16-byte aligned
  // experts: position p of the sorted (token, slot) pairs is pair order[p] = token * top_k + slot
  const int32_t* order;
  const X8Tile* tiles;
  const int32_t* ntiles;
  int top_k;
  const float* pair_w;
  int64_t pair_w_stride;
  uint8_t* h8;       // kX8Up: [positions, n / 2] e4m3 and its scales [positions, n / 256]
  float* hs;
};

// Four results of a row at element o.  a.vec: rows and base allow whole-vector stores.
__device__ __forceinline__ void store_quad(const X8Args& a, int64_t o, float (&v)[4]) {
  if (a.y_add) {  // fp32
    float* yp = static_cast<float*>(a.y) + o;
#pragma unroll
    for (int i = 0; i < 4; ++i) yp[i] = add_rn(yp[i], v[i]);
  } else if (!a.vec) {
#pragma unroll
    for (int i = 0; i < 4; ++i) store_act_dt(a.y, o + i, v[i], a.y_dtype);
  } else if (a.y_dtype == RIA_DT_F32) {
    store_act4<RIA_DT_F32>(a.y, o, v);
  } else if (a.y_dtype == RIA_DT_F16) {
    store_act4<RIA_DT_F16>(a.y, o, v);
  } else {
    store_act4<RIA_DT_BF16>(a.y, o, v);
  }
}

// A workgroup takes BN = 32 WF NF features x BM = 32 WT NT rows of x, a wave
// 32 WF x 32 WT of them.  Weights are the A operand: a lane's results are one
// row of x (lane % 32) and, of each 32 features, 8 q + 4 (lane / 32) + i.  Each
// step stages one block of K, 128 bytes a row, in LDS by direct copies, chunk
// c of row r at chunk c ^ ((r >> 1) & 7), so that the 16 lanes of a read's
// phase meet all 64 banks.
template <int MODE, int WF, int WT, int NF, int NT, bool WIDE>
__global__ __launch_bounds__(64 * NF * NT) void x8_tile_kernel(const X8Args a) {
  constexpr int NW = NF * NT;
  constexpr int BN = 32 * WF * NF, BM = 32 * WT * NT;
  constexpr int WL = BN / 8 / NW, XL = BM / 8 / NW;  // 1 KiB copies of a wave per step
  static_assert(WL * 8 * NW == BN && XL * 8 * NW == BM, "whole copies");
  static_assert(MODE != kX8Up || (BN == 256 && WF % 2 == 0), "one block of 128 gate and 128 up features");
  constexpr int kHalf = (BN + BM) * kX8Block;  // bytes of a step
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * kHalf];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wf = wave % NF, wt = wave / NF;
  const int l32 = lane & 31, half = lane >> 5;

  int expert = 0, first = 0, rows = 0;
  if constexpr (MODE == kX8Dense) {
    first = blockIdx.y * BM;
    rows = min(BM, a.m - first);
  } else {
    if (static_cast<int>(blockIdx.y) >= *a.ntiles) return;
    const X8Tile t = a.tiles[blockIdx.y];
    expert = t.expert;
    first = t.first;
    rows = t.rows;
  }
  const int n0 = blockIdx.x * BN;
  const int kblocks = a.k / kX8Block;
  const int nblocks = (a.n + kX8Block - 1) / kX8Block;
  const uint8_t* w = a.w + (int64_t)expert * a.n * a.k;
  const float* ws = a.ws + (int64_t)expert * nblocks * kblocks;

  // row of w behind tile row r: kX8Up takes 16 WF gate and 16 WF up rows for each wave
  auto weight_row = [&](int r) {
    if constexpr (MODE == kX8Up) {
      const int g = r / (32 * WF), i = r % (32 * WF);
      const int f = blockIdx.x * 128 + g * 16 * WF + i % (16 * WF);
      return i < 16 * WF ? f : a.n / 2 + f;
    } else {
      return min(n0 + r, a.n - 1);  // features past n repeat the last one: computed, never stored
    }
  };
  auto x_row = [&](int r) -> int64_t {  // rows past the last likewise
    const int p = first + min(r, rows - 1);
    if constexpr (MODE == kX8Up)
      return a.order[p] / a.top_k;
    else
      return p;
  };
  const uint8_t* wp[WL];
  const uint8_t* xp[XL];
#pragma unroll
  for (int i = 0; i < WL; ++i) {
    const int r = (wave * WL + i) * 8 + (lane >> 3);
    wp[i] = w + (int64_t)weight_row(r) * a.k + 16 * ((lane & 7) ^ ((r >> 1) & 7));
  }
#pragma unroll
  for (int i = 0; i < XL; ++i) {
    const int r = (wave * XL + i) * 8 + (lane >> 3);
    xp[i] = a.x + x_row(r) * a.x_stride + 16 * ((lane & 7) ^ ((r >> 1) & 7));
  }
  auto issue = [&](int kb, int buf) {
    uint8_t* d = lds + buf * kHalf;
#pragma unroll
    for (int i = 0; i < WL; ++i)
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(wp[i] + kb * kX8Block),
                                       (__attribute__((address_space(3))) void*)(d + (wave * WL + i) * 1024), 16, 0, 0);
#pragma unroll
    for (int i = 0; i < XL; ++i)
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(xp[i] + kb * kX8Block),
                                       (__attribute__((address_space(3))) void*)(d + BN * kX8Block + (wave * XL + i) * 1024),
                                       16, 0, 0);
  };
  // this lane's rows of x: their scales
  const float* xsp[WT];
#pragma unroll
  for (int t = 0; t < WT; ++t) xsp[t] = a.xs + x_row((wt * WT + t) * 32 + l32) * a.xs_stride;
  // the scale rows of the wave's features: one block of 128 (kX8Up: one of gate, one of up rows)
  const float *wsp0, *wsp1;
  if constexpr (MODE == kX8Up) {
    wsp0 = ws + (int64_t)blockIdx.x * kblocks;
    wsp1 = ws + (int64_t)(nblocks / 2 + blockIdx.x) * kblocks;
  } else {
    static_assert(128 % (32 * WF) == 0, "a wave's features lie in one block");
    wsp0 = wsp1 = ws + (int64_t)min((n0 + wf * 32 * WF) / kX8Block, nblocks - 1) * kblocks;
  }

  f32x16 acc[WF][WT];
#pragma unroll
  for (int f = 0; f < WF; ++f)
#pragma unroll
    for (int t = 0; t < WT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[f][t][i] = 0.f;

  auto operand = [&](const uint8_t* base, int r, int s) {  // 32 bytes of row r: chunks 4 s + 2 half, + 1
    const int z = (r >> 1) & 7, c = 4 * s + 2 * half;
    const u32x4 lo = *reinterpret_cast<const u32x4*>(base + r * kX8Block + 16 * (c ^ z));
    const u32x4 hi = *reinterpret_cast<const u32x4*>(base + r * kX8Block + 16 * ((c + 1) ^ z));
    return join_x8(lo, hi);
  };

  // scales of a step, loaded ahead of its copies: the wait for them is the barrier's
  float xs[WT], sw0, sw1;
  auto load_scales = [&](int kb) {
#pragma unroll
    for (int t = 0; t < WT; ++t) xs[t] = xsp[t][kb];
    sw0 = wsp0[kb];
    sw1 = wsp1[kb];
  };
  load_scales(0);
  issue(0, 0);
  for (int kb = 0; kb < kblocks; ++kb) {
    __syncthreads();  // step kb is in LDS, step kb - 1 is done with
    float s0[WT], s1[WT];
#pragma unroll
    for (int t = 0; t < WT; ++t) {
      s0[t] = xs[t] * sw0;
      s1[t] = xs[t] * sw1;
    }
    if (kb + 1 < kblocks) {
      load_scales(kb + 1);
      issue(kb + 1, (kb + 1) & 1);
    }
    const uint8_t* d = lds + (kb & 1) * kHalf;
    i32x8 b[WT][2];
#pragma unroll
    for (int t = 0; t < WT; ++t)
#pragma unroll
      for (int s = 0; s < 2; ++s) b[t][s] = operand(d + BN * kX8Block, (wt * WT + t) * 32 + l32, s);
#pragma unroll
    for (int f = 0; f < WF; ++f) {
      const i32x8 a0 = operand(d, (wf * WF + f) * 32 + l32, 0), a1 = operand(d, (wf * WF + f) * 32 + l32, 1);
#pragma unroll
      for (int t = 0; t < WT; ++t) {
        f32x16 part;
#pragma unroll
        for (int i = 0; i < 16; ++i) part[i] = 0.f;
        part = mfma_x8_32<WIDE>(a0, b[t][0], part);
        part = mfma_x8_32<WIDE>(a1, b[t][1], part);
        const float sc = f < WF / 2 ? s0[t] : s1[t];
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[f][t][i] = fmaf(part[i], sc, acc[f][t][i]);
      }
    }
  }

  if constexpr (MODE == kX8Up) {
    // a = SiLU(gate) up, then one scale over the 128 features of a row: the
    // waves' parts of its largest value meet in LDS
    __syncthreads();
    float* top = reinterpret_cast<float*>(lds);  // [NF][BM]
    constexpr int HF = WF / 2;
#pragma unroll
    for (int t = 0; t < WT; ++t) {
      float m = 0.f;
#pragma unroll
      for (int f = 0; f < HF; ++f)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float v = silu_f(acc[f][t][i]) * acc[HF + f][t][i];
          acc[f][t][i] = v;
          m = fmaxf(m, finite_abs(v));
        }
      const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
      m = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
      if (half == 0) top[wf * BM + (wt * WT + t) * 32 + l32] = m;
    }
    __syncthreads();
    const int inter = a.n / 2;
#pragma unroll
    for (int t = 0; t < WT; ++t) {
      const int r = (wt * WT + t) * 32 + l32;
      float m = 0.f;
#pragma unroll
      for (int j = 0; j < NF; ++j) m = fmaxf(m, top[j * BM + r]);
      const uint32_t e = x8_scale_exp(m);
      const float inv = x8_inverse(e);
      if (r >= rows) continue;
      const int64_t p = first + r;
      if (wf == 0 && half == 0) a.hs[p * (inter / kX8Block) + blockIdx.x] = x8_scale(e);
#pragma unroll
      for (int f = 0; f < HF; ++f)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = x8_value(acc[f][t][4 * q + i], inv);
          *reinterpret_cast<uint32_t*>(a.h8 + p * inter + blockIdx.x * 128 + (wf * HF + f) * 32 + 8 * q + 4 * half) =
              pack_x8(v[0], v[1], v[2], v[3]);
        }
    }
  } else {
#pragma unroll
    for (int t = 0; t < WT; ++t) {
      const int r = (wt * WT + t) * 32 + l32;
      if (r >= rows) continue;
      int64_t row = first + r;
      float pw = 1.f;
      if constexpr (MODE == kX8Down) {
        row = a.order[first + r];
        pw = a.pair_w[row / a.top_k * a.pair_w_stride + row % a.top_k];
      }
#pragma unroll
      for (int f = 0; f < WF; ++f)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int n = n0 + (wf * WF + f) * 32 + 8 * q + 4 * half;
          if (n >= a.n) continue;  // n is a multiple of 16: four features are in or out
          float v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = MODE == kX8Down ? pw * acc[f][t][4 * q + i] : acc[f][t][4 * q + i];
          store_quad(a, row * a.y_stride + n, v);
        }
    }
  }
}

// Host side (linear_x8.hip).
bool x8_dtype_ok(int dt);
int launch_quant_fp8(const char* who, int64_t rows, int cols, const void* x, int x_dtype, int64_t x_row_stride,
                     void* out, float* scale, hipStream_t st);

}  // namespace ria
