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

// 16x16 results over one block of K, both operands widened to fp16.
__device__ __forceinline__ f32x4 mfma_x8_16(const u32x4 (&a)[2], const u32x4 (&b)[2]) {
  f32x4 c{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    c = Kv16<RIA_DT_F16>::mfma_k32(x8_to_f16x8(a[i / 2][2 * (i % 2)], a[i / 2][2 * (i % 2) + 1]),
                                   x8_to_f16x8(b[i / 2][2 * (i % 2)], b[i / 2][2 * (i % 2) + 1]), c);
  return c;
}

// This lane's 32 bytes of a 128-byte row block: chunks l / 16 and l / 16 + 4 of
// 16 bytes, so that one load takes 64 whole bytes of each of 16 rows.
__device__ __forceinline__ void load_chunks(const uint8_t* row, int lane, u32x4 (&v)[2]) {
  const u32x4* p = reinterpret_cast<const u32x4*>(row) + (lane >> 4);
  v[0] = p[0];
  v[1] = p[4];
}
// 16 rows of w at block kb of K (row l % 16 in this lane).
__device__ __forceinline__ void load_rows16(const uint8_t* w, int k, int kb, int lane, u32x4 (&v)[2]) {
  const u32x4* p = reinterpret_cast<const u32x4*>(w + (int64_t)(lane & 15) * k + kb * kX8Block) + (lane >> 4);
  v[0] = p[0];
  v[1] = p[4];
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

// SiLU(g) u.  The hardware's exp2 and reciprocal are within an ulp; rounding -g
// log2(e) before the exp2 adds |g| 2^-24 relative, 2^-20 where SiLU still
// matters (g > -16): the e4m3 rounding that follows is 2^-4.
__device__ __forceinline__ float x8_swiglu(float g, float u) {
  return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.44269504f)) * u;
}

// Biased exponent of the scale of a slot's 64 terms whose largest finite |y| is
// top: the largest becomes 2^14 to 2^15, so fp16 keeps 11 bits of every term
// down to 2^-28 of it, whatever the range of x's type.
__device__ __forceinline__ uint32_t term_scale_exp(float top) {
  const uint32_t u = __float_as_uint(top);
  return u == 0 ? 127u : static_cast<uint32_t>(max(static_cast<int>(u >> 23) - 14, 1));
}

// Eight values of a block to e4m3 at d; the first of its 16 lanes stores the scale.
__device__ __forceinline__ void quant_eight(float (&v)[8], uint8_t* d, float* s, int lane) {
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

struct QuantArgs {
  int64_t units;     // rows * per_row
  int per_row;       // 8 values each
  const void* x;
  int64_t x_stride;
  uint8_t* out;
  float* scale;
};

// One thread per 8 values, 16 threads per block of 128 (units are whole blocks).
template <int XT>
__device__ __forceinline__ void quant_unit(const QuantArgs& a, int64_t u) {
  if (u >= a.units) return;
  const int64_t r = u / a.per_row;
  const int c = static_cast<int>(u - r * a.per_row) * 8;
  float v[8];
  load_act8<XT>(a.x, r * a.x_stride + c, v);
  quant_eight(v, a.out + u * 8, a.scale + u / 16, static_cast<int>(u & 15));
}

// ---- the tiled product
enum X8Mode {
  kX8Dense = 0,  // y [m, n]
  kX8Up = 1,     // an expert's gate and up rows of its tokens, SwiGLU, quantised
  kX8Down = 2    // an expert's down rows of its pairs, times the router's weight, to the pairs' positions
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
  uint8_t* ye;       // kX8Down with RIA_DT_F16: y holds term / 2^(e - 127), e [positions, ye_stride] one per 64 features
  int ye_stride;
  uint8_t* h8;       // kX8Up: [positions, n / 2] e4m3 and its scales [positions, n / 256]
  float* hs;
};

// Direct copies into LDS (16 bytes a lane, lane l at d + 16 l) through a buffer
// resource, so that a lane's part of the address is one 32-bit offset.  (Device
// functions of their own: the host pass of a kernel template refuses the builtins.)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t x8_rsrc(const uint8_t* p, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, static_cast<int>(static_cast<uint32_t>(bytes)),
                                           kBufferWord3);
}
template <bool STREAM = false>  // read once: not kept in the caches
__device__ __forceinline__ void x8_copy(__amdgpu_buffer_rsrc_t r, uint8_t* d, uint32_t lane_offset, int offset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, d, 16, lane_offset, offset, 0, STREAM ? 2 : 0);
}

// One fp32 through a resource: 32-bit offsets, as the copies beside it have.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t x8_rsrc_f32(const float* p, int64_t count) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(p), 0, static_cast<int>(static_cast<uint32_t>(4 * count)),
                                           kBufferWord3);
}
__device__ __forceinline__ float x8_load_f32(__amdgpu_buffer_rsrc_t r, uint32_t lane_offset, int offset) {
  return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, lane_offset, offset, 0));
}

// Four results of a row at element o (n is a multiple of 16).
__device__ __forceinline__ void store_four(const X8Args& a, int64_t o, const f32x4& v) {
  if (a.y_add) {  // fp32
    float* yp = static_cast<float*>(a.y) + o;
#pragma unroll
    for (int i = 0; i < 4; ++i) yp[i] = add_rn(yp[i], v[i]);
  } else if (!a.vec) {
#pragma unroll
    for (int i = 0; i < 4; ++i) store_act_dt(a.y, o + i, v[i], a.y_dtype);
  } else if (a.y_dtype == RIA_DT_F32) {
    *reinterpret_cast<f32x4*>(static_cast<float*>(a.y) + o) = v;
  } else {
    const bool h = a.y_dtype == RIA_DT_F16;
    *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.y) + o) =
        h ? u32x2{Kv16<RIA_DT_F16>::pack2(v[0], v[1]), Kv16<RIA_DT_F16>::pack2(v[2], v[3])}
          : u32x2{Kv16<RIA_DT_BF16>::pack2(v[0], v[1]), Kv16<RIA_DT_BF16>::pack2(v[2], v[3])};
  }
}

// Eight results of a row at element o.  a.vec: rows and base allow whole-vector
// stores.  STREAM: 16-bit results past the caches, where they outgrow them.
template <bool STREAM = false>
__device__ __forceinline__ void store_eight(const X8Args& a, int64_t o, const float (&v)[8]) {
  if (a.y_add) {  // fp32
    float* yp = static_cast<float*>(a.y) + o;
    if (a.vec) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        f32x4 t = reinterpret_cast<f32x4*>(yp)[h];
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = add_rn(t[i], v[4 * h + i]);
        reinterpret_cast<f32x4*>(yp)[h] = t;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) yp[i] = add_rn(yp[i], v[i]);
    }
  } else if (!a.vec) {
#pragma unroll
    for (int i = 0; i < 8; ++i) store_act_dt(a.y, o + i, v[i], a.y_dtype);
  } else if (a.y_dtype == RIA_DT_F32) {
    f32x4* yp = reinterpret_cast<f32x4*>(static_cast<float*>(a.y) + o);
    yp[0] = f32x4{v[0], v[1], v[2], v[3]};
    yp[1] = f32x4{v[4], v[5], v[6], v[7]};
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = a.y_dtype == RIA_DT_F16 ? Kv16<RIA_DT_F16>::pack2(v[2 * i], v[2 * i + 1])
                                     : Kv16<RIA_DT_BF16>::pack2(v[2 * i], v[2 * i + 1]);
    u32x4* yp = reinterpret_cast<u32x4*>(static_cast<uint16_t*>(a.y) + o);
    if constexpr (STREAM)
      __builtin_nontemporal_store(u32x4{w[0], w[1], w[2], w[3]}, yp);
    else
      *yp = u32x4{w[0], w[1], w[2], w[3]};
  }
}

// Workgroup b of a launch takes tile x8_order(b, total): the workgroups that
// one XCD runs (b % 8) take consecutive tiles, whose operands meet in its L2.
__device__ __forceinline__ int x8_order(int b, int total) {
  const int per = (total + 7) / 8;
  return b / 8 < per ? (b % 8) * per + b / 8 : total;
}

// A workgroup takes BN = 32 WF NF features x BM = 32 WT NT rows of x, a wave
// 32 WF x 32 WT of them.  Weights are the A operand: a lane's results are one
// row of x (lane % 32) and, of each 32 features, 8 q + 4 (lane / 32) + i.  Each
// step stages one block of K, 128 bytes a row, in LDS by direct copies, chunk
// c of row r at chunk c ^ ((r >> 1) & 7), so that the 16 lanes of a read's
// phase meet all 64 banks; the next step's copies run beside the products.
//
// Large tiles (4, 2, 2, 4: 256 x 256, one workgroup a CU) are bound by the matrix
// cores at the clock they allow, beside 64 KB of LDS copies, 128 KB of LDS reads
// and the scaling's FMAs a step: some 2 us a step, 6 outside the steps.  16384 x
// 8192 x 2048 to fp16 in 295 us, 1.86 PFLOP/s; 128 x 256 tiles with one LDS
// buffer, two workgroups a CU: 330 (and the experts' products the same as now).
// Small tiles (32 or 64 rows) are bound by the weights' way from HBM.
//
// ONE: one LDS buffer, and registers for ONE waves a SIMD: a step's copies are
// covered by the CU's other workgroups, where there are more than two for it.
// 4096 x 2048 x 4096 in tiles of 128 x 128: 46 us, 51 with two buffers; but with
// one tile a CU (2048 x 2048 x 4096) 41 and 32.
template <int MODE, int WF, int WT, int NF, int NT, bool WIDE, bool STREAM = false, int ONE = 0>
__global__ __launch_bounds__(64 * NF * NT, ONE ? ONE : 1) void x8_tile_kernel(const X8Args a) {
  constexpr int NW = NF * NT;
  constexpr int BN = 32 * WF * NF, BM = 32 * WT * NT;
  constexpr int WL = BN / 8 / NW, XL = BM / 8 / NW;  // 1 KiB copies of a wave per step
  static_assert(WL * 8 * NW == BN && XL * 8 * NW == BM, "whole copies");
  static_assert(MODE != kX8Up || (BN == 256 && WF % 2 == 0), "one block of 128 gate and 128 up features");
  constexpr int kStep = (BN + BM) * kX8Block;  // bytes of a step
  constexpr int kPitch = 64 + 4;               // fp32 values of a row that a wave stages for its stores
  constexpr int kStage = 32 * kPitch * 4;
  __shared__ __attribute__((aligned(16))) uint8_t lds[(ONE ? 1 : 2) * kStep > NW * kStage ? (ONE ? 1 : 2) * kStep : NW * kStage];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wf = wave % NF, wt = wave / NF;
  const int l32 = lane & 31, half = lane >> 5;

  const int ntn = MODE == kX8Up ? a.n / 256 : (a.n + BN - 1) / BN;  // feature tiles
  int expert = 0, first = 0, rows = 0, tn = 0;
  if constexpr (MODE == kX8Dense) {
    const int ntm = (a.m + BM - 1) / BM;
    const int at = x8_order(blockIdx.x, ntm * ntn);
    if (at >= ntm * ntn) return;
    // four row tiles by all feature tiles at a time
    const int g0 = at / (4 * ntn) * 4, gs = min(4, ntm - g0), in = at - g0 * ntn;
    first = (g0 + in % gs) * BM;
    tn = in / gs;
    rows = min(BM, a.m - first);
  } else {
    const int total = *a.ntiles * ntn;
    const int at = x8_order(blockIdx.x, total);
    if (at >= total) return;
    const X8Tile t = a.tiles[at / ntn];
    tn = at % ntn;
    expert = t.expert;
    first = t.first;
    rows = t.rows;
  }
  const int n0 = tn * BN;
  const int kblocks = a.k / kX8Block;
  const int nblocks = (a.n + kX8Block - 1) / kX8Block;
  const uint8_t* w = a.w + (int64_t)expert * a.n * a.k;
  const float* ws = a.ws + (int64_t)expert * nblocks * kblocks;

  // Tile row r of the weights: kX8Up takes 16 WF gate and 16 WF up rows for
  // each wave; features past n and rows past the last repeat the last one
  // (computed, never stored).
  auto weight_row = [&](int r) {
    if constexpr (MODE == kX8Up) {
      const int g = r / (32 * WF), i = r % (32 * WF);
      return g * 16 * WF + i % (16 * WF) + (i < 16 * WF ? 0 : a.n / 2);
    } else {
      return min(r, a.n - 1 - n0);
    }
  };
  auto x_row = [&](int r) -> int64_t {
    const int p = first + min(r, rows - 1);
    if constexpr (MODE == kX8Up)
      return a.order[p] / a.top_k;
    else
      return p;
  };
  const int64_t x0 = MODE == kX8Up ? 0 : first;  // the resource starts at this row
  const __amdgpu_buffer_rsrc_t wr =
      MODE == kX8Up ? x8_rsrc(w + (int64_t)tn * 128 * a.k, (int64_t)(a.n - tn * 128) * a.k)
                    : x8_rsrc(w + (int64_t)n0 * a.k, (int64_t)min(BN, a.n - n0) * a.k);
  const __amdgpu_buffer_rsrc_t xr =
      x8_rsrc(a.x + x0 * a.x_stride, MODE == kX8Up ? a.m * a.x_stride : (rows - 1) * a.x_stride + a.k);
  uint32_t wo[WL], xo[XL];
#pragma unroll
  for (int i = 0; i < WL; ++i) {
    const int r = (wave * WL + i) * 8 + (lane >> 3);
    wo[i] = static_cast<uint32_t>(weight_row(r)) * a.k + 16 * ((lane & 7) ^ ((r >> 1) & 7));
  }
#pragma unroll
  for (int i = 0; i < XL; ++i) {
    const int r = (wave * XL + i) * 8 + (lane >> 3);
    xo[i] = static_cast<uint32_t>((x_row(r) - x0) * a.x_stride) + 16 * ((lane & 7) ^ ((r >> 1) & 7));
  }
  auto issue = [&](int kb) __attribute__((always_inline)) {
    uint8_t* d = lds + (ONE ? 0 : (kb & 1) * kStep);
#pragma unroll
    for (int i = 0; i < WL; ++i) x8_copy<STREAM>(wr, d + (wave * WL + i) * 1024, wo[i], kb * kX8Block);
#pragma unroll
    for (int i = 0; i < XL; ++i) x8_copy(xr, d + BN * kX8Block + (wave * XL + i) * 1024, xo[i], kb * kX8Block);
  };
  // this lane's rows of x: their scales
  const float* xsp[WT];
#pragma unroll
  for (int t = 0; t < WT; ++t) xsp[t] = a.xs + x_row((wt * WT + t) * 32 + l32) * a.xs_stride;
  // the scale rows of the wave's features: one block of 128 (kX8Up: one of gate, one of up rows)
  const float *wsp0, *wsp1;
  if constexpr (MODE == kX8Up) {
    wsp0 = ws + (int64_t)tn * kblocks;
    wsp1 = ws + (int64_t)(nblocks / 2 + tn) * kblocks;
  } else {
    static_assert(128 % (32 * WF) == 0, "a wave's features lie in one block");
    wsp0 = wsp1 = ws + (int64_t)min((n0 + wf * 32 * WF) / kX8Block, nblocks - 1) * kblocks;
  }
  // scales of a step, loaded ahead of its copies: the wait for them is the barrier's
  float xs[WT], sw0, sw1;
  auto load_scales = [&](int kb) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < WT; ++t) xs[t] = xsp[t][kb];
    sw0 = wsp0[kb];
    sw1 = wsp1[kb];
  };

  f32x16 acc[WF][WT];
#pragma unroll
  for (int f = 0; f < WF; ++f)
#pragma unroll
    for (int t = 0; t < WT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[f][t][i] = 0.f;

  auto operand = [&](const uint8_t* base, int r, int s) __attribute__((always_inline)) {  // chunks 4 s + 2 half, + 1 of row r
    const int z = (r >> 1) & 7, c = 4 * s + 2 * half;
    const u32x4 lo = *reinterpret_cast<const u32x4*>(base + r * kX8Block + 16 * (c ^ z));
    const u32x4 hi = *reinterpret_cast<const u32x4*>(base + r * kX8Block + 16 * ((c + 1) ^ z));
    return join_x8(lo, hi);
  };
  const bool live = wt * 32 * WT < rows;  // a wave whose rows are all past the last only copies

  load_scales(0);
  issue(0);
  for (int kb = 0; kb < kblocks; ++kb) {
    // step kb's copies are in LDS (a barrier alone does not wait for them), step kb - 1 is done with
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    float s0[WT], s1[WT];
#pragma unroll
    for (int t = 0; t < WT; ++t) {
      s0[t] = xs[t] * sw0;
      s1[t] = xs[t] * sw1;
    }
    if (kb + 1 < kblocks) {
      load_scales(kb + 1);
      if (!ONE) issue(kb + 1);
    }
    if constexpr (!ONE) {
      if (!live) continue;
    }
    if (!ONE || live) {
      const uint8_t* d = lds + (ONE ? 0 : (kb & 1) * kStep);
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
    if (ONE && kb + 1 < kblocks) {
      __syncthreads();  // the step is read before the next is copied over it
      issue(kb + 1);
    }
  }
  __syncthreads();

  if constexpr (MODE == kX8Up) {
    // a = SiLU(gate) up, then one scale over the 128 features of a row: the
    // waves' parts of its largest value meet in LDS
    float* top = reinterpret_cast<float*>(lds);               // [NF][BM]
    uint8_t* stage = lds + NF * BM * 4;                       // [BM][128] quantised, chunks swizzled
    static_assert(NF * BM * 4 + BM * 128 <= (ONE ? 1 : 2) * kStep, "both fit");
    constexpr int HF = WF / 2;
#pragma unroll
    for (int t = 0; t < WT; ++t) {
      float m = 0.f;
#pragma unroll
      for (int f = 0; f < HF; ++f)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float v = x8_swiglu(acc[f][t][i], acc[HF + f][t][i]);
          acc[f][t][i] = v;
          m = fmaxf(m, fabsf(v));
        }
      if (__ballot(m == __builtin_inff())) {  // infinities set no scale, and are NaN in e4m3
        m = 0.f;
#pragma unroll
        for (int f = 0; f < HF; ++f)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float v = acc[f][t][i];
            m = fmaxf(m, finite_abs(v));
            acc[f][t][i] = x8_value(v, 1.f);
          }
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
      if (wf == 0 && half == 0 && r < rows) a.hs[(int64_t)(first + r) * (inter / kX8Block) + tn] = x8_scale(e);
#pragma unroll
      for (int f = 0; f < HF; ++f)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = acc[f][t][4 * q + i] * inv;
          const int o = (wf * HF + f) * 32 + 8 * q + 4 * half;  // byte of the row
          *reinterpret_cast<uint32_t*>(stage + r * 128 + (((o >> 4) ^ (r & 7)) << 4) + (o & 15)) =
              pack_x8(v[0], v[1], v[2], v[3]);
        }
    }
    __syncthreads();
    for (int u = tid; u < BM * 8; u += 64 * NW) {
      const int r = u >> 3, c = u & 7;
      if (r < rows)
        *reinterpret_cast<u32x4*>(a.h8 + (int64_t)(first + r) * inter + tn * 128 + 16 * c) =
            *reinterpret_cast<const u32x4*>(stage + r * 128 + 16 * (c ^ (r & 7)));
    }
  } else {
    // 32 rows x 64 features at a time through the wave's own LDS, out in whole rows' pieces
    if (!live) return;
    float* st = reinterpret_cast<float*>(lds + wave * kStage);
#pragma unroll
    for (int t = 0; t < WT; ++t) {
      float pw = 1.f;
      if constexpr (MODE == kX8Down) {
        const int64_t pair = a.order[first + min((wt * WT + t) * 32 + l32, rows - 1)];
        pw = a.pair_w[pair / a.top_k * a.pair_w_stride + pair % a.top_k];
      }
#pragma unroll
      for (int f0 = 0; f0 < WF; f0 += 2) {
        float scale = 1.f;
        if constexpr (MODE == kX8Down) {
          float top = 0.f;
#pragma unroll
          for (int f = 0; f < 2; ++f)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float v = pw * acc[f0 + f][t][i];
              acc[f0 + f][t][i] = v;
              top = fmaxf(top, fabsf(v));
            }
          if (a.y_dtype != RIA_DT_F32) {
            if (__ballot(top == __builtin_inff())) {  // infinities set no scale
              top = 0.f;
#pragma unroll
              for (int f = 0; f < 2; ++f)
#pragma unroll
                for (int i = 0; i < 16; ++i) top = fmaxf(top, finite_abs(acc[f0 + f][t][i]));
            }
            const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
            const uint32_t e = term_scale_exp(fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])));
            scale = x8_inverse(e);
            const int rr = (wt * WT + t) * 32 + l32, g = (n0 + (wf * WF + f0) * 32) / 64;
            if (half == 0 && rr < rows && g < a.ye_stride)
              a.ye[(int64_t)(first + rr) * a.ye_stride + g] = static_cast<uint8_t>(e);
          }
        }
#pragma unroll
        for (int f = 0; f < 2; ++f)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            f32x4 v;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = MODE == kX8Down ? acc[f0 + f][t][4 * q + i] * scale : acc[f0 + f][t][4 * q + i];
            *reinterpret_cast<f32x4*>(st + l32 * kPitch + f * 32 + 8 * q + 4 * half) = v;
          }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = 8 * j + (lane >> 3), c = 8 * (lane & 7);
          const f32x4 v0 = *reinterpret_cast<const f32x4*>(st + r * kPitch + c);
          const f32x4 v1 = *reinterpret_cast<const f32x4*>(st + r * kPitch + c + 4);
          const float v[8] = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
          const int rr = (wt * WT + t) * 32 + r, n = n0 + (wf * WF + f0) * 32 + c;
          if (rr >= rows || n >= a.n) continue;  // n is a multiple of 16: eight features are in or out
          store_eight<(BM == 256)>(a, (int64_t)(first + rr) * a.y_stride + n, v);
        }
      }
    }
  }
}

// Host side (linear_x8.hip).
bool x8_dtype_ok(int dt);

}  // namespace ria
