// Activations quantised to e4m3 and their products with block-FP8 weights.
//
//   quant_fp8_kernel   x [rows, cols] -> e4m3 values and one power-of-two
//                      scale per 128 values of a row.
//   x8_tile_kernel     y = (x8 xs) (w8 ws)^T (x8_tile.h).
//
// The block-FP8 checkpoints whose weights linear_fp8.hip dequantises to fp16
// name this as the way to run them: activations in e4m3, a scale for each
// 128 values of a row, found as they come.  The reference multiplies in fp16
// (qwen36_attention_cache.py:232-247), which linear_fp8.hip reproduces; here
// both operands stay in 8 bits and the matrix cores run at twice the rate.
#include <algorithm>

#include "x8_tile.h"

namespace ria {

template <int XT>
__global__ __launch_bounds__(256) void quant_fp8_kernel(const QuantArgs a) {
  quant_unit<XT>(a, (int64_t)blockIdx.x * 256 + threadIdx.x);
}

// A few rows: 16 features x up to 16 MT rows a workgroup, NW waves sharing K.
// The weights stream from HBM straight into MFMA operands (16 rows x 128 bytes a
// product, widened to fp16), all of a wave's kFewAhead blocks in flight at once.
constexpr int kFewAhead = 4;
template <int MT, int NW>
__global__ __launch_bounds__(64 * NW) void x8_few_kernel(const X8Args a) {
  __shared__ f32x4 red[NW][MT][64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MT;
  const int rows = min(16 * MT, a.m - m0);
  const int kblocks = a.k / kX8Block;
  const uint8_t* w = a.w + (int64_t)n0 * a.k;
  const float* ws = a.ws + (int64_t)(n0 / kX8Block) * kblocks;
  const uint8_t* x[MT];
  const float* xs[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {  // rows past the last repeat it: computed, never stored
    const int64_t row = m0 + min(16 * t + (lane & 15), rows - 1);
    x[t] = a.x + row * a.x_stride;
    xs[t] = a.xs + row * a.xs_stride;
  }
  u32x4 v[kFewAhead][2], b[kFewAhead][MT][2];
  float fw[kFewAhead], fx[kFewAhead][MT];
  auto load = [&](int kb0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kFewAhead; ++i) load_rows16(w, a.k, min(kb0 + i, kblocks - 1), lane, v[i]);
#pragma unroll
    for (int i = 0; i < kFewAhead; ++i) {
      const int kb = min(kb0 + i, kblocks - 1);
      fw[i] = ws[kb];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        load_chunks(x[t] + kb * kX8Block, lane, b[i][t]);
        fx[i][t] = xs[t][kb];
      }
    }
    __builtin_amdgcn_sched_barrier(0);  // all of them in flight before the first product
  };
  load(wave * kFewAhead);
  f32x4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int kb0 = wave * kFewAhead; kb0 < kblocks; kb0 += NW * kFewAhead) {
#pragma unroll
    for (int i = 0; i < kFewAhead; ++i) {
      if (kb0 + i >= kblocks) break;
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const f32x4 part = mfma_x8_16(v[i], b[i][t]);
        const float s = fx[i][t] * fw[i];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[t][j] = fmaf(part[j], s, acc[t][j]);
      }
    }
    if (kb0 + NW * kFewAhead < kblocks) load(kb0 + NW * kFewAhead);
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) red[wave][t][lane] = acc[t];
  __syncthreads();
  // lane l of a product: row l % 16, features 4 (l / 16) .. + 3
  for (int u = tid; u < 64 * MT; u += 64 * NW) {
    const int t = u >> 6, l = ((u & 3) << 4) | ((u >> 2) & 15);  // neighbours in a row are neighbours here
    const int row = 16 * t + (l & 15);
    if (row >= rows) continue;
    f32x4 s = red[0][t][l];
#pragma unroll
    for (int j = 1; j < NW; ++j) s += red[j][t][l];
    store_four(a, (int64_t)(m0 + row) * a.y_stride + n0 + 4 * (l >> 4), s);
  }
}

// Some hundred rows: 64 x 64 tiles, the blocks of K dealt to the workgroup's
// waves.  Each wave copies a block into LDS of its own and multiplies it with no
// barrier; the waves' sums meet in LDS at the end.  Bound by the loads' latency
// and, with two waves a SIMD to cover it, by the CU's 64 bytes a clock into LDS:
// 333 x 2048 x 4096 to fp32 11.8 us, of it 5 outside the blocks; four waves with
// two buffers each 14.1.  Operands straight into registers (16 rows x 64 bytes a
// load, two to four blocks ahead) 25: half lines.
template <bool WIDE, int NW>
__global__ __launch_bounds__(64 * NW) void x8_deal_kernel(const X8Args a) {
  constexpr int kStep = 128 * kX8Block;  // 64 rows of w, 64 of x
  __shared__ __attribute__((aligned(16))) uint8_t lds[NW * kStep];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, half = lane >> 5;
  const int ntn = (a.n + 63) / 64, ntm = (a.m + 63) / 64;
  const int at = x8_order(blockIdx.x, ntn * ntm);
  if (at >= ntn * ntm) return;
  const int n0 = at / ntm * 64, m0 = at % ntm * 64;  // neighbours share their weights
  const int rows = min(64, a.m - m0), feats = min(64, a.n - n0);
  const int kblocks = a.k / kX8Block;
  const __amdgpu_buffer_rsrc_t wr = x8_rsrc(a.w + (int64_t)n0 * a.k, (int64_t)feats * a.k);
  const __amdgpu_buffer_rsrc_t xr = x8_rsrc(a.x + m0 * a.x_stride, (rows - 1) * a.x_stride + a.k);
  uint32_t wo[8], xo[8];  // rows past the last repeat it
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = 8 * i + (lane >> 3), c = 16 * ((lane & 7) ^ ((r >> 1) & 7));
    wo[i] = static_cast<uint32_t>(min(r, feats - 1)) * a.k + c;
    xo[i] = static_cast<uint32_t>(min(r, rows - 1) * a.x_stride) + c;
  }
  const __amdgpu_buffer_rsrc_t xsr = x8_rsrc_f32(a.xs + m0 * a.xs_stride, (rows - 1) * a.xs_stride + kblocks);
  const __amdgpu_buffer_rsrc_t wsr = x8_rsrc_f32(a.ws + (int64_t)(n0 / kX8Block) * kblocks, kblocks);
  uint32_t xso[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) xso[t] = static_cast<uint32_t>(4 * min(32 * t + l32, rows - 1) * a.xs_stride);
  uint8_t* own = lds + wave * kStep;
  float xs[2], sw;
  auto issue = [&](int kb) __attribute__((always_inline)) {
    xs[0] = x8_load_f32(xsr, xso[0], 4 * kb);
    xs[1] = x8_load_f32(xsr, xso[1], 4 * kb);
    sw = x8_load_f32(wsr, 0, 4 * kb);
#pragma unroll
    for (int i = 0; i < 8; ++i) x8_copy(wr, own + i * 1024, wo[i], kb * kX8Block);
#pragma unroll
    for (int i = 0; i < 8; ++i) x8_copy(xr, own + (8 + i) * 1024, xo[i], kb * kX8Block);
  };
  f32x16 acc[2][2];
#pragma unroll
  for (int f = 0; f < 2; ++f)
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[f][t][i] = 0.f;
  auto operand = [&](const uint8_t* base, int r, int s) __attribute__((always_inline)) {
    const int z = (r >> 1) & 7, c = 4 * s + 2 * half;
    return join_x8(*reinterpret_cast<const u32x4*>(base + r * kX8Block + 16 * (c ^ z)),
                   *reinterpret_cast<const u32x4*>(base + r * kX8Block + 16 * ((c + 1) ^ z)));
  };
  auto step = [&]() __attribute__((always_inline)) {
    const uint8_t* d = own;
    i32x8 b[2][2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int s = 0; s < 2; ++s) b[t][s] = operand(d + 64 * kX8Block, 32 * t + l32, s);
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      const i32x8 a0 = operand(d, 32 * f + l32, 0), a1 = operand(d, 32 * f + l32, 1);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        f32x16 part;
#pragma unroll
        for (int i = 0; i < 16; ++i) part[i] = 0.f;
        part = mfma_x8_32<WIDE>(a0, b[t][0], part);
        part = mfma_x8_32<WIDE>(a1, b[t][1], part);
        const float sc = xs[t] * sw;
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[f][t][i] = fmaf(part[i], sc, acc[f][t][i]);
      }
    }
  };
  for (int kb = wave; kb < kblocks; kb += NW) {
    issue(kb);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    step();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the block is read before the next is copied over it
  }
  __syncthreads();
  // sums [wave][row of x][64 features], chunks of four swizzled
  f32x4* sum = reinterpret_cast<f32x4*>(lds);
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = 32 * t + l32;
        sum[(wave * 64 + r) * 16 + ((8 * f + 2 * q + half) ^ (r & 15))] =
            f32x4{acc[f][t][4 * q], acc[f][t][4 * q + 1], acc[f][t][4 * q + 2], acc[f][t][4 * q + 3]};
      }
  __syncthreads();
  for (int u = tid; u < 64 * 16; u += 64 * NW) {
    const int r = u >> 4, c = u & 15, at_c = c ^ (r & 15);
    if (r >= rows || n0 + 4 * c >= a.n) continue;
    f32x4 s = sum[r * 16 + at_c];
#pragma unroll
    for (int j = 1; j < NW; ++j) s += sum[(j * 64 + r) * 16 + at_c];
    store_four(a, (int64_t)(m0 + r) * a.y_stride + n0 + 4 * c, s);
  }
}

// The kernel of a product.  Up to 32 rows the weights' way from HBM is all there
// is.  Past that the kernel of the least time by rounds of its tiles over the
// CUs, in microseconds measured on MI355X (kk = K / 2048): a round of 64 x 64
// tiles with K dealt to the waves 1.6 + 4.6 kk; of 128 x 128 tiles 5 + 12 kk with
// one a CU, 4 + 22.5 kk with two, between them where some CUs have two, 3 + 28 kk
// with three of one LDS buffer (no rounds: they start one by one); of 256 x 256
// tiles 6 + 32 kk.  Measured on both sides, 64 / 128 tiles, N = 8192, K = 2048:
// 256 rows 14.7 / 18.1, 384 rows 20.9 / 18.9, 2048 rows 107 / 54 (41 with 256);
// N = 2048, K = 4096: 512 rows 11.1 / 30.0, 1024 rows 22.4 / 30.9, 1536 rows 35.7 /
// 31.3, 8192 rows 189 / 98 (72 with 256); N = 4096, K = 1024: 512 rows 10.5 / 11.4,
// 768 rows 15.0 / 11.9.  Wide (fp32 results): N = 8192, K = 2048: 384 rows 23.9 /
// 26.1, 512 rows 30.0 / 27.6; N = 2048, K = 4096: 512 rows 12.6 / 40.7, 3000 rows
// 81 / 66.  Tiles of 128 with one buffer / two: N = 8192, K = 2048: 512 rows 23.5 /
// 19.7, 1024 rows 26.5 / 27.2, 3000 rows 76 / 78; N = 2048, K = 4096: 2048 rows 41 /
// 32, 3000 rows 43.5 / 47, 4096 rows 46 / 51; N = 4096, K = 1024: 2048 rows 17.2 /
// 16.9, 3000 rows 22.5 / 22.5.
enum class X8Plan { kFew, kDeal, kTile128, kTile128Many, kTile256 };
static X8Plan plan_x8(int m, int64_t t256, int64_t t128, int64_t t64, int k, bool wide) {
  if (m <= 32) return X8Plan::kFew;
  const int64_t cus = device_cus();
  const double kk = k / 2048.0;
  auto rounds = [&](int64_t tiles) { return static_cast<double>((tiles + cus - 1) / cus); };
  const double one = wide ? 7 + 18 * kk : 5 + 12 * kk, two = wide ? 5 + 36 * kk : 4 + 22.5 * kk;
  const double deal = 2 + rounds(t64) * (wide ? 1.8 + 5.3 * kk : 1.6 + 4.6 * kk);
  const double tile256 = 2 + rounds(t256) * (6 + 32 * kk);
  const bool many = !wide && t128 > cus;
  double tile128;
  if (many) {
    tile128 = std::max(0.9 * two, 4 + (3 + 28 * kk) * static_cast<double>(t128) / static_cast<double>(3 * cus));
  } else {
    const int64_t rest = t128 % (2 * cus);
    const double last = rest == 0 ? 0 : rest <= cus ? one : two - 0.6 * (two - one) * (2 * cus - rest) / cus;
    tile128 = 1 + static_cast<double>(t128 / (2 * cus)) * two + last;
  }
  if (!wide && tile256 < tile128 && tile256 < deal) return X8Plan::kTile256;
  if (deal <= tile128) return X8Plan::kDeal;
  return many ? X8Plan::kTile128Many : X8Plan::kTile128;
}

bool x8_dtype_ok(int dt) { return dt == RIA_DT_BF16 || dt == RIA_DT_F16 || dt == RIA_DT_F32; }

}  // namespace ria

using namespace ria;

extern "C" int ria_quant_fp8(int64_t rows, int cols, const void* x, int x_dtype, int64_t x_row_stride, void* out,
                             float* scale, void* stream) {
  const char* who = "ria_quant_fp8";
  if (rows < 0 || cols <= 0 || cols % kX8Block)
    return set_error(RIA_ERR_INVALID, "%s: cols must be a positive multiple of %d (got %d)", who, kX8Block, cols);
  if (!x8_dtype_ok(x_dtype)) return set_error(RIA_ERR_INVALID, "%s: unknown dtype code", who);
  if (rows == 0) return RIA_OK;
  if (!x || !out || !scale) return set_error(RIA_ERR_INVALID, "%s: null pointer", who);
  if (x_row_stride < cols || x_row_stride % 8 || reinterpret_cast<uintptr_t>(x) % 16)
    return set_error(RIA_ERR_INVALID, "%s: x must be 16-byte aligned with a row stride of at least cols, a multiple of 8", who);
  if (reinterpret_cast<uintptr_t>(out) % 16) return set_error(RIA_ERR_INVALID, "%s: out must be 16-byte aligned", who);
  const QuantArgs a{rows * (cols / 8), cols / 8, x, x_row_stride, static_cast<uint8_t*>(out), scale};
  const int64_t blocks = (a.units + 255) / 256;
  if (blocks > 0x7fffffff) return set_error(RIA_ERR_INVALID, "%s: too many values", who);
  const dim3 grid(static_cast<unsigned>(blocks));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (x_dtype == RIA_DT_BF16)
    hipLaunchKernelGGL((quant_fp8_kernel<RIA_DT_BF16>), grid, dim3(256), 0, st, a);
  else if (x_dtype == RIA_DT_F16)
    hipLaunchKernelGGL((quant_fp8_kernel<RIA_DT_F16>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((quant_fp8_kernel<RIA_DT_F32>), grid, dim3(256), 0, st, a);
  return check_launch(who);
}

extern "C" int ria_linear_fp8_x8(int m, int n, int k, const void* x, int64_t x_row_stride, const float* x_scale,
                                 int64_t x_scale_row_stride, const void* weight, const float* scale_inv, void* y,
                                 int y_dtype, int64_t y_row_stride, int y_add, void* stream) {
  const char* who = "ria_linear_fp8_x8";
  if (m < 0 || n <= 0 || n % 16) return set_error(RIA_ERR_INVALID, "%s: N must be a positive multiple of 16 (got %d)", who, n);
  if (k <= 0 || k % kX8Block || k > 32768)
    return set_error(RIA_ERR_INVALID, "%s: K must be a multiple of %d up to 32768 (got %d)", who, kX8Block, k);
  if (!x8_dtype_ok(y_dtype)) return set_error(RIA_ERR_INVALID, "%s: unknown dtype code", who);
  if (y_add && y_dtype != RIA_DT_F32) return set_error(RIA_ERR_INVALID, "%s: y_add needs an fp32 y", who);
  if (m == 0) return RIA_OK;
  if (!x || !x_scale || !weight || !scale_inv || !y) return set_error(RIA_ERR_INVALID, "%s: null pointer", who);
  if (x_row_stride < k || x_row_stride % 16 || reinterpret_cast<uintptr_t>(x) % 16)
    return set_error(RIA_ERR_INVALID, "%s: x must be 16-byte aligned with a row stride of at least K, a multiple of 16", who);
  if (x_scale_row_stride > (1 << 23)) return set_error(RIA_ERR_INVALID, "%s: x_scale row stride over 2^23", who);
  if (x_scale_row_stride < k / kX8Block) return set_error(RIA_ERR_INVALID, "%s: x_scale row stride too small", who);
  if (y_row_stride < n) return set_error(RIA_ERR_INVALID, "%s: y row stride too small", who);
  if (reinterpret_cast<uintptr_t>(weight) % 16) return set_error(RIA_ERR_INVALID, "%s: weight must be 16-byte aligned", who);
  X8Args a{};
  a.x = static_cast<const uint8_t*>(x);
  a.x_stride = x_row_stride;
  a.xs = x_scale;
  a.xs_stride = x_scale_row_stride;
  a.w = static_cast<const uint8_t*>(weight);
  a.ws = scale_inv;
  a.m = m;
  a.n = n;
  a.k = k;
  a.y = y;
  a.y_stride = y_row_stride;
  a.y_dtype = y_dtype;
  a.y_add = y_add;
  a.vec = reinterpret_cast<uintptr_t>(y) % 16 == 0 && y_row_stride % 8 == 0;
  if (x_row_stride > (1 << 23)) return set_error(RIA_ERR_INVALID, "%s: x row stride over 8 MiB", who);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t t256 = (int64_t)((m + 255) / 256) * ((n + 255) / 256), t128 = (int64_t)((m + 127) / 128) * ((n + 127) / 128);
  const int64_t t64 = (int64_t)((m + 63) / 64) * ((n + 63) / 64);
  if (t64 > 0x7ffffff0) return set_error(RIA_ERR_INVALID, "%s: too many rows", who);
  auto grid = [](int64_t tiles) { return dim3(static_cast<unsigned>((tiles + 7) / 8 * 8)); };
  const bool wide = y_dtype == RIA_DT_F32;
  const X8Plan plan = plan_x8(m, t256, t128, t64, k, wide);
  if (plan == X8Plan::kFew) {
    const bool deep = k > 4 * kFewAhead * kX8Block;  // more blocks of K than four waves hold
    const dim3 few(n / 16, 1);
    if (m <= 16 && deep)
      hipLaunchKernelGGL((x8_few_kernel<1, 8>), few, dim3(512), 0, st, a);
    else if (m <= 16)
      hipLaunchKernelGGL((x8_few_kernel<1, 4>), few, dim3(256), 0, st, a);
    else if (deep)
      hipLaunchKernelGGL((x8_few_kernel<2, 8>), few, dim3(512), 0, st, a);
    else
      hipLaunchKernelGGL((x8_few_kernel<2, 4>), few, dim3(256), 0, st, a);
  } else if (plan == X8Plan::kTile256) {
    hipLaunchKernelGGL((x8_tile_kernel<kX8Dense, 4, 2, 2, 4, false>), grid(t256), dim3(512), 0, st, a);
  } else if (plan == X8Plan::kTile128Many) {
    hipLaunchKernelGGL((x8_tile_kernel<kX8Dense, 2, 2, 2, 2, false, false, 3>), grid(t128), dim3(256), 0, st, a);
  } else if (plan == X8Plan::kTile128 && !wide) {
    hipLaunchKernelGGL((x8_tile_kernel<kX8Dense, 2, 2, 2, 2, false>), grid(t128), dim3(256), 0, st, a);
  } else if (plan == X8Plan::kTile128) {
    hipLaunchKernelGGL((x8_tile_kernel<kX8Dense, 2, 2, 2, 2, true>), grid(t128), dim3(256), 0, st, a);
  } else {
    // a wave for each block of K up to eight: K = 512 with eight waves, half of them idle, takes 0.6 us more
    const bool deep = k > 4 * kX8Block;
    if (wide && deep)
      hipLaunchKernelGGL((x8_deal_kernel<true, 8>), grid(t64), dim3(512), 0, st, a);
    else if (wide)
      hipLaunchKernelGGL((x8_deal_kernel<true, 4>), grid(t64), dim3(256), 0, st, a);
    else if (deep)
      hipLaunchKernelGGL((x8_deal_kernel<false, 8>), grid(t64), dim3(512), 0, st, a);
    else
      hipLaunchKernelGGL((x8_deal_kernel<false, 4>), grid(t64), dim3(256), 0, st, a);
  }
  return check_launch(who);
}
