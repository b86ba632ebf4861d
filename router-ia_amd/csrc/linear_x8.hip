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
#include "x8_tile.h"

namespace ria {

template <int XT>
__global__ __launch_bounds__(256) void quant_fp8_kernel(const QuantArgs a) {
  quant_unit<XT>(a, (int64_t)blockIdx.x * 256 + threadIdx.x);
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
  if (t128 > 0x7ffffff0) return set_error(RIA_ERR_INVALID, "%s: too many rows", who);
  const dim3 g256(static_cast<unsigned>((t256 + 7) / 8 * 8)), g128(static_cast<unsigned>((t128 + 7) / 8 * 8));
  if (y_dtype == RIA_DT_F32)
    hipLaunchKernelGGL((x8_tile_kernel<kX8Dense, 2, 2, 2, 2, true>), g128, dim3(256), 0, st, a);
  else if (t256 >= 256)
    hipLaunchKernelGGL((x8_tile_kernel<kX8Dense, 4, 2, 2, 4, false>), g256, dim3(512), 0, st, a);
  else
    hipLaunchKernelGGL((x8_tile_kernel<kX8Dense, 2, 2, 2, 2, false>), g128, dim3(256), 0, st, a);
  return check_launch(who);
}
