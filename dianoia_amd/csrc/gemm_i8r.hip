// y[t][r] = xs[t] ws[r] sum_k xq[t][k] wq[r][k]: int8 rows times int8 weight
// rows with one scale each, on the int8 matrix cores. The sums are whole
// numbers, exact in int32 (|q| <= 128: K up to 131040), so no order of adding
// changes a result; each output is rounded to float32 three times (the sum,
// the product of the scales, their product).

#include "common.h"
#include "dnx_kernels.h"

using namespace dnx;

namespace {

typedef int v16i __attribute__((ext_vector_type(16)));

constexpr int64_t kMaxK = 131040;   // fewer than 2^17 products of 2^14 or less: below 2^31

// A wave takes 32 tokens x 32 weight rows, a workgroup 2 x 2 of them; one
// v_mfma_i32_32x32x32_i8 per 32 of K, both operands straight from memory
// (lane l: row l % 32, the 16 bytes at k = 16 (l / 32)). Tokens and rows past
// the last read the last, and are not stored.
__global__ void __launch_bounds__(256)
gemm_i8r_kernel(const int8_t* __restrict__ w, const float* __restrict__ w_scale,
                const int8_t* __restrict__ x, const float* __restrict__ x_scale,
                float* __restrict__ y, int rows, int cols, int n) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int t0 = blockIdx.y * 64 + (wave >> 1) * 32, r0 = blockIdx.x * 64 + (wave & 1) * 32;
  const int half = lane >> 5, l32 = lane & 31;
  const int8_t* xp = x + (size_t)min(t0 + l32, n - 1) * cols + 16 * half;
  const int8_t* wp = w + (size_t)min(r0 + l32, rows - 1) * cols + 16 * half;
  v16i acc = {};
#pragma unroll 4
  for (int k = 0; k < cols; k += 32) {
    acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(*(const i32x4*)(xp + k), *(const i32x4*)(wp + k),
                                                acc, 0, 0, 0);
  }
  const int r = r0 + l32;
  if (r >= rows) return;
  const float ws = w_scale[r];
#pragma unroll
  for (int v = 0; v < 16; v++) {
    const int t = t0 + 8 * (v >> 2) + 4 * half + (v & 3);
    if (t < n) y[(size_t)t * rows + r] = (float)acc[v] * (x_scale[t] * ws);
  }
}

}  // namespace

extern "C" {

int dnx_gemm_i8r(const int8_t* w, const float* w_scale, const int8_t* x, const float* x_scale,
                 float* y, int64_t rows, int64_t cols, int64_t n, dnx_stream_t stream) {
  if (rows <= 0 || rows > 0x7fffffff || n < 0 || n > 65535 * 64 || cols <= 0 ||
      cols % kBlock != 0 || cols > kMaxK) {
    return DNX_EINVAL;
  }
  if (n == 0) return DNX_OK;
  if (w == nullptr || w_scale == nullptr || x == nullptr || x_scale == nullptr || y == nullptr ||
      (((uintptr_t)w | (uintptr_t)x) & 15) != 0 ||
      (((uintptr_t)w_scale | (uintptr_t)x_scale | (uintptr_t)y) & 3) != 0) {
    return DNX_EINVAL;
  }
  const dim3 grid((unsigned)((rows + 63) / 64), (unsigned)((n + 63) / 64));
  hipLaunchKernelGGL(gemm_i8r_kernel, grid, dim3(256), 0, (hipStream_t)stream, w, w_scale, x,
                     x_scale, y, (int)rows, (int)cols, (int)n);
  return hipGetLastError() == hipSuccess ? DNX_OK : DNX_ELAUNCH;
}

}  // extern "C"
