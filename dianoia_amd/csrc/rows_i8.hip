// Rows as int8 with one float32 scale a row: the activations and the weights
// of the products in gemm_i8r.hip. Per row, with y the row's values,
//   y_j = x_j                                   (quantize: weights, any rows)
//   y_j = w_j (s_j r), r = 1 / sqrt(mean(s^2) + eps), s = x + m or x  (norm)
//   top = max |y_j|, scale = top / 127, code_j = y_j / scale rounded to the
//   nearest whole number, halves away from zero; zeros past cols.
// No counterpart in the reference, whose 8-bit rows have a scale per 32
// values.
//
// The codes of a normed row do not depend on r: code_j = 127 w_j s_j / max
// |w s|. They are formed in 64 bits, where the product of two floats is
// exact, so a code is that of the formula, not of the order of a float sum.
// The factor 127 / top is rounded up by 2^-50: a value on the border of two
// codes (which bf16 weights meet: 254 x = (2 k + 1) top) then goes away from
// zero whatever the division's last bit, and no float strictly inside reaches
// the border: 254 x - (2 k + 1) top is a whole multiple of 2^-34 top or more.
// 64-bit multiply-adds run at the rate of 32-bit ones on this chip, so the
// rows stay bound by their bytes.

#include "codes_i8.h"
#include "common.h"
#include "dnx_kernels.h"

#include <math.h>

using namespace dnx;

namespace {

constexpr int kMaxThreads = 1024;
constexpr int kMaxV = 16;                                // four values each, per thread
constexpr int64_t kManyRows = 512;
constexpr int64_t kMaxRows = 1 << 22;                    // 2^32 threads in a launch
constexpr int64_t kMaxCols = (int64_t)kMaxThreads * kMaxV * 4;

// A wave's sum and maximum in 64 bits, and the maximum of unsigned words, on
// DPP (as wave_sum_dpp): every lane gets the same bits. All lanes active.
DNX_DEV double lane_value64(double v, int lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint64_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, lane);
  const uint64_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(b >> 32), lane);
  return __builtin_bit_cast(double, hi << 32 | lo);
}
DNX_DEV double wave_sum64(double v) {
  v += dpp64<kQuadXor1>(v);
  v += dpp64<kQuadXor2>(v);
  v += dpp64<kHalfRowMirror>(v);
  v += dpp64<kRowMirror>(v);
  return (lane_value64(v, 0) + lane_value64(v, 16)) + (lane_value64(v, 32) + lane_value64(v, 48));
}
DNX_DEV double wave_max64(double v) {
  v = fmax(v, dpp64<kQuadXor1>(v));
  v = fmax(v, dpp64<kQuadXor2>(v));
  v = fmax(v, dpp64<kHalfRowMirror>(v));
  v = fmax(v, dpp64<kRowMirror>(v));
  return fmax(fmax(lane_value64(v, 0), lane_value64(v, 16)),
              fmax(lane_value64(v, 32), lane_value64(v, 48)));
}
DNX_DEV uint32_t wave_max_u32(uint32_t v) {
  v = max(v, (uint32_t)dpp<kQuadXor1>((int)v));
  v = max(v, (uint32_t)dpp<kQuadXor2>((int)v));
  v = max(v, (uint32_t)dpp<kHalfRowMirror>((int)v));
  v = max(v, (uint32_t)dpp<kRowMirror>((int)v));
  auto lane = [&](int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); };
  return max(max(lane(0), lane(16)), max(lane(32), lane(48)));
}

DNX_DEV float4 load4(const float* p) { return *(const float4*)p; }
DNX_DEV float4 load4(const uint16_t* p) {
  const uint2 b = *(const uint2*)p;
  return make_float4(__uint_as_float(b.x << 16), __uint_as_float(b.x & 0xffff0000u),
                     __uint_as_float(b.y << 16), __uint_as_float(b.y & 0xffff0000u));
}

// Four normed values' part of a row's sum of squares and top = max |y| without
// r. The sum also tells of an infinity or NaN: it is finite in 64 bits for
// finite floats, and nothing times a product is added to it, for one in w.
DNX_DEV void norm4(float4 s4, float4 w4, double& sum, double& top) {
#pragma unroll
  for (int c = 0; c < 4; c++) {
    const double s = (&s4.x)[c], y = s * (double)(&w4.x)[c];
    sum = fma(y, 0.0, fma(s, s, sum));
    top = fmax(top, fabs(y));
  }
}

// The workgroup's sum and top.
DNX_DEV void norm_reduce(double& sum, double& top) {
  __shared__ double part[2][kMaxThreads / 64];
  const int tid = threadIdx.x;
  sum = wave_sum64(sum);
  top = wave_max64(top);
  if ((tid & 63) == 0) {
    part[0][tid >> 6] = sum;
    part[1][tid >> 6] = top;
  }
  __syncthreads();
  sum = part[0][0];
  top = part[1][0];
  for (int k = 1; k < (int)blockDim.x / 64; k++) {
    sum += part[0][k];
    top = fmax(top, part[1][k]);
  }
}

DNX_DEV float norm_scale(double sum, double top, int cols, float eps) {
  return (float)(top / 127.0 * (1.0 / sqrt(sum / (double)cols + (double)eps)));
}

// A normed row of more values than registers hold: read again for the codes.
// 512 x 32768 with addition and norm: 60 us, 3.7 TB/s (with 16 steps in registers,
// most of them spilled, 153).
template <bool kAdd>
__global__ void __launch_bounds__(kMaxThreads)
long_rows_i8_kernel(const float* x, const float* m, float* x_out, const float* __restrict__ w,
                    int8_t* __restrict__ qs, float* __restrict__ scales, int cols, int cols_pad,
                    float eps) {
  constexpr int U = 4;                    // steps whose loads are in flight together
  const int quads = cols / 4, threads = blockDim.x, tid = threadIdx.x;
  const size_t at = (size_t)blockIdx.x * cols;
  const float4 zero = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  double sum = 0.0, top = 0.0;
  for (int i0 = tid; i0 < quads; i0 += U * threads) {
    float4 s[U], u[U], a[U];
#pragma unroll
    for (int e = 0; e < U; e++) {
      const int i = i0 + e * threads;
      s[e] = u[e] = a[e] = zero;
      if (i < quads) {
        s[e] = load4(x + at + 4 * i);
        u[e] = load4(w + 4 * i);
        if constexpr (kAdd) a[e] = load4(m + at + 4 * i);
      }
    }
#pragma unroll
    for (int e = 0; e < U; e++) {
      const int i = i0 + e * threads;
      if constexpr (kAdd) {
        s[e] = make_float4(s[e].x + a[e].x, s[e].y + a[e].y, s[e].z + a[e].z, s[e].w + a[e].w);
        if (i < quads) *(float4*)(x_out + at + 4 * i) = s[e];
      }
      norm4(s[e], u[e], sum, top);
    }
  }
  norm_reduce(sum, top);
  const bool fine = sum < INFINITY;
  const double inv = code_factor(top, fine);
  const float* from = kAdd ? x_out : x;
  int* out = (int*)(qs + (size_t)blockIdx.x * cols_pad);
  for (int i0 = tid; i0 < quads; i0 += U * threads) {
    float4 s[U], u[U];
#pragma unroll
    for (int e = 0; e < U; e++) {
      const int i = i0 + e * threads;
      s[e] = u[e] = zero;
      if (i < quads) {
        s[e] = load4(from + at + 4 * i);
        u[e] = load4(w + 4 * i);
      }
    }
#pragma unroll
    for (int e = 0; e < U; e++) {
      int q[4];
#pragma unroll
      for (int c = 0; c < 4; c++)
        q[c] = code1((double)(&s[e].x)[c] * (double)(&u[e].x)[c], inv);
      const int i = i0 + e * threads;
      if (i < quads) out[i] = fine ? pack4(q[0], q[1], q[2], q[3]) : 0;
    }
  }
  for (int i = quads + tid; i < cols_pad / 4; i += threads) out[i] = 0;
  if (tid == 0) scales[blockIdx.x] = fine ? norm_scale(sum, top, cols, eps) : NAN;
}

// One workgroup a row, four values per thread and step e (V steps cover the
// row): the row stays in registers between the reduction and the codes, so
// each byte is read once. 4099 x 4096 with addition and norm: 44 us, 5.0 TB/s
// (a large copy reaches 4.6); 8192 x 4096 bf16 weights 24.5 us, 4.1 TB/s (69
// with 1024 threads a row and the reductions through LDS lanes: too few rows
// at once); 16 x 2048 with addition and norm 2.9 us, of which 2.0 are an empty
// launch's.
template <typename S, int V, bool kNorm, bool kAdd>
__global__ void __launch_bounds__(kMaxThreads)
rows_i8_kernel(const S* x, const float* __restrict__ m, float* x_out, const float* __restrict__ w,
               int8_t* __restrict__ qs, float* __restrict__ scales, int cols, int cols_pad,
               float eps) {
  const int quads = cols / 4, threads = blockDim.x, tid = threadIdx.x;
  const size_t at = (size_t)blockIdx.x * cols;
  // Every load of the row before the first store: x_out may be x.
  float4 xv[V], wv[V], mv[V];
#pragma unroll
  for (int e = 0; e < V; e++) {
    const int i = e * threads + tid;
    xv[e] = wv[e] = mv[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (i < quads) {
      xv[e] = load4(x + at + 4 * i);
      if constexpr (kNorm) wv[e] = load4(w + 4 * i);
      if constexpr (kAdd) mv[e] = load4(m + at + 4 * i);
    }
  }
  if constexpr (kAdd) {
#pragma unroll
    for (int e = 0; e < V; e++) {
      const int i = e * threads + tid;
      xv[e] = make_float4(xv[e].x + mv[e].x, xv[e].y + mv[e].y, xv[e].z + mv[e].z,
                          xv[e].w + mv[e].w);
      if (i < quads) *(float4*)(x_out + at + 4 * i) = xv[e];
    }
  }
  // top = max |y| without r; `fine`: the row holds no infinity or NaN. As they
  // are, the rows' sizes order as their bits do, infinities and NaN above all.
  double sum = 0.0, top = 0.0;
  bool fine;
  if constexpr (kNorm) {
#pragma unroll
    for (int e = 0; e < V; e++) norm4(xv[e], wv[e], sum, top);
    norm_reduce(sum, top);
    fine = sum < INFINITY;
  } else {
    __shared__ uint32_t part[kMaxThreads / 64];
    uint32_t bits = 0;
#pragma unroll
    for (int e = 0; e < V; e++)
#pragma unroll
      for (int c = 0; c < 4; c++) bits = max(bits, __float_as_uint((&xv[e].x)[c]) & 0x7fffffffu);
    bits = wave_max_u32(bits);
    if ((tid & 63) == 0) part[tid >> 6] = bits;
    __syncthreads();
    bits = part[0];
    for (int k = 1; k < threads / 64; k++) bits = max(bits, part[k]);
    fine = bits < 0x7f800000u;
    top = __uint_as_float(bits);
  }
  const double inv = code_factor(top, fine);
  int* out = (int*)(qs + (size_t)blockIdx.x * cols_pad);
#pragma unroll
  for (int e = 0; e < V; e++) {
    const int i = e * threads + tid;
    if (i >= quads) break;
    int q[4];
#pragma unroll
    for (int c = 0; c < 4; c++) {
      const double s = (&xv[e].x)[c];
      q[c] = code1(kNorm ? s * (double)(&wv[e].x)[c] : s, inv);
    }
    out[i] = fine ? pack4(q[0], q[1], q[2], q[3]) : 0;
  }
  for (int i = quads + tid; i < cols_pad / 4; i += threads) out[i] = 0;
  if (tid == 0) {
    const float scale = kNorm ? norm_scale(sum, top, cols, eps) : (float)(top / 127.0);
    scales[blockIdx.x] = fine ? scale : NAN;
  }
}

template <typename S, bool kNorm, bool kAdd>
int launch_rows(const S* x, const float* m, float* x_out, const float* w, int8_t* qs,
                float* scales, int64_t rows, int64_t cols, int64_t cols_pad, float eps,
                dnx_stream_t stream) {
  if (rows < 0 || rows >= kMaxRows || cols <= 0 || cols % 4 != 0 || cols > kMaxCols ||
      cols_pad < cols || cols_pad % kBlock != 0 || cols_pad > kMaxCols) {
    return DNX_EINVAL;
  }
  if (rows == 0) return DNX_OK;
  if (x == nullptr || qs == nullptr || scales == nullptr ||
      (((uintptr_t)x | (uintptr_t)m | (uintptr_t)x_out | (uintptr_t)w | (uintptr_t)qs) & 15) != 0 ||
      ((uintptr_t)scales & 3) != 0) {
    return DNX_EINVAL;
  }
  const int64_t quads = cols / 4;
  const int64_t steps = (quads + kMaxThreads - 1) / kMaxThreads;
  // Few rows: as many threads as hold a row (latency). Many: four steps a
  // thread, more rows at once.
  const int V = rows >= kManyRows && steps <= 4 ? 4
                : steps <= 1 ? 1 : steps <= 2 ? 2 : steps <= 4 ? 4 : kMaxV;
  const unsigned threads = (unsigned)(((quads + V - 1) / V + 63) / 64 * 64);
  auto launch = [&](auto k, unsigned n) {
    hipLaunchKernelGGL(k, dim3((unsigned)rows), dim3(n), 0, (hipStream_t)stream, x, m, x_out, w, qs,
                       scales, (int)cols, (int)cols_pad, eps);
  };
  if (V == 1) {
    launch(rows_i8_kernel<S, 1, kNorm, kAdd>, threads);
  } else if (V == 2) {
    launch(rows_i8_kernel<S, 2, kNorm, kAdd>, threads);
  } else if (V == 4) {
    launch(rows_i8_kernel<S, 4, kNorm, kAdd>, threads);
  } else if constexpr (kNorm) {
    launch(long_rows_i8_kernel<kAdd>, kMaxThreads);
  } else {
    launch(rows_i8_kernel<S, kMaxV, kNorm, kAdd>, threads);
  }
  return hipGetLastError() == hipSuccess ? DNX_OK : DNX_ELAUNCH;
}

}  // namespace

extern "C" {

int dnx_quantize_i8r(const float* x, int8_t* qs, float* scales, int64_t rows, int64_t cols,
                     int64_t cols_pad, dnx_stream_t stream) {
  return launch_rows<float, false, false>(x, nullptr, nullptr, nullptr, qs, scales, rows, cols,
                                          cols_pad, 0.0f, stream);
}

int dnx_quantize_i8r_bf16(const uint16_t* x, int8_t* qs, float* scales, int64_t rows, int64_t cols,
                          int64_t cols_pad, dnx_stream_t stream) {
  return launch_rows<uint16_t, false, false>(x, nullptr, nullptr, nullptr, qs, scales, rows, cols,
                                             cols_pad, 0.0f, stream);
}

int dnx_rms_norm_i8r(const float* x, const float* m, float* x_out, const float* w, int8_t* qs,
                     float* scales, int64_t rows, int64_t cols, int64_t cols_pad, float eps,
                     dnx_stream_t stream) {
  if (rows != 0 && (w == nullptr || (m == nullptr) != (x_out == nullptr))) return DNX_EINVAL;
  if (m != nullptr) {
    return launch_rows<float, true, true>(x, m, x_out, w, qs, scales, rows, cols, cols_pad, eps,
                                          stream);
  }
  return launch_rows<float, true, false>(x, nullptr, nullptr, w, qs, scales, rows, cols, cols_pad,
                                         eps, stream);
}

}  // extern "C"
