// The append of new tokens' keys and values to a paged cache, with their
// per-head norm and rotation, and the reading of its places as float32. No
// counterpart in the reference, which serves one sequence from one contiguous
// cache.

#include "bf16_pieces.h"
#include "codes_i8.h"
#include "common.h"
#include "paged.h"

#include <math.h>

using namespace dnx;

namespace {

constexpr int kThreads = 256;

struct AppendArgs {
  const float *q, *k, *v, *q_norm, *k_norm, *rope;
  float* q_out;
  const int32_t *positions, *slots;
  int64_t q_stride, k_stride, v_stride, rope_rows, places;
  void *keys, *values;
  float *key_scales, *value_scales;
  int n, heads, kv_heads, page_bits;
  float eps;
};

DNX_DEV void store4(float* p, float4 v) { *(float4*)p = v; }
DNX_DEV void store4(uint16_t* p, float4 v) {
  const f32x2 a = {v.x, v.y}, b = {v.z, v.w};
  *(uint2*)p = make_uint2(__builtin_bit_cast(uint32_t, __builtin_convertvector(a, bf2)),
                          __builtin_bit_cast(uint32_t, __builtin_convertvector(b, bf2)));
}

// Sum over an aligned group of LT = 8 or 16 lanes, by DPP.
template <int LT>
DNX_DEV float lanes_sum(float v) {
  v += dppf<kQuadXor1>(v);
  v += dppf<kQuadXor2>(v);
  v += dppf<kHalfRowMirror>(v);
  if constexpr (LT == 16) v += dppf<kRowMirror>(v);
  return v;
}
template <int LT>
DNX_DEV double lanes_sum(double v) {
  v += dpp64<kQuadXor1>(v);
  v += dpp64<kQuadXor2>(v);
  v += dpp64<kHalfRowMirror>(v);
  if constexpr (LT == 16) v += dpp64<kRowMirror>(v);
  return v;
}
template <int LT>
DNX_DEV double lanes_max(double v) {
  v = fmax(v, dpp64<kQuadXor1>(v));
  v = fmax(v, dpp64<kQuadXor2>(v));
  v = fmax(v, dpp64<kHalfRowMirror>(v));
  if constexpr (LT == 16) v = fmax(v, dpp64<kRowMirror>(v));
  return v;
}

// A key or value head as int8 codes and one scale. In 64 bits, so that a code
// is that of the formula and not of the order of a float sum: the product of
// two floats is exact there, the norm's factor r drops out of the codes
// (127 y / max |y|) and is left to the scale. The 64-bit work hides behind the
// bytes: 4093 tokens of 32 / 8 heads, hd 128, 36 us, 4.9 TB/s (to bf16 36 too);
// one token of 16 / 8 heads 2.5, of which 2.0 are an empty launch's.
template <int HD>
DNX_DEV void append_codes(float4 x, float4 y, const float* norm, const float* rope, float eps,
                          int l, int8_t* dst, float* scale) {
  constexpr int LT = HD / 8;
  double u[4], w[4], r = 1.0;
#pragma unroll
  for (int c = 0; c < 4; c++) {
    u[c] = (double)(&x.x)[c];
    w[c] = (double)(&y.x)[c];
  }
  if (norm != nullptr) {
    const float4 f = *(const float4*)(norm + 4 * l), g = *(const float4*)(norm + HD / 2 + 4 * l);
    double sum = 0.0;
#pragma unroll
    for (int c = 0; c < 4; c++) {
      sum = fma(u[c], u[c], fma(w[c], w[c], sum));
      u[c] *= (double)(&f.x)[c];
      w[c] *= (double)(&g.x)[c];
    }
    r = 1.0 / sqrt(lanes_sum<LT>(sum) / (double)HD + (double)eps);
  }
  if (rope != nullptr) {
    const float4 cs = *(const float4*)(rope + 4 * l), sn = *(const float4*)(rope + HD / 2 + 4 * l);
#pragma unroll
    for (int c = 0; c < 4; c++) {
      const double a = u[c], b = w[c], co = (double)(&cs.x)[c], si = (double)(&sn.x)[c];
      u[c] = fma(a, co, -(b * si));
      w[c] = fma(b, co, a * si);
    }
  }
  double top = 0.0, check = 0.0;
#pragma unroll
  for (int c = 0; c < 4; c++) {
    top = fmax(top, fmax(fabs(u[c]), fabs(w[c])));
    check = fma(u[c], 0.0, fma(w[c], 0.0, check));   // NaN for an infinity or NaN
  }
  top = lanes_max<LT>(top);
  const float s = (float)(top / 127.0 * r);
  const bool fine = lanes_sum<LT>(check) == 0.0 && s < INFINITY;
  const double inv = code_factor(top, fine);
  int a[4], b[4];
#pragma unroll
  for (int c = 0; c < 4; c++) {
    a[c] = fine ? code1(u[c], inv) : 0;
    b[c] = fine ? code1(w[c], inv) : 0;
  }
  *(int*)(dst + 4 * l) = pack4(a[0], a[1], a[2], a[3]);
  *(int*)(dst + HD / 2 + 4 * l) = pack4(b[0], b[1], b[2], b[3]);
  if (l == 0) *scale = fine ? s : NAN;
}

// HD / 8 lanes a head of a token: lane l holds dims 4 l .. 4 l + 3 and their
// partners HD / 2 further, 16 bytes each, so a pair of the rotation lies in
// one lane. The heads of a token follow each other: the queries (where there
// are any), the keys, the values. Every byte is read and written once, and that
// is what it costs: 4093 tokens of 32 / 8 heads, hd 128, to bf16 36 us, 5.1 TB/s
// (a large copy reaches 4.6); one token of 16 / 8 heads 2.4 us, of which 2.0 are
// an empty launch's.
template <typename C, int HD>
__global__ void __launch_bounds__(kThreads) append_kernel(AppendArgs a) {
  constexpr int LT = HD / 8;
  const int per = (a.q != nullptr ? a.heads : 0) + 2 * a.kv_heads;
  const int64_t unit = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / LT;
  if (unit >= (int64_t)a.n * per) return;   // whole groups of lanes
  const int l = threadIdx.x % LT;
  const int t = (int)(unit / per);
  int h = (int)(unit - (int64_t)t * per);
  const int64_t slot = a.slots[t];
  const int64_t pos = a.rope != nullptr ? a.positions[t] : 0;
  if (slot < 0 || slot >= a.places || pos < 0 || (a.rope != nullptr && pos >= a.rope_rows)) return;
  const float* src;
  const float* norm = nullptr;
  float* dst_q = nullptr;
  C* dst = nullptr;
  float* scale = nullptr;
  bool turn = a.rope != nullptr;
  const int nq = per - 2 * a.kv_heads;
  // int8: where the scale of this place and head 0 lies.
  const int64_t scale_at = ((slot >> a.page_bits) * a.kv_heads << a.page_bits) +
                           (slot & ((1 << a.page_bits) - 1));
  if (h < nq) {
    src = a.q + t * a.q_stride + h * HD;
    norm = a.q_norm;
    dst_q = a.q_out + ((int64_t)t * nq + h) * HD;
  } else if ((h -= nq) < a.kv_heads) {
    src = a.k + t * a.k_stride + h * HD;
    norm = a.k_norm;
    dst = (C*)a.keys + (slot * a.kv_heads + h) * HD;
    scale = a.key_scales + scale_at + ((int64_t)h << a.page_bits);
  } else {
    h -= a.kv_heads;
    src = a.v + t * a.v_stride + h * HD;
    turn = false;
    dst = (C*)a.values + (slot * a.kv_heads + h) * HD;
    scale = a.value_scales + scale_at + ((int64_t)h << a.page_bits);
  }
  float4 x = *(const float4*)(src + 4 * l), y = *(const float4*)(src + HD / 2 + 4 * l);
  if constexpr (sizeof(C) == 1) {
    if (dst_q == nullptr) {
      append_codes<HD>(x, y, norm, turn ? a.rope + pos * HD : nullptr, a.eps, l, dst, scale);
      return;
    }
  }
  if (norm != nullptr) {
    float s = (x.x * x.x + y.x * y.x) + (x.y * x.y + y.y * y.y) + (x.z * x.z + y.z * y.z) +
              (x.w * x.w + y.w * y.w);
    s = lanes_sum<LT>(s);
    const float r = 1.0f / sqrtf(s / (float)HD + a.eps);
    const float4 u = *(const float4*)(norm + 4 * l), w = *(const float4*)(norm + HD / 2 + 4 * l);
    x = make_float4(u.x * (x.x * r), u.y * (x.y * r), u.z * (x.z * r), u.w * (x.w * r));
    y = make_float4(w.x * (y.x * r), w.y * (y.y * r), w.z * (y.z * r), w.w * (y.w * r));
  }
  if (turn) {
    const float* row = a.rope + pos * HD + 4 * l;
    const float4 c = *(const float4*)row, s = *(const float4*)(row + HD / 2);
    const float4 p = x;
    x = make_float4(p.x * c.x - y.x * s.x, p.y * c.y - y.y * s.y, p.z * c.z - y.z * s.z,
                    p.w * c.w - y.w * s.w);
    y = make_float4(y.x * c.x + p.x * s.x, y.y * c.y + p.y * s.y, y.z * c.z + p.z * s.z,
                    y.w * c.w + p.w * s.w);
  }
  if (dst_q != nullptr) {
    store4(dst_q + 4 * l, x);
    store4(dst_q + HD / 2 + 4 * l, y);
  } else if constexpr (sizeof(C) > 1) {
    store4(dst + 4 * l, x);
    store4(dst + HD / 2 + 4 * l, y);
  }
}

struct ReadArgs {
  const void *keys, *values;
  const float *key_scales, *value_scales;
  const int32_t* slots;
  float *k, *v;
  int64_t k_stride, v_stride, places;
  int n, kv_heads, page_bits;
};

DNX_DEV float4 widen4(const float* p) { return *(const float4*)p; }
DNX_DEV float4 widen4(const uint16_t* p) {
  const uint2 b = *(const uint2*)p;
  return make_float4(__uint_as_float(b.x << 16), __uint_as_float(b.x & 0xffff0000u),
                     __uint_as_float(b.y << 16), __uint_as_float(b.y & 0xffff0000u));
}
DNX_DEV float4 widen4(const int8_t* p) {
  const int b = *(const int*)p;
  return make_float4((float)(int8_t)b, (float)(int8_t)(b >> 8), (float)(int8_t)(b >> 16),
                     (float)(b >> 24));
}

// Four dims of one place's key head and value head a thread: 16-byte stores, in
// order of the outputs, which are most of the bytes. int8, 8191 places of 8 heads, hd
// 128: 15.4 us, 5.5 TB/s (a large copy reaches 5.0); the same places again, which the
// caches hold in part, int8 12.9, bf16 14.0, float32 18.1; 37 places of 2 heads, hd
// 64, 2.2 to 2.4 from each type, of which 2.0 are an empty launch's.
template <typename C, int HD>
__global__ void __launch_bounds__(kThreads) read_kernel(ReadArgs a) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t unit = i / (HD / 4);
  if (unit >= (int64_t)a.n * a.kv_heads) return;
  const int c = (int)(i % (HD / 4)), t = (int)(unit / a.kv_heads);
  const int h = (int)(unit - (int64_t)t * a.kv_heads);
  const int64_t slot = a.slots[t];
  if (slot < 0 || slot >= a.places) return;
  const int64_t at = (slot * a.kv_heads + h) * HD + 4 * c;
  const int64_t scale_at = (((slot >> a.page_bits) * a.kv_heads + h) << a.page_bits) +
                           (slot & ((1 << a.page_bits) - 1));
  auto one = [&](const void* from, const float* scales, float* to) {
    float4 x = widen4((const C*)from + at);
    if constexpr (sizeof(C) == 1) {
      const float s = scales[scale_at];
      x = make_float4(x.x * s, x.y * s, x.z * s, x.w * s);
    }
    *(float4*)to = x;
  };
  if (a.k != nullptr) one(a.keys, a.key_scales, a.k + t * a.k_stride + h * HD + 4 * c);
  if (a.v != nullptr) one(a.values, a.value_scales, a.v + t * a.v_stride + h * HD + 4 * c);
}

}  // namespace

extern "C" {

int dnx_paged_append(const dnx_paged_cache* cache, const float* q, int64_t q_stride, float* q_out,
                     const float* k, int64_t k_stride, const float* v, int64_t v_stride,
                     const float* q_norm, const float* k_norm, const float* rope,
                     int64_t rope_rows, const int32_t* positions, const int32_t* slots,
                     int64_t heads, int64_t n, float eps, dnx_stream_t stream) {
  if (!cache_ok(cache) || n < 0 || n > (1 << 22) || heads < 0 || heads > 65535) return DNX_EINVAL;
  if (n == 0) return DNX_OK;
  const int64_t kv_dim = (int64_t)cache->kv_heads * cache->hd;
  const uintptr_t all = (uintptr_t)q | (uintptr_t)q_out | (uintptr_t)k | (uintptr_t)v |
                        (uintptr_t)q_norm | (uintptr_t)k_norm | (uintptr_t)rope;
  if (k == nullptr || v == nullptr || slots == nullptr || (all & 15) != 0 ||
      (((uintptr_t)positions | (uintptr_t)slots) & 3) != 0 || k_stride < kv_dim ||
      v_stride < kv_dim || k_stride % 4 != 0 || v_stride % 4 != 0 ||
      (rope != nullptr && (positions == nullptr || rope_rows <= 0)) ||
      (q != nullptr && (q_out == nullptr || heads == 0 || q_stride < heads * cache->hd ||
                        q_stride % 4 != 0))) {
    return DNX_EINVAL;
  }
  const CacheScales scales = cache_scales(cache);
  const AppendArgs a{q, k, v, q_norm, k_norm, rope, q_out, positions, slots, q_stride, k_stride,
                     v_stride, rope_rows, cache->pages * cache->page, cache->keys, cache->values,
                     scales.keys, scales.values, (int)n, (int)heads, cache->kv_heads,
                     __builtin_ctz((unsigned)cache->page), eps};
  const int64_t units = n * ((q != nullptr ? heads : 0) + 2 * cache->kv_heads);
  const int64_t per = kThreads / (cache->hd / 8);
  const int64_t grid = (units + per - 1) / per;
  if (grid > kLaunchThreads / kThreads) return DNX_EINVAL;
  constexpr decltype(&append_kernel<float, 64>) kernels[] = {
      append_kernel<float, 64>,     append_kernel<float, 128>,  append_kernel<uint16_t, 64>,
      append_kernel<uint16_t, 128>, append_kernel<int8_t, 64>, append_kernel<int8_t, 128>};
  hipLaunchKernelGGL(kernels[2 * cache->type + (cache->hd == 128)], dim3((unsigned)grid),
                     dim3(kThreads), 0, (hipStream_t)stream, a);
  return hipGetLastError() == hipSuccess ? DNX_OK : DNX_ELAUNCH;
}

int dnx_paged_read(const dnx_paged_cache* cache, const int32_t* slots, float* k, int64_t k_stride,
                   float* v, int64_t v_stride, int64_t n, dnx_stream_t stream) {
  if (!cache_ok(cache) || n < 0 || n > (1 << 22)) return DNX_EINVAL;
  if (n == 0) return DNX_OK;
  const int64_t kv_dim = (int64_t)cache->kv_heads * cache->hd;
  if (slots == nullptr || ((uintptr_t)slots & 3) != 0 || (k == nullptr && v == nullptr) ||
      (((uintptr_t)k | (uintptr_t)v) & 15) != 0 ||
      (k != nullptr && (k_stride < kv_dim || k_stride % 4 != 0)) ||
      (v != nullptr && (v_stride < kv_dim || v_stride % 4 != 0))) {
    return DNX_EINVAL;
  }
  const CacheScales scales = cache_scales(cache);
  const ReadArgs a{cache->keys, cache->values, scales.keys, scales.values, slots, k, v,
                   k_stride, v_stride, cache->pages * cache->page, (int)n, cache->kv_heads,
                   __builtin_ctz((unsigned)cache->page)};
  const int64_t grid = (n * kv_dim / 4 + kThreads - 1) / kThreads;
  if (grid > kLaunchThreads / kThreads) return DNX_EINVAL;
  constexpr decltype(&read_kernel<float, 64>) kernels[] = {
      read_kernel<float, 64>,     read_kernel<float, 128>,  read_kernel<uint16_t, 64>,
      read_kernel<uint16_t, 128>, read_kernel<int8_t, 64>, read_kernel<int8_t, 128>};
  hipLaunchKernelGGL(kernels[2 * cache->type + (cache->hd == 128)], dim3((unsigned)grid),
                     dim3(kThreads), 0, (hipStream_t)stream, a);
  return hipGetLastError() == hipSuccess ? DNX_OK : DNX_ELAUNCH;
}

}  // extern "C"
