// The append of new tokens' keys and values to a paged cache, with their
// per-head norm and rotation. No counterpart in the reference, which serves
// one sequence from one contiguous cache.

#include "bf16_pieces.h"
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
  int n, heads, kv_heads;
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
  bool turn = a.rope != nullptr;
  const int nq = per - 2 * a.kv_heads;
  if (h < nq) {
    src = a.q + t * a.q_stride + h * HD;
    norm = a.q_norm;
    dst_q = a.q_out + ((int64_t)t * nq + h) * HD;
  } else if ((h -= nq) < a.kv_heads) {
    src = a.k + t * a.k_stride + h * HD;
    norm = a.k_norm;
    dst = (C*)a.keys + (slot * a.kv_heads + h) * HD;
  } else {
    h -= a.kv_heads;
    src = a.v + t * a.v_stride + h * HD;
    turn = false;
    dst = (C*)a.values + (slot * a.kv_heads + h) * HD;
  }
  float4 x = *(const float4*)(src + 4 * l), y = *(const float4*)(src + HD / 2 + 4 * l);
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
  } else {
    store4(dst + 4 * l, x);
    store4(dst + HD / 2 + 4 * l, y);
  }
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
  const AppendArgs a{q, k, v, q_norm, k_norm, rope, q_out, positions, slots, q_stride, k_stride,
                     v_stride, rope_rows, cache->pages * cache->page, cache->keys, cache->values,
                     (int)n, (int)heads, cache->kv_heads, eps};
  const int64_t units = n * ((q != nullptr ? heads : 0) + 2 * cache->kv_heads);
  const int64_t per = kThreads / (cache->hd / 8);
  const int64_t grid = (units + per - 1) / per;
  if (grid > kLaunchThreads / kThreads) return DNX_EINVAL;
  auto k_ = cache->type == DNX_F32
                ? (cache->hd == 128 ? append_kernel<float, 128> : append_kernel<float, 64>)
                : (cache->hd == 128 ? append_kernel<uint16_t, 128> : append_kernel<uint16_t, 64>);
  hipLaunchKernelGGL(k_, dim3((unsigned)grid), dim3(kThreads), 0, (hipStream_t)stream, a);
  return hipGetLastError() == hipSuccess ? DNX_OK : DNX_ELAUNCH;
}

}  // extern "C"
