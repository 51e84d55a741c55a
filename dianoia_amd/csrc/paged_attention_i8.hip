// The attention of paged_attention.hip over int8 caches: keys and values are
// codes from -127 to 127 with a float32 scale for each place and head. For a
// row (a query head of a token) and the keys j it sees,
//   s_j = ks_j (q.c_j) / sqrt(hd),
//   out = sum_j e^(s_j - m) vs_j d_j / sum_j e^(s_j - m).

#include "common.h"
#include "paged.h"
#include "paged_i8.h"

#include <math.h>

using namespace dnx;

namespace {

struct SimpleArgs {
  dnx_paged_cache c;
  dnx_paged_batch b;
  const float *q, *gate;
  float* out;
  int64_t max_own, window;
  int heads, group, page_bits;
  float scale;
};

// One wave a row: 64 keys a step, one a lane, then the step's values, the dims
// dealt to the lanes.
template <int HD>
__global__ void __launch_bounds__(64) simple_kernel(SimpleArgs a) {
  __shared__ float q[HD];
  const int64_t row = blockIdx.x;
  const int token = (int)(row / a.heads), head = (int)(row % a.heads), kvh = head / a.group;
  const int lane = threadIdx.x, seqs = (int)a.b.seqs, kv = a.c.kv_heads;
  const int live = max(0, min(a.b.starts[seqs], (int)a.b.tokens));
  if (token >= live) return;
  int lo = 0, hi = seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.b.starts[mid] <= token) lo = mid; else hi = mid;
  }
  for (int i = lane; i < HD; i += 64) q[i] = a.q[row * HD + i] * a.scale;
  __syncthreads();
  const int64_t prefix = a.b.prefix_len, len = a.b.lens[lo];
  const int64_t place = prefix + len - min(a.b.starts[lo + 1], live) + token;
  const int64_t from = a.window > 0 ? max(place, (int64_t)0) - a.window + 1 : 0;
  const int64_t own = max(min(len, a.max_own), (int64_t)0);
  const int64_t to = prefix + max(min(own, place + 1 - prefix), (int64_t)0);
  const int mask = (1 << a.page_bits) - 1;
  float m = -INFINITY, l = 0.0f, o[HD / 64] = {};
  for (int64_t k0 = max(from, (int64_t)0) / 64 * 64; k0 < to; k0 += 64) {
    const int64_t key = k0 + lane;
    bool seen = key >= from && key < to;
    int64_t slot = 0, scale_at = 0;
    if (seen) {
      const bool first = key < prefix;
      const int64_t at = first ? key : key - prefix;
      const int64_t page = first ? a.b.prefix_pages[at >> a.page_bits]
                                 : a.b.tables[lo * a.b.table_stride + (at >> a.page_bits)];
      seen = page >= 0 && page < a.c.pages;
      slot = (page << a.page_bits) + (at & mask);
      scale_at = ((page * kv + kvh) << a.page_bits) + (at & mask);
    }
    float s = -INFINITY, vs = 0.0f;
    if (seen) {
      const int8_t* k = (const int8_t*)a.c.keys + (slot * kv + kvh) * HD;
      s = 0.0f;
      for (int i = 0; i < HD; i++) s = fmaf(q[i], (float)k[i], s);
      s *= a.c.key_scales[scale_at];
      vs = a.c.value_scales[scale_at];
    }
    const float top = fmaxf(m, wave_max_dpp(s)), ref = top == -INFINITY ? 0.0f : top;
    const float alpha = expf(m - ref), p = expf(s - ref);
    l = l * alpha + wave_sum_dpp(p);
    m = top;
    for (int j = 0; j < HD / 64; j++) o[j] *= alpha;
    const uint64_t with = __ballot(seen);
    for (int i = 0; i < 64; i++) {
      if (!((with >> i) & 1)) continue;
      const float w = lane_value(p, i) * lane_value(vs, i);
      const int64_t at = __shfl(slot, i);
      const int8_t* v = (const int8_t*)a.c.values + (at * kv + kvh) * HD;
      for (int j = 0; j < HD / 64; j++) o[j] = fmaf(w, (float)v[lane + 64 * j], o[j]);
    }
  }
  float f = l == 0.0f ? 0.0f : 1.0f / l;
  if (a.gate != nullptr) f /= 1.0f + expf(-a.gate[row]);
  for (int j = 0; j < HD / 64; j++) a.out[row * HD + lane + 64 * j] = o[j] * f;
}

}  // namespace

namespace dnx {

int paged_attention_i8(const dnx_paged_cache* cache, const dnx_paged_batch* batch, const float* q,
                       const float* gate, float* out, int64_t heads, int64_t window,
                       int64_t max_own, hipStream_t stream) {
  const SimpleArgs a{*cache, *batch, q, gate, out, max_own, window, (int)heads,
                     (int)(heads / cache->kv_heads), __builtin_ctz((unsigned)cache->page),
                     (float)(1.0 / sqrt((double)cache->hd))};
  auto k = cache->hd == 128 ? simple_kernel<128> : simple_kernel<64>;
  hipLaunchKernelGGL(k, dim3((unsigned)(batch->tokens * heads)), dim3(64), 0, stream, a);
  return hipGetLastError() == hipSuccess ? DNX_OK : DNX_ELAUNCH;
}

}  // namespace dnx
