// Keys and values in pages: the append of new tokens with their per-head norm
// and rotation, and the attention of a batch of sequences over a shared
// beginning and their own pages. No counterpart in the reference, which
// serves one sequence from one contiguous cache.

#include "common.h"
#include "dnx_kernels.h"
#include "paged_split.h"

#include <algorithm>

#include <math.h>

using namespace dnx;

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));

bool cache_ok(const dnx_paged_cache* c) {
  return c != nullptr && c->keys != nullptr && c->values != nullptr &&
         (((uintptr_t)c->keys | (uintptr_t)c->values) & 15) == 0 && c->pages > 0 &&
         c->page >= 16 && c->page <= 4096 && (c->page & (c->page - 1)) == 0 &&
         c->pages * c->page <= 0x7fffffff && (c->hd == 64 || c->hd == 128) && c->kv_heads > 0 &&
         c->kv_heads <= 1024 && (c->type == DNX_F32 || c->type == DNX_BF16);
}

// ---------------------------------------------------------------- the append

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
// are any), the keys, the values.
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

// ------------------------------------------------------------- the attention

struct PagedArgs {
  const void *keys, *values;
  int64_t pages;
  int page_bits, kv_heads, heads, group;
  const int32_t *starts, *lens, *tables, *prefix_pages;
  int64_t table_stride;
  int prefix_len, seqs, tokens, max_len;
  const float *q, *gate;
  float *out, *stat, *part;   // partials: stat [rows][splits][2], part [rows][splits][hd]
  int window, splits, prefix_splits, own_splits;
  int prefix_run, own_run, prefix_rows, own_rows;
  int64_t prefix_items;
  float scale;
};

// Max and sum over lanes i, i ^ 16, i ^ 32, i ^ 48, on the VALU lane swaps.
DNX_DEV float quarter_max(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
DNX_DEV float quarter_sum(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// The factor that takes a partial sum (m, l) to the maximum `top`. A partial
// without a weight (l = 0: no key seen, or every score -inf) counts for
// nothing; its m is -inf, which a partial whose scores are all NaN has too.
DNX_DEV float partial_factor(float m, float l, float top) {
  return l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - top);
}

// A row's output: o / l times its gate, zeros where no key had a weight.
DNX_DEV float row_scale(float l, const float* gate, int64_t row) {
  const float s = l == 0.0f ? 0.0f : 1.0f / l;
  return gate != nullptr ? s / (1.0f + expf(-gate[row])) : s;
}

// E values of a row of the cache as floats: 16 bytes, or 8 where E is 4 and
// the cache holds bf16.
template <typename C, int E>
DNX_DEV void load_row(i32x4 rsrc, int offset, float* x) {
  if constexpr (sizeof(C) == 4) {
    const float4 v = buffer_load_f4(rsrc, offset);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else {
    uint32_t b[E / 2];
    if constexpr (E == 8) {
      const uint4 v = buffer_load16(rsrc, offset);
      b[0] = v.x, b[1] = v.y, b[2] = v.z, b[3] = v.w;
    } else {
      const i32x2 v = dnx_raw_buffer_load_v2i32(rsrc, offset, 0, 0);
      b[0] = (uint32_t)v.x, b[1] = (uint32_t)v.y;
    }
#pragma unroll
    for (int j = 0; j < E / 2; j++) {
      x[2 * j] = __uint_as_float(b[j] << 16);
      x[2 * j + 1] = __uint_as_float(b[j] & 0xffff0000u);
    }
  }
}

// One workgroup: 16 rows of one key head against a run of keys, each wave
// taking every fourth 16 of them, on the float32 matrix cores straight from
// memory. Products are exact, sums float32.
// * S^T = K Q^T, 16 keys x 16 rows: lane l holds key l % 16 and row l % 16 at
//   the dims that its quarter g = l / 16 takes, and ends with the scores of
//   row l % 16 for keys 4 g + 0..3;
// * O^T += V^T P^T: step v takes the keys 4 g + v, whose weights lane l has
//   just formed; lane l loads dims EV (l % 16) .. of those keys' values.
// The resources of a 16-key step end with the last key, so that what lies
// behind it in its page is never read; the page is the same for all 16.
template <typename C, int HD>
__global__ void __launch_bounds__(kThreads) paged_attention_kernel(PagedArgs a) {
  constexpr int EK = 16 / sizeof(C), ND = HD / (4 * EK);     // K: ND loads of EK dims
  constexpr int EV = EK < HD / 16 ? EK : HD / 16, NH = HD / (16 * EV);   // V: NH loads a key
  const int lane = threadIdx.x & 63, l16 = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int live = max(0, min(a.starts[a.seqs], a.tokens));

  // What this workgroup takes: rows r0 .. of key head kvh, keys k_lo .. k_hi.
  int64_t item = blockIdx.x;
  const bool own = item >= a.prefix_items;
  if (own) item -= a.prefix_items;
  const int nrb = own ? a.own_rows : a.prefix_rows, nsp = own ? a.own_splits : a.prefix_splits;
  const int rb = (int)(item % nrb);
  item /= nrb;
  const int split = (int)(item % nsp);
  item /= nsp;
  const int kvh = (int)(item % a.kv_heads), b = (int)(item / a.kv_heads);
  int t0 = 0, t1 = live, count = a.prefix_len, run = a.prefix_run, first = 0;
  const int32_t* table = a.prefix_pages;
  if (own) {
    t0 = max(0, min(a.starts[b], live));
    t1 = max(t0, min(a.starts[b + 1], live));
    const int len = a.lens[b];
    first = len - (t1 - t0);    // the own place of the sequence's first new token
    table = a.tables + b * a.table_stride;
    count = (int)min((int64_t)min(len, a.max_len), a.table_stride << a.page_bits);
    run = a.own_run;
  }
  const int row_lo = rb * kPagedRows, rows = (t1 - t0) * a.group;
  if (row_lo >= rows) return;
  const int k_lo = split * run, k_hi = min(count, k_lo + run);

  // The lane's row: its query, and the keys that it sees.
  const int row = min(row_lo + l16, rows - 1);
  const int token = t0 + row / a.group;
  const int64_t at = (int64_t)token * a.heads + kvh * a.group + row % a.group;
  int see_lo = 0, see_hi = count;
  if (own) {
    const int place = first + token - t0;
    see_hi = min(count, place + 1);
    see_lo = a.window > 0 ? place - a.window + 1 : 0;
  } else if (a.window > 0) {
    int lo = 0, hi = a.seqs;              // the token's sequence: starts[lo] <= token < starts[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (a.starts[mid] <= token) lo = mid; else hi = mid;
    }
    const int place = a.prefix_len + a.lens[lo] - a.starts[lo + 1] + token;
    see_lo = place - a.window + 1;
  }
  float q[ND][EK];
#pragma unroll
  for (int d = 0; d < ND; d++)
#pragma unroll
    for (int j = 0; j < EK; j += 4) {
      const float4 v = *(const float4*)(a.q + at * HD + 4 * EK * d + EK * g4 + j);
      q[d][j] = v.x, q[d][j + 1] = v.y, q[d][j + 2] = v.z, q[d][j + 3] = v.w;
    }

  const float sl = a.scale * 1.44269504088896341f;   // scores in units of log2
  const int stride = a.kv_heads * HD * (int)sizeof(C);
  float m = -INFINITY, l = 0.0f;
  v4f o[NH][EV];
#pragma unroll
  for (int h = 0; h < NH; h++)
#pragma unroll
    for (int c = 0; c < EV; c++) o[h][c] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

  for (int kt = k_lo + 16 * wave; kt < k_hi; kt += 16 * kWaves) {
    const int page = table[kt >> a.page_bits];
    if ((uint32_t)page >= (uint64_t)a.pages) continue;   // no such page: its keys are not seen
    const int left = min(16, k_hi - kt);
    if (!__any(see_lo < kt + left && see_hi > kt)) continue;
    const int64_t base =
        ((((int64_t)page << a.page_bits) + (kt & ((1 << a.page_bits) - 1))) * a.kv_heads + kvh) * HD;
    const i32x4 krs = buffer_rsrc((const C*)a.keys + base, (uint32_t)(left * stride));
    const i32x4 vrs = buffer_rsrc((const C*)a.values + base, (uint32_t)(left * stride));
    float k[ND][EK], x[4][NH][EV];
#pragma unroll
    for (int d = 0; d < ND; d++)
      load_row<C, EK>(krs, l16 * stride + (4 * EK * d + EK * g4) * (int)sizeof(C), k[d]);
#pragma unroll
    for (int v = 0; v < 4; v++)
#pragma unroll
      for (int h = 0; h < NH; h++)
        load_row<C, EV>(vrs, (4 * g4 + v) * stride + (16 * EV * h + EV * l16) * (int)sizeof(C),
                        x[v][h]);
    v4f s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
      for (int j = 0; j < EK; j++)
        s = __builtin_amdgcn_mfma_f32_16x16x4f32(k[d][j], q[d][j], s, 0, 0, 0);
    float mt = -INFINITY;
    bool hidden = false;
    float weight[4];
#pragma unroll
    for (int v = 0; v < 4; v++) {
      const int key = kt + 4 * g4 + v;
      const bool see = key >= see_lo && key < see_hi && key < k_hi;
      hidden |= !see;
      weight[v] = see ? 1.0f : 0.0f;
      s[v] = see ? s[v] * sl : -INFINITY;
      mt = fmaxf(mt, s[v]);
    }
    const float m_new = fmaxf(m, quarter_max(mt)), ref = m_new == -INFINITY ? 0.0f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m - ref);
    float ps = 0.0f;
#pragma unroll
    for (int v = 0; v < 4; v++) {
      s[v] = __builtin_amdgcn_exp2f(s[v] - ref);
      ps += s[v];
      if (s[v] == 0.0f) weight[v] *= 16384.0f;
    }
    l = l * alpha + quarter_sum(ps);
    m = m_new;
    const bool edge = __any(hidden);
#pragma unroll
    for (int h = 0; h < NH; h++)
#pragma unroll
      for (int c = 0; c < EV; c++) {
        v4f d = {0.0f, 0.0f, 0.0f, 0.0f};
        bool finite = true;
        if (edge) {
#pragma unroll
          for (int v = 0; v < 4; v++) finite &= fabsf(x[v][h][c]) < INFINITY;
        }
        // An infinity or NaN that a row does not see counts for nothing in
        // it, but zero times it is NaN: zero in the products, and a code for
        // it (1: +inf, 128: -inf, 129: NaN) summed over the keys that are
        // seen, times 1 where p > 0 and 2^14 where p is zero (zero times an
        // infinity is NaN; 16 codes stay below 2^14).
        if (__builtin_expect(__any(!finite), 0)) {
          v4f codes = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int v = 0; v < 4; v++) {
            const float xv = x[v][h][c];
            const float code = xv == INFINITY ? 1.0f : xv == -INFINITY ? 128.0f
                               : xv != xv ? 129.0f : 0.0f;
            codes = __builtin_amdgcn_mfma_f32_16x16x4f32(code, weight[v], codes, 0, 0, 0);
            x[v][h][c] = code == 0.0f ? xv : 0.0f;
          }
#pragma unroll
          for (int v = 0; v < 4; v++) {
            const float minus = floorf(codes[v] * (1.0f / 128.0f));
            const float up = codes[v] - 128.0f * minus > 0.0f ? INFINITY : 0.0f;
            const float down = minus > 0.0f ? INFINITY : 0.0f;
            d[v] = codes[v] >= 16384.0f ? NAN : up - down;
          }
        }
#pragma unroll
        for (int v = 0; v < 4; v++)
          d = __builtin_amdgcn_mfma_f32_16x16x4f32(x[v][h][c], s[v], d, 0, 0, 0);
#pragma unroll
        for (int v = 0; v < 4; v++) o[h][c][v] = fmaf(o[h][c][v], alpha, d[v]);
      }
  }

  // The four waves' sums, added in wave order.
  __shared__ float ml[kWaves][2][16];
  __shared__ __align__(16) float sums[kWaves][16][HD + 4];
  if (g4 == 0) {
    ml[wave][0][l16] = m;
    ml[wave][1][l16] = l;
  }
#pragma unroll
  for (int h = 0; h < NH; h++)
#pragma unroll
    for (int v = 0; v < 4; v++)
#pragma unroll
      for (int c = 0; c < EV; c += 4)
        *(float4*)&sums[wave][l16][16 * EV * h + EV * (4 * g4 + v) + c] =
            make_float4(o[h][c][v], o[h][c + 1][v], o[h][c + 2][v], o[h][c + 3][v]);
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * HD / 4; i += kThreads) {
    const int r = i / (HD / 4), c = i % (HD / 4);
    if (row_lo + r >= rows) break;
    float top = -INFINITY, total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; w++) top = fmaxf(top, ml[w][0][r]);
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
      if (ml[w][1][r] == 0.0f) continue;
      const float f = partial_factor(ml[w][0][r], ml[w][1][r], top);
      const float4 y = *(const float4*)&sums[w][r][4 * c];
      total = fmaf(ml[w][1][r], f, total);
      acc = make_float4(fmaf(y.x, f, acc.x), fmaf(y.y, f, acc.y), fmaf(y.z, f, acc.z),
                        fmaf(y.w, f, acc.w));
    }
    const int tr = t0 + (row_lo + r) / a.group;
    const int64_t head = (int64_t)tr * a.heads + kvh * a.group + (row_lo + r) % a.group;
    if (a.splits == 1) {
      const float f = row_scale(total, a.gate, head);
      *(float4*)(a.out + head * HD + 4 * c) = make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f);
    } else {
      const int64_t p = head * a.splits + (own ? a.prefix_splits : 0) + split;
      *(float4*)(a.part + p * HD + 4 * c) = acc;
      if (c == 0) *(float2*)(a.stat + 2 * p) = make_float2(top, total);
    }
  }
}

// A row's partial results added in order, one wave a row: lane s holds the
// statistics of run s, lane i sums dims ND i .. (at most 64 runs).
template <int HD>
__global__ void __launch_bounds__(kThreads) paged_combine_kernel(PagedArgs a) {
  constexpr int ND = HD / 64;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t r = (int64_t)blockIdx.x * kWaves + wave;
  const int live = max(0, min(a.starts[a.seqs], a.tokens));
  if (r >= (int64_t)live * a.heads) return;
  float m = -INFINITY, l = 0.0f;
  if (lane < a.splits) {
    const float2 s = *(const float2*)(a.stat + 2 * (r * a.splits + lane));
    m = s.x;
    l = s.y;
  }
  const float top = wave_max_dpp(m);
  const float f = partial_factor(m, l, top);
  const float total = wave_sum_dpp(l * f);
  float acc[ND] = {};
  for (int s = 0; s < a.splits; s++) {
    if (lane_value(l, s) == 0.0f) continue;
    const float fs = lane_value(f, s);
#pragma unroll
    for (int i = 0; i < ND; i++)
      acc[i] = fmaf(a.part[(r * a.splits + s) * HD + ND * lane + i], fs, acc[i]);
  }
  const float g = row_scale(total, a.gate, r);
#pragma unroll
  for (int i = 0; i < ND; i++) a.out[r * HD + ND * lane + i] = acc[i] * g;
}

bool batch_ok(const dnx_paged_batch* b) {
  return b != nullptr && b->seqs > 0 && b->seqs <= (1 << 20) && b->tokens >= 0 &&
         b->tokens <= (1 << 22) && b->max_tokens > 0 && b->max_tokens <= (1 << 22) &&
         b->max_len >= 0 && b->max_len <= (1 << 30) && b->prefix_len >= 0 &&
         b->prefix_len <= (1 << 30) && b->table_stride >= 0 && b->table_stride <= (1 << 26) &&
         b->starts != nullptr && b->lens != nullptr &&
         (b->tables != nullptr || b->max_len == 0 || b->table_stride == 0) &&
         (b->prefix_pages != nullptr || b->prefix_len == 0);
}

PagedSplit split_of(const dnx_paged_cache* c, const dnx_paged_batch* b, int64_t heads) {
  return paged_split(b->seqs, b->tokens, std::min(b->max_tokens, std::max<int64_t>(1, b->tokens)),
                     heads / c->kv_heads, c->kv_heads, b->prefix_len, b->max_len);
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
  if (grid > 0x7fffffff) return DNX_EINVAL;
  auto k_ = cache->type == DNX_F32
                ? (cache->hd == 128 ? append_kernel<float, 128> : append_kernel<float, 64>)
                : (cache->hd == 128 ? append_kernel<uint16_t, 128> : append_kernel<uint16_t, 64>);
  hipLaunchKernelGGL(k_, dim3((unsigned)grid), dim3(kThreads), 0, (hipStream_t)stream, a);
  return hipGetLastError() == hipSuccess ? DNX_OK : DNX_ELAUNCH;
}

int64_t dnx_paged_attention_workspace_bytes(const dnx_paged_cache* cache,
                                            const dnx_paged_batch* batch, int64_t heads) {
  if (!cache_ok(cache) || !batch_ok(batch) || heads <= 0 || heads % cache->kv_heads != 0 ||
      heads > 65535 || batch->tokens * heads > (1 << 30)) {
    return -1;
  }
  const int64_t splits = split_of(cache, batch, heads).splits();
  return splits <= 1 ? 0 : batch->tokens * heads * splits * (cache->hd + 2) * 4;
}

int dnx_paged_attention(const dnx_paged_cache* cache, const dnx_paged_batch* batch,
                        const float* q, const float* gate, float* out, int64_t heads,
                        int64_t window, void* workspace, int64_t workspace_bytes,
                        dnx_stream_t stream) {
  const int64_t need = dnx_paged_attention_workspace_bytes(cache, batch, heads);
  if (need < 0 || window < 0 || window > 0x7fffffff) return DNX_EINVAL;
  if (batch->tokens == 0) return DNX_OK;
  if (q == nullptr || out == nullptr || (((uintptr_t)q | (uintptr_t)out) & 15) != 0 ||
      ((uintptr_t)gate & 3) != 0 || workspace_bytes < need ||
      (need > 0 && (workspace == nullptr || ((uintptr_t)workspace & 15) != 0))) {
    return DNX_EINVAL;
  }
  const PagedSplit s = split_of(cache, batch, heads);
  PagedArgs a{};
  a.keys = cache->keys;
  a.values = cache->values;
  a.pages = cache->pages;
  a.page_bits = __builtin_ctz((unsigned)cache->page);
  a.kv_heads = cache->kv_heads;
  a.heads = (int)heads;
  a.group = (int)(heads / cache->kv_heads);
  a.starts = batch->starts;
  a.lens = batch->lens;
  a.tables = batch->tables;
  a.prefix_pages = batch->prefix_pages;
  a.table_stride = batch->table_stride;
  a.prefix_len = (int)batch->prefix_len;
  a.seqs = (int)batch->seqs;
  a.tokens = (int)batch->tokens;
  a.max_len = (int)batch->max_len;
  a.q = q;
  a.gate = gate;
  a.out = out;
  a.splits = (int)s.splits();
  a.part = (float*)workspace;
  a.stat = a.part + batch->tokens * heads * a.splits * cache->hd;
  a.window = (int)window;
  a.prefix_splits = (int)s.prefix_splits;
  a.own_splits = (int)s.own_splits;
  a.prefix_run = (int)s.prefix_run;
  a.own_run = (int)s.own_run;
  a.prefix_rows = (int)s.prefix_rows;
  a.own_rows = (int)s.own_rows;
  a.prefix_items = s.prefix_rows * s.prefix_splits * cache->kv_heads;
  a.scale = (float)(1.0 / sqrt((double)cache->hd));
  const int64_t grid = a.prefix_items + s.own_rows * s.own_splits * cache->kv_heads * batch->seqs;
  if (grid > 0x7fffffff) return DNX_EINVAL;
  const hipStream_t st = (hipStream_t)stream;
  if (grid > 0) {
    auto k = cache->type == DNX_F32 ? (cache->hd == 128 ? paged_attention_kernel<float, 128>
                                                        : paged_attention_kernel<float, 64>)
                                    : (cache->hd == 128 ? paged_attention_kernel<uint16_t, 128>
                                                        : paged_attention_kernel<uint16_t, 64>);
    hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(kThreads), 0, st, a);
    if (hipGetLastError() != hipSuccess) return DNX_ELAUNCH;
  }
  if (a.splits != 1) {
    const int64_t blocks = (batch->tokens * heads + kWaves - 1) / kWaves;
    if (blocks > 0x7fffffff) return DNX_EINVAL;
    auto k = cache->hd == 128 ? paged_combine_kernel<128> : paged_combine_kernel<64>;
    hipLaunchKernelGGL(k, dim3((unsigned)blocks), dim3(kThreads), 0, st, a);
  }
  return hipGetLastError() == hipSuccess ? DNX_OK : DNX_ELAUNCH;
}

}  // extern "C"
