// The attention of a batch of sequences over a shared beginning and their own
// pages. No counterpart in the reference, which serves one sequence from one
// contiguous cache.
//
// For a row (a query head of a token) and the keys j it sees,
//   s_j = q.k_j / sqrt(hd), out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m).
// Keys are taken in runs; a run gives its maximum m, its sum l and its
// unnormalised o, and runs are added as o = sum o_r e^(m_r - M), l likewise.
// The prefix's keys meet the rows of all sequences at once: they are read for
// blocks of rows, not for sequences.

#include <algorithm>

#include "bf16_pieces.h"
#include "common.h"
#include "paged.h"
#include "paged_attention.h"

#include <math.h>

using namespace dnx;

namespace {

// 16 keys of an item from kt on (a page holds whole sixteens) as resources
// over one head's rows of the cache: what lies behind the last key, or in a
// page outside the cache, reads as zeros without touching memory.
struct Block {
  i32x4 keys, values;
  int end;      // its keys lie before this key (none: not after the first)
};
// Blocks as seen from `behind` keys before them: the offset of key i of the
// block is that of row behind + i.
template <typename C, int HD, bool kJoined>
DNX_DEV Block block_at(const PagedArgs& a, const Item& w, int kt, int page, int keys = 16,
                       int behind = 0) {
  Block b;
  const bool own = !kJoined || kt >= w.joined;
  const int left = min(keys, (own ? w.k_hi : a.prefix_len) - kt);
  const bool there = left > 0 && (uint32_t)page < (uint32_t)a.pages;
  b.end = there ? kt + left : kt;
  const uint32_t range = there ? (uint32_t)((left + behind) * a.row_bytes) : 0u;
  // Not used where the range is empty.
  const uint32_t in_page = (uint32_t)((kJoined && own ? kt - w.joined : kt) & ((1 << a.page_bits) - 1));
  const uint64_t at = (uint64_t)(uint32_t)page * ((uint32_t)a.row_bytes << a.page_bits) +
                      (uint64_t)(in_page * (uint32_t)a.row_bytes) -
                      (uint64_t)((uint32_t)behind * (uint32_t)a.row_bytes);
  const uint32_t head = (uint32_t)(w.kvh * HD * (int)sizeof(C));
  b.keys = buffer_rsrc((const uint8_t*)a.keys + head + at, range);
  b.values = buffer_rsrc((const uint8_t*)a.values + head + at, range);
  return b;
}

// ---- 16 rows, 16 or 32 keys at a time in one wave, straight from memory.
//
// Lane l (quarter g = l / 16) holds key l % 16 and row l % 16 at the dims EK
// (4 d + g) .., d < ND: 16 bytes of the cache each; and the values of keys 4 g
// + 0..3 at dims EV (l % 16 + 16 h) .., h < NH.
template <typename C, int HD>
struct Lanes {
  static constexpr int EK = 16 / sizeof(C), ND = HD / (4 * EK);
  static constexpr int EV = EK < HD / 16 ? EK : HD / 16, NH = HD / (16 * EV);
};

template <typename C, int HD>
struct Raw {
  using L = Lanes<C, HD>;
  uint4 k[L::ND], v[4][L::NH];
};

template <typename C, int HD>
DNX_DEV void load_keys(const Block& b, int stride, int l16, int g4, Raw<C, HD>& x) {
#pragma unroll
  for (int d = 0; d < Lanes<C, HD>::ND; d++)
    x.k[d] = buffer_load16(b.keys, l16 * stride + (4 * d + g4) * 16);
}
template <typename C, int HD>
DNX_DEV void load_values(const Block& b, int stride, int l16, int g4, Raw<C, HD>& x) {
  using L = Lanes<C, HD>;
  constexpr int S = sizeof(C);
#pragma unroll
  for (int v = 0; v < 4; v++)
#pragma unroll
    for (int h = 0; h < L::NH; h++) {
      const int at = (4 * g4 + v) * stride + L::EV * S * (l16 + 16 * h);
      if constexpr (L::EV * S == 16) {
        x.v[v][h] = buffer_load16(b.values, at);
      } else {
        const i32x2 y = dnx_raw_buffer_load_v2i32(b.values, at, 0, 0);
        x.v[v][h] = make_uint4((uint32_t)y.x, (uint32_t)y.y, 0, 0);
      }
    }
}

DNX_DEV uint32_t word(const uint4& u, int i) { return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w; }

// Element i of 16 bytes of the cache.
template <typename C>
DNX_DEV float element(const uint4& u, int i) {
  if constexpr (sizeof(C) == 4) {
    return __uint_as_float(word(u, i));
  } else {
    const uint32_t w = word(u, i / 2);
    return __uint_as_float(i % 2 == 0 ? w << 16 : w & 0xffff0000u);
  }
}

// The running sums of a wave's 16 rows: o[h][c][v] of row l % 16 at dim EV (4
// g + v + 16 h) + c.
template <typename C, int HD>
struct Sums {
  using L = Lanes<C, HD>;
  float m, l;
  v4f o[L::NH][L::EV];
  __device__ __forceinline__ void clear() {
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int h = 0; h < L::NH; h++)
#pragma unroll
      for (int c = 0; c < L::EV; c++) o[h][c] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  }
};

// 16 keys from kt on, on the float32 matrix cores: exact products, float32
// sums, whatever the operands are.
// * S^T = K Q^T: the lane ends with the scores of row l % 16 for keys 4 g ..;
// * O^T += V^T P^T: step v takes the keys 4 g + v, whose weights the lane has.
// An infinity or NaN among the values of keys that a row does not see counts
// for nothing in it, but zero times it is NaN: zero in the products, and a
// code for it (1: +inf, 128: -inf, 129: NaN) summed over the keys that are
// seen, times 1 where p > 0 and 2^14 where p is zero (zero times an infinity
// is NaN; 16 codes stay below 2^14).
//
// `between` runs when the keys' registers are free.
template <typename C, int HD, typename F>
DNX_DEV void exact_step(const Raw<C, HD>& x, const float (*q)[Lanes<C, HD>::EK], int kt, int end,
                        Seen see, float sl, int g4, Sums<C, HD>& a, F between) {
  using L = Lanes<C, HD>;
  v4f s = {0.0f, 0.0f, 0.0f, 0.0f}, s2 = s;     // two chains
#pragma unroll
  for (int d = 0; d < L::ND; d++)
#pragma unroll
    for (int j = 0; j < L::EK; j += 2) {
      s = __builtin_amdgcn_mfma_f32_16x16x4f32(element<C>(x.k[d], j), q[d][j], s, 0, 0, 0);
      s2 = __builtin_amdgcn_mfma_f32_16x16x4f32(element<C>(x.k[d], j + 1), q[d][j + 1], s2, 0, 0, 0);
    }
  between();
#pragma unroll
  for (int v = 0; v < 4; v++) s[v] += s2[v];
  float mt = -INFINITY;
  bool hidden = false;
  float weight[4];
#pragma unroll
  for (int v = 0; v < 4; v++) {
    const int key = kt + 4 * g4 + v;
    const bool sees = key >= see.lo && key < see.hi && key < end;
    hidden |= !sees;
    weight[v] = sees ? 1.0f : 0.0f;
    s[v] = sees ? s[v] * sl : -INFINITY;
    mt = fmaxf(mt, s[v]);
  }
  const float m_new = fmaxf(a.m, rows4_max(mt)), ref = m_new == -INFINITY ? 0.0f : m_new;
  const float alpha = __builtin_amdgcn_exp2f(a.m - ref);
  float ps = 0.0f;
#pragma unroll
  for (int v = 0; v < 4; v++) {
    s[v] = __builtin_amdgcn_exp2f(s[v] - ref);
    ps += s[v];
    if (s[v] == 0.0f) weight[v] *= 16384.0f;
  }
  a.l = a.l * alpha + rows4_sum(ps);
  a.m = m_new;
  bool finite = true;
  if (__any(hidden)) {
#pragma unroll
    for (int h = 0; h < L::NH; h++)
#pragma unroll
      for (int c = 0; c < L::EV; c++)
#pragma unroll
        for (int v = 0; v < 4; v++) finite &= fabsf(element<C>(x.v[v][h], c)) < INFINITY;
  }
  const bool codes_wanted = __any(!finite);
#pragma unroll
  for (int h = 0; h < L::NH; h++)
#pragma unroll
    for (int c = 0; c < L::EV; c++) {
      v4f d = {0.0f, 0.0f, 0.0f, 0.0f};
      float y[4];
#pragma unroll
      for (int v = 0; v < 4; v++) y[v] = element<C>(x.v[v][h], c);
      if (__builtin_expect(codes_wanted, 0)) {
        v4f codes = d;
#pragma unroll
        for (int v = 0; v < 4; v++) {
          const float code = y[v] == INFINITY ? 1.0f : y[v] == -INFINITY ? 128.0f
                             : y[v] != y[v] ? 129.0f : 0.0f;
          codes = __builtin_amdgcn_mfma_f32_16x16x4f32(code, weight[v], codes, 0, 0, 0);
          if (code != 0.0f) y[v] = 0.0f;
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
        d = __builtin_amdgcn_mfma_f32_16x16x4f32(y[v], s[v], d, 0, 0, 0);
#pragma unroll
      for (int v = 0; v < 4; v++) a.o[h][c][v] = fmaf(a.o[h][c][v], alpha, d[v]);
    }
}

// The row's query at the lane's dims.
template <typename C, int HD>
DNX_DEV void load_query(const float* q, int g4, float (*x)[Lanes<C, HD>::EK]) {
  using L = Lanes<C, HD>;
#pragma unroll
  for (int d = 0; d < L::ND; d++)
#pragma unroll
    for (int j = 0; j < L::EK; j += 4) {
      const float4 v = *(const float4*)(q + L::EK * (4 * d + g4) + j);
      x[d][j] = v.x, x[d][j + 1] = v.y, x[d][j + 2] = v.z, x[d][j + 3] = v.w;
    }
}

// Keys first .. first + width - 1, then `stride` further, to the item's end,
// in exact steps.
template <typename C, int HD, bool kJoined>
DNX_DEV void exact_walk(const PagedArgs& a, const Item& w, const float* qp, Seen see, float sl,
                        int first, int width, int stride, int l16, int g4, Sums<C, HD>& sums) {
  float q[Lanes<C, HD>::ND][Lanes<C, HD>::EK];
  load_query<C, HD>(qp, g4, q);
  sums.clear();
#pragma unroll 1
  for (int k0 = first; k0 < w.k_hi; k0 += stride)
#pragma unroll 1
    for (int kt = k0; kt < min(w.k_hi, k0 + width); kt += 16) {
      const Block b = block_at<C, HD, kJoined>(a, w, kt, page_at<kJoined>(a, w, kt));
      if (b.end == kt || !__any(see.lo < kt + 16 && see.hi > kt)) continue;
      Raw<C, HD> x;
      load_keys<C, HD>(b, a.row_bytes, l16, g4, x);
      load_values<C, HD>(b, a.row_bytes, l16, g4, x);
      exact_step<C, HD>(x, q, kt, b.end, see, sl, g4, sums, [] {});
    }
}

// ---- 16 rows a workgroup, each wave other keys (decode: few rows read many
// keys, and what it costs is to read them).
//
// float32 caches take 16 keys a step in exact steps. bf16 caches take 32 on
// the bf16 matrix cores: a key's or value's 16 bits are exact there, the query
// and the weights are sums of three bf16 pieces, of which every product with
// it is formed. The sums start from zero in each step. The values' fragments
// (eight keys of one dim a lane) come from rows of eight dims by one byte
// permute for two values. An infinity or NaN has no pieces: a wave that ends
// with one in its sums walks its keys again in exact steps.
//
// bf16, 64 sequences of 1088 keys, 32 / 8 heads, hd 128: 54 us, 5.3 TB/s (a
// large copy reaches 4.6, this library's best reader 6.1): bound by the bytes.
// Of unequal lengths (128 to 2048) 69 us, 4.1 TB/s: the longest ends last.
// Dealing all sequences' keys to the workgroups in equal parts gave 69 too: a
// prologue for each part and a second launch took what it saved.
template <typename C, int HD, bool kJoined>
DNX_DEV void narrow(const PagedArgs& a, const Item& w, uint8_t* lds) {
  using L = Lanes<C, HD>;
  constexpr bool kF32 = sizeof(C) == 4;
  constexpr int U = kF32 ? 1 : 2, KS = 16 * U;     // keys of a wave's step
  const int lane = threadIdx.x & 63, l16 = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = min(w.row0 + l16, w.rows - 1);
  const Seen see = row_sees(a, w, row);
  const float* qp = a.q + row_at(a, w, row) * HD;
  const float sl = a.scale * 1.44269504088896341f;   // scores in units of log2
  Sums<C, HD> sums;
  sums.clear();

  // The next step's keys are requested when this step's scores are formed, its
  // values when this step's are added: one step's registers, and requests in
  // flight during all of the math; its pages one step before that. Steps that
  // no row sees are passed over.
  constexpr int kStride = KS * kWaves;
  const int first = w.k_lo + KS * wave;
  Raw<C, HD> x[U];
  Block block[U];
  int page[U];
  auto pages = [&](int at) {
#pragma unroll
    for (int u = 0; u < U; u++) page[u] = page_at<kJoined>(a, w, at + 16 * u);
  };
  auto blocks = [&](int at) {
#pragma unroll
    for (int u = 0; u < U; u++) block[u] = block_at<C, HD, kJoined>(a, w, at + 16 * u, page[u]);
  };
  auto request_keys = [&] {
#pragma unroll
    for (int u = 0; u < U; u++) load_keys<C, HD>(block[u], a.row_bytes, l16, g4, x[u]);
  };
  auto request_values = [&] {
#pragma unroll
    for (int u = 0; u < U; u++) load_values<C, HD>(block[u], a.row_bytes, l16, g4, x[u]);
  };
  auto next = [&](int at) {
    while (at < w.k_hi && !__any(see.lo < at + KS && see.hi > at)) at += kStride;
    return at;
  };
  float q[L::ND][L::EK];
  int kt = next(first), after = kt;
  if (kt < w.k_hi) {
    if (kt == first) {
#pragma unroll
      for (int u = 0; u < U; u++) page[u] = w.page[u];
    } else {
      pages(kt);
    }
    load_query<C, HD>(qp, g4, q);
    blocks(kt);
    request_keys();
    request_values();
    after = next(kt + kStride);
    pages(after);
  }
  if constexpr (kF32) {
    while (kt < w.k_hi) {
      const int end = block[0].end;
      const int then = next(after + kStride);
      blocks(after);
      pages(then);
      exact_step<C, HD>(x[0], q, kt, end, see, sl, g4, sums, request_keys);
      request_values();
      kt = after;
      after = then;
    }
  } else {
    uint4 qf[L::ND][3];
#pragma unroll
    for (int d = 0; d < L::ND; d++) {
      if (kt < w.k_hi) split_pieces(q[d], qf[d]);
    }
    while (kt < w.k_hi) {
      int end[U];
#pragma unroll
      for (int u = 0; u < U; u++) end[u] = block[u].end;
      const int then = next(after + kStride);
      blocks(after);
      pages(then);
      auto mfma = [](const uint4& p, const uint4& r, v4f acc) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, p),
                                                       __builtin_bit_cast(bf8, r), acc, 0, 0, 0);
      };
      v4f s[U], low[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        s[u] = low[u] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int d = 0; d < L::ND; d++) {
          s[u] = mfma(x[u].k[d], qf[d][0], s[u]);
          low[u] = mfma(x[u].k[d], qf[d][2], low[u]);
          low[u] = mfma(x[u].k[d], qf[d][1], low[u]);
        }
      }
      request_keys();
      float mt = -INFINITY, p[8];
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int v = 0; v < 4; v++) {
          const int key = kt + 16 * u + 4 * g4 + v;
          const bool sees = key >= see.lo && key < see.hi && key < end[u];
          p[4 * u + v] = sees ? (s[u][v] + low[u][v]) * sl : -INFINITY;
          mt = fmaxf(mt, p[4 * u + v]);
        }
      const float m_new = fmaxf(sums.m, rows4_max(mt)), ref = m_new == -INFINITY ? 0.0f : m_new;
      const float alpha = __builtin_amdgcn_exp2f(sums.m - ref);
      float ps = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        p[i] = __builtin_amdgcn_exp2f(p[i] - ref);
        ps += p[i];
      }
      sums.l = sums.l * alpha + rows4_sum(ps);
      sums.m = m_new;
      uint4 pf[3];
      split_pieces(p, pf);
#pragma unroll
      for (int c = 0; c < L::EV; c++) {
        // Dim c of the lane's eight keys: the low or high half of word c / 2.
        auto two = [&](int u, int v) {
          return __builtin_amdgcn_perm(word(x[u].v[v + 1][0], c / 2), word(x[u].v[v][0], c / 2),
                                       c % 2 == 0 ? 0x05040100u : 0x07060302u);
        };
        const uint4 vf = make_uint4(two(0, 0), two(0, 2), two(U - 1, 0), two(U - 1, 2));
        // The small products before the large one: they round at their size.
        v4f d = {0.0f, 0.0f, 0.0f, 0.0f};
        d = mfma(vf, pf[2], d);
        d = mfma(vf, pf[1], d);
        d = mfma(vf, pf[0], d);
#pragma unroll
        for (int v = 0; v < 4; v++) sums.o[0][c][v] = fmaf(sums.o[0][c][v], alpha, d[v]);
      }
      request_values();
      kt = after;
      after = then;
    }
    float check = sums.l - sums.l;
#pragma unroll
    for (int c = 0; c < L::EV; c++)
#pragma unroll
      for (int v = 0; v < 4; v++) check += sums.o[0][c][v] - sums.o[0][c][v];
    if (__builtin_expect(__any(check != check), 0))
      exact_walk<C, HD, kJoined>(a, w, qp, see, sl, first, KS, kStride, l16, g4, sums);
  }

  float* all = (float*)lds;
  float* ml = wave_stats<HD>(lds, wave);
  if (g4 == 0) {
    ml[l16] = sums.m;
    ml[16 + l16] = sums.l;
  }
#pragma unroll
  for (int h = 0; h < L::NH; h++)
#pragma unroll
    for (int v = 0; v < 4; v++)
#pragma unroll
      for (int c = 0; c < L::EV; c += 4)
        *(float4*)&all[(wave * 16 + l16) * kSumRow<HD> + L::EV * (4 * g4 + v + 16 * h) + c] =
            make_float4(sums.o[h][c][v], sums.o[h][c + 1][v], sums.o[h][c + 2][v],
                        sums.o[h][c + 3][v]);
  merge_waves<HD, 16>(a, w, lds);
}

// ---- One token's R <= 2 or 4 rows on a float32 cache, each wave other keys
// (decode steps). The float32
// matrix cores would form 16 rows for them; vector instructions form R.
//
// Lanes as above: a lane sums its dims of key l % 16 for each row, the four
// lanes of the key are added, and the weights of keys 4 g .. 4 g + 3 are
// fetched from their lanes. A row's sums are relative to one maximum, which
// follows where a score has passed it by kSlack: weights up to 2^kSlack are as
// exact as those up to one. Values that the token does not see are zeros.
//
// 64 sequences of 128 to 1500 keys, 16 / 4 heads, hd 128: 52 us, 4.1 TB/s
// (on the matrix cores 63), hd 64 33 (44); 3 sequences of up to 200, hd 128,
// two rows 7.1 (9.5). The same scheme on bf16 caches, whose elements it has to
// unpack, took 41 us for 29 on the matrix cores.
template <int HD, int R, bool kJoined>
DNX_DEV void few(const PagedArgs& a, const Item& w, uint8_t* lds) {
  using L = Lanes<float, HD>;
  constexpr int KS = 16, kStride = KS * kWaves;
  const int lane = threadIdx.x & 63, l16 = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const float sl = a.scale * 1.44269504088896341f;   // scores in units of log2
  const Seen see = row_sees(a, w, 0);
  const int lo = __builtin_amdgcn_readfirstlane(see.lo);
  const int hi = __builtin_amdgcn_readfirstlane(see.hi);
  float m[R], l[R], o[R][L::NH][4];
#pragma unroll
  for (int r = 0; r < R; r++) {
    m[r] = -INFINITY;
    l[r] = 0.0f;
#pragma unroll
    for (int h = 0; h < L::NH; h++)
#pragma unroll
      for (int c = 0; c < 4; c++) o[r][h][c] = 0.0f;
  }

  // The queries in LDS: four rows of 32 dims a lane are more registers than
  // there are.
  float* q = (float*)(lds + kMergeBytes<HD>);     // [R][HD]
  if (threadIdx.x < R * HD / 4) {
    const int r = threadIdx.x / (HD / 4), c = threadIdx.x % (HD / 4);
    *(float4*)&q[4 * threadIdx.x] =
        *(const float4*)(a.q + row_at(a, w, min(w.row0 + r, w.rows - 1)) * HD + 4 * c);
  }

  // Requests as above: a step's keys and values while the step before is added.
  Raw<float, HD> x;
  Block block;
  int page;
  auto next = [&](int at) {
    while (at < w.k_hi && (lo >= at + KS || hi <= at)) at += kStride;
    return at;
  };
  const int first = w.k_lo + KS * wave;
  int kt = next(first), after = kt;
  if (kt < w.k_hi) {
    page = kt == first ? w.page[0] : page_at<kJoined>(a, w, kt);
    block = block_at<float, HD, kJoined>(a, w, kt, page);
    load_keys<float, HD>(block, a.row_bytes, l16, g4, x);
    load_values<float, HD>(block, a.row_bytes, l16, g4, x);
    after = next(kt + kStride);
    page = page_at<kJoined>(a, w, after);
  }
  __syncthreads();
  int q_at = 4 * g4;
  while (kt < w.k_hi) {
    const int end = block.end;
    const int then = next(after + kStride);
    block = block_at<float, HD, kJoined>(a, w, after, page);
    page = page_at<kJoined>(a, w, then);
    float s[R];
    float4 y[2][R];
    auto read = [&](int d) {
#pragma unroll
      for (int r = 0; r < R; r++) y[d & 1][r] = *(const float4*)&q[q_at + r * HD + 16 * d];
    };
    read(0);
#pragma unroll
    for (int d = 0; d < L::ND; d++) {
      if (d + 1 < L::ND) read(d + 1);
      __builtin_amdgcn_sched_barrier(0);   // or all are read at once
#pragma unroll
      for (int r = 0; r < R; r++) {
        const float4 z = y[d & 1][r];
        s[r] = d == 0 ? element<float>(x.k[0], 0) * z.x : fmaf(element<float>(x.k[d], 0), z.x, s[r]);
        s[r] = fmaf(element<float>(x.k[d], 1), z.y, s[r]);
        s[r] = fmaf(element<float>(x.k[d], 2), z.z, s[r]);
        s[r] = fmaf(element<float>(x.k[d], 3), z.w, s[r]);
      }
    }
    asm("" : "+v"(q_at));                  // nor kept for the next step
    load_keys<float, HD>(block, a.row_bytes, l16, g4, x);
    auto sees = [&](int key) { return key >= lo && key < min(hi, end); };
    const bool seen = sees(kt + l16);
    bool grows = false;
#pragma unroll
    for (int r = 0; r < R; r++) {
      s[r] = rows4_sum(s[r]) * sl;
      s[r] = seen ? s[r] : -INFINITY;
      grows |= s[r] > m[r] + kSlack;
    }
    if (__any(grows)) {
#pragma unroll
      for (int r = 0; r < R; r++) {
        float top = s[r];
        top = fmaxf(top, dppf<kQuadXor1>(top));
        top = fmaxf(top, dppf<kQuadXor2>(top));
        top = fmaxf(top, dppf<kHalfRowMirror>(top));
        top = fmaxf(top, dppf<kRowMirror>(top));
        top = fmaxf(top, m[r]);
        const float alpha = top == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[r] - top);
        m[r] = top;
        l[r] *= alpha;
#pragma unroll
        for (int h = 0; h < L::NH; h++)
#pragma unroll
          for (int c = 0; c < 4; c++) o[r][h][c] *= alpha;
      }
    }
    float p[R][4];
#pragma unroll
    for (int r = 0; r < R; r++) {
      s[r] = __builtin_amdgcn_exp2f(s[r] - (m[r] == -INFINITY ? 0.0f : m[r]));
      l[r] += s[r];
#pragma unroll
      for (int v = 0; v < 4; v++) p[r][v] = __shfl(s[r], 4 * g4 + v);
    }
    if (lo > kt || min(hi, end) < kt + KS) {
#pragma unroll
      for (int v = 0; v < 4; v++)
#pragma unroll
        for (int h = 0; h < L::NH; h++)
          if (!sees(kt + 4 * g4 + v)) x.v[v][h] = make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int h = 0; h < L::NH; h++)
#pragma unroll
      for (int c = 0; c < 4; c++)
#pragma unroll
        for (int v = 0; v < 4; v++)
#pragma unroll
          for (int r = 0; r < R; r++)
            o[r][h][c] = fmaf(element<float>(x.v[v][h], c), p[r][v], o[r][h][c]);
    load_values<float, HD>(block, a.row_bytes, l16, g4, x);
    kt = after;
    after = then;
  }

  float* all = (float*)lds;
  float* ml = wave_stats<HD>(lds, wave);
#pragma unroll
  for (int r = 0; r < R; r++) {
    l[r] += dppf<kQuadXor1>(l[r]);
    l[r] += dppf<kQuadXor2>(l[r]);
    l[r] += dppf<kHalfRowMirror>(l[r]);
    l[r] += dppf<kRowMirror>(l[r]);
    if (lane == 0) {
      ml[r] = m[r];
      ml[16 + r] = l[r];
    }
#pragma unroll
    for (int h = 0; h < L::NH; h++) {
#pragma unroll
      for (int c = 0; c < 4; c++) o[r][h][c] = rows4_sum(o[r][h][c]);
      if (g4 == 0)
        *(float4*)&all[(wave * 16 + r) * kSumRow<HD> + 4 * (l16 + 16 * h)] =
            make_float4(o[r][h][0], o[r][h][1], o[r][h][2], o[r][h][3]);
    }
  }
  merge_waves<HD, R>(a, w, lds);
}

// ---- 64 rows a workgroup, 16 a wave, which share tiles of KT keys in LDS (a
// batch's rows over the prefix, a prompt's rows over its own keys).
//
// The scheme of the bf16 steps above on tiles in LDS: keys as [8 dims][key],
// values as [8 keys][dim] in the order in which a lane's weights stand (k slot
// j of quarter g: key 4 g + j, or 16 + 4 g + j - 4), 16 bytes each. float32
// caches are split into three pieces on the way (PC = 3), each product formed
// from the six largest products of pieces; of the three left out two reach 2^-25
// of it, all together 2^-24 (a float's half step). The pieces of an operand below
// 2^-110 are not all of it. The next tile is in registers meanwhile.
//
// A prefix of 8192 keys, bf16, for 64 tokens of 32 / 8 heads, hd 128: 40 us
// for 16 tiles of 64 keys a wave, 0.6 PFLOP/s of bf16 products, three for each
// of the formula's. Waits bound it, not one unit: a tile takes a lone wave of a
// SIMD 1.8 us, and two waves 1.2 each.
template <typename C, int HD>
struct WideTile {
  static constexpr int PC = sizeof(C) == 4 ? 3 : 1;
  static constexpr int KT = sizeof(C) == 4 && HD == 128 ? 32 : 64;
  static constexpr int KS = KT * 16 + 16;         // K: 8 dims of all keys, + pad
  static constexpr int VS = HD * 16;              // V: 8 keys of all dims
  static constexpr int kK = PC * (HD / 8) * KS, kV = PC * (KT / 8) * VS;
  static constexpr int KU = KT * HD / 8 / kThreads;    // K: 8 dims of a key, per thread
  static constexpr int VD = KT / 8 * HD / kThreads;    // V: dims of 8 keys, per thread
};

template <typename C, int HD>
DNX_DEV void wide(const PagedArgs& a, const Item& w, uint8_t* lds) {
  using T = WideTile<C, HD>;
  constexpr int KT = T::KT, NB = KT / 16, NE = HD / 16, ND = HD / 32, PC = T::PC;
  constexpr int S = sizeof(C);
  uint8_t* Kp = lds;
  uint8_t* Vp = lds + T::kK;
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wave_row = w.row0 + 16 * wave;
  const bool live = wave_row < w.rows;
  const int row = min(wave_row + l16, w.rows - 1);
  const Seen see = row_sees(a, w, row);
  const float* qp = a.q + row_at(a, w, row) * HD;
  const float sl = a.scale * 1.44269504088896341f;
  const int stride = a.row_bytes;

  // The keys that any row of the workgroup sees.
  int* span = (int*)(lds + T::kK + T::kV);
  int lo = see.lo, hi = see.hi;
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    lo = min(lo, __shfl_xor(lo, o));
    hi = max(hi, __shfl_xor(hi, o));
  }
  if (lane == 0) {
    span[2 * wave] = lo;
    span[2 * wave + 1] = hi;
  }
  const int wave_lo = __builtin_amdgcn_readfirstlane(lo);
  const int wave_hi = __builtin_amdgcn_readfirstlane(hi);
  __syncthreads();
  int all_lo = span[0], all_hi = span[1];
#pragma unroll
  for (int k = 1; k < kWaves; k++) {
    all_lo = min(all_lo, span[2 * k]);
    all_hi = max(all_hi, span[2 * k + 1]);
  }
  const int from = __builtin_amdgcn_readfirstlane(
      w.k_lo + (max(all_lo, w.k_lo) - w.k_lo) / KT * KT);
  const int to = __builtin_amdgcn_readfirstlane(min(w.k_hi, all_hi));

  // Staging. A wave's part of a load lies in one block of 16 keys.
  constexpr int KC = HD / 8, VC = HD / T::VD;     // threads a key, threads a key group
  const int vg = tid / VC, vd = tid % VC;         // V: dims VD vd.., key group vg
  constexpr int KW = S == 4 ? 2 : 1;              // 16-byte words of 8 dims
  uint4 kr[T::KU][KW];
  uint32_t vr[8][T::VD * S / 4];
  uint32_t there = 0, there_next = 0;             // which blocks of 16 keys there are
  int page[NB];                                   // of the tile to load next
  auto pages = [&](int kt) {
#pragma unroll
    for (int i = 0; i < NB; i++) page[i] = page_at<false>(a, w, kt + 16 * i);
  };

  // The offsets are those within the tile: one resource serves it where a page
  // holds it whole, else one for each of its blocks.
  auto load_key = [&](int j, const Block& b) {
    const int unit = j * kThreads + tid, key = unit / KC, c = unit % KC;
#pragma unroll
    for (int i = 0; i < KW; i++) kr[j][i] = buffer_load16(b.keys, key * stride + c * 8 * S + 16 * i);
  };
  auto load_value = [&](int j, const Block& b) {
    const int key = 32 * (vg >> 2) + 16 * (j >> 2) + 4 * (vg & 3) + (j & 3);
    const int at = key * stride + vd * T::VD * S;
    if constexpr (T::VD * S == 8) {
      const i32x2 x = dnx_raw_buffer_load_v2i32(b.values, at, 0, 0);
      vr[j][0] = (uint32_t)x.x, vr[j][1] = (uint32_t)x.y;
    } else {
      vr[j][0] = (uint32_t)dnx_raw_buffer_load_i32(b.values, at, 0, 0);
    }
  };
  auto load_tile = [&](int kt) {
    if ((1 << a.page_bits) >= KT) {
      const Block b = block_at<C, HD, false>(a, w, kt, page[0], KT);
      there_next = b.end > kt ? (1u << NB) - 1 : 0u;
#pragma unroll
      for (int j = 0; j < T::KU; j++) load_key(j, b);
#pragma unroll
      for (int j = 0; j < 8; j++) load_value(j, b);
    } else {
      const bool second = wave >= kWaves / 2;
      Block b[NB];
      there_next = 0;
#pragma unroll
      for (int i = 0; i < NB; i++) {
        b[i] = block_at<C, HD, false>(a, w, kt + 16 * i, page[i], 16, 16 * i);
        there_next |= b[i].end > kt + 16 * i ? 1u << i : 0u;
      }
      // Of the second half of the waves the blocks of key groups 4 .. 7, and
      // where 32 keys are loaded at once those of the latter 16.
      auto of = [&](int i, int d) { return second ? b[i + d] : b[i]; };
#pragma unroll
      for (int j = 0; j < T::KU; j++) load_key(j, KC == 16 ? b[j] : of(2 * j, 1));
      constexpr int kHalf = NB == 4 ? 2 : 0;
#pragma unroll
      for (int j = 0; j < 8; j++) load_value(j, of(j >> 2, kHalf));
    }
  };
  // A dim's place in the rows of V^T is turned by bits 3 and 4 of the dim, as
  // rows a few dims apart would meet in the same banks.
  auto v_slot = [](int dim) { return dim ^ ((dim >> 3) & 3); };
  auto store_tile = [&] {
#pragma unroll
    for (int j = 0; j < T::KU; j++) {
      const int unit = j * kThreads + tid, key = unit / KC, c = unit % KC;
      if constexpr (PC == 1) {
        *(uint4*)(Kp + c * T::KS + key * 16) = kr[j][0];
      } else {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = __uint_as_float(word(kr[j][i >> 2], i & 3));
        uint4 p[3];
        split_pieces(x, p);
#pragma unroll
        for (int i = 0; i < 3; i++) *(uint4*)(Kp + (i * KC + c) * T::KS + key * 16) = p[i];
      }
    }
#pragma unroll
    for (int d = 0; d < T::VD; d++) {
      uint8_t* at = Vp + vg * T::VS + v_slot(T::VD * vd + d) * 16;
      if constexpr (PC == 1) {
        auto two = [&](int j) {
          return __builtin_amdgcn_perm(vr[j + 1][d / 2], vr[j][d / 2],
                                       d % 2 == 0 ? 0x05040100u : 0x07060302u);
        };
        *(uint4*)at = make_uint4(two(0), two(2), two(4), two(6));
      } else {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = __uint_as_float(vr[j][d]);
        uint4 p[3];
        split_pieces(x, p);
#pragma unroll
        for (int i = 0; i < 3; i++) *(uint4*)(at + i * (KT / 8) * T::VS) = p[i];
      }
    }
  };
  auto mfma = [](const uint4& p, const uint4& r, v4f acc) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, p),
                                                   __builtin_bit_cast(bf8, r), acc, 0, 0, 0);
  };
  // The products of pieces but that of the first ones, the smallest first.
  constexpr int kSmall = PC == 3 ? 5 : 2;
  auto small = [&](int i, const uint4* x, const uint4* y, v4f acc) {
    if constexpr (PC == 3) {
      constexpr int kx[] = {2, 1, 0, 1, 0}, ky[] = {0, 1, 2, 0, 1};
      return mfma(x[kx[i]], y[ky[i]], acc);
    } else {
      return mfma(x[0], y[2 - i], acc);
    }
  };
  constexpr int EG = PC == 3 && KT == 64 ? 1 : 2;   // 16-dim blocks of a step of the sums

  uint4 qf[ND][3];
  {
    float4 qv[2 * ND];
#pragma unroll
    for (int d = 0; d < ND; d++) {
      qv[2 * d] = *(const float4*)(qp + 32 * d + 8 * g4);
      qv[2 * d + 1] = *(const float4*)(qp + 32 * d + 8 * g4 + 4);
    }
    if (from < to) {
      pages(from);
      load_tile(from);
      pages(from + KT);
    }
#pragma unroll
    for (int d = 0; d < ND; d++) {
      const float4 x = qv[2 * d], y = qv[2 * d + 1];
      const float f[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
      split_pieces(f, qf[d]);
    }
  }
  float m = -INFINITY, l = 0.0f;
  v4f o[NE];
#pragma unroll
  for (int e = 0; e < NE; e++) o[e] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  for (int kt = from; kt < to; kt += KT) {
    __syncthreads();   // every wave is done with the tile before
    store_tile();
    there = there_next;
    __syncthreads();
    if (kt + KT < to) {        // in flight during this tile's math
      load_tile(kt + KT);
      pages(kt + 2 * KT);
    }
    if (!live || wave_lo >= kt + KT || wave_hi <= kt) continue;
    // Scores. The fragments of a step are read while the step before is
    // multiplied; nothing is moved across, or each read is waited for at once.
    v4f s[NB];
#pragma unroll
    for (int u = 0; u < NB; u++) s[u] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    uint4 kf[2][NB][PC];
    auto read_keys = [&](int d) {
#pragma unroll
      for (int u = 0; u < NB; u++)
#pragma unroll
        for (int i = 0; i < PC; i++)
          kf[d & 1][u][i] =
              *(const uint4*)(Kp + (i * KC + 4 * d + g4) * T::KS + (16 * u + l16) * 16);
    };
    read_keys(0);
#pragma unroll
    for (int d = 0; d < ND; d++) {
      if (d + 1 < ND) read_keys(d + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < kSmall; i++)
#pragma unroll
        for (int u = 0; u < NB; u++) s[u] = small(i, kf[d & 1][u], qf[d], s[u]);
#pragma unroll
      for (int u = 0; u < NB; u++) s[u] = mfma(kf[d & 1][u][0], qf[d][0], s[u]);
      __builtin_amdgcn_sched_barrier(0);
    }
    uint4 vf[2][EG][KT / 32][PC];
    auto read_values = [&](int e0) {
#pragma unroll
      for (int e = 0; e < EG; e++)
#pragma unroll
        for (int h = 0; h < KT / 32; h++)
#pragma unroll
          for (int i = 0; i < PC; i++)
            vf[e0 / EG & 1][e][h][i] =
                *(const uint4*)(Vp + (i * (KT / 8) + 4 * h + g4) * T::VS +
                                v_slot(16 * (e0 + e) + l16) * 16);
    };
    read_values(0);
    __builtin_amdgcn_sched_barrier(0);
    const bool edge = there != (1u << NB) - 1 || kt + KT > w.k_hi ||
                      __any(see.lo > kt || see.hi < kt + KT);
    if (edge) {
#pragma unroll
      for (int u = 0; u < NB; u++)
#pragma unroll
        for (int v = 0; v < 4; v++) {
          const int key = kt + 16 * u + 4 * g4 + v;
          const bool sees = (there >> u & 1) && key >= see.lo && key < see.hi && key < w.k_hi;
          s[u][v] = sees ? s[u][v] : -INFINITY;
        }
    }
    float mt = -INFINITY;
#pragma unroll
    for (int u = 0; u < NB; u++)
#pragma unroll
      for (int v = 0; v < 4; v++) mt = fmaxf(mt, s[u][v]);
    // The sums are kept relative to m, which follows the maximum only where
    // that has grown by more than 2^kSlack: weights up to 2^kSlack are as exact
    // as those up to one, and the sums are seldom scaled anew.
    const float mx = rows4_max(mt) * sl;
    const float m_new = mx > m + kSlack ? mx : m, ref = m_new == -INFINITY ? 0.0f : m_new;
    if (__any(m_new != m)) {
      const float alpha = __builtin_amdgcn_exp2f(m - ref);
      l *= alpha;
#pragma unroll
      for (int e = 0; e < NE; e++)
#pragma unroll
        for (int v = 0; v < 4; v++) o[e][v] *= alpha;
      m = m_new;
    }
    float ps = 0.0f;
#pragma unroll
    for (int u = 0; u < NB; u++)
#pragma unroll
      for (int v = 0; v < 4; v++) {
        s[u][v] = __builtin_amdgcn_exp2f(fmaf(s[u][v], sl, -ref));
        ps += s[u][v];
      }
    l += rows4_sum(ps);
    uint4 pf[KT / 32][3];
#pragma unroll
    for (int h = 0; h < KT / 32; h++) {
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; j++) x[j] = s[2 * h + (j >> 2)][j & 3];
      split_pieces(x, pf[h]);
    }
    // Sums, EG times 16 dims a step.
#pragma unroll
    for (int e0 = 0; e0 < NE; e0 += EG) {
      if (e0 + EG < NE) read_values(e0 + EG);
      __builtin_amdgcn_sched_barrier(0);
      const auto& x = vf[e0 / EG & 1];
#pragma unroll
      for (int h = 0; h < KT / 32; h++)
#pragma unroll
        for (int i = 0; i < kSmall; i++)
#pragma unroll
          for (int e = 0; e < EG; e++) o[e0 + e] = small(i, x[e][h], pf[h], o[e0 + e]);
#pragma unroll
      for (int h = 0; h < KT / 32; h++)
#pragma unroll
        for (int e = 0; e < EG; e++) o[e0 + e] = mfma(x[e][h][0], pf[h][0], o[e0 + e]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  if (!live) return;
  const bool mine = wave_row + l16 < w.rows;
  const int64_t out_row = row_at(a, w, row);
  float check = l - l;
#pragma unroll
  for (int e = 0; e < NE; e++)
#pragma unroll
    for (int v = 0; v < 4; v++) check += o[e][v] - o[e][v];
  if (__builtin_expect(__any(check != check), 0)) {
    using L = Lanes<C, HD>;
    Sums<C, HD> x;
    exact_walk<C, HD, false>(a, w, qp, see, sl, w.k_lo, w.k_hi - w.k_lo, w.k_hi - w.k_lo, l16, g4, x);
#pragma unroll
    for (int h = 0; h < L::NH; h++)
#pragma unroll
      for (int v = 0; v < 4; v++)
#pragma unroll
        for (int c = 0; c < L::EV; c += 4)
          if (mine)
            write_row4(a, w, out_row, HD, L::EV * (4 * g4 + v + 16 * h) + c,
                       make_float4(x.o[h][c][v], x.o[h][c + 1][v], x.o[h][c + 2][v],
                                   x.o[h][c + 3][v]),
                       x.m, x.l, g4 == 0);
    return;
  }
#pragma unroll
  for (int e = 0; e < NE; e++)
    if (mine)
      write_row4(a, w, out_row, HD, 16 * e + 4 * g4, make_float4(o[e][0], o[e][1], o[e][2], o[e][3]),
                 m, l, g4 == 0);
}

template <typename C, int HD>
constexpr int attention_lds() {
  using T = WideTile<C, HD>;
  constexpr int w = T::kK + T::kV + kWaves * 8, n = kMergeBytes<HD> + 4 * HD * 4;
  return w > n ? w : n;
}

template <typename C, int HD>
struct FloatBody {
  static constexpr int kKeys = sizeof(C) == 4 ? 16 : 32;
  static constexpr bool kTogether = false, kLastFirst = false;
  static __device__ __forceinline__ void wide(const PagedArgs& a, const Item& w, uint8_t* lds) {
    ::wide<C, HD>(a, w, lds);
  }
  template <bool kJoined>
  static __device__ __forceinline__ void block_of_16(const PagedArgs& a, const Item& w, int rows, uint8_t* lds) {
    if constexpr (sizeof(C) == 4) {
      if (rows == 2) return few<HD, 2, kJoined>(a, w, lds);
      if (rows == 4) return few<HD, 4, kJoined>(a, w, lds);
    }
    narrow<C, HD, kJoined>(a, w, lds);
  }
};

template <typename C, int HD, bool kPacked>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2, 2)))
paged_attention_kernel(PagedArgs a) {
  __shared__ __align__(16) uint8_t lds[attention_lds<C, HD>()];
  paged_workgroup<FloatBody<C, HD>, kPacked>(a, lds);
}

// A row's partial results added in order by W waves, an equal part of the runs
// each (at most 64): lane s holds the statistics of the part's run s, lane i
// sums dims ND i .., eight runs' values requested at once. What runs without a
// weight hold does not count. Under a trace 5.0 us for 64 tokens of 32 heads,
// hd 128, 9 runs by one wave a row (5.8 by four); 4.0 for 16 tokens of 16, 18
// runs, by four (by one 0.6 more): the launch and two
// waits for memory.
template <int HD, int W>
__global__ void __launch_bounds__(kThreads) paged_combine_kernel(PagedArgs a) {
  constexpr int ND = HD / 64, U = 8;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t r =
      ((int64_t)blockIdx.y * a.combine_x + blockIdx.x) * (kWaves / W) + wave / W;
  if (r >= (int64_t)a.tokens * a.heads) return;
  const int live = max(0, min(a.starts[a.seqs], a.tokens));
  const int per = (a.splits + W - 1) / W, first = W == 1 ? 0 : wave * per;
  const int runs = max(0, min(per, a.splits - first));
  // Resources that end with the part's runs: lanes and runs past them read 0.
  const int64_t at0 = r * a.splits + first;
  const i32x4 srs = buffer_rsrc(a.stat + 2 * at0, (uint32_t)runs * 8u);
  const i32x4 prs = buffer_rsrc(a.part + at0 * HD, (uint32_t)(runs * HD) * 4u);
  const i32x2 ml = dnx_raw_buffer_load_v2i32(srs, lane * 8, 0, 0);
  float v[U][ND];
  auto load = [&](int s0) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int at = ((s0 + u) * HD + ND * lane) * 4;
      if constexpr (ND == 2) {
        const i32x2 x = dnx_raw_buffer_load_v2i32(prs, at, 0, 0);
        v[u][0] = __int_as_float(x.x);
        v[u][1] = __int_as_float(x.y);
      } else {
        v[u][0] = __int_as_float(dnx_raw_buffer_load_i32(prs, at, 0, 0));
      }
    }
  };
  load(0);
  __builtin_amdgcn_sched_barrier(0);   // all requested before the first wait
  if (r >= (int64_t)live * a.heads) return;   // behind the last sequence
  const float l = __int_as_float(ml.y), m = lane < runs ? __int_as_float(ml.x) : -INFINITY;
  float top = wave_max_dpp(m);
  const float f = partial_factor(m, l, top);
  float total = wave_sum_dpp(l * f);
  const uint64_t with = __ballot(l != 0.0f);
  float acc[ND] = {};
  for (int s0 = 0; s0 < runs; s0 += U) {
    if (s0 > 0) load(s0);
#pragma unroll
    for (int u = 0; u < U; u++) {
      const float fs = lane_value(f, s0 + u);
      const bool counts = (with >> (s0 + u)) & 1;
#pragma unroll
      for (int i = 0; i < ND; i++) acc[i] = fmaf(counts ? v[u][i] : 0.0f, fs, acc[i]);
    }
  }
  if constexpr (W > 1) {
    __shared__ float stats[W][2], sums[W][HD];
    if (lane == 0) stats[wave][0] = top, stats[wave][1] = total;
#pragma unroll
    for (int i = 0; i < ND; i++) sums[wave][ND * lane + i] = acc[i];
    __syncthreads();
    if (wave > 0) return;
    top = stats[0][0];
#pragma unroll
    for (int k = 1; k < W; k++) top = fmaxf(top, stats[k][0]);
    total = 0.0f;
#pragma unroll
    for (int i = 0; i < ND; i++) acc[i] = 0.0f;
#pragma unroll
    for (int k = 0; k < W; k++) {
      const float part = stats[k][1];
      if (part == 0.0f) continue;
      const float fk = partial_factor(stats[k][0], part, top);
      total = fmaf(part, fk, total);
#pragma unroll
      for (int i = 0; i < ND; i++) acc[i] = fmaf(sums[k][ND * lane + i], fk, acc[i]);
    }
  }
  const float g = row_scale(total, a.gate, r);
#pragma unroll
  for (int i = 0; i < ND; i++) a.out[r * HD + ND * lane + i] = acc[i] * g;
}

PartArgs part_of(const PagedPart& p) {
  return {p.wide, p.few, (int)p.blocks, (int)p.runs, (int)p.keys, p.together};
}

// The most own keys of a sequence that can be seen.
int64_t most_own(const dnx_paged_cache* c, const dnx_paged_batch* b) {
  return std::min(b->max_len, b->table_stride * c->page);
}

PagedSplit split_of(const dnx_paged_cache* c, const dnx_paged_batch* b, int64_t heads) {
  return paged_split(b->seqs, b->tokens, std::min(b->max_tokens, b->tokens), heads / c->kv_heads,
                     c->kv_heads, b->prefix_len, most_own(c, b), c->type == DNX_F32,
                     c->type == DNX_I8 ? c->hd : 0);
}

}  // namespace

extern "C" {

int64_t dnx_paged_attention_workspace_bytes(const dnx_paged_cache* cache,
                                            const dnx_paged_batch* batch, int64_t heads) {
  if (!cache_ok(cache) || !batch_ok(batch) || heads <= 0 || heads % cache->kv_heads != 0 ||
      heads > 65535 || batch->tokens * heads >= (1 << 26)) {
    return -1;
  }
  const PagedSplit s = split_of(cache, batch, heads);
  if (s.prefix_items + s.own_items > kPagedItems) return -1;
  return s.splits() <= 1 ? 0 : batch->tokens * heads * s.splits() * (cache->hd + 2) * 4;
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
  a.pages = (int)cache->pages;
  a.page_bits = __builtin_ctz((unsigned)cache->page);
  a.row_bytes = cache->kv_heads * cache->hd * (cache->type == DNX_F32 ? 4 : cache->type == DNX_BF16 ? 2 : 1);
  a.key_scales = cache_scales(cache).keys;
  a.value_scales = cache_scales(cache).values;
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
  a.max_len = (int)most_own(cache, batch);
  a.q = q;
  a.gate = gate;
  a.out = out;
  a.splits = (int)s.splits();
  a.part = (float*)workspace;
  a.stat = a.part + batch->tokens * heads * a.splits * cache->hd;
  a.window = (int)window;
  a.joined = (int)s.joined;
  a.prefix = part_of(s.prefix);
  a.own = part_of(s.own);
  a.slots = (uint32_t)s.slots;
  a.prefix_items = s.prefix_items;
  a.scale = (float)(1.0 / sqrt((double)cache->hd));
  static_assert(kPagedItems == kLaunchThreads / kThreads, "the launch's limit");
  const int64_t grid = s.prefix_items + s.own_items;
  const hipStream_t st = (hipStream_t)stream;
  if (grid > 0) {
    const int kind = (s.slots > 0 ? 4 : 0) + (cache->type == DNX_BF16 ? 2 : 0) + (cache->hd == 128);
    constexpr decltype(&paged_attention_kernel<float, 64, false>) kernels[] = {
        paged_attention_kernel<float, 64, false>,    paged_attention_kernel<float, 128, false>,
        paged_attention_kernel<uint16_t, 64, false>, paged_attention_kernel<uint16_t, 128, false>,
        paged_attention_kernel<float, 64, true>,     paged_attention_kernel<float, 128, true>,
        paged_attention_kernel<uint16_t, 64, true>,  paged_attention_kernel<uint16_t, 128, true>,
    };
    const PagedKernel k = cache->type == DNX_I8 ? paged_attention_i8(cache->hd, s.slots > 0)
                                                : kernels[kind];
    hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(kThreads), 0, st, a);
    if (hipGetLastError() != hipSuccess) return DNX_ELAUNCH;
  }
  if (a.splits != 1) {
    const int64_t rows = batch->tokens * heads;
    const bool split = rows < kPagedManyRows && a.splits > (rows < 2048 ? 8 : 16);
    const int64_t blocks = split ? rows : (rows + kWaves - 1) / kWaves;
    // One dimension holds the workgroups of 2^26 - 4 rows; calls have up to 2^26 - 1.
    const int64_t x = std::min(blocks, kLaunchThreads / kThreads);
    a.combine_x = (int)x;
    auto k = cache->hd == 128 ? (split ? paged_combine_kernel<128, kWaves>
                                       : paged_combine_kernel<128, 1>)
                              : (split ? paged_combine_kernel<64, kWaves>
                                       : paged_combine_kernel<64, 1>);
    hipLaunchKernelGGL(k, dim3((unsigned)x, (unsigned)((blocks + x - 1) / x)), dim3(kThreads), 0, st,
                       a);
  }
  return hipGetLastError() == hipSuccess ? DNX_OK : DNX_ELAUNCH;
}

}  // extern "C"
