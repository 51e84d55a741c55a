// The attention of paged_attention.hip over int8 caches: keys c_j and values d_j
// are codes from -127 to 127 with a float32 scale for each place and head. For
// a row (a query head of a token) and the keys j it sees,
//   s_j = ks_j (q.c_j) / sqrt(hd),
//   out = sum_j e^(s_j - m) vs_j d_j / sum_j e^(s_j - m).
//
// Both products run on the int8 matrix cores, on the codes as they lie in the
// cache. The other operand is a whole number in digits of base 256 from -128 to 127
// (the highest up to 127), a product each:
// * a query row is a number of 31 bits in four digits, in units of 2^(e - 31), 2^e
//   the power of two above 1.004 times its largest value: off by half a unit, 2^-32
//   of 2^e. With three digits a row with one channel 3000 times the others, whose
//   keys are as much smaller, is off by 1.2e-4 (2000 keys, hd 128), with four by
//   5e-7; the fourth takes 3% of a prompt's time and none of a decode step's.
// * the weights e^(s_j - m) vs_j of a row and step are numbers of 23 bits in three,
//   2^e above the largest of that step: relative to the step, not to the running
//   maximum, so that a long tail of small weights is kept. 64 keys times half a
//   unit times codes of 127 are 2^-9 of half a code of that largest one, which
//   is what its value was rounded by when it was appended.
// The int32 sums are exact (128 products of 7 by 8 bits are below 2^21). A bf16
// form would convert every code (1.5 instructions each) and take three
// products of half the depth.

#include "paged.h"
#include "paged_attention.h"

#include "bf16_pieces.h"

using namespace dnx;

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

DNX_DEV v4i mfma8(const uint4& x, const uint4& y, v4i acc) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(v4i, x), __builtin_bit_cast(v4i, y),
                                               acc, 0, 0, 0);
}

// Sums of products of digits as one number: 2^24 a + 65536 b + 256 c + d.
DNX_DEV float of_digits(int a, int b, int c, int d) {
  return fmaf((float)(int)(((uint32_t)a << 8) + (uint32_t)b), 65536.0f,
              (float)(int)(((uint32_t)c << 8) + (uint32_t)d));
}
// 65536 a + 256 b + c.
DNX_DEV float of_digits(int a, int b, int c) {
  return fmaf((float)a, 65536.0f, (float)(int)(((uint32_t)b << 8) + (uint32_t)c));
}

// 2^e for -126 <= e <= 127.
DNX_DEV float power2(int e) { return __int_as_float((e + 127) << 23); }

// The digits below the highest are bytes less 128: 0x80 in each, taken off by an xor.
constexpr int kMiddle = 0x8080, kMiddle4 = 0x808080;
constexpr uint32_t kSigns = 0x80808080u;
// 127 (65536 + 256 + 1) is the largest number of three digits: 2^23 / 1.00394; of
// four 2^31 / 1.00394.
constexpr float kRoom = 1.004f;
constexpr int kQ = 4, kQBits = 31;   // digits of a query's values, bits of them

// Bytes of four words turned: word c of the result holds byte c of each.
DNX_DEV void turn4(uint32_t x0, uint32_t x1, uint32_t x2, uint32_t x3, uint32_t* y) {
  const uint32_t a = __builtin_amdgcn_perm(x1, x0, 0x05010400u);
  const uint32_t b = __builtin_amdgcn_perm(x3, x2, 0x05010400u);
  const uint32_t c = __builtin_amdgcn_perm(x1, x0, 0x07030602u);
  const uint32_t d = __builtin_amdgcn_perm(x3, x2, 0x07030602u);
  y[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
  y[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
  y[2] = __builtin_amdgcn_perm(d, c, 0x05040100u);
  y[3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}

// Word k of the result holds byte k of each of four words; of the lower two bytes
// the digits.
DNX_DEV void bytes_of(const uint32_t* y, uint32_t* d) {
  const uint32_t a = __builtin_amdgcn_perm(y[1], y[0], 0x05010400u);
  const uint32_t b = __builtin_amdgcn_perm(y[3], y[2], 0x05010400u);
  d[0] = __builtin_amdgcn_perm(b, a, 0x05040100u) ^ kSigns;
  d[1] = __builtin_amdgcn_perm(b, a, 0x07060302u) ^ kSigns;
  d[2] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(y[3], y[2], 0x0c0c0602u),
                               __builtin_amdgcn_perm(y[1], y[0], 0x0c0c0602u), 0x05040100u);
}

// The larger of |x| and |y|, NaN if either is.
DNX_DEV float abs_max(float x, float y) {
  return __builtin_elementwise_maximum(fabsf(x), fabsf(y));
}

// What takes a sum of products of a query row's digits to a score in units of
// log2: `first` before the key's scale and `c` after it, powers of two but for c's
// part of the formula. Their product may be too small for a float (rows of small
// values), and a sum times a large key's scale too large: with both, which are
// normal numbers, a score up to 2^60 is reached from any row and any scale.
struct QueryFactor {
  float c, first;
};
DNX_DEV QueryFactor query_factor(float scale, int e, float nan) {
  const int a = max(min(e - kQBits, 0), -120);
  return {__builtin_amdgcn_ldexpf(scale * 1.44269504088896341f, e - kQBits - a) + nan, power2(a)};
}

// The digits of a query row at the lane's dims, 16 from `dim` on and each `step`
// further. A row with an infinity or NaN: a factor of NaN.
template <int HD>
DNX_DEV QueryFactor query_digits(const float* q, int dim, int step, float scale, uint4 (*qd)[kQ]) {
  constexpr int ND = HD / 64;
  float x[ND][16], top = 0.0f;
#pragma unroll
  for (int d = 0; d < ND; d++)
#pragma unroll
    for (int j = 0; j < 16; j += 4) {
      const float4 v = *(const float4*)(q + dim + step * d + j);
      x[d][j] = v.x, x[d][j + 1] = v.y, x[d][j + 2] = v.z, x[d][j + 3] = v.w;
    }
#pragma unroll
  for (int d = 0; d < ND; d++)
#pragma unroll
    for (int j = 0; j < 16; j++) top = abs_max(top, x[d][j]);
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(top), __float_as_uint(top), false,
                                                  false);
  top = abs_max(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false,
                                                  false);
  top = abs_max(__uint_as_float(b[0]), __uint_as_float(b[1]));
  top *= kRoom;
  const int e = __builtin_amdgcn_frexp_expf(top);
#pragma unroll
  for (int d = 0; d < ND; d++) {
    uint32_t w[kQ][4];
#pragma unroll
    for (int j = 0; j < 16; j += 4) {
      uint32_t y[4], t[kQ];
#pragma unroll
      for (int i = 0; i < 4; i++)
        y[i] = (uint32_t)(int)rintf(__builtin_amdgcn_ldexpf(x[d][j + i], kQBits - e)) + kMiddle4;
      turn4(y[0], y[1], y[2], y[3], t);
#pragma unroll
      for (int k = 0; k < kQ; k++) w[k][j / 4] = k < kQ - 1 ? t[k] ^ kSigns : t[k];
    }
#pragma unroll
    for (int k = 0; k < kQ; k++) qd[d][k] = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
  }
  return query_factor(scale, e, top - top);
}

// Sums of products to scores over c.
DNX_DEV void to_scores(v4f* s, const QueryFactor& f, const float4* ks) {
#pragma unroll
  for (int u = 0; u < 4; u++)
#pragma unroll
    for (int v = 0; v < 4; v++) s[u][v] = s[u][v] * f.first * (&ks[u].x)[v];
}

// The digits of four weights up to 2^e / kRoom, unit = 2^(23 - e), word k those of
// place k: the float 2^23 + 0x8080 + w 2^(23 - e), below 2^24, has them as its bytes.
DNX_DEV void weight_digits(const float* w, float unit, uint32_t* d) {
  uint32_t y[4];
#pragma unroll
  for (int i = 0; i < 4; i++) y[i] = __float_as_uint(fmaf(w[i], unit, 8388608.0f + kMiddle));
  bytes_of(y, d);
}

// 16 keys of an item from kt on, as paged_attention.hip's blocks: where their
// codes of one head lie, how many bytes of them there are, and where their
// scales lie. A page holds whole sixteens, so the sixteen scales may be read
// whatever keys there are. The resources over them are made at each use: sixteen
// for a step's blocks are more registers than there are.
struct Block {
  uint64_t at, scale;
  uint32_t range;
  int end;      // its keys lie before this key (none: not after the first)
};
DNX_DEV i32x4 codes_of(const Block& b, const void* from) {
  return buffer_rsrc((const uint8_t*)from + b.at, b.range);
}
DNX_DEV i32x4 scales_of(const Block& b, const float* from) {
  return buffer_rsrc(from + b.scale, b.range > 0 ? 64u : 0u);
}
template <int HD, bool kJoined>
DNX_DEV Block block_at(const PagedArgs& a, const Item& w, int kt, int page) {
  Block b;
  const bool own = !kJoined || kt >= w.joined;
  const int left = min(16, (own ? w.k_hi : a.prefix_len) - kt);
  const bool there = left > 0 && (uint32_t)page < (uint32_t)a.pages;
  b.end = there ? kt + left : kt;
  b.range = there ? (uint32_t)(left * a.row_bytes) : 0u;
  // Not used where the range is empty.
  const uint32_t in_page = (uint32_t)((kJoined && own ? kt - w.joined : kt) & ((1 << a.page_bits) - 1));
  b.at = (uint64_t)(uint32_t)page * ((uint32_t)a.row_bytes << a.page_bits) +
         (uint64_t)(in_page * (uint32_t)a.row_bytes) + (uint32_t)(w.kvh * HD);
  b.scale =
      (((uint64_t)(uint32_t)page * (uint32_t)a.kv_heads + (uint32_t)w.kvh) << a.page_bits) + in_page;
  return b;
}

// The running sums of a wave's 16 rows: o[c][v] of row l % 16 at the dim that row 4
// g + v of product c is of, l the lane's part of the row's sum.
template <int HD>
struct Sums {
  float m, l;
  v4f o[HD / 16];
};

// A step's 64 scores and weights of row l % 16, of which the lane has keys kt +
// 16 u + 4 g + v. In: the scores' sums of products times the key's scale. Out:
// the weights' digits, whose word u of digit k is d[k][u]; the running sums
// are scaled anew where the maximum has grown by 2^kSlack, and the factor is
// returned that takes this step's sums of products to theirs.
// edge: the step holds keys that some row does not see.
template <int HD, typename F>
DNX_DEV float step_weights(v4f* s, float c, const float4* vs, bool edge, F sees, Sums<HD>& a,
                           uint32_t (*d)[4]) {
  float mt = -INFINITY;
  if (edge) {
#pragma unroll
    for (int u = 0; u < 4; u++)
#pragma unroll
      for (int v = 0; v < 4; v++) s[u][v] = sees(u, v) ? s[u][v] : -INFINITY;
  }
#pragma unroll
  for (int u = 0; u < 4; u++)
#pragma unroll
    for (int v = 0; v < 4; v++) mt = fmaxf(mt, s[u][v]);
  const float mx = rows4_max(mt) * c;
  const float m_new = mx > a.m + kSlack ? mx : a.m, ref = m_new == -INFINITY ? 0.0f : m_new;
  if (__any(m_new != a.m)) {
    const float alpha = __builtin_amdgcn_exp2f(a.m - ref);
    a.l *= alpha;
#pragma unroll
    for (int e = 0; e < HD / 16; e++)
#pragma unroll
      for (int v = 0; v < 4; v++) a.o[e][v] *= alpha;
    a.m = m_new;
  }
  float ps = 0.0f, top = 0.0f;
#pragma unroll
  for (int u = 0; u < 4; u++)
#pragma unroll
    for (int v = 0; v < 4; v++) {
      const float p = __builtin_amdgcn_exp2f(fmaf(s[u][v], c, -ref));
      ps += p;
      s[u][v] = p * (&vs[u].x)[v];
    }
  a.l += ps;
  if (edge) {   // what an unseen place's scale holds does not matter
#pragma unroll
    for (int u = 0; u < 4; u++)
#pragma unroll
      for (int v = 0; v < 4; v++) s[u][v] = sees(u, v) ? s[u][v] : 0.0f;
  }
#pragma unroll
  for (int u = 0; u < 4; u++)
#pragma unroll
    for (int v = 0; v < 4; v += 2) top = abs_max(top, abs_max(s[u][v], s[u][v + 1]));
  const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(top), __float_as_uint(top), false,
                                                  false);
  top = abs_max(__uint_as_float(x[0]), __uint_as_float(x[1]));
  const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false,
                                                  false);
  top = abs_max(__uint_as_float(y[0]), __uint_as_float(y[1]));
  top *= kRoom;
  const int e = max(__builtin_amdgcn_frexp_expf(top), -100);
  const float unit = power2(23 - e);
#pragma unroll
  for (int u = 0; u < 4; u++) {
    const float w[4] = {s[u][0], s[u][1], s[u][2], s[u][3]};
    uint32_t t[3];
    weight_digits(w, unit, t);
    d[0][u] = t[0], d[1][u] = t[1], d[2][u] = t[2];
  }
  return power2(e - 23) + (top - top);   // NaN where a weight is no finite number
}

// ---- 16 rows a workgroup, each wave other keys, 64 a step.
//
// Lane l (quarter g = l / 16) takes key 16 u + l % 16 at 16 dims of each 64, whose
// products with row l % 16's digits leave it with the scores of keys 16 u + 4 g
// + v: the sixteen keys whose values it takes at HD / 16 dims, turned in
// registers into bytes of one dim, and whose weights' digits are then the other
// operand as they are.
//
// What bounds it is the reading, and how fast that goes depends on what one load
// instruction covers (537 MB of keys and values read and dropped, hd 128, 8 key
// heads: 4.8 TB/s by half lines of 16 keys, 5.1 by whole lines of 8, 5.9 by whole
// lines marked as read once). So at hd 128 a load covers the 128 bytes of eight
// keys, half of what a lane gets is for the lane 8 further in its quarter, and
// the two trade it: K arrives as key l % 8 (+ 8) at dims 32 g + 16 (l / 8 % 2)
// .., V as dims 16 (l % 8) .. of key 16 u + 4 g + l / 8 % 2 (+ 2). At hd 64 the
// lines hold two heads: those of a run run on one XCD, through one L2 (64
// sequences of 1088 keys, 28 -> 19.5 us; at hd 128 3% slower).
//
// 64 sequences, 32 / 8 heads, hd 128, of 4096 keys 108 us, 5.1 TB/s (reading alone
// 98), of 1088 32 us, 4.6; one of 131072 56, of which 5 are the second launch. A
// step of 64 keys takes about 630 vector instructions and 56 matrix ones (the bf16
// form of paged_attention.hip 1000 vector ones for as many), which a decode step
// hides behind the reading; forming the products of one part beside the sums of
// another gained nothing. In a prompt they are what bounds it: 4096 tokens, 32 / 8
// heads, hd 128, 610 us, 225 TFLOP/s of the formula's products; 725 of 4099 keys, 16 /
// 8 heads, 107.
template <int HD>
struct Raw {
  uint4 k[4][HD / 64];
  uint32_t v[4][4][HD / 64];
  float4 ks[4], vs[4];
};

// Lanes 0 .. 7 of 16 keep x and take the x of 8 .. 15 into y; those keep their y
// and take the y of 0 .. 7 into x.
DNX_DEV void trade8(uint32_t& x, uint32_t& y) {
  constexpr int kRor8 = 0x128;
  const uint32_t a = x, b = y;
  x = (uint32_t)__builtin_amdgcn_update_dpp((int)a, (int)b, kRor8, 0xf, 0xc, false);
  y = (uint32_t)__builtin_amdgcn_update_dpp((int)b, (int)a, kRor8, 0xf, 0x3, false);
}

template <int HD, bool kJoined>
DNX_DEV void narrow(const PagedArgs& a, const Item& w, uint8_t* lds) {
  constexpr int ND = HD / 64, EV = HD / 16, KS = 64, kStride = KS * kWaves;
  const int lane = threadIdx.x & 63, l16 = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = min(w.row0 + l16, w.rows - 1);
  const Seen see = row_sees(a, w, row);
  const float* qp = a.q + row_at(a, w, row) * HD;
  Sums<HD> sums;
  sums.m = -INFINITY;
  sums.l = 0.0f;
#pragma unroll
  for (int e = 0; e < EV; e++) sums.o[e] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

  // As in paged_attention.hip: the next step's keys are requested when this
  // step's scores are formed, its values when this step's are added, its pages
  // one step before that.
  Raw<HD> x;
  Block block[4];
  int page[4];
  auto pages = [&](int at) {
#pragma unroll
    for (int u = 0; u < 4; u++) page[u] = page_at<kJoined>(a, w, at + 16 * u);
  };
  auto blocks = [&](int at) {
#pragma unroll
    for (int u = 0; u < 4; u++) block[u] = block_at<HD, kJoined>(a, w, at + 16 * u, page[u]);
  };
  const int l8 = l16 & 7, b8 = l16 >> 3;
  auto request_keys = [&] {
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const i32x4 r = codes_of(block[u], a.keys);
      if constexpr (ND == 2) {
#pragma unroll
        for (int d = 0; d < 2; d++)
          x.k[u][d] = buffer_load16_stream(r, (8 * d + l8) * a.row_bytes + 32 * g4 + 16 * b8);
      } else {
        x.k[u][0] = buffer_load16(r, l16 * a.row_bytes + 16 * g4);
      }
      x.ks[u] = buffer_load_f4(scales_of(block[u], a.key_scales), 16 * g4);
    }
  };
  auto request_values = [&] {
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const i32x4 r = codes_of(block[u], a.values);
      if constexpr (ND == 2) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const uint4 y = buffer_load16_stream(r, (4 * g4 + 2 * j + b8) * a.row_bytes + 16 * l8);
          x.v[u][2 * j][0] = y.x, x.v[u][2 * j][1] = y.y;
          x.v[u][2 * j + 1][0] = y.z, x.v[u][2 * j + 1][1] = y.w;
        }
      } else {
#pragma unroll
        for (int v = 0; v < 4; v++)
          x.v[u][v][0] = (uint32_t)dnx_raw_buffer_load_i32(r, (4 * g4 + v) * a.row_bytes + EV * l16, 0, 0);
      }
      x.vs[u] = buffer_load_f4(scales_of(block[u], a.value_scales), 16 * g4);
    }
  };
  auto next = [&](int at) {
    while (at < w.k_hi && !__any(see.lo < at + KS && see.hi > at)) at += kStride;
    return at;
  };
  uint4 qd[ND][kQ];
  QueryFactor factor{};
  const int first = w.k_lo + KS * wave;
  int kt = next(first), after = kt;
  if (kt < w.k_hi) {
    if (kt == first) {
#pragma unroll
      for (int u = 0; u < 4; u++) page[u] = w.page[u];
    } else {
      pages(kt);
    }
    blocks(kt);
    request_keys();
    request_values();
    after = next(kt + kStride);
    pages(after);
    factor = ND == 2 ? query_digits<HD>(qp, 32 * g4, 16, a.scale, qd)
                     : query_digits<HD>(qp, 16 * g4, 64, a.scale, qd);
  }
  while (kt < w.k_hi) {
    int end[4];
#pragma unroll
    for (int u = 0; u < 4; u++) end[u] = block[u].end;
    const int then = next(after + kStride);
    blocks(after);
    pages(then);
    v4f s[4];
#pragma unroll
    for (int u = 0; u < 4; u++) {
      if constexpr (ND == 2) {     // (the key of the first eight, dims of b8) for (own key, first dims)
        trade8(x.k[u][0].x, x.k[u][1].x);
        trade8(x.k[u][0].y, x.k[u][1].y);
        trade8(x.k[u][0].z, x.k[u][1].z);
        trade8(x.k[u][0].w, x.k[u][1].w);
      }
      v4i t[kQ];
#pragma unroll
      for (int k = 0; k < kQ; k++) {
        t[k] = v4i{0, 0, 0, 0};
#pragma unroll
        for (int d = 0; d < ND; d++) t[k] = mfma8(x.k[u][d], qd[d][k], t[k]);
      }
#pragma unroll
      for (int v = 0; v < 4; v++) s[u][v] = of_digits(t[3][v], t[2][v], t[1][v], t[0][v]);
    }
    to_scores(s, factor, x.ks);
    request_keys();
    bool edge = __any(see.lo > kt || see.hi < kt + KS);
#pragma unroll
    for (int u = 0; u < 4; u++) edge |= end[u] != kt + 16 * u + 16;
    auto sees = [&](int u, int v) {
      const int key = kt + 16 * u + 4 * g4 + v;
      return key >= see.lo && key < see.hi && key < end[u];
    };
    uint32_t pd[3][4];
    const float beta = step_weights<HD>(s, factor.c, x.vs, edge, sees, sums, pd);
    if constexpr (ND == 2) {       // (key of b8, its first dims) for (first key, own dims)
#pragma unroll
      for (int u = 0; u < 4; u++)
#pragma unroll
        for (int v = 0; v < 4; v += 2)
#pragma unroll
          for (int h = 0; h < 2; h++) trade8(x.v[u][v][h], x.v[u][v + 1][h]);
    }
#pragma unroll
    for (int h = 0; h < ND; h++) {
      uint32_t f[4][4];
#pragma unroll
      for (int u = 0; u < 4; u++) {
        uint32_t y[4];
        turn4(x.v[u][0][h], x.v[u][1][h], x.v[u][2][h], x.v[u][3][h], y);
#pragma unroll
        for (int e = 0; e < 4; e++) f[e][u] = y[e];
      }
#pragma unroll
      for (int e = 0; e < 4; e++) {
        v4i t[3];
#pragma unroll
        for (int k = 0; k < 3; k++)
          t[k] = mfma8(make_uint4(f[e][0], f[e][1], f[e][2], f[e][3]),
                       make_uint4(pd[k][0], pd[k][1], pd[k][2], pd[k][3]), v4i{0, 0, 0, 0});
#pragma unroll
        for (int v = 0; v < 4; v++)
          sums.o[4 * h + e][v] =
              fmaf(of_digits(t[2][v], t[1][v], t[0][v]), beta, sums.o[4 * h + e][v]);
      }
    }
    request_values();
    kt = after;
    after = then;
  }
  sums.l = rows4_sum(sums.l);

  // The dims of which row i of the products is: EV from here on.
  auto dim_of = [](int i) { return ND == 2 ? 16 * (i & 7) + 8 * (i >> 3) : EV * i; };
  float* all = (float*)lds;
  float* ml = wave_stats<HD>(lds, wave);
  if (g4 == 0) {
    ml[l16] = sums.m;
    ml[16 + l16] = sums.l;
  }
#pragma unroll
  for (int v = 0; v < 4; v++)
#pragma unroll
    for (int e = 0; e < EV; e += 4)
      *(float4*)&all[(wave * 16 + l16) * kSumRow<HD> + dim_of(4 * g4 + v) + e] =
          make_float4(sums.o[e][v], sums.o[e + 1][v], sums.o[e + 2][v], sums.o[e + 3][v]);
  merge_waves<HD, 16>(a, w, lds);
}

// ---- 64 rows a workgroup, 16 a wave, which share tiles of 64 keys in LDS.
//
// Keys as [16 dims][key], values as [quarter][dim], 16 bytes each: the bytes of
// a quarter and dim are those of its sixteen keys, turned on the way. The next
// tile is in registers meanwhile.
//
// Sixteen prompts of 512 tokens, 32 / 8 heads, hd 128: 226 us, 152 TFLOP/s of the
// formula's products; 64 of 64 tokens 48 us. For a wave's 64 keys of 16 rows it takes
// about 450 vector instructions, 18 a score (digits to a float, exp2, float to digits)
// and 5 a sum (digits to a float, into the running sum), beside 56 matrix ones, and
// about 60 to stage its part of the tile: the four blocks of a tile lie in scratch
// memory (112 bytes a lane), since a load's block is chosen at run time, and the
// loads' addresses wait for it. That, the two barriers and the digits bound it; a
// staging that looks up a wave's own block alone and tiles of 128 keys (half the sums)
// are not tried.
template <int HD>
struct WideTile {
  static constexpr int KT = 64, KC = HD / 16;      // 16-byte chunks of a key
  static constexpr int KS = KT * 16 + 16;          // K: a chunk of all keys, + pad
  static constexpr int kK = KC * KS, kV = KT * HD; // bytes
  static constexpr int kScales = 2 * KT * 4;
  static constexpr int KU = KT * KC / kThreads;    // K: chunks a thread
  static constexpr int UV = HD / 64;               // V: of the four u, a thread
};

template <int HD>
DNX_DEV void wide(const PagedArgs& a, const Item& w, uint8_t* lds) {
  using T = WideTile<HD>;
  constexpr int KT = T::KT, ND = HD / 64, NE = HD / 16;
  uint8_t* Kp = lds;
  uint8_t* Vp = lds + T::kK;
  float* scales = (float*)(Vp + T::kV);            // of the keys, of the values
  int* span = (int*)(lds + T::kK + T::kV + T::kScales);
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wave_row = w.row0 + 16 * wave;
  const bool live = wave_row < w.rows;
  const int row = min(wave_row + l16, w.rows - 1);
  const Seen see = row_sees(a, w, row);
  const float* qp = a.q + row_at(a, w, row) * HD;

  // The keys that any row of the workgroup sees.
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

  // Staging. A thread's values: dims 4 vt .. of the keys 16 u + 4 vg + 0..3, u
  // from vu on; a wave's part of a load may lie in two blocks of 16 keys.
  constexpr int VT = HD / 4;
  const int vt = tid % VT, vg = tid / VT % 4, vu = tid / VT / 4 * T::UV;
  uint4 kr[T::KU];
  uint32_t vr[T::UV][4];
  float sr = 0.0f;
  uint32_t there = 0, there_next = 0;              // which blocks of 16 keys there are
  int page[4];
  auto pages = [&](int kt) {
#pragma unroll
    for (int i = 0; i < 4; i++) page[i] = page_at<false>(a, w, kt + 16 * i);
  };
  auto load_tile = [&](int kt) {
    Block b[4];
    there_next = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      b[i] = block_at<HD, false>(a, w, kt + 16 * i, page[i]);
      there_next |= b[i].end > kt + 16 * i ? 1u << i : 0u;
    }
    const int stride = a.row_bytes;
    auto of = [&](int i, const void* from) {
      const uint64_t at = i == 0 ? b[0].at : i == 1 ? b[1].at : i == 2 ? b[2].at : b[3].at;
      const uint32_t range = i == 0 ? b[0].range : i == 1 ? b[1].range
                             : i == 2 ? b[2].range : b[3].range;
      return buffer_rsrc((const uint8_t*)from + at, range);
    };
    // Keys: the 64 chunks of a wave's load lie in one block (HD 64: 16 keys of
    // 4 chunks) or in half of one.
#pragma unroll
    for (int j = 0; j < T::KU; j++) {
      const int unit = j * kThreads + tid, key = unit / T::KC, ch = unit % T::KC;
      const int at = (key & 15) * stride + ch * 16;
      constexpr int kPer = 16 * T::KC / 64;        // waves a block
      const int i = (j * kWaves + wave) / kPer;
      kr[j] = buffer_load16(of(i, a.keys), at);
    }
#pragma unroll
    for (int j = 0; j < T::UV; j++) {
      const int first = wave * 64 / VT / 4 * T::UV + j;     // u of the wave's values
      const i32x4 r = of(first, a.values);
#pragma unroll
      for (int v = 0; v < 4; v++)
        vr[j][v] = (uint32_t)dnx_raw_buffer_load_i32(r, (4 * vg + v) * stride + 4 * vt, 0, 0);
    }
    if (wave < 2) {   // the scales: a wave the keys', a wave the values'
      const int i = lane / 16;
      float f[4];
#pragma unroll
      for (int k = 0; k < 4; k++)
        f[k] = __int_as_float(dnx_raw_buffer_load_i32(
            scales_of(b[k], wave == 0 ? a.key_scales : a.value_scales), 4 * l16, 0, 0));
      sr = i == 0 ? f[0] : i == 1 ? f[1] : i == 2 ? f[2] : f[3];
    }
  };
  // A dim's place among its quarter's is turned by bits 4 and 5 of the dim, or
  // the stores of dims 16 apart would meet in the same banks.
  auto v_slot = [](int dim) { return dim ^ ((dim >> 4) & 3); };
  auto store_tile = [&] {
#pragma unroll
    for (int j = 0; j < T::KU; j++) {
      const int unit = j * kThreads + tid, key = unit / T::KC, ch = unit % T::KC;
      *(uint4*)(Kp + ch * T::KS + key * 16) = kr[j];
    }
    uint32_t y[T::UV][4];
#pragma unroll
    for (int j = 0; j < T::UV; j++) turn4(vr[j][0], vr[j][1], vr[j][2], vr[j][3], y[j]);
#pragma unroll
    for (int e = 0; e < 4; e++) {
      uint8_t* at = Vp + (vg * HD + v_slot(4 * vt + e)) * 16 + 4 * vu;
      if constexpr (T::UV == 2) {
        *(uint2*)at = make_uint2(y[0][e], y[1][e]);
      } else {
        *(uint32_t*)at = y[0][e];
      }
    }
    if (wave < 2) scales[tid] = sr;
  };

  uint4 qd[ND][kQ];
  if (from < to) {
    pages(from);
    load_tile(from);
    pages(from + KT);
  }
  const QueryFactor factor = query_digits<HD>(qp, 16 * g4, 64, a.scale, qd);
  Sums<HD> sums;
  sums.m = -INFINITY;
  sums.l = 0.0f;
#pragma unroll
  for (int e = 0; e < NE; e++) sums.o[e] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
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
    v4f s[4];
    float4 ks[4], vs[4];
#pragma unroll
    for (int u = 0; u < 4; u++) {
      ks[u] = *(const float4*)&scales[16 * u + 4 * g4];
      vs[u] = *(const float4*)&scales[KT + 16 * u + 4 * g4];
      v4i t[kQ] = {};
#pragma unroll
      for (int d = 0; d < ND; d++) {
        const uint4 kf = *(const uint4*)(Kp + (4 * d + g4) * T::KS + (16 * u + l16) * 16);
#pragma unroll
        for (int k = 0; k < kQ; k++) t[k] = mfma8(kf, qd[d][k], t[k]);
      }
#pragma unroll
      for (int v = 0; v < 4; v++) s[u][v] = of_digits(t[3][v], t[2][v], t[1][v], t[0][v]);
    }
    to_scores(s, factor, ks);
    const bool edge = there != 15u || kt + KT > w.k_hi || __any(see.lo > kt || see.hi < kt + KT);
    auto sees = [&](int u, int v) {
      const int key = kt + 16 * u + 4 * g4 + v;
      return (there >> u & 1) && key >= see.lo && key < see.hi && key < w.k_hi;
    };
    uint32_t pd[3][4];
    const float beta = step_weights<HD>(s, factor.c, vs, edge, sees, sums, pd);
#pragma unroll
    for (int e = 0; e < NE; e++) {
      const uint4 vf = *(const uint4*)(Vp + (g4 * HD + v_slot(16 * e + l16)) * 16);
      v4i t[3];
#pragma unroll
      for (int k = 0; k < 3; k++)
        t[k] = mfma8(vf, make_uint4(pd[k][0], pd[k][1], pd[k][2], pd[k][3]), v4i{0, 0, 0, 0});
#pragma unroll
      for (int v = 0; v < 4; v++)
        sums.o[e][v] = fmaf(of_digits(t[2][v], t[1][v], t[0][v]), beta, sums.o[e][v]);
    }
  }
  if (!live) return;
  const float l = rows4_sum(sums.l);
  const int64_t out_row = row_at(a, w, row);
  if (wave_row + l16 < w.rows) {
#pragma unroll
    for (int e = 0; e < NE; e++)
      write_row4(a, w, out_row, HD, 16 * e + 4 * g4,
                 make_float4(sums.o[e][0], sums.o[e][1], sums.o[e][2], sums.o[e][3]), sums.m, l,
                 g4 == 0);
  }
}

template <int HD>
constexpr int attention_lds() {
  using T = WideTile<HD>;
  constexpr int w = T::kK + T::kV + T::kScales + kWaves * 8;
  return w > kMergeBytes<HD> ? w : kMergeBytes<HD>;
}

template <int HD>
struct Int8Body {
  static constexpr int kKeys = 64;
  static constexpr bool kTogether = HD == 64, kLastFirst = true;
  static __device__ __forceinline__ void wide(const PagedArgs& a, const Item& w, uint8_t* lds) {
    ::wide<HD>(a, w, lds);
  }
  template <bool kJoined>
  static __device__ __forceinline__ void block_of_16(const PagedArgs& a, const Item& w, int,
                                                     uint8_t* lds) {
    narrow<HD, kJoined>(a, w, lds);
  }
};

template <int HD, bool kPacked>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2, 2)))
paged_attention_i8_kernel(PagedArgs a) {
  __shared__ __align__(16) uint8_t lds[attention_lds<HD>()];
  paged_workgroup<Int8Body<HD>, kPacked>(a, lds);
}

}  // namespace

namespace dnx {

PagedKernel paged_attention_i8(int hd, bool packed) {
  if (hd == 128) return packed ? paged_attention_i8_kernel<128, true> : paged_attention_i8_kernel<128, false>;
  return packed ? paged_attention_i8_kernel<64, true> : paged_attention_i8_kernel<64, false>;
}

}  // namespace dnx
