// What the attention kernels over the paged cache's types share: how a
// workgroup finds its rows and keys, and what becomes of their sums.
#pragma once

#include "common.h"
#include "paged_split.h"

#include <math.h>

namespace dnx {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr float kSlack = 8.0f;   // of a running maximum, in units of log2

struct PartArgs {
  int wide, few, blocks, runs, keys, together;
};

struct PagedArgs {
  const void *keys, *values;
  int pages, page_bits, row_bytes;   // row_bytes: of all heads of one place
  int kv_heads, heads, group;
  const int32_t *starts, *lens, *tables, *prefix_pages;
  int64_t table_stride;
  int prefix_len, seqs, tokens, max_len;   // max_len: within the tables too
  const float *key_scales, *value_scales;   // of an int8 cache
  const float *q, *gate;
  float *out, *stat, *part;   // partials: stat [rows][splits][2], part [rows][splits][hd]
  int window, splits, joined;
  PartArgs prefix, own;
  int64_t prefix_items;
  uint32_t slots;  // of all sequences' blocks together, or 0
  int combine_x;   // of the second launch's workgroups, whose y counts the rest
  float scale;
};

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

// What a workgroup takes: rows row0 .. of the `rows` of tokens t0 .. that
// share key head kvh, and keys k_lo .. k_hi - 1 of a list of pages. Where the
// prefix is joined to a sequence's own keys, these begin at key `joined`; the
// keys from prefix_len to there do not exist.
struct Item {
  bool own;
  int kvh, run, row0, rows, t0, first;   // first: the place of token t0 among the keys
  int k_lo, k_hi, count, joined;
  int most;                 // of the list's keys, whatever lens says
  int page[4];              // of a wave's first keys in a narrow block, and 16 further, ..
  const int32_t* table;
};

// The output row of row r of an item.
DNX_DEV int64_t row_at(const PagedArgs& a, const Item& w, int r) {
  return (int64_t)(w.t0 + r / a.group) * a.heads + w.kvh * a.group + r % a.group;
}

// The first key under the window of a token that stands at `place`: a place
// before the first key (down to minus the new tokens) sees no less than that
// key's, and one far behind the last (a length past its bound) nothing. In 64
// bits: a place less the widest window, and a prefix's length and any other,
// leave 32. kBehind is behind every key (2^30 of a prefix, 2^30 own).
constexpr int64_t kBehind = 0x7fff0000;
DNX_DEV int window_begin(int64_t place, int window) {
  return (int)min(max(place, (int64_t)0) - window + 1, kBehind);
}

// The keys of an item that its row r sees: lo .. hi - 1.
struct Seen {
  int lo, hi;
};
DNX_DEV Seen row_sees(const PagedArgs& a, const Item& w, int r) {
  const int token = w.t0 + r / a.group;
  if (w.own) {
    const int place = w.first + token - w.t0;
    const int hi = w.joined + min(w.count, max(place + 1, 0));
    if (a.window == 0) return {0, hi};
    if (w.joined == 0) return {window_begin(place, a.window), hi};
    const int lo = window_begin((int64_t)a.prefix_len + place, a.window);
    return {lo < a.prefix_len ? lo : lo - a.prefix_len + w.joined, hi};
  }
  if (a.window == 0) return {0, w.count};
  int lo = 0, hi = a.seqs;              // the token's sequence: starts[lo] <= token < starts[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.starts[mid] <= token) lo = mid; else hi = mid;
  }
  const int64_t place = (int64_t)a.prefix_len + a.lens[lo] - a.starts[lo + 1] + token;
  return {window_begin(place, a.window), w.count};
}

// The page of the 16 keys from kt on, looked up ahead of its use (past the
// list's end its last one) and without a branch or the sequence's length, so
// that no load waits for another.
template <bool kJoined>
DNX_DEV int page_at(const PagedArgs& a, const Item& w, int kt) {
  const bool own = !kJoined || kt >= w.joined;
  const int32_t* table = own ? w.table : a.prefix_pages;
  const int place = own ? min(kJoined ? kt - w.joined : kt, w.most - 1)
                        : min(kt, a.prefix_len - 1);
  // Constant memory to the kernel: a scalar load wherever it stands (behind a
  // store or a barrier the compiler would wait for a vector load instead).
  typedef const __attribute__((address_space(4))) int32_t* Constant;
  return __builtin_amdgcn_readfirstlane(((Constant)(uintptr_t)table)[place >> a.page_bits]);
}
// A row's partial result (or, with one run, its output), EV values from dim
// `dim` on at a time; `stats`: this lane also writes m and l.
DNX_DEV void write_row4(const PagedArgs& a, const Item& w, int64_t row, int hd, int dim, float4 o,
                        float m, float l, bool stats) {
  if (a.splits == 1) {
    const float f = row_scale(l, a.gate, row);
    *(float4*)(a.out + row * hd + dim) = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
  } else {
    const int64_t p = row * a.splits + (w.own ? a.prefix.runs : 0) + w.run;
    *(float4*)(a.part + p * hd + dim) = o;
    if (stats) *(float2*)(a.stat + 2 * p) = make_float2(m, l);
  }
}

// Rows of four waves' sums in LDS: [wave][16][kSumRow] and, behind them, each
// wave's maxima and sums of weights [wave][2][16].
template <int HD>
constexpr int kSumRow = HD + 4;
template <int HD>
DNX_DEV float* wave_stats(uint8_t* lds, int wave) {
  return (float*)lds + kWaves * 16 * kSumRow<HD> + wave * 32;
}

template <int HD>
constexpr int kMergeBytes = kWaves * (16 * kSumRow<HD> + 32) * 4;

// The four waves' sums of the first N rows, added in wave order.
template <int HD, int N>
DNX_DEV void merge_waves(const PagedArgs& a, const Item& w, uint8_t* lds) {
  const float* all = (const float*)lds;
  const float* ml = wave_stats<HD>(lds, 0);
  __syncthreads();
  for (int i = threadIdx.x; i < N * HD / 4; i += kThreads) {
    const int r = i / (HD / 4), c = i % (HD / 4);
    if (w.row0 + r >= w.rows) break;
    float top = -INFINITY, total = 0.0f;
#pragma unroll
    for (int k = 0; k < kWaves; k++) top = fmaxf(top, ml[2 * k * 16 + r]);
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < kWaves; k++) {
      const float l = ml[(2 * k + 1) * 16 + r];
      if (l == 0.0f) continue;
      const float f = partial_factor(ml[2 * k * 16 + r], l, top);
      const float4 y = *(const float4*)&all[(k * 16 + r) * kSumRow<HD> + 4 * c];
      total = fmaf(l, f, total);
      acc = make_float4(fmaf(y.x, f, acc.x), fmaf(y.y, f, acc.y), fmaf(y.z, f, acc.z),
                        fmaf(y.w, f, acc.w));
    }
    write_row4(a, w, row_at(a, w, w.row0 + r), HD, 4 * c, acc, top, total, c == 0);
  }
}

// Whether none of an own block's rows, up to `end`, sees a key of its run: the
// run lies behind the sequence's keys (where the bound on the lengths is far
// above them), or the window or the rows' own places end before it. Such a run
// only says so; its sums are not written. 64 sequences of 200 keys, bound 32768,
// 32 / 8 heads, hd 128, bf16: 65 us without this and with a sequence's runs side
// by side in the launch, 33 with both (13 with the bound at 200).
DNX_DEV bool unseen(const PagedArgs& a, const Item& w, int end) {
  int lo = w.k_lo, hi = w.k_hi;
  if (lo < hi && (a.window > 0 || w.rows > a.group)) {
    if (a.window > 0) lo = max(lo, window_begin(w.first + w.row0 / a.group, a.window));
    hi = min(hi, w.first + (end - 1) / a.group + 1);
  }
  return lo >= hi;
}

// The prefix's workgroups, then the sequences' own: both kinds in one launch,
// so that the matrix cores' work on the prefix runs beside the reading of the
// sequences' keys (64 tokens, 8192 shared keys, 128 to 2048 own, 32 / 8 heads,
// hd 128, bf16: 93 us, alone 41 and 69; the own ones first 100, with 16384
// shared and up to 400 own 78 against 105). Workgroups go round the eight XCDs, each with an L2 of its
// own: the blocks of rows that read the same keys go to one of them.
// kPacked: the own blocks of all sequences lie in a row (paged_fit). A kernel of
// its own: the choice in one kernel cost every call 0.1 us (44 calls, geometric
// mean: 9.11 us against 8.98).
// Body: the blocks of one cache type and head size. kKeys: of a wave's step in a
// block of 16. kTogether: paged_together's order. kLastFirst: a prompt's last rows,
// which see the most keys, begin first (int8, hd 128: 4096 tokens, 32 / 8 heads, 632
// -> 610 us; four prompts of 1024 190 -> 160, sixteen of 512 222 -> 226; 725 tokens of
// 4099 keys, 16 / 8 heads, 111 -> 107).
template <typename Body, bool kPacked>
DNX_DEV void paged_workgroup(const PagedArgs& a, uint8_t* lds) {
  Item w;
  uint32_t id = blockIdx.x;
  w.own = id >= (uint32_t)a.prefix_items;
  if (w.own) id -= (uint32_t)a.prefix_items;
  const PartArgs part = w.own ? a.own : a.prefix;
  const bool packed = kPacked && w.own;   // its blocks lie among all sequences'
  uint32_t unit = id, sets = a.slots;
  int block = 0;
  if (!packed) {
    const uint32_t turn = id / 8;
    unit = turn / (uint32_t)part.blocks * 8 + id % 8;
    block = (int)(turn % (uint32_t)part.blocks);
    if (Body::kLastFirst) block = part.blocks - 1 - block;   // they see the most keys
    sets = w.own ? (uint32_t)a.seqs : 1;
  }
  // The sequences' first runs before their second ones: where the bound on the
  // lengths is far above them, those that have keys start at once.
  uint32_t set = unit / (uint32_t)a.kv_heads;
  w.kvh = (int)(unit % (uint32_t)a.kv_heads);
  if (Body::kTogether && part.together) {   // all heads of a run to one XCD
    set = unit / 8 / (uint32_t)a.kv_heads * 8 + unit % 8;
    w.kvh = (int)(unit / 8 % (uint32_t)a.kv_heads);
  }
  uint32_t b = set % sets;
  w.run = (int)(set / sets);
  if (w.run >= part.runs) return;
  if (packed) {
    const int rows = part.wide ? kPagedWide : kPagedNarrow, slot = (int)b;
    const int live = max(0, min(a.starts[a.seqs], a.tokens));
    b = (uint32_t)paged_sequence(a.starts, a.seqs, live, a.group, rows, slot);
    block = slot - paged_slot(a.starts, (int)b, live, a.group, rows);
    if (block < 0) return;   // before the first sequence's rows
  }
  w.k_lo = w.run * part.keys;
  w.joined = w.own ? a.joined : 0;
  w.table = w.own ? a.tables + b * a.table_stride : a.prefix_pages;
  w.most = w.own ? a.max_len : a.prefix_len;
  // One wait for everything that the first keys' addresses and rows need.
  int all = a.starts[a.seqs], s0 = a.starts[b], s1 = a.starts[b + 1], len = a.lens[b];
  {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int first = w.k_lo + Body::kKeys * wave;
    w.page[0] = page_at<true>(a, w, first);
    w.page[1] = page_at<true>(a, w, first + 16);
    if constexpr (Body::kKeys > 32) {
      w.page[2] = page_at<true>(a, w, first + 32);
      w.page[3] = page_at<true>(a, w, first + 48);
      asm("" : "+s"(w.page[2]), "+s"(w.page[3]));
    }
    asm("" : "+s"(all), "+s"(s0), "+s"(s1), "+s"(len), "+s"(w.page[0]), "+s"(w.page[1]));
  }
  const int live = max(0, min(all, a.tokens));
  w.t0 = w.own ? max(0, min(s0, live)) : 0;
  const int t1 = w.own ? max(w.t0, min(s1, live)) : live;
  w.first = w.own ? len - (t1 - w.t0) : 0;
  w.count = w.own ? max(min(len, a.max_len), 0) : a.prefix_len;
  w.row0 = block * (part.wide ? kPagedWide : kPagedNarrow);
  w.rows = (t1 - w.t0) * a.group;
  if (w.row0 >= w.rows) return;
  w.k_hi = min(w.joined > 0 && w.count == 0 ? a.prefix_len : w.joined + w.count,
               w.k_lo + part.keys);
  const int end = min(w.row0 + (part.wide ? kPagedWide : kPagedNarrow), w.rows);
  if (w.own && a.splits > 1 && unseen(a, w, end)) {
    const int r = w.row0 + threadIdx.x;
    if (r < end) {
      const int64_t p = row_at(a, w, r) * a.splits + a.prefix.runs + w.run;
      *(float2*)(a.stat + 2 * p) = make_float2(-INFINITY, 0.0f);
    }
    return;
  }
  if (part.wide) {
    Body::wide(a, w, lds);
    return;
  }
  if (w.joined > 0) {
    Body::template block_of_16<true>(a, w, part.few, lds);
  } else {
    Body::template block_of_16<false>(a, w, part.few, lds);
  }
}

// The kernel over an int8 cache of that head size.
typedef void (*PagedKernel)(PagedArgs);
PagedKernel paged_attention_i8(int hd, bool packed);

}  // namespace dnx
