// How the paged attention deals rows and keys to workgroups. Without HIP: host
// code, and (constexpr) how a workgroup finds its sequence.
#pragma once

#include <algorithm>
#include <stdint.h>

namespace dnx {

// A row is one query head of one token. A workgroup takes a block of rows that
// share a key head and a run of keys: of the prefix (all tokens' rows), or of
// one sequence's own keys (that sequence's rows). `wide` blocks hold 64 rows,
// 16 a wave, whose waves share the keys' tiles; the others 16 rows, of which
// each wave takes other keys. The rows' partial results are added by a second
// launch unless there is one run in all.
// `few`: 2 or 4 where a block of a float32 cache holds one token's rows, at
// most that many (a kernel of their own), else 0.
struct PagedPart {
  bool wide;
  int few;
  bool together;                // all key heads of a run to one XCD (paged_together)
  int64_t blocks, runs, keys;   // blocks of rows, runs of that many keys
};
// `joined` (a multiple of kPagedStep): the prefix is walked with each
// sequence's own keys in one run, in which the own keys begin at that place.
// `slots`: 0 where each sequence has own.blocks blocks, else the blocks of all
// sequences together (paged_slot).
struct PagedSplit {
  PagedPart prefix, own;
  int64_t joined, slots;
  int64_t prefix_items, own_items;   // workgroups of the launch
  int64_t splits() const { return prefix.runs + own.runs; }
};

constexpr int kPagedNarrow = 16, kPagedWide = 64;   // rows of a workgroup
constexpr int kPagedStep = 64;       // runs are whole steps
// Runs of the prefix, and of a sequence: up to 32, and more (256 in all) where
// they hold 128 keys each and the call has few rows (whose partial results are
// then added by four waves each). One token after 131072 keys, 8 heads over
// one, hd 128, bf16: 45 us with 32 runs, 19 with 128 or 256; f32 147, 46, 34.
// (At least 256 keys each: 8192 keys of one key head, f32, 14.3 us against 11.4,
// bf16 9.1 against 8.5, but 32768 keys 11.0 against 11.7.)
constexpr int kPagedRuns = 32, kPagedMaxRuns = 256, kPagedLong = 128;
constexpr int64_t kPagedManyRows = 1 << 20;
constexpr int64_t kPagedItems = 0xffffffff / 256;   // workgroups that a launch may have

// Wide blocks read the keys for 64 rows at once and take fewer products, but
// one after another; narrow ones of the same rows run side by side and find
// the keys in the L2. So narrow up to 32 rows, and up to 128 where the whole
// is small (us, narrow against wide; 32 query heads over 8 key heads, hd 128):
// f32 64 rows x 512 keys 11.6 / 13.4, 64 x 2048 18.3 / 17.7, 64 x 8192 39.6 /
// 30.9, 128 x 512 13.7 / 15.4, 128 x 2048 25 / 22; bf16 (whose narrow blocks
// take the bf16 matrix cores too) 64 x 8192 19.9 / 21, 128 x 2048 14.9 / 15.9,
// 128 x 8192 28.2 / 28.4.
inline bool paged_wide(int64_t rows, int64_t units, int64_t keys, bool f32) {
  if (rows <= 32) return false;
  return rows > 128 || rows * keys * units > (f32 ? 1200000 : 4000000);
}

// int8: a wide block takes the keys' products for 64 rows one step after another,
// with two barriers each; narrow ones have no barrier in a step, but join four
// waves' sums for every 16 rows. So wide where all rows together fill the card with
// them and the keys are no more than they are: there what a narrow block costs
// besides its steps is felt. (All rows, not the bound on a sequence's: 64 sequences,
// one of 20 new tokens and the others of one, 200 keys, 8 / 2 heads, hd 128, 9.5 us
// narrow, 15.3 wide.) And wide on a prefix of up to four key heads that narrow blocks
// would read in as many runs, of one XCD each. us, narrow / wide, 32 / 8 heads, hd
// 128: 1 sequence of 64 new tokens and 256 keys 9.9 / 19.7, 1 of 512 and 2048 keys 67 /
// 113 (16 / 8: 36 / 67), 1 of 2048 and 2048 161 / 145, 16 of 256 and 256 139 / 76, 64
// of 64 and 64 115 / 49, of 64 and 1024 324 / 321; 256 tokens over 1000 shared keys 55
// / 57, 512 over 16384 on 8 heads over one 834 / 275, 128 68 / 67. At hd 64, 12 / 4:
// 16 of 64 and 64 11.7 / 8.7, 1 of 1024 and 16384 266 / 334. (544 calls, geometric mean:
// narrow alone 43.9 us, wide alone 50.5, bf16's rule 49.1, this one 40.9, the better
// of both 40.8; 128 or 256 workgroups at least 41.0.)
// rows: of a unit; all: of a key head in all sequences.
inline bool paged_wide_i8(int64_t rows, int64_t all, int64_t kv_heads, int64_t keys, bool prefix) {
  if (rows <= 32) return false;
  return kv_heads * ((all + kPagedWide - 1) / kPagedWide) >= std::max<int64_t>(192, keys) ||
         (prefix && kv_heads <= 4 && rows >= 1024);
}

// At most that many runs of whole steps.
inline void paged_deal(PagedPart& p, int64_t keys, int64_t runs) {
  p.keys = ((keys + runs - 1) / runs + kPagedStep - 1) / kPagedStep * kPagedStep;
  p.runs = (keys + p.keys - 1) / p.keys;
}

// The workgroups of a part: for each unit (a key head, of a sequence) its runs
// and blocks, in whole rounds of the eight XCDs.
inline int64_t paged_items(const PagedPart& p, int64_t units) {
  return (units * p.runs + 7) / 8 * 8 * p.blocks;
}

inline PagedPart paged_part(int64_t tokens, int64_t group, int64_t units, int64_t keys, bool wide,
                            bool f32, int64_t least, int64_t most, int64_t max_runs) {
  PagedPart p{};
  const int64_t rows = tokens * group;
  p.wide = wide;
  p.few = !f32 || tokens > 1 || rows > 4 ? 0 : rows <= 2 ? 2 : 4;
  const int64_t block = p.wide ? kPagedWide : kPagedNarrow;
  p.blocks = (rows + block - 1) / block;
  p.keys = kPagedStep;
  if (keys <= 0 || units <= 0 || rows <= 0) return p;
  // Runs that make about 256 workgroups, of `least` to `most` keys (49 calls,
  // geometric mean: 13.7 us; with 192 or 384 workgroups 13.9 and 14.0, with 128
  // keys at least 14.1; int8, 44 calls: 10.7, with 192 10.8, 384 and 512 10.9).
  const int64_t wgs = units * p.blocks;
  int64_t runs = (256 + wgs - 1) / wgs;
  runs = std::min(std::max(runs, (keys + most - 1) / most), std::max<int64_t>(1, keys / least));
  runs = std::min(runs, std::max<int64_t>(kPagedRuns, keys / kPagedLong));
  runs = std::min<int64_t>(std::max<int64_t>(runs, 1), max_runs);
  paged_deal(p, keys, runs);
  return p;
}

// The blocks of all sequences in a row: sequence b's begin at this place. It
// has floor((s + n) / block) - floor(s / block) + 1 places for its n rows from
// s on, at least ceil(n / block), and all sequences together have
// floor(tokens * group / block) + seqs, however the tokens lie.
constexpr int paged_slot(const int32_t* starts, int b, int live, int group, int block) {
  const int64_t s = starts[b] < 0 ? 0 : starts[b] > live ? live : starts[b];
  return (int)(s * group / block) + b;
}

// The sequence whose blocks hold place `slot`: the last that begins at or
// before it.
constexpr int paged_sequence(const int32_t* starts, int seqs, int live, int group, int block,
                             int slot) {
  int lo = 0, hi = seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (paged_slot(starts, mid, live, group, block) <= slot) lo = mid; else hi = mid;
  }
  return lo;
}

// Bounds may lie far above what a batch holds: each of many sequences might
// have max_tokens new ones, of which there are `tokens` in all. Where a place for
// every block of every sequence, in rounds of the XCDs, makes kPagedEmpty more
// workgroups than all sequences' blocks in a row, they lie in a row: to find its
// sequence takes a workgroup up to 0.7 us, but full workgroups wait behind empty
// ones (us, a place for every block against a row; bf16, 32 / 8 heads, hd 128:
// 24 sequences of up to 48 tokens, one each, 250 keys, 360 more, 13.5 / 14.1;
// 24 of up to 16, 240 keys, 528 more, 16.8 / 9.4; 64 of up to 512, one of 512
// among them, 1000 keys, 15592 more, 132 / 60; one prompt of 2048 tokens on
// 8 heads over one, whose blocks a place each puts on one XCD, 213 / 69).
// Runs become longer where a launch may not have as many workgroups. What still
// does not fit has more than 2^22 key heads of sequences.
constexpr int64_t kPagedEmpty = 512;

inline void paged_fit(PagedSplit& s, int64_t seqs, int64_t tokens, int64_t group,
                      int64_t kv_heads, int64_t prefix_len, int64_t max_len) {
  const int64_t units = seqs * kv_heads;
  const int64_t row = kv_heads * (tokens * group / (s.own.wide ? kPagedWide : kPagedNarrow) + seqs);
  const auto own_items = [&] { return s.slots > 0 ? row * s.own.runs : paged_items(s.own, units); };
  if (paged_items(s.own, units) - row * s.own.runs >= kPagedEmpty) s.slots = row / kv_heads;
  s.prefix_items = paged_items(s.prefix, kv_heads);
  s.own_items = own_items();
  if (s.prefix_items + s.own_items <= kPagedItems) return;
  const auto longer = [](PagedPart& p, int64_t keys, int64_t runs) {
    if (p.runs > std::max<int64_t>(runs, 1)) paged_deal(p, keys, std::max<int64_t>(runs, 1));
  };
  longer(s.prefix, prefix_len, kPagedItems / 2 / s.prefix.blocks / 8 * 8 / kv_heads);
  s.prefix_items = paged_items(s.prefix, kv_heads);
  const int64_t left = kPagedItems - s.prefix_items;
  if (s.own_items > left) {
    if (row < (units + 7) / 8 * 8 * s.own.blocks) s.slots = row / kv_heads;
    longer(s.own, max_len, s.slots > 0 ? left / row : left / s.own.blocks / 8 * 8 / units);
    s.own_items = own_items();
  }
}

// int8 at head size 64: a line of the cache holds two heads. Where the runs are
// whole rounds of the XCDs, or many, all heads of one go to the same XCD: the
// workgroups that this takes, or 0.
inline int64_t paged_together(int64_t sets, int64_t kv_heads, int64_t blocks) {
  return sets > 0 && (sets % 8 == 0 || sets >= 64) ? (sets + 7) / 8 * 8 * kv_heads * blocks : 0;
}

// i8: the head size of an int8 cache, else 0.
inline PagedSplit paged_split(int64_t seqs, int64_t tokens, int64_t max_tokens, int64_t group,
                              int64_t kv_heads, int64_t prefix_len, int64_t max_len, bool f32,
                              int i8 = 0) {
  // Without a prefix, keys that one workgroup walks in about the time of the
  // second launch (3 us) stay in one run: up to 256 (int8, 63 calls of up to 512
  // keys, geometric mean: 8.2 us; up to 64 9.0, 128 8.7, 384 and 512 8.3).
  const int64_t least = prefix_len == 0 && max_len <= 256 ? 256 : kPagedStep;
  const int64_t max_runs = tokens * group * kv_heads >= kPagedManyRows ? kPagedRuns
                           : prefix_len > 0 ? kPagedMaxRuns / 2 : kPagedMaxRuns;
  const int64_t rows = tokens * group, own_rows = max_tokens * group;
  const bool own_wide = i8 > 0 ? paged_wide_i8(own_rows, rows, kv_heads, max_len, false)
                               : paged_wide(own_rows, seqs * kv_heads, max_len, f32);
  const bool prefix_wide = i8 > 0 ? paged_wide_i8(rows, rows, kv_heads, prefix_len, true)
                                  : paged_wide(rows, kv_heads, prefix_len, f32);
  const PagedPart own =
      paged_part(max_tokens, group, seqs * kv_heads, max_len, own_wide, f32, least, 2048, max_runs);
  PagedSplit s{paged_part(tokens, group, kv_heads, prefix_len, prefix_wide, f32, kPagedStep, 1 << 20,
                          max_runs),
               own, 0, 0, 0, 0};
  // A short prefix is joined to them where a CU for each workgroup is left: its
  // keys are then read once for each block of rows, but without the second
  // launch. Up to 384 keys, or 256 where the float32 matrix cores take 16 rows
  // (us, apart against joined: 1 sequence of 83 keys after 238, f32 hd 64, 8.1 /
  // 6.8; 31 tokens each of 6 after 235, bf16 hd 128, 11.9 / 8.8; 6 tokens each of
  // 12 after 276, f32 hd 128, 11.3 / 15.4; limits of 512 keys change nothing). int8,
  // 216 calls, geometric mean: apart 9.6, up to 256 keys 8.6, up to 384 8.6 (hd 128, 32
  // sequences of 60 keys after 250, 32 / 8 heads, 12.5 / 11.5, one of them 10.1 / 10.9).
  const auto steps = [](int64_t keys) { return (keys + kPagedStep - 1) / kPagedStep * kPagedStep; };
  const int64_t joined = steps(prefix_len), keys = joined + steps(max_len);
  if (joined > 0 && s.own.runs > 0 && !s.own.wide && keys <= (f32 && s.own.few == 0 ? 256 : 384) &&
      seqs * kv_heads * s.own.blocks <= 256) {
    s.joined = joined;
    s.own.runs = 1;
    s.own.keys = keys;
    s.prefix.runs = 0;
  }
  paged_fit(s, seqs, tokens, group, kv_heads, prefix_len, max_len);
  if (i8 == 64) {
    const int64_t prefix = paged_together(s.prefix.runs, kv_heads, s.prefix.blocks);
    if (prefix > 0 && prefix + s.own_items <= kPagedItems) {
      s.prefix.together = true;
      s.prefix_items = prefix;
    }
    const int64_t own = paged_together((s.slots > 0 ? s.slots : seqs) * s.own.runs, kv_heads,
                                       s.slots > 0 ? 1 : s.own.blocks);
    if (own > 0 && s.prefix_items + own <= kPagedItems) {
      s.own.together = true;
      s.own_items = own;
    }
  }
  return s;
}

}  // namespace dnx
