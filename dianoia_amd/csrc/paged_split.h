// How the paged attention deals rows and keys to workgroups. Host code alone,
// without HIP.
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
  int64_t blocks, runs, keys;   // blocks of rows, runs of that many keys
};
// `joined` (a multiple of kPagedStep): the prefix is walked with each
// sequence's own keys in one run, in which the own keys begin at that place.
struct PagedSplit {
  PagedPart prefix, own;
  int64_t joined;
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

inline PagedPart paged_part(int64_t tokens, int64_t group, int64_t units, int64_t keys, bool f32,
                            int64_t least, int64_t most, int64_t max_runs) {
  PagedPart p{};
  const int64_t rows = tokens * group;
  p.wide = paged_wide(rows, units, keys, f32);
  p.few = !f32 || tokens > 1 || rows > 4 ? 0 : rows <= 2 ? 2 : 4;
  const int64_t block = p.wide ? kPagedWide : kPagedNarrow;
  p.blocks = (rows + block - 1) / block;
  p.keys = kPagedStep;
  if (keys <= 0 || units <= 0 || rows <= 0) return p;
  // Runs that make about 256 workgroups, of `least` to `most` keys (49 calls,
  // geometric mean: 13.7 us; with 192 or 384 workgroups 13.9 and 14.0, with 128
  // keys at least 14.1).
  const int64_t wgs = units * p.blocks;
  int64_t runs = (256 + wgs - 1) / wgs;
  runs = std::min(std::max(runs, (keys + most - 1) / most), std::max<int64_t>(1, keys / least));
  runs = std::min(runs, std::max<int64_t>(kPagedRuns, keys / kPagedLong));
  runs = std::min<int64_t>(std::max<int64_t>(runs, 1), max_runs);
  p.keys = ((keys + runs - 1) / runs + kPagedStep - 1) / kPagedStep * kPagedStep;
  p.runs = (keys + p.keys - 1) / p.keys;
  return p;
}

inline PagedSplit paged_split(int64_t seqs, int64_t tokens, int64_t max_tokens, int64_t group,
                              int64_t kv_heads, int64_t prefix_len, int64_t max_len, bool f32) {
  // Without a prefix, keys that one workgroup walks in about the time of the
  // second launch (3 us) stay in one run: up to 256.
  const int64_t least = prefix_len == 0 && max_len <= 256 ? 256 : kPagedStep;
  const int64_t max_runs = tokens * group * kv_heads >= kPagedManyRows ? kPagedRuns
                           : prefix_len > 0 ? kPagedMaxRuns / 2 : kPagedMaxRuns;
  PagedSplit s{paged_part(tokens, group, kv_heads, prefix_len, f32, kPagedStep, 1 << 20, max_runs),
               paged_part(max_tokens, group, seqs * kv_heads, max_len, f32, least, 2048, max_runs), 0};
  // A short prefix is joined to them where a CU for each workgroup is left: its
  // keys are then read once for each block of rows, but without the second
  // launch. Up to 384 keys, or 256 where the float32 matrix cores take 16 rows
  // (us, apart against joined: 1 sequence of 83 keys after 238, f32 hd 64, 8.1 /
  // 6.8; 31 tokens each of 6 after 235, bf16 hd 128, 11.9 / 8.8; 6 tokens each of
  // 12 after 276, f32 hd 128, 11.3 / 15.4; limits of 512 keys change nothing).
  const auto steps = [](int64_t keys) { return (keys + kPagedStep - 1) / kPagedStep * kPagedStep; };
  const int64_t joined = steps(prefix_len), keys = joined + steps(max_len);
  if (joined > 0 && s.own.runs > 0 && !s.own.wide && keys <= (f32 && s.own.few == 0 ? 256 : 384) &&
      seqs * kv_heads * s.own.blocks <= 256) {
    s.joined = joined;
    s.own.runs = 1;
    s.own.keys = keys;
    s.prefix.runs = 0;
  }
  return s;
}

}  // namespace dnx
