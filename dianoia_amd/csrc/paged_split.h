// How the paged attention deals its keys to workgroups. Host code alone,
// without HIP.
#pragma once

#include <algorithm>
#include <stdint.h>

namespace dnx {

// A row is one query head of one token. A workgroup takes kRowsBlock rows
// that share a key head, and a run of the prefix's keys (`prefix_run`,
// prefix_splits of them) or of one sequence's own keys (own_run, own_splits).
// The rows' partial results are added by a second launch unless there is one
// run in all.
struct PagedSplit {
  int64_t prefix_rows, own_rows;     // blocks of rows: all tokens', one sequence's
  int64_t prefix_splits, prefix_run;
  int64_t own_splits, own_run;
  int64_t splits() const { return prefix_splits + own_splits; }
};

constexpr int kPagedRows = 16;       // rows of a workgroup
constexpr int kPagedStep = 64;       // keys a workgroup takes at once: 16 a wave
constexpr int kPagedMaxSplits = 32;  // of the prefix, and of a sequence

inline PagedSplit paged_split(int64_t seqs, int64_t tokens, int64_t max_tokens, int64_t group,
                              int64_t kv_heads, int64_t prefix_len, int64_t max_len) {
  auto blocks = [](int64_t rows) { return (rows + kPagedRows - 1) / kPagedRows; };
  PagedSplit s{blocks(tokens * group), blocks(max_tokens * group), 0, kPagedStep, 0, kPagedStep};
  // Runs that make about `target` workgroups, of at least two steps.
  constexpr int64_t target = 512;
  auto deal = [&](int64_t units, int64_t keys, int64_t& splits, int64_t& run) {
    if (keys <= 0 || units <= 0) return;
    const int64_t steps = (keys + kPagedStep - 1) / kPagedStep;
    int64_t want = std::min<int64_t>((target + units - 1) / units, kPagedMaxSplits);
    want = std::max<int64_t>(1, std::min(want, steps / 2));
    const int64_t per = (steps + want - 1) / want;
    run = per * kPagedStep;
    splits = (steps + per - 1) / per;
  };
  deal(kv_heads * s.prefix_rows, prefix_len, s.prefix_splits, s.prefix_run);
  deal(seqs * kv_heads * s.own_rows, max_len, s.own_splits, s.own_run);
  return s;
}

}  // namespace dnx
