// Which kernel the int8 row product (gemm_i8r.hip) takes for a shape. Host
// code alone, without HIP.
#pragma once

#include <algorithm>
#include <stdint.h>

namespace dnx {

// A tile kernel: its tokens x weight rows, the parts of K that a workgroup's
// wave groups share, and what it costs (us): a launch with prologue and
// epilogue, a stage of 64 of K for a workgroup that has a CU to itself, and
// for each of the workgroups that share one.
struct I8RTile {
  int tokens, rows, parts;
  float fixed, alone, shared;
};

// Fitted to 179 shapes (n 17 .. 2048, rows 512 .. 8192, K 512 .. 4096), timed
// with weights rotated past the L2: the estimates are off by 7 to 10% (rms),
// and the kernel they choose is 0.6% slower than the best of the seven in the
// mean, 17% at worst (48 x 4096 x 4096: 9.2 against 7.8 us). Each is the
// fastest somewhere: e.g. (us, in this order, n x rows x K) 17 x 512 x 4096:
// 6.8 8.1 11.5 - - - -; 128 x 4096 x 2048: - 7.1 8.5 10.4 15.4 15.5 23.1; 256
// x 4096 x 2048: - 10.4 9.0 10.7 15.8 19.4 25.0; 512 x 4096 x 4096: - 27.6
// 20.9 17.5 25.3 31.8 41.7; 2048 x 2048 x 4096: - 73 40.7 31.7 27.4 33.5 41.9;
// 1024 x 8192 x 4096: - 107 79 62 52 45.7 53.4; 2048 x 8192 x 4096: - 288 161
// 122 93 84.5 73.5.
constexpr I8RTile kI8RTiles[] = {
    {32, 32, 4, 3.25f, 0.200f, 0.320f},  {64, 32, 2, 3.50f, 0.148f, 0.216f},
    {64, 64, 1, 3.90f, 0.120f, 0.152f},  {128, 64, 1, 4.20f, 0.175f, 0.217f},
    {128, 128, 1, 5.90f, 0.282f, 0.340f}, {256, 128, 1, 5.70f, 0.351f, 0.569f},
    {256, 256, 1, 7.75f, 0.488f, 0.867f},
};
constexpr int kI8RCount = sizeof(kI8RTiles) / sizeof(kI8RTiles[0]);
constexpr int kI8RFew = -1;

// The index of the tile kernel, or kI8RFew for batches of up to 16 tokens: the
// kernel without LDS for its operands (13 x 1024 x 4096: 6.2 us against 6.8 of
// the smallest tile, 1 x 6144 x 2048 5.5 against 5.8; 16 x 6144 x 2048 6.7
// against 6.0).
inline int i8r_route(int64_t n, int64_t rows, int64_t cols) {
  if (n <= 16) return kI8RFew;
  int best = 0;
  double least = 0.0;
  for (int i = 0; i < kI8RCount; i++) {
    const I8RTile& t = kI8RTiles[i];
    const int64_t tiles = ((n + t.tokens - 1) / t.tokens) * ((rows + t.rows - 1) / t.rows);
    const int64_t stages = ((cols + 63) / 64 + t.parts - 1) / t.parts;
    const double fill = tiles / 256.0;   // workgroups a CU
    const double stage = std::max(t.alone + (t.shared - t.alone) * std::min(1.0, fill),
                                  t.shared * fill);
    const double us = t.fixed + stages * stage;
    if (i == 0 || us < least) {
      best = i;
      least = us;
    }
  }
  return best;
}

}  // namespace dnx
