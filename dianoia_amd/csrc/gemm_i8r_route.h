// Which kernel the int8 row product (gemm_i8r.hip) takes for a shape. Host
// code alone, without HIP.
#pragma once

#include <cmath>
#include <stdint.h>

namespace dnx {

// A tile kernel: its tokens x weight rows, the parts of K that a workgroup's
// wave groups share, and what it costs (us): a launch with prologue and
// epilogue, a stage of 64 of K for a workgroup that has a CU to itself, and
// for each of the workgroups that share one; and how much of a last round of
// workgroups that does not reach all CUs is waited for.
struct I8RTile {
  int tokens, rows, parts;
  float fixed, alone, shared, last;
};

// Fitted to 240 shapes (n 17 .. 2048, rows 512 .. 8192, K 512 .. 4096), timed
// with weights rotated past the L2: the estimates are off by 8 to 12% (rms),
// and the kernel they choose is 1.1% slower than the best of the seven (in two
// or three depths of their rings each) in the mean, 31% at worst (777 x 4304 x
// 4096: 33.3 against 25.5 us). Each is the fastest somewhere (us, in this
// order, n x rows x K): 64 x 512 x 4096 7.4 9.4 12 14 19 - -; 64 x 4304 x 2048
// 8.4 6.9 8.4 9.4 12 - -; 128 x 6144 x 4096 - 21.5 17.0 23.7 28.9 35.3 48; 256
// x 6144 x 4096 - - 27.9 24.0 28.5 43 55; 512 x 8192 x 4096 - - 48.5 40 30.6 44
// 54; 1024 x 6144 x 4096 - - - 57 46.8 40.5 52.7; 2048 x 8192 x 4096 - - - 135
// 92 81 72.6.
constexpr I8RTile kI8RTiles[] = {
    {32, 32, 4, 3.73f, 0.154f, 0.357f, 0.52f},   {64, 32, 2, 3.53f, 0.146f, 0.256f, 0.36f},
    {64, 64, 1, 3.91f, 0.121f, 0.173f, 0.33f},   {128, 64, 1, 4.13f, 0.154f, 0.267f, 0.28f},
    {128, 128, 1, 5.80f, 0.206f, 0.382f, 0.34f}, {256, 128, 1, 6.45f, 0.345f, 0.602f, 0.63f},
    {256, 256, 1, 8.70f, 0.457f, 0.987f, 0.55f},
};
constexpr int kI8RCount = sizeof(kI8RTiles) / sizeof(kI8RTiles[0]);
constexpr int kI8RFew = -1;

// Tiles of 16 weight rows of a workgroup of the few-token kernel. Two read the
// tokens half as often, which counts from about five of them on, but not where
// they leave some CUs more rows than one would (us, one against two: 13 x 6144
// x 2048 5.66 / 5.40, 16 x 128256 x 4096 139 / 128, 4 x 6144 x 2048 5.10 / 5.21,
// 16 x 4096 x 2048 4.10 / 5.15, 16 x 12288 x 4096 16.7 / 17.7).
inline int i8r_few_tiles(int64_t n, int64_t rows) {
  const auto rounds = [&](int64_t wg_rows) { return ((rows + wg_rows - 1) / wg_rows + 255) / 256; };
  return n > 4 && (2 * rounds(32) <= rounds(16) || rows > 32768) ? 2 : 1;
}

// The index of the tile kernel, or kI8RFew for batches of up to 16 tokens: the
// kernel without LDS for its operands (13 x 1024 x 4096: 6.2 us against 6.8 of
// the smallest tile, 1 x 6144 x 2048 5.5 against 5.8; 16 x 6144 x 2048 5.5
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
    const double stage = fill <= 1.0 ? t.alone + (t.shared - t.alone) * fill
                                     : t.shared * (fill + t.last * (std::ceil(fill) - fill));
    const double us = t.fixed + stages * stage;
    if (i == 0 || us < least) {
      best = i;
      least = us;
    }
  }
  return best;
}

}  // namespace dnx
