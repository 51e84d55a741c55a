// Values as int8 codes of a scale: code = 127 y / top rounded to the nearest
// whole number, halves away from zero, formed in 64 bits.
#pragma once

#include "common.h"

namespace dnx {

template <int Ctrl>
DNX_DEV double dpp64(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint64_t lo = (uint32_t)dpp<Ctrl>((int)(uint32_t)b), hi = (uint32_t)dpp<Ctrl>((int)(b >> 32));
  return __builtin_bit_cast(double, hi << 32 | lo);
}

// One code: the nearest whole number to y * inv, halves away from zero.
DNX_DEV int code1(double y, double inv) {
  const double t = y * inv;
  return (int)(t + __builtin_copysign(0.5, t));
}

DNX_DEV int pack4(int a, int b, int c, int d) {
  return (a & 0xff) | ((b & 0xff) << 8) | ((c & 0xff) << 16) | (int)((uint32_t)d << 24);
}

// 127 / top, rounded up by 2^-50.
DNX_DEV double code_factor(double top, bool fine) {
  return fine && top > 0.0 ? 127.0 / top * (1.0 + 0x1p-50) : 0.0;
}

}  // namespace dnx
