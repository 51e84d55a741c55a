// Floats as sums of bf16 pieces for the bf16 matrix cores, and the reductions
// over the four rows of 16 lanes that the attention kernels use.
#pragma once

#include "common.h"

namespace dnx {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));

// Max / sum over lanes i, i ^ 16, i ^ 32 and i ^ 48 (lane i % 16 of the four
// 16-lane rows), every lane getting the result, on gfx950's VALU lane swaps:
// with both operands v, permlane16_swap pairs each lane with lane ^ 16 and
// permlane32_swap with lane ^ 32. No LDS round trip.
DNX_DEV float rows4_max(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

DNX_DEV float rows4_sum(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Eight floats as three bf16 fragments (piece i of value j in element j),
// each piece the rest rounded to nearest: the terms that are not formed are
// then as often too small as too large. An infinity, a NaN and a float that
// rounds to an infinity have NaN among their pieces.
DNX_DEV void split_pieces(const float* x, uint4* p) {
  uint32_t w[3][4];
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    f32x2 v = {x[j], x[j + 1]};
#pragma unroll
    for (int i = 0; i < 3; i++) {
      w[i][j / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf2));
      if (i == 2) break;
      v.x -= __uint_as_float(w[i][j / 2] << 16);
      v.y -= __uint_as_float(w[i][j / 2] & 0xffff0000u);
    }
  }
#pragma unroll
  for (int i = 0; i < 3; i++) p[i] = make_uint4(w[i][0], w[i][1], w[i][2], w[i][3]);
}

}  // namespace dnx
