// Weights of logits as whole numbers, for sampling.hip; host code can include it too, which is how its arithmetic is tested without a GPU.
//
// w = 2^-y, y >= 0, is held as the nearest whole number of units of 2^-fraction, 2^fraction * V < 2^62, so that sums do not depend on their
// order.  A weight is off by half a unit and 2^-38 of itself at most, what rounds to zero included, so the sum of n logits by n / 2 units
// and 2^-38 of itself: of 131072 logits 2^-28 of the largest weight, of 2^20 2^-22.  That is with every rounding to one side;
// as they fall, sums of 2^20 normally distributed logits are off by some 2^10 units.  (Cut off instead of rounded all of them were too small, by
// 2^19 units there, and about one row in a thousand got a neighbour of its token.)
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#define TAMD_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define TAMD_HOST_DEVICE inline
#endif

namespace tamd {

// Bits of a weight of one: a row's weights together stay below 2^62, one below 2^52.
TAMD_HOST_DEVICE int fraction_bits(int V) {
  const int b = 62 - (32 - __builtin_clz((uint32_t)V));
  return b < 51 ? b : 51;
}

// 2^(fraction - y) to the nearest whole number, of y < fraction + 1 (of another: any number).  powers[j] = 2^(fraction - j / 256).  y in units of 2^-40
// (the low bits of y + 1.5 * 2^12) is a whole number of its own, eight bits for the table and the rest r for the series of 2^-r, whose
// first four terms leave 2.3e-12 of w; adding 2^52 rounds the product.  (With exp() and conversions this took longer than reading the
// logits.  Fused by hand: the histogram and the candidates have to agree to the last unit in every kernel.)
TAMD_HOST_DEVICE uint64_t weight_units(double y, const double *powers) {
#ifdef __clang__
#pragma clang fp contract(off)
#endif
  const uint64_t fixed = __builtin_bit_cast(uint64_t, y + 6144.0);   // 6144 = 1.5 * 2^12: the lowest bit is 2^-40
  const uint32_t high = (uint32_t)(fixed >> 32);
  const double r = (double)(uint32_t)fixed * (0.6931471805599453 * 0x1p-40);
  double p = __builtin_fma(r, -1.0 / 6.0, 0.5);
  p = __builtin_fma(r, p, -1.0);
  p = __builtin_fma(r, p, 1.0);
  // (the whole part of y, six bits, is taken from the power's exponent)
  const uint64_t power = __builtin_bit_cast(uint64_t, powers[high & 0xFFu]) - ((uint64_t)(high << 12 & 0x03F00000u) << 32);
  const double x = __builtin_fma(__builtin_bit_cast(double, power), p, 0x1p52);
  return __builtin_bit_cast(uint64_t, x) & 0xFFFFFFFFFFFFFull;
}

}  // namespace tamd
