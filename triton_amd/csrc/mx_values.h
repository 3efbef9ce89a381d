// Groups of 32 microscaled values: their scale, their 8-bit codes, and where a group lies.
#pragma once
#include "common.h"

namespace tamd {

// Value kinds of a microscaled tensor: e2m1 codes (two per byte), or fp8 bytes.  Largest magnitude and
// largest power of two of each (mxfp.py:206-209, mxfp_details/_downcast_to_mxfp.py:24-31).
constexpr int QK_E2M1 = 0, QK_E4M3 = 1, QK_E5M2 = 2;
template <int QK>
constexpr float kMaxQ = QK == QK_E2M1 ? 6.0f : (QK == QK_E4M3 ? 448.0f : 57344.0f);
template <int QK>
constexpr float kInvPow2Q = QK == QK_E2M1 ? 0.25f : (QK == QK_E4M3 ? 1.0f / 256.0f : 1.0f / 32768.0f);

// e8m0 byte of a group with the largest magnitude gmax.
template <int QK>
TAMD_DEVICE uint32_t group_scale_byte(float gmax, int mode) {
  constexpr int DT = QK == QK_E2M1 ? TAMD_MXFP4 : (QK == QK_E4M3 ? TAMD_FP8_E4M3 : TAMD_FP8_E5M2);
  return mode == TAMD_ROUND_UP ? ceil_scale_byte<DT>(gmax) : f32_to_bits(gmax * kInvPow2Q<QK>) >> 23;
}
// 1 / 2^(e-127): 2^(127-e), of which the one for e = 254 is a subnormal; 0 for e = 0 (an empty group) and for infinity
TAMD_DEVICE float scale_reciprocal(uint32_t e) {
  return bits_to_f32(e == 0u || e == 255u ? 0u : (e == 254u ? 0x00400000u : (254u - e) << 23));
}
// Returns the multiplier 1/scale and writes the e8m0 byte.
template <int QK = QK_E2M1>
TAMD_DEVICE float group_scale(float gmax, int mode, uint32_t &scale_byte) {
  scale_byte = group_scale_byte<QK>(gmax, mode);
  return scale_reciprocal(scale_byte);
}

// q (already multiplied by 1/scale) -> fp8 byte: clamp to the finite range, round to nearest even (mxfp.py:313-316)
template <int QK>
TAMD_DEVICE uint32_t fp8_code(float q) {
  if (q != q) return 0x7Fu;
  const float c = __builtin_fminf(__builtin_fmaxf(q, -kMaxQ<QK>), kMaxQ<QK>);
  if constexpr (QK == QK_E4M3) return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, c, 0, false) & 0xFFu;
  return (uint32_t)__builtin_amdgcn_cvt_pk_bf8_f32(c, c, 0, false) & 0xFFu;
}
template <int QK>
TAMD_DEVICE float fp8_value(uint32_t byte) {
  if constexpr (QK == QK_E4M3) return __builtin_amdgcn_cvt_f32_fp8((int)byte, 0);
  return __builtin_amdgcn_cvt_f32_bf8((int)byte, 0);
}

// Division of an index below 2^31 by a divisor fixed for the launch: q = (mulhi(n, mul) + n) >> shift (Granlund and
// Montgomery, "Division by invariant integers using multiplication").  The row kernels below have 16 bytes of work per
// thread, and the two 64-bit divisions that placed a group were most of their instructions.
struct FastDiv {
  uint32_t d, mul, shift;
};
inline FastDiv fast_div(int64_t d) {
  if (d < 1 || d >= ((int64_t)1 << 31)) return FastDiv{0, 0, 0};   // (not used: the launch takes 64-bit divisions)
  uint32_t sh = 0;
  while (((uint64_t)1 << sh) < (uint64_t)d) ++sh;
  return FastDiv{(uint32_t)d, (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << sh) - (uint64_t)d)) / (uint64_t)d + 1), sh};
}
TAMD_DEVICE uint32_t div_by(uint32_t n, const FastDiv &f) { return (__umulhi(n, f.mul) + n) >> f.shift; }

// Where group number `gid` of `total` lies: (batch entry, row, group of the row).
struct GroupDiv {
  int64_t total, G, nr;
  FastDiv by_g, by_nr;
  int wide;    // 2^31 groups or more
};
inline GroupDiv group_div(int64_t nb, int64_t nr, int64_t G) {
  const int64_t total = nb * nr * G;
  return GroupDiv{total, G, nr, fast_div(G), fast_div(nr), total >= ((int64_t)1 << 31)};
}
TAMD_DEVICE void place_group(const GroupDiv &d, int64_t gid, int64_t &b, int64_t &r, int64_t &g) {
  if (d.wide) {
    const int64_t run = gid / d.G;
    g = gid - run * d.G;
    b = run / d.nr;
    r = run - b * d.nr;
  } else {
    const uint32_t run = div_by((uint32_t)gid, d.by_g);
    g = (uint32_t)gid - run * d.by_g.d;
    const uint32_t bb = div_by(run, d.by_nr);
    b = bb;
    r = run - bb * d.by_nr.d;
  }
}

}  // namespace tamd
