// A few rows times a matrix of 4-bit weights with a scale (and possibly a zero point) per group of 32, 64 or 128 along K:
//
//   y[m, n] = sum_g s[g, n] * sum_{k in g} x[m, k] (q[k, n] - z[g, n]) + bias[n]         q, z in 0..15; z = 8 where there are none
//
// Every weight byte is used for a handful of rows, so the product is bound by HBM: half a byte per weight and the scales.
//
// Weights lie in blocks of 16 columns x 128 K, 1 KB each, the blocks of a strip of 16 columns one after the other along K: a wave reads a
// block with one load of 16 bytes per lane.  Lane (c = lane % 16, h = lane / 16) holds column c; its dword t is K 32 t + 8 h .. + 8, the B operand
// of one v_mfma_f32_16x16x32, so that an MFMA stays inside one group whatever the group's size, and a group's scale
// multiplies float32 sums: no weight is ever rounded.  In a dword the code of K 2 i is in bits 4 i, that of K 2 i + 1 in bits 16 + 4 i: a shift and an
// and-or turn a pair into the 16-bit numbers 16 + q (the code is the top of the mantissa).  What is too much, (16 + z) times
// the sum of the group's x, is what the group's accumulators start from; the sums of x come from one more MFMA against
// ones.  (With 128 + q or 1024 + q the shift could go, but the difference would lose four or seven bits of the float32 sums.)
#pragma once
#include "moe_layer.h"

namespace tamd {

constexpr int kMatvecRows = 64;   // rows of a workgroup's tiles: more rows read the weights again

template <int XDT>
struct Int4;
template <>
struct Int4<TAMD_BF16> {
  static constexpr uint32_t kMask = 0x00780078u, kSixteen = 0x41804180u, kOne = 0x3F803F80u;
  static constexpr int kUp = 3;   // place of a code in the mantissa
};
template <>
struct Int4<TAMD_F16> {
  static constexpr uint32_t kMask = 0x03C003C0u, kSixteen = 0x4C004C00u, kOne = 0x3C003C00u;
  static constexpr int kUp = 6;
};

// eight codes -> 16 + q
template <int XDT>
TAMD_DEVICE typename Mma<XDT>::frag_t codes_plus_16(uint32_t d) {
  typedef Int4<XDT> I;
  u32x4_t v;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int by = 4 * i - I::kUp;
    v[i] = ((by < 0 ? d << -by : d >> by) & I::kMask) | I::kSixteen;
  }
  return as_frag<XDT>(v);
}

// MT tiles of 16 rows; PER = groups of a block (4, 2, 1); eight waves split K, U blocks requested together.
template <int XDT, int MT, int PER, bool ZEROS, int U>
__global__ __launch_bounds__(512, MT == 1 ? 4 : 2) void matvec_kernel(tamd_matvec_args a) {
  __shared__ f32x4_t red[8][kWave];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  const uint32_t c = lane & 15, h = lane >> 4;
  const int64_t strip = blockIdx.x;
  const int m0 = blockIdx.y * kMatvecRows, rows = a.M - m0 < kMatvecRows ? a.M - m0 : kMatvecRows;
  const uint32_t K = (uint32_t)a.K, n_kb = (K + 127) / 128;
  const Buffer x((const uint8_t *)a.x + m0 * a.x_stride_m * 2, (int64_t)(rows - 1) * a.x_stride_m * 2 + 2 * (int64_t)K);
  const Buffer codes(a.codes + strip * n_kb * 1024, (int64_t)n_kb * 1024);
  const Buffer scales((const uint8_t *)a.scales + strip * n_kb * (32 * PER), (int64_t)n_kb * (32 * PER));
  const Buffer zeros((const uint8_t *)a.zeros + (ZEROS ? strip * n_kb * (16 * PER) : 0), ZEROS ? (int64_t)n_kb * (16 * PER) : 0);
  const bool scale_f16 = a.scale_dtype == TAMD_F16;
  uint32_t x_row[MT];
  f32x4_t y[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    x_row[t] = 16 * t + (int)c < rows ? (uint32_t)((16 * t + c) * (uint32_t)a.x_stride_m * 2u) + 16u * h : kMoeOob;
    y[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  const u32x4_t ones = {Int4<XDT>::kOne, Int4<XDT>::kOne, Int4<XDT>::kOne, Int4<XDT>::kOne};
  const uint32_t end = n_kb * (uint32_t)(wave + 1) / 8u;
  for (uint32_t kb = n_kb * (uint32_t)wave / 8u; kb < end; kb += U) {
    u32x4_t q[U];
    uint32_t s[U][PER > 2 ? 2 : 1], z[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (kb + i < end) {
        q[i] = codes.template load16<2>(16u * lane, (kb + i) * 1024u);
        if constexpr (PER == 4) {
          const u32x2_t v = scales.load8(8u * c, (kb + i) * 128u);
          s[i][0] = v.x, s[i][1] = v.y;
        } else if constexpr (PER == 2) {
          s[i][0] = scales.load4(4u * c, (kb + i) * 64u);
        } else {
          s[i][0] = scales.load2(2u * c, (kb + i) * 32u);
        }
        if constexpr (ZEROS) {
          if constexpr (PER == 4) z[i] = zeros.load4(4u * c, (kb + i) * 64u);
          else if constexpr (PER == 2) z[i] = zeros.load2(2u * c, (kb + i) * 32u);
          else z[i] = zeros.load1(c, (kb + i) * 16u);
        }
      }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      u32x4_t xr[U][4];
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (kb + i < end) {
#pragma unroll
          for (int j = 0; j < 4; ++j) xr[i][j] = x.load16(128u * (kb + i) + 32u * j < K ? x_row[t] + 256u * (kb + i) + 64u * j : kMoeOob);
        }
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (kb + i < end) {
#pragma unroll
          for (int g = 0; g < PER; ++g) {
            const uint32_t bits = s[i][g / 2] >> (16 * (g & 1)) & 0xFFFFu;
            const float scale = scale_f16 ? f16_bits_to_f32(bits) : bf16_bits_to_f32(bits);
            const float offset = ZEROS ? -16.f - (float)(z[i] >> (8 * g) & 0xFFu) : -24.f;
            f32x4_t of_x = {0.f, 0.f, 0.f, 0.f}, p;
#pragma unroll
            for (int j = 0; j < 4 / PER; ++j) of_x = Mma16<XDT>::mma(as_frag<XDT>(xr[i][g * (4 / PER) + j]), as_frag<XDT>(ones), of_x);
#pragma unroll
            for (int v = 0; v < 4; ++v) p[v] = offset * of_x[v];
#pragma unroll
            for (int j = 0; j < 4 / PER; ++j)
              p = Mma16<XDT>::mma(as_frag<XDT>(xr[i][g * (4 / PER) + j]), codes_plus_16<XDT>(q[i][g * (4 / PER) + j]), p);
#pragma unroll
            for (int v = 0; v < 4; ++v) y[t][v] = __builtin_fmaf(scale, p[v], y[t][v]);
          }
        }
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    red[wave][lane] = y[t];
    sync_threads();
    const int m = tid >> 4, col = tid & 15;
    const int64_t n = 16 * strip + col;
    if (m < 16 && 16 * t + m < rows && n < a.N) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) v += ((const float *)&red[w][(m >> 2) * 16 + col])[m & 3];
      if (a.bias) v += load_any_f32(a.bias, a.bias_dtype, n);
      store_any(a.y, a.y_dtype, (m0 + 16 * t + m) * a.y_stride_m + n, v);
    }
    sync_threads();
  }
}

template <int XDT, int PER, bool ZEROS>
int launch_matvec(const tamd_matvec_args &a, hipStream_t st) {
  const dim3 grid((unsigned)((a.N + 15) / 16), (unsigned)((a.M + kMatvecRows - 1) / kMatvecRows));
  if (a.M <= 16) matvec_kernel<XDT, 1, PER, ZEROS, 4><<<grid, 512, 0, st>>>(a);
  else if (a.M <= 32) matvec_kernel<XDT, 2, PER, ZEROS, 4><<<grid, 512, 0, st>>>(a);
  else matvec_kernel<XDT, 4, PER, ZEROS, 2><<<grid, 512, 0, st>>>(a);
  return launch_status();
}

template <int XDT>
int matvec_of(const tamd_matvec_args &a, hipStream_t st) {
  if (a.zeros) return a.group == 32 ? launch_matvec<XDT, 4, true>(a, st) : a.group == 64 ? launch_matvec<XDT, 2, true>(a, st) : launch_matvec<XDT, 1, true>(a, st);
  return a.group == 32 ? launch_matvec<XDT, 4, false>(a, st) : a.group == 64 ? launch_matvec<XDT, 2, false>(a, st) : launch_matvec<XDT, 1, false>(a, st);
}

int matvec_bf16(const tamd_matvec_args &a, hipStream_t st);
int matvec_f16(const tamd_matvec_args &a, hipStream_t st);

}  // namespace tamd
