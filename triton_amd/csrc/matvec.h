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
//
// With bf16 rows all of these numbers, and the ones, are 2^-12 of that, and the result is 2^12 times the sums: 128 values of up to 2^128 times up to
// 31 stay within float32, so every finite row has finite sums before its scales come in.  (Without it one x from 1e37 on, or a
// group of one sign from 1e35 on, made a row infinite or NaN.  At the other end the matrix unit keeps subnormal numbers: products are exact down to
// bf16's smallest, and sums of 2^-149 steps leave results to a multiple of 2^-137.)
#pragma once
#include "moe_layer.h"

namespace tamd {

constexpr int kMatvecRows = 64;   // rows that are addressed together

template <int XDT>
struct Int4;
template <>
struct Int4<TAMD_BF16> {
  static constexpr uint32_t kMask = 0x00780078u, kSixteen = 0x3B803B80u, kOne = 0x39803980u;   // 16 and 1 times 2^-12
  static constexpr float kTimes = 0x1p12f;   // what the sums are multiplied by at last
  static constexpr int kUp = 3;   // place of a code in the mantissa
};
template <>
struct Int4<TAMD_F16> {
  static constexpr uint32_t kMask = 0x03C003C0u, kSixteen = 0x4C004C00u, kOne = 0x3C003C00u;
  static constexpr float kTimes = 1.f;
  static constexpr int kUp = 6;
};

// eight codes -> 16 + q, over kTimes
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

// Where the blocks of a wave lie in K: n of the n_kb blocks from kb0 on, an eighth of them.
struct MatvecPart {
  uint32_t kb0, n;
  TAMD_DEVICE MatvecPart(uint32_t n_kb, uint32_t wave) : kb0(n_kb * wave / 8u), n(n_kb * (wave + 1u) / 8u - kb0) {}
};

// A strip's sums over the eight waves: row m of a tile, column `col`, from the waves' accumulators of that tile.
template <int XDT>
TAMD_DEVICE float matvec_sum(const f32x4_t (*red)[kWave], int m, int col) {
  float v = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) v += ((const float *)&red[w][(m >> 2) * 16 + col])[m & 3];
  return Int4<XDT>::kTimes * v;
}
// A mask for a buffer's length (a uniform value), hidden from the compiler as in dead_unless.
TAMD_DEVICE uint32_t all_ones_if(bool b) {
  uint32_t v = (uint32_t)__builtin_amdgcn_readfirstlane(b ? 0x7FFFFFFF : 0);
  asm volatile("" : "+s"(v));
  return v;
}
// A scale of either type; f16 is all ones or zero, hidden from the compiler: behind a branch per scale it put off what the
// accumulators are used for, until the registers did not suffice.
TAMD_DEVICE uint32_t scale_type(int dtype) {
  uint32_t v = (uint32_t)__builtin_amdgcn_readfirstlane(dtype == TAMD_F16 ? -1 : 0);
  asm volatile("" : "+s"(v));
  return v;
}
TAMD_DEVICE float scale_of(uint32_t bits, uint32_t f16) { return bits_to_f32((f32_to_bits(f16_bits_to_f32(bits)) & f16) | (bits << 16 & ~f16)); }

// Up to 16 rows and NB blocks per wave.  A workgroup per CU (two where a wave has few blocks) walks over a contiguous part of the
// strips; its eight waves split K, and a wave's part of x stays in registers.  The codes of D strips are in flight, the waves'
// sums meet in LDS, a barrier per strip.  Scales and zero points of four blocks come with one request, each quarter of the lanes bringing
// those of one block, and change lanes from there: a request costs the CU about 20 cycles whatever it brings.
// One strip per workgroup, x requested with the codes: 70 us for 1 x 4096 x 131072, 43 to 46 now.
template <int XDT, int PER, bool ZEROS, int NB, int D>
__global__ __launch_bounds__(512, D == 1 ? 4 : 2) void matvec_kernel(tamd_matvec_args a) {
  constexpr int SQ = (NB + 3) / 4, STEPS = 4 / PER;
  constexpr bool KEEP = D > 1 && NB * PER <= 8;   // the sums of x stay in registers too
  __shared__ f32x4_t red[2][8][kWave];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  const uint32_t c = lane & 15, h = lane >> 4, K = (uint32_t)a.K, n_kb = (K + 127) / 128;
  const MatvecPart part(n_kb, (uint32_t)wave);
  const int64_t strips = (a.N + 15) / 16;
  const int64_t begin = strips * blockIdx.x / gridDim.x, end = strips * (blockIdx.x + 1) / gridDim.x;
  const uint32_t scale_f16 = scale_type(a.scale_dtype);
  const u32x4_t ones = {Int4<XDT>::kOne, Int4<XDT>::kOne, Int4<XDT>::kOne, Int4<XDT>::kOne};

  struct Stage {
    u32x4_t q[NB];
    uint32_t s[SQ][PER == 4 ? 2 : 1], z[SQ];
  };
  uint32_t code_off[NB], group_off[SQ];   // of the lane; group_off in groups
#pragma unroll
  for (int i = 0; i < NB; ++i) code_off[i] = (uint32_t)i < part.n ? (part.kb0 + i) * 1024u + 16u * lane : kMoeOob;
#pragma unroll
  for (int i = 0; i < SQ; ++i) group_off[i] = 4u * i + h < part.n ? ((part.kb0 + 4u * i + h) * 16u + c) * PER : kMoeOob / 4u;
  int64_t ask = begin;
  const auto request = [&](Stage &st) {   // (an empty buffer past the last strip: no branch around requests)
    const bool live = ask < end;
    const int64_t at = live ? ask : 0, blocks = live ? n_kb : 0;
    const Buffer codes(a.codes + at * n_kb * 1024, blocks * 1024), scales((const uint8_t *)a.scales + at * n_kb * (32 * PER), blocks * (32 * PER));
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      st.q[i] = codes.template load16<2>(code_off[i]);
      __builtin_amdgcn_sched_barrier(0);   // (one order wherever this is expanded: the waits are counted from it)
    }
#pragma unroll
    for (int i = 0; i < SQ; ++i) {
      if constexpr (PER == 4) {
        const u32x2_t v = scales.load8(2u * group_off[i]);
        st.s[i][0] = v.x, st.s[i][1] = v.y;
      } else if constexpr (PER == 2) {
        st.s[i][0] = scales.load4(2u * group_off[i]);
      } else {
        st.s[i][0] = scales.load2(2u * group_off[i]);
      }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (ZEROS) {
        const Buffer zeros(a.zeros + at * n_kb * (16 * PER), blocks * (16 * PER));
        if constexpr (PER == 4) st.z[i] = zeros.load4(group_off[i]);
        else if constexpr (PER == 2) st.z[i] = zeros.load2(group_off[i]);
        else st.z[i] = zeros.load1(group_off[i]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    ++ask;
  };

  Stage st[D];
#pragma unroll
  for (int d = 0; d < D; ++d) request(st[d]);
  // ---- x, and the sums of its groups
  u32x4_t xr[NB][4];
  {
    const Buffer x(a.x, (int64_t)(a.M - 1) * a.x_stride_m * 2 + 2 * (int64_t)K);
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t k = 128u * (part.kb0 + i) + 32u * j;
        xr[i][j] = x.load16((int)c < a.M && (uint32_t)i < part.n && k < K ? c * (uint32_t)a.x_stride_m * 2u + 2u * k + 16u * h : kMoeOob);
      }
  }
  const auto x_sum = [&](int i, int g) {
    f32x4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < STEPS; ++j) v = Mma16<XDT>::mma(as_frag<XDT>(xr[i][g * STEPS + j]), as_frag<XDT>(ones), v);
    return v;
  };
  f32x4_t kept[KEEP ? NB : 1][PER];
  if constexpr (KEEP) {
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int g = 0; g < PER; ++g) kept[i][g] = x_sum(i, g);
  }

  int64_t now = begin;
  int turn = 0;
  const auto multiply = [&](const Stage &st) {
    f32x4_t y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int from = 4 * (int)(16u * (i & 3) + c);
      const uint32_t s0 = (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)st.s[i / 4][0]);
      const uint32_t s1 = PER == 4 ? (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)st.s[i / 4][PER == 4 ? 1 : 0]) : 0u;
      const uint32_t z = ZEROS ? (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)st.z[i / 4]) : 0u;
#pragma unroll
      for (int g = 0; g < PER; ++g) {
        const float scale = scale_of((g < 2 ? s0 : s1) >> (16 * (g & 1)) & 0xFFFFu, scale_f16);
        const float offset = ZEROS ? -16.f - (float)(z >> (8 * g) & 0xFFu) : -24.f;
        f32x4_t p;
        if constexpr (KEEP) p = kept[i][g];
        else p = x_sum(i, g);
#pragma unroll
        for (int v = 0; v < 4; ++v) p[v] *= offset;
#pragma unroll
        for (int j = 0; j < STEPS; ++j) p = Mma16<XDT>::mma(as_frag<XDT>(xr[i][g * STEPS + j]), codes_plus_16<XDT>(st.q[i][g * STEPS + j]), p);
#pragma unroll
        for (int v = 0; v < 4; ++v) y[v] = __builtin_fmaf(scale, p[v], y[v]);
      }
    }
    red[turn][wave][lane] = y;
    sync_threads();
    const int m = tid >> 4, col = tid & 15;
    const int64_t n = 16 * now + col;
    if (m < a.M && n < a.N) {
      float v = matvec_sum<XDT>(red[turn], m, col);
      if (a.bias) v += load_any_f32(a.bias, a.bias_dtype, n);
      store_any(a.y, a.y_dtype, m * a.y_stride_m + n, v);
    }
    turn ^= 1;   // (one barrier between two uses of either half)
    ++now;
  };
  if constexpr (D == 1) {   // (a workgroup per strip)
    multiply(st[0]);
  } else {
    while (now < end) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
        if (now < end) multiply(st[d]);
        request(st[d]);
      }
    }
  }
}

// Any number of rows and any K: a workgroup has C strips and MT tiles of 16 rows, its eight waves split K and read their part of x once,
// with the codes, U blocks at a time and twice that in flight.  Each block of x serves C strips.
// (One strip, U = 2 and nothing ahead: 51 us for 48 x 8192 x 8192, 21 now.)
template <int XDT, int MT, int XI, int C, int PER, bool ZEROS, int U>
__global__ __launch_bounds__(512, MT == 1 ? 4 : 2) void matvec_rows_kernel(tamd_matvec_args a) {
  constexpr int STEPS = 4 / PER, PITCH = 256 + 16;   // bytes of a row of a block in LDS: rows 16 bytes apart on the banks
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  f32x4_t (*const red)[kWave] = (f32x4_t (*)[kWave])lds;   // (used after the loop)
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  const uint32_t c = lane & 15, h = lane >> 4, K = (uint32_t)a.K, n_kb = (K + 127) / 128;
  const MatvecPart part(n_kb, (uint32_t)wave);
  const int64_t strips = (a.N + 15) / 16, strip = (int64_t)blockIdx.x * C;
  const int m0 = blockIdx.y * (16 * MT), rows = a.M - m0 < 16 * MT ? a.M - m0 : 16 * MT;
  const uint32_t scale_f16 = scale_type(a.scale_dtype);
  const u32x4_t ones = {Int4<XDT>::kOne, Int4<XDT>::kOne, Int4<XDT>::kOne, Int4<XDT>::kOne};
  const int64_t here = strips - strip < C ? strips - strip : C, blocks = here * n_kb;
  const uint8_t *const x_at = (const uint8_t *)a.x + m0 * a.x_stride_m * 2, *const codes_at = a.codes + strip * n_kb * 1024;
  const uint8_t *const scales_at = (const uint8_t *)a.scales + strip * n_kb * (32 * PER), *const zeros_at = ZEROS ? a.zeros + strip * n_kb * (16 * PER) : nullptr;
  const int64_t x_bytes = (int64_t)(rows - 1) * a.x_stride_m * 2 + 2 * (int64_t)K;
  // A block's part of x: request i of a tile's XI brings rows 16 t + 4 i .. + 3, 256 bytes each, which go through LDS to the lanes that
  // multiply them.  (Requested where they are multiplied, 64 bytes of 16 rows at a time, 48 rows of 8192 took 18 of 31 us.)
  uint8_t *const x_lds = lds + wave * (U * MT * 4 * XI * PITCH);
  const uint32_t x_read = wave_lds_offset((c & (4u * XI - 1u)) * PITCH + 16u * h);   // (rows past the last repeat)
  uint32_t x_row[MT][XI];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int i = 0; i < XI; ++i) {
      const int row = 16 * t + 4 * i + (int)h;
      x_row[t][i] = row < rows ? (uint32_t)row * (uint32_t)a.x_stride_m * 2u + 16u * c : kMoeOob;
    }
  const uint32_t tail = K - 128u * (n_kb - 1u);   // K of the last block
  struct Stage {
    u32x4_t q[U][C], x[U][MT][XI];
    uint32_t s[U][C][PER == 4 ? 2 : 1], z[U][C];
  };
  uint32_t ask = 0;
  const auto request = [&](Stage &st) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      // (what is not there comes from an empty buffer: no branch around requests)
      const uint32_t kb = part.kb0 + ask + i, there = all_ones_if(ask + i < part.n);
      const Buffer x(x_at, x_bytes & (int64_t)there);
      const uint32_t beyond = all_ones_if(kb + 1u == n_kb) & (8u * c >= tail ? kMoeOob : 0u);   // (K past the last block's)
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int j = 0; j < XI; ++j) {
          st.x[i][t][j] = x.load16(x_row[t][j] | beyond, 256u * kb);
          __builtin_amdgcn_sched_barrier(0);   // (one order wherever this is expanded: the waits are counted from it)
        }
#pragma unroll
      for (int s = 0; s < C; ++s) {   // (the scalar offset is no part of the range check)
        const int64_t mask = (int64_t)(there & all_ones_if(s < here));
        const Buffer codes(codes_at, (blocks * 1024) & mask), scales(scales_at, (blocks * 32 * PER) & mask);
        st.q[i][s] = codes.template load16<2>(16u * lane, (s * n_kb + kb) * 1024u);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (PER == 4) {
          const u32x2_t v = scales.load8(8u * c, (s * n_kb + kb) * 128u);
          st.s[i][s][0] = v.x, st.s[i][s][1] = v.y;
        } else if constexpr (PER == 2) {
          st.s[i][s][0] = scales.load4(4u * c, (s * n_kb + kb) * 64u);
        } else {
          st.s[i][s][0] = scales.load2(2u * c, (s * n_kb + kb) * 32u);
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (ZEROS) {
          const Buffer zeros(zeros_at, (blocks * 16 * PER) & mask);
          if constexpr (PER == 4) st.z[i][s] = zeros.load4(4u * c, (s * n_kb + kb) * 64u);
          else if constexpr (PER == 2) st.z[i][s] = zeros.load2(2u * c, (s * n_kb + kb) * 32u);
          else st.z[i][s] = zeros.load1(c, (s * n_kb + kb) * 16u);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    ask += U;
  };
  f32x4_t y[MT][C];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int s = 0; s < C; ++s) y[t][s] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const auto multiply = [&](const Stage &st) {
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int j = 0; j < XI; ++j) *(u32x4_t *)(x_lds + ((i * MT + t) * 4 * XI + 4 * j + h) * PITCH + 16u * c) = st.x[i][t][j];
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int g = 0; g < PER; ++g) {
        f32x4_t of_x[MT];
        u32x4_t xf[MT][STEPS];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
#pragma unroll
          for (int j = 0; j < STEPS; ++j) xf[t][j] = *(const u32x4_t *)(x_lds + x_read + (i * MT + t) * 4 * XI * PITCH + 64u * (g * STEPS + j));
          of_x[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < STEPS; ++j) of_x[t] = Mma16<XDT>::mma(as_frag<XDT>(xf[t][j]), as_frag<XDT>(ones), of_x[t]);
        }
#pragma unroll
        for (int s = 0; s < C; ++s) {
          const float scale = scale_of(st.s[i][s][g / 2] >> (16 * (g & 1)) & 0xFFFFu, scale_f16);
          const float offset = ZEROS ? -16.f - (float)(st.z[i][s] >> (8 * g) & 0xFFu) : -24.f;
          typename Mma<XDT>::frag_t w[STEPS];
#pragma unroll
          for (int j = 0; j < STEPS; ++j) w[j] = codes_plus_16<XDT>(st.q[i][s][g * STEPS + j]);
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            f32x4_t p;
#pragma unroll
            for (int v = 0; v < 4; ++v) p[v] = offset * of_x[t][v];
#pragma unroll
            for (int j = 0; j < STEPS; ++j) p = Mma16<XDT>::mma(as_frag<XDT>(xf[t][j]), w[j], p);
#pragma unroll
            for (int v = 0; v < 4; ++v) y[t][s][v] = __builtin_fmaf(scale, p[v], y[t][s][v]);
          }
        }
        if constexpr (U > 1) __builtin_amdgcn_sched_barrier(0);   // (or a later group's x is read at once, and 128 registers do not suffice)
      }
  };
  Stage s0, s1;
  request(s0);
  request(s1);
  for (uint32_t k = 0; k < part.n; k += 2 * U) {   // (blocks past the wave's last: zeros)
    multiply(s0);
    request(s0);
    multiply(s1);
    request(s1);
  }
  sync_threads();
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int s = 0; s < C; ++s) {
      red[wave][lane] = y[t][s];
      sync_threads();
      const int m = tid >> 4, col = tid & 15;
      const int64_t n = 16 * (strip + s) + col;
      if (m < 16 && 16 * t + m < rows && n < a.N) {
        float v = matvec_sum<XDT>(red, m, col);
        if (a.bias) v += load_any_f32(a.bias, a.bias_dtype, n);
        store_any(a.y, a.y_dtype, (m0 + 16 * t + m) * a.y_stride_m + n, v);
      }
      sync_threads();
    }
}

// Many columns: a workgroup has MT tiles of 16 rows and C WN strips.  Its waves are WN, with C strips each, times 8 / WN parts of K;
// a block of x goes through LDS once for all waves of its part, two blocks deep, and with the codes is requested two blocks ahead.
// (64 x 4096 x 131072: 269 us by matvec_rows_kernel, where x comes from the caches for every second strip, 125 so; 149 with three blocks
// ahead, which leave room for one workgroup per CU.  The matrix products, the codes' arithmetic and LDS take about 40 us each.)
template <int XDT, int MT, int WN, int C, int PER, bool ZEROS>
__global__ __launch_bounds__(512, 2) void matvec_wide_kernel(tamd_matvec_args a) {
  constexpr int D = 2, WK = 8 / WN, STEPS = 4 / PER, PITCH = 256 + 16, XL = (4 * MT + WN - 1) / WN;
  constexpr uint32_t TILE = XL * 4 * WN * PITCH;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  const uint32_t c = lane & 15, h = lane >> 4, K = (uint32_t)a.K, n_kb = (K + 127) / 128;
  const uint32_t n = (n_kb + WK - 1) / WK, kb0 = (uint32_t)(wave / WN) * n;
  const int64_t strips = (a.N + 15) / 16, strip = ((int64_t)blockIdx.x * WN + wave % WN) * C;
  const int m0 = blockIdx.y * (16 * MT), rows = a.M - m0 < 16 * MT ? a.M - m0 : 16 * MT;
  const uint32_t scale_f16 = scale_type(a.scale_dtype);
  const u32x4_t ones = {Int4<XDT>::kOne, Int4<XDT>::kOne, Int4<XDT>::kOne, Int4<XDT>::kOne};
  const int64_t here = strips - strip < C ? (strips > strip ? strips - strip : 0) : C, first = here ? strip : 0, blocks = here * n_kb;
  const uint8_t *const x_at = (const uint8_t *)a.x + m0 * a.x_stride_m * 2, *const codes_at = a.codes + first * n_kb * 1024;
  const uint8_t *const scales_at = (const uint8_t *)a.scales + first * n_kb * (32 * PER), *const zeros_at = ZEROS ? a.zeros + first * n_kb * (16 * PER) : nullptr;
  const int64_t x_bytes = (int64_t)(rows - 1) * a.x_stride_m * 2 + 2 * (int64_t)K;
  uint8_t *const x_lds = lds + (wave / WN) * 2 * TILE;
  uint32_t x_row[XL];   // request i of a wave brings four rows
#pragma unroll
  for (int i = 0; i < XL; ++i) {
    const int row = 4 * (i * WN + wave % WN) + (int)h;
    x_row[i] = row < rows ? (uint32_t)row * (uint32_t)a.x_stride_m * 2u + 16u * c : kMoeOob;
  }
  const uint32_t tail = K - 128u * (n_kb - 1u);   // K of the last block
  struct Stage {
    u32x4_t q[C], x[XL];
    uint32_t s[C][PER == 4 ? 2 : 1], z[C];
  };
  uint32_t ask = 0;
  const auto request = [&](Stage &st) {   // (what is not there comes from an empty buffer: no branch around requests)
    const uint32_t kb = kb0 + ask, there = all_ones_if(ask < n && kb < n_kb);
    const Buffer x(x_at, x_bytes & (int64_t)there);
    const uint32_t beyond = all_ones_if(kb + 1u == n_kb) & (8u * c >= tail ? kMoeOob : 0u);   // (K past the last block's)
#pragma unroll
    for (int j = 0; j < XL; ++j) {
      st.x[j] = x.load16(x_row[j] | beyond, 256u * kb);
      __builtin_amdgcn_sched_barrier(0);   // (one order wherever this is expanded: the waits are counted from it)
    }
#pragma unroll
    for (int s = 0; s < C; ++s) {   // (the scalar offset is no part of the range check)
      const int64_t mask = (int64_t)(there & all_ones_if(s < here));
      const Buffer codes(codes_at, (blocks * 1024) & mask), scales(scales_at, (blocks * 32 * PER) & mask);
      st.q[s] = codes.template load16<2>(16u * lane, (s * n_kb + kb) * 1024u);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (PER == 4) {
        const u32x2_t v = scales.load8(8u * c, (s * n_kb + kb) * 128u);
        st.s[s][0] = v.x, st.s[s][1] = v.y;
      } else if constexpr (PER == 2) {
        st.s[s][0] = scales.load4(4u * c, (s * n_kb + kb) * 64u);
      } else {
        st.s[s][0] = scales.load2(2u * c, (s * n_kb + kb) * 32u);
      }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (ZEROS) {
        const Buffer zeros(zeros_at, (blocks * 16 * PER) & mask);
        if constexpr (PER == 4) st.z[s] = zeros.load4(4u * c, (s * n_kb + kb) * 64u);
        else if constexpr (PER == 2) st.z[s] = zeros.load2(2u * c, (s * n_kb + kb) * 32u);
        else st.z[s] = zeros.load1(c, (s * n_kb + kb) * 16u);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    ++ask;
  };
  f32x4_t y[MT][C];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int s = 0; s < C; ++s) y[t][s] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const auto keep = [&](const Stage &st, uint32_t at) {
#pragma unroll
    for (int i = 0; i < XL; ++i) *(u32x4_t *)(x_lds + at + (4 * (i * WN + wave % WN) + h) * PITCH + 16u * c) = st.x[i];
  };
  const auto multiply = [&](const Stage &st, uint32_t at) {
#pragma unroll
    for (int g = 0; g < PER; ++g) {
      f32x4_t of_x[MT], p[MT][C];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        of_x[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < C; ++s) p[t][s] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int j = 0; j < STEPS; ++j) {
        u32x4_t xf[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) xf[t] = *(const u32x4_t *)(x_lds + at + (16 * t + c) * PITCH + 64u * (g * STEPS + j) + 16u * h);
        typename Mma<XDT>::frag_t w[C];
#pragma unroll
        for (int s = 0; s < C; ++s) w[s] = codes_plus_16<XDT>(st.q[s][g * STEPS + j]);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          of_x[t] = Mma16<XDT>::mma(as_frag<XDT>(xf[t]), as_frag<XDT>(ones), of_x[t]);
#pragma unroll
          for (int s = 0; s < C; ++s) p[t][s] = Mma16<XDT>::mma(as_frag<XDT>(xf[t]), w[s], p[t][s]);
        }
      }
#pragma unroll
      for (int s = 0; s < C; ++s) {
        const float scale = scale_of(st.s[s][g / 2] >> (16 * (g & 1)) & 0xFFFFu, scale_f16);
        const float offset = ZEROS ? -16.f - (float)(st.z[s] >> (8 * g) & 0xFFu) : -24.f;
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int v = 0; v < 4; ++v) y[t][s][v] = __builtin_fmaf(scale, __builtin_fmaf(offset, of_x[t][v], p[t][s][v]), y[t][s][v]);
      }
      __builtin_amdgcn_sched_barrier(0);   // (or a later group's x is read at once, and the registers do not suffice)
    }
  };
  Stage st[D];
#pragma unroll
  for (int d = 0; d < D; ++d) request(st[d]);
  keep(st[0], 0);
  sync_threads();
  uint32_t at = 0;
  for (uint32_t k = 0; k < n; k += D) {   // (blocks past the last: zeros.  One barrier between two uses of either half of the part's LDS)
#pragma unroll
    for (int d = 0; d < D; ++d) {
      keep(st[(d + 1) % D], TILE - at);
      __builtin_amdgcn_sched_barrier(0);
      multiply(st[d], at);
      request(st[d]);
      at = TILE - at;
      sync_threads();
    }
  }
  f32x4_t (*const red)[MT][C][kWave] = (f32x4_t (*)[MT][C][kWave])lds;
  if constexpr (WK > 1) {
    if (wave >= WN) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int s = 0; s < C; ++s) red[wave - WN][t][s][lane] = y[t][s];
    }
    sync_threads();
    if (wave >= WN) return;
  }
#pragma unroll
  for (int s = 0; s < C; ++s) {
    const int64_t col = 16 * (strip + s) + c;
    if (col >= a.N) continue;
    const float bias = a.bias ? load_any_f32(a.bias, a.bias_dtype, col) : 0.f;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
#pragma unroll
      for (int q = 1; q < WK; ++q) y[t][s] += red[(q - 1) * WN + wave][t][s][lane];
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int m = 16 * t + 4 * (int)h + v;
        if (m < rows) store_any(a.y, a.y_dtype, (m0 + m) * a.y_stride_m + col, Int4<XDT>::kTimes * y[t][s][v] + bias);
      }
    }
  }
}

template <int XDT, int PER, bool ZEROS, int NB, int D>
int launch_matvec_kept(const tamd_matvec_args &a, int cus, hipStream_t st) {
  const int64_t strips = (a.N + 15) / 16;
  // up to two strips per CU: a workgroup each, side by side (1 x 2880 x 5120: 5.7 us, 9.0 with one per CU that walks)
  if constexpr (NB <= 4)
    if (strips <= 2 * cus) {
      matvec_kernel<XDT, PER, ZEROS, NB, 1><<<(unsigned)strips, 512, 0, st>>>(a);
      return launch_status();
    }
  matvec_kernel<XDT, PER, ZEROS, NB, D><<<(unsigned)(strips < cus ? strips : cus), 512, 0, st>>>(a);
  return launch_status();
}
template <int XDT, int PER, bool ZEROS, int MT, int C, int U, int XI = 4>
int launch_matvec_rows(const tamd_matvec_args &a, hipStream_t st) {
  const int64_t strips = (a.N + 15) / 16;
  const dim3 grid((unsigned)((strips + C - 1) / C), (unsigned)((a.M + 16 * MT - 1) / (16 * MT)));
  const auto kernel = matvec_rows_kernel<XDT, MT, XI, C, PER, ZEROS, U>;
  constexpr int for_x = 8 * U * MT * 4 * XI * (256 + 16), lds = for_x > 8 * kWave * 16 ? for_x : 8 * kWave * 16;
  static_assert(lds <= 160 * 1024);
  if (lds > 64 * 1024)
    if (int rc = raise_lds_limit_once((const void *)kernel)) return rc;
  kernel<<<grid, 512, lds, st>>>(a);
  return launch_status();
}

template <int XDT, int PER, bool ZEROS, int MT, int WN, int C>
int launch_matvec_wide(const tamd_matvec_args &a, hipStream_t st) {
  const int64_t strips = (a.N + 15) / 16;
  const dim3 grid((unsigned)((strips + C * WN - 1) / (C * WN)), (unsigned)((a.M + 16 * MT - 1) / (16 * MT)));
  const auto kernel = matvec_wide_kernel<XDT, MT, WN, C, PER, ZEROS>;
  constexpr int WK = 8 / WN, for_x = WK * 2 * ((4 * MT + WN - 1) / WN) * 4 * WN * (256 + 16), for_sums = (8 - WN) * MT * C * kWave * 16;
  constexpr int lds = for_x > for_sums ? for_x : for_sums;
  static_assert(lds <= 160 * 1024);
  if (lds > 64 * 1024)
    if (int rc = raise_lds_limit_once((const void *)kernel)) return rc;
  kernel<<<grid, 512, lds, st>>>(a);
  return launch_status();
}

template <int XDT, int PER, bool ZEROS, int C>
int launch_matvec_wide_of(const tamd_matvec_args &a, hipStream_t st) {
  if (a.M <= 32) return launch_matvec_wide<XDT, PER, ZEROS, 2, 4, C>(a, st);
  if (a.M <= 48) return launch_matvec_wide<XDT, PER, ZEROS, 3, 4, C>(a, st);
  return launch_matvec_wide<XDT, PER, ZEROS, 4, 4, C>(a, st);
}

template <int XDT, int PER, bool ZEROS>
int launch_matvec(const tamd_matvec_args &a, hipStream_t st) {
  int cus = 0;
  if (int rc = cu_count(cus)) return rc;
  const int64_t strips = (a.N + 15) / 16;
  if (a.M <= 16) {   // x of a wave in registers, up to six blocks
    const int nb = ((a.K + 127) / 128 + 7) / 8;
    if (nb <= 1) return launch_matvec_kept<XDT, PER, ZEROS, 1, 4>(a, cus, st);
    if (nb <= 2) return launch_matvec_kept<XDT, PER, ZEROS, 2, 4>(a, cus, st);
    if (nb <= 3) return launch_matvec_kept<XDT, PER, ZEROS, 3, 4>(a, cus, st);
    if (nb <= 4) return launch_matvec_kept<XDT, PER, ZEROS, 4, 3>(a, cus, st);
    if constexpr (PER < 4)
      if (nb <= 6 && strips > 2 * cus) return launch_matvec_kept<XDT, PER, ZEROS, 6, 2>(a, cus, st);
    if (a.M <= 4) return launch_matvec_rows<XDT, PER, ZEROS, 1, 1, PER < 2 ? 2 : 1, 1>(a, st);
    if (a.M <= 8) return launch_matvec_rows<XDT, PER, ZEROS, 1, 1, 1, 2>(a, st);
    // (16 x 8192 x 28672: 33 us, 43 by the next; 5 rows take 39 and 34)
    if (strips >= 5 * cus) return launch_matvec_wide<XDT, PER, ZEROS, 1, 4, 2>(a, st);
    return launch_matvec_rows<XDT, PER, ZEROS, 1, 1, 1>(a, st);
  }
  // Waves with strips of their own where there are more than two for a CU, from five on two for each: 64 x 4096 x 14336 takes 23 us so and 35
  // with the other kernel, 48 x 512 x 16384 7 and 15, 64 x 4096 x 20480 32 and 45; at two per CU 48 x 8192 x 8192 takes 33 and 21.
  if (strips >= 5 * cus) return launch_matvec_wide_of<XDT, PER, ZEROS, 2>(a, st);
  if (strips > 2 * cus) return launch_matvec_wide_of<XDT, PER, ZEROS, 1>(a, st);
  // Few strips: every 16 rows a workgroup of their own, two of which a CU holds; the weights come again from the caches.  Up to three for two CUs:
  // 33 x 5120 x 530 takes 6.3 us so and 11.2 as one, 48 x 4096 x 2048 7.7 and 10.4, at four for two 20 x 14336 x 4096 19.8 and 17.4.
  if (2 * strips * ((a.M + 15) / 16) <= 3 * cus) return launch_matvec_rows<XDT, PER, ZEROS, 1, 1, 1>(a, st);
  // Two strips share x where one each would be more than one workgroup per CU (24 x 2880 x 5120: 9.8 us, 13.2 with one each).  (Three tiles
  // with groups of 32, and four of any, do not fit the registers with two strips: one strip, and above 48 rows parts of
  // 32, which read the weights again from the caches.)
  const bool two = strips > cus;
  if (a.M > 32 && a.M <= 48) return PER < 4 && two ? launch_matvec_rows<XDT, PER, ZEROS, 3, PER < 4 ? 2 : 1, 1>(a, st) : launch_matvec_rows<XDT, PER, ZEROS, 3, 1, 1>(a, st);
  return two ? launch_matvec_rows<XDT, PER, ZEROS, 2, 2, 1>(a, st) : launch_matvec_rows<XDT, PER, ZEROS, 2, 1, 1>(a, st);
}

template <int XDT>
int matvec_of(const tamd_matvec_args &a, hipStream_t st) {
  if (a.zeros) return a.group == 32 ? launch_matvec<XDT, 4, true>(a, st) : a.group == 64 ? launch_matvec<XDT, 2, true>(a, st) : launch_matvec<XDT, 1, true>(a, st);
  return a.group == 32 ? launch_matvec<XDT, 4, false>(a, st) : a.group == 64 ? launch_matvec<XDT, 2, false>(a, st) : launch_matvec<XDT, 1, false>(a, st);
}

int matvec_bf16(const tamd_matvec_args &a, hipStream_t st);
int matvec_f16(const tamd_matvec_args &a, hipStream_t st);

}  // namespace tamd
