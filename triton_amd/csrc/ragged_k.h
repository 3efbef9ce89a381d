// Products over ragged rows: y[e] = x[rows of slice e]^T d[rows of slice e], the gradient of every expert's weights.
//
// Both operands lie row by row, so the axis that is summed over is the strided one of both.  A stage is BK rows of BM columns of x and of BN
// columns of d, copied to LDS as they lie (16 bytes per lane, without registers); `ds_read_b64_tr_b16` hands a lane four rows of its column, which is
// the order that the matrix instruction wants.  Its sixteen lanes read 32 bytes each of four rows: 64-byte pieces of a row change places
// with the row's number, so that these lie in different banks.
//
//   LDS image of an operand: row r (0 .. BK - 1), 16-byte chunk c at r * 2 B + 16 * (c ^ ((r & 3) * 4))
//   instruction (d's fragment, x's fragment): lane l holds m = l % 32 and n = 8 (i / 4) + 4 (l / 32) + i % 4 of 32 x 32 results
//
// Rows past the slice's end are zeros by the buffer descriptors' bounds (or the loads' own), so what lies there, NaN included, takes no part;
// columns past M or N make results that are not stored.  Sums are float32, rounded once.
#pragma once
#include "common.h"

namespace tamd {

struct RaggedK {
  const void *x, *d;
  int64_t x_pitch, d_pitch;           // elements
  const int32_t *offs;                // [E + 1]
  void *y;
  int64_t y_stride_e, y_stride_m, y_stride_split;
  int64_t K;                          // rows of x and d
  int M, N, E, y_dtype, whole_stores; // whole_stores: 16 bytes of a row of y at a time
  int tiles_m, tiles_n, splits;
};

constexpr int kRaggedBK = 32;
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef short s16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_by2_t __attribute__((ext_vector_type(4), aligned(2)));
typedef int s32x4_t __attribute__((ext_vector_type(4)));

// 16 bytes per lane from memory to LDS, lane l's to lds_at + 16 l; offsets past the descriptor's end deliver zeros.  (The wait states cover the
// scalar registers that the compiler may have written just before, and M0.)
TAMD_DEVICE void copy_to_lds(s32x4_t rsrc, uint32_t lds_at, uint32_t offset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds_at)), "v"(offset), "s"(rsrc)
               : "memory", "m0");
}
template <int N>
TAMD_DEVICE void wait_copies() {
  static_assert(N >= 0 && N < 64, "a counter of 6 bits");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

template <int DT>
TAMD_DEVICE f32x16_t mma(s16x8_t a, s16x8_t b, f32x16_t c) {
  if constexpr (DT == TAMD_BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// One operand of a tile: B of its columns from c0 on, of C there are.
template <int B, int WAVES, bool DMA>
struct Operand {
  static constexpr int ROW = 2 * B, CHUNKS = B / 8, PER = 64 / CHUNKS;        // bytes and chunks of a row, rows of a wave's copy
  static constexpr int COPIES = kRaggedBK / PER / WAVES;                      // copies of a wave per stage
  static constexpr int BYTES = kRaggedBK * ROW;
  static_assert(COPIES * PER * WAVES == kRaggedBK, "the copies of a stage are dealt out evenly");

  const uint8_t *base;
  int64_t pitch;       // bytes
  int C, row[COPIES], col, wave;
  uint32_t offset[COPIES];
  u32x4_t held[DMA ? 1 : COPIES];

  TAMD_DEVICE Operand(const void *p, int64_t pitch_elements, int c0, int C_, int wave_, int lane)
      : base((const uint8_t *)p), pitch(pitch_elements * 2), C(C_), wave(wave_) {
    const int slot = lane % CHUNKS;
#pragma unroll
    for (int u = 0; u < COPIES; ++u) {
      row[u] = (wave + u * WAVES) * PER + lane / CHUNKS;
      col = c0 + 8 * (slot ^ ((row[u] & 3) * 4));   // (the same for all u: a wave's copies start at rows that agree in their last two bits)
      offset[u] = col < C ? (uint32_t)(row[u] * pitch + 2 * col) : 0x7FFFFFFFu;
    }
  }
  // the rows r0 .. of which `rows` are there
  TAMD_DEVICE void request(int64_t r0, int64_t rows, uint32_t lds_at) {
    if constexpr (DMA) {
      const uint64_t at = (uint64_t)(base + r0 * pitch);
      const int64_t n = rows < kRaggedBK ? rows : kRaggedBK;
      const s32x4_t rsrc = {(int)(uint32_t)at, (int)((uint32_t)(at >> 32) & 0xFFFFu), n > 0 ? (int)((n - 1) * pitch + 2 * C) : 0, 0x00020000};
#pragma unroll
      for (int u = 0; u < COPIES; ++u) copy_to_lds(rsrc, lds_at + (wave + u * WAVES) * 1024, offset[u]);
    } else {
#pragma unroll
      for (int u = 0; u < COPIES; ++u) {
        u32x4_t q = {0, 0, 0, 0};
        const uint16_t *p = (const uint16_t *)(base + (r0 + row[u]) * pitch) + col;
        if (row[u] < rows && col < C) {
          if (col + 8 <= C) {
            q = *(const u32x4_by2_t *)p;
          } else {
#pragma unroll
            for (int e = 0; e < 7; ++e)
              if (col + e < C) q[e / 2] |= (uint32_t)p[e] << (16 * (e & 1));
          }
        }
        held[u] = q;
      }
    }
  }
  TAMD_DEVICE void put(uint8_t *lds, int lane) {   // what request() left in registers
    if constexpr (!DMA) {
#pragma unroll
      for (int u = 0; u < COPIES; ++u) *(u32x4_t *)(lds + (wave + u * WAVES) * 1024 + lane * 16) = held[u];
    }
  }
};

template <int BM, int BN, int WM, int WN, int RING_, bool DMA>
struct RaggedShape {
  static constexpr int WAVES = WM * WN, RING = DMA ? RING_ : 2;
  static constexpr int MF = BM / WM / 32, NF = BN / WN / 32;
  static constexpr int STAGE = (BM + BN) * 2 * kRaggedBK;
  static constexpr int OUT = 32 * (NF * 128 + 16);                       // a wave's 32 rows of results, float32
  static constexpr int LDS = RING * STAGE > WAVES * OUT ? RING * STAGE : WAVES * OUT;
  static_assert(BM % 128 == 0 && BN % 128 == 0 && LDS <= 160 * 1024, "pieces change places among four");
};

template <int DT, int BM, int BN, int WM, int WN, int RING_, bool DMA>
__global__ __launch_bounds__(64 * WM * WN) void ragged_k_kernel(RaggedK a) {
  typedef RaggedShape<BM, BN, WM, WN, RING_, DMA> S;
  constexpr int WAVES = S::WAVES, RING = S::RING, MF = S::MF, NF = S::NF, STAGE = S::STAGE;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = wave / WN, wn = wave % WN;

  // ---- the tile: 32 neighbours of a slice (8 x 4 tiles) go to one XCD, whose L2 then holds their rows once
  const uint32_t per = (uint32_t)a.tiles_m * a.tiles_n, total = per * a.E * a.splits;
  const uint32_t run = blockIdx.x / 256u, in = blockIdx.x % 256u;
  const uint32_t id = run * 256u + (in % 8u) * 32u + in / 8u;
  if (id >= total) return;
  const uint32_t es = id / per, t = id - es * per;
  const int e = (int)(es / a.splits), split = (int)(es - (uint32_t)e * a.splits);
  const uint32_t g = t / (4u * a.tiles_m), tg = t - g * 4u * a.tiles_m;
  const uint32_t w = a.tiles_n - 4u * g < 4u ? a.tiles_n - 4u * g : 4u;
  const int m0 = (int)(tg / w) * BM, n0 = (int)(4u * g + tg % w) * BN;

  int64_t begin = a.offs[e], end = a.offs[e + 1];
  begin = begin < 0 ? 0 : begin;
  end = end > a.K ? a.K : end;
  const int64_t stages = end > begin ? (end - begin + kRaggedBK - 1) / kRaggedBK : 0;
  const int64_t first = stages * split / a.splits, last = stages * (split + 1) / a.splits;
  const int n_k = (int)(last - first);
  const int64_t r0 = begin + first * kRaggedBK;

  Operand<BM, WAVES, DMA> x(a.x, a.x_pitch, m0, a.M, wave, lane);
  Operand<BN, WAVES, DMA> d(a.d, a.d_pitch, n0, a.N, wave, lane);
  const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;

  // ---- where a lane reads: its sixteen's rows i / 4 (of four), its columns 4 (i % 4) ..
  const int grp = lane >> 4, i = lane & 15, r = i >> 2;
  const uint32_t at = (uint32_t)((grp >> 1) * 8 + r), piece = (uint32_t)((grp & 1) * 32 + (i & 3) * 8);
  uint32_t x_at[MF], d_at[NF];
#pragma unroll
  for (int f = 0; f < MF; ++f) x_at[f] = lds_base + at * (2 * BM) + (uint32_t)((wm * MF + f) ^ r) * 64 + piece;
#pragma unroll
  for (int f = 0; f < NF; ++f) d_at[f] = lds_base + (uint32_t)(BM * 2 * kRaggedBK) + at * (2 * BN) + (uint32_t)((wn * NF + f) ^ r) * 64 + piece;
  const auto fragment = [](uint32_t p, int row_bytes) {
    typedef __attribute__((address_space(3))) s16x4_t lds_t;
    const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t *)p), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t *)(p + 4 * row_bytes));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };

  f32x16_t acc[MF][NF];
#pragma unroll
  for (int f = 0; f < MF; ++f)
#pragma unroll
    for (int h = 0; h < NF; ++h)
#pragma unroll
      for (int j = 0; j < 16; ++j) acc[f][h][j] = 0.f;

  const auto multiply = [&](uint32_t slot) {
#pragma unroll
    for (int k = 0; k < kRaggedBK / 16; ++k) {
      s16x8_t xf[MF], df[NF];
#pragma unroll
      for (int f = 0; f < NF; ++f) df[f] = fragment(d_at[f] + slot + k * 16 * 2 * BN, 2 * BN);
#pragma unroll
      for (int f = 0; f < MF; ++f) xf[f] = fragment(x_at[f] + slot + k * 16 * 2 * BM, 2 * BM);
#pragma unroll
      for (int f = 0; f < MF; ++f)
#pragma unroll
        for (int h = 0; h < NF; ++h) acc[f][h] = mma<DT>(df[h], xf[f], acc[f][h]);
    }
  };
  const auto request = [&](int s, uint32_t slot) {
    const int64_t row = r0 + (int64_t)s * kRaggedBK, rows = s < n_k ? end - row : 0;
    x.request(row, rows, lds_base + slot);
    d.request(row, rows, lds_base + slot + BM * 2 * kRaggedBK);
  };
  const auto put = [&](uint32_t slot) {
    x.put(lds + slot, lane);
    d.put(lds + slot + BM * 2 * kRaggedBK, lane);
  };

  if (n_k > 0) {
    if constexpr (DMA) {
#pragma unroll
      for (int s = 0; s < RING - 1; ++s) request(s, s * STAGE);
      uint32_t rd = 0, wr = (RING - 1) * STAGE;
      for (int s = 0; s < n_k; ++s) {
        // (copies complete in the order of their requests: all but those of the newest stages have landed)
        wait_copies<(RING - 2) * (Operand<BM, WAVES, DMA>::COPIES + Operand<BN, WAVES, DMA>::COPIES)>();
        sync_threads();   // stage s is visible; every wave is done with the slot that is filled now
        request(s + RING - 1, wr);
        multiply(rd);
        rd = rd + STAGE == RING * STAGE ? 0 : rd + STAGE;
        wr = wr + STAGE == RING * STAGE ? 0 : wr + STAGE;
      }
      wait_copies<0>();
    } else {
      request(0, 0);
      put(0);
      for (int s = 0; s < n_k; ++s) {
        sync_threads();   // stage s is visible; every wave is done with the other slot
        request(s + 1, 0);
        multiply((s & 1) * STAGE);
        put(((s + 1) & 1) * STAGE);
      }
    }
  }
  sync_threads();

  // ---- results: 32 rows of the wave's strip at a time through its part of LDS, then whole pieces of rows
  uint8_t *const out_lds = lds + wave * S::OUT;
  const bool wide = a.y_dtype == TAMD_F32;
  const int size = wide ? 4 : 2, chunks = NF * 2 * size, row_pitch = NF * 32 * size + 16;     // 16-byte pieces and bytes of a row
  uint8_t *const y = (uint8_t *)a.y + ((int64_t)e * a.y_stride_e + split * a.y_stride_split) * size;
  const int per_row = 16 / size;
#pragma unroll
  for (int f = 0; f < MF; ++f) {
    const int mine = (lane & 31) * row_pitch + (lane >> 5) * 4 * size;
#pragma unroll
    for (int h = 0; h < NF; ++h)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x16_t &c = acc[f][h];
        const int to = mine + (h * 32 + q * 8) * size;
        if (wide) {
          *(u32x4_t *)(out_lds + to) = u32x4_t{f32_to_bits(c[4 * q]), f32_to_bits(c[4 * q + 1]), f32_to_bits(c[4 * q + 2]), f32_to_bits(c[4 * q + 3])};
        } else if (a.y_dtype == TAMD_BF16) {
          *(uint2 *)(out_lds + to) = make_uint2(f32_to_bf16_bits(c[4 * q]) | (f32_to_bf16_bits(c[4 * q + 1]) << 16),
                                                f32_to_bf16_bits(c[4 * q + 2]) | (f32_to_bf16_bits(c[4 * q + 3]) << 16));
        } else {
          *(uint2 *)(out_lds + to) = make_uint2(f32_to_f16_bits(c[4 * q]) | (f32_to_f16_bits(c[4 * q + 1]) << 16),
                                                f32_to_f16_bits(c[4 * q + 2]) | (f32_to_f16_bits(c[4 * q + 3]) << 16));
        }
      }
    for (int p = lane; p < 32 * chunks; p += 64) {
      const int row = p / chunks, chunk = p % chunks;
      const uint32_t from = wave_lds_offset((uint32_t)(row * row_pitch + chunk * 16));
      const u32x4_t v = *(const u32x4_t *)(out_lds + from + 0);
      const int m = m0 + (wm * MF + f) * 32 + row, n = n0 + wn * NF * 32 + chunk * per_row;
      if (m >= a.M || n >= a.N) continue;
      uint8_t *const to = y + ((int64_t)m * a.y_stride_m + n) * size;
      if (a.whole_stores) {
        *(u32x4_t *)to = v;
      } else {
#pragma unroll
        for (int b = 0; b < 8; ++b) {
          if (b >= per_row || n + b >= a.N) continue;
          if (wide) ((uint32_t *)to)[b] = v[b & 3];
          else ((uint16_t *)to)[b] = (uint16_t)(v[b / 2] >> (16 * (b & 1)));
        }
      }
    }
  }
}

int ragged_k_bf16(const RaggedK &a, int tile, bool dma, void *stream);
int ragged_k_f16(const RaggedK &a, int tile, bool dma, void *stream);

template <int DT, int BM, int BN, int WM, int WN, int RING, bool DMA>
inline int ragged_k_launch(const RaggedK &a, hipStream_t st) {
  const auto kern = ragged_k_kernel<DT, BM, BN, WM, WN, RING, DMA>;
  if (int rc = raise_lds_limit_once((const void *)kern)) return rc;
  const uint64_t total = (uint64_t)a.tiles_m * a.tiles_n * a.E * a.splits;
  kern<<<(unsigned)((total + 255) / 256 * 256), 64 * WM * WN, RaggedShape<BM, BN, WM, WN, RING, DMA>::LDS, st>>>(a);
  return launch_status();
}
template <int DT>
inline int ragged_k_typed(const RaggedK &a, int tile, bool dma, hipStream_t st) {
  if (tile == 256) return dma ? ragged_k_launch<DT, 256, 256, 2, 4, 4, true>(a, st) : ragged_k_launch<DT, 256, 256, 2, 4, 4, false>(a, st);
  return dma ? ragged_k_launch<DT, 128, 128, 2, 2, 4, true>(a, st) : ragged_k_launch<DT, 128, 128, 2, 2, 4, false>(a, st);
}

}  // namespace tamd
