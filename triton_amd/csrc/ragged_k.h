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
// Rows past the slice's end are zeros by the buffer descriptors' bounds, so what lies there, NaN included, takes no part;
// columns past M or N make results that are not stored.  Sums are float32, rounded once.
#pragma once
#include "common.h"
#include <type_traits>

namespace tamd {

struct RaggedK {
  const void *x, *d;
  int64_t x_pitch, d_pitch;           // elements, a multiple of 8, no less than the columns that can be read
  int x_cols, d_cols;                 // columns that can be read: M and N, filled up to a multiple of 8
  const int32_t *offs, *sizes;        // [E]
  void *y;
  int64_t y_stride_e, y_stride_m, y_stride_split;
  int64_t K;                          // rows of x and d
  int M, N, E, y_dtype;
  int whole_lines, past_caches;       // y's rows begin on lines of 128 bytes, and are results; others are stored past the caches
  int tiles_m, tiles_n, splits;
  int longest_first;                  // slices in the order of their rows (at most 64)
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

// (The copies take 16-byte pieces at 16-byte addresses; operands that are not made of these are laid out so first, by a launch of its own, which
// also fills their rows up with zeros: 66000 rows over 16 slices, 1000 x 1001, 244 us so, of which the pass takes
// 43; with unaligned loads through registers 558, where the pass gave 272.)

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
template <int B, int WAVES>
struct Operand {
  static constexpr int ROW = 2 * B, CHUNKS = B / 8, PER = 64 / CHUNKS;        // bytes and chunks of a row, rows of a wave's copy
  static constexpr int COPIES = kRaggedBK / PER / WAVES;                      // copies of a wave per stage
  static_assert(COPIES * PER * WAVES == kRaggedBK, "the copies of a stage are dealt out evenly");
  static_assert(PER * WAVES % 4 == 0, "the rows of a lane's copies agree in their last two bits");

  const uint8_t *base;
  int64_t pitch;       // bytes
  int C, wave;
  uint32_t offset[COPIES];

  TAMD_DEVICE Operand(const void *p, int64_t pitch_elements, int c0, int C_, int wave_, int lane)
      : base((const uint8_t *)p), pitch(pitch_elements * 2), C(C_), wave(wave_) {
#pragma unroll
    for (int u = 0; u < COPIES; ++u) {
      const int row = (wave + u * WAVES) * PER + lane / CHUNKS, col = c0 + 8 * ((lane % CHUNKS) ^ ((row & 3) * 4));
      offset[u] = col < C ? (uint32_t)(row * pitch + 2 * col) : 0x7FFFFFFFu;
    }
  }
  // what bounds the copies of the rows r0 .., of which `rows` are there
  TAMD_DEVICE s32x4_t bounds(int64_t r0, int64_t rows) const {
    const uint64_t at = (uint64_t)(base + r0 * pitch);
    const int64_t n = rows < kRaggedBK ? rows : kRaggedBK;
    return s32x4_t{(int)(uint32_t)at, (int)((uint32_t)(at >> 32) & 0xFFFFu), n > 0 ? (int)((n - 1) * pitch + 2 * C) : 0, 0x00020000};
  }
  TAMD_DEVICE void copy(s32x4_t rsrc, int u, uint32_t lds_at) const { copy_to_lds(rsrc, lds_at + (wave + u * WAVES) * 1024, offset[u]); }
};

template <int BM, int BN, int WM, int WN, int RING_>
struct RaggedShape {
  static constexpr int WAVES = WM * WN, RING = RING_;
  static constexpr int MF = BM / WM / 32, NF = BN / WN / 32;
  static constexpr int STAGE = (BM + BN) * 2 * kRaggedBK;
  static constexpr int OUT = BM * (BN * 2 + 16);                         // the tile's rows in 16 bits, or half of them in 32
  static constexpr int LDS = RING * STAGE > OUT ? RING * STAGE : OUT;
  static_assert(BM % 128 == 0 && BN % 128 == 0 && LDS <= 160 * 1024 && WAVES * 32 * (NF * 128 + 16) <= LDS, "pieces change places among four");
};

template <int DT, int BM, int BN, int WM, int WN, int RING_>
__global__ __launch_bounds__(64 * WM * WN, 2) void ragged_k_kernel(RaggedK a) {
  typedef RaggedShape<BM, BN, WM, WN, RING_> S;
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
  const int turn = (int)(es / a.splits), split = (int)(es - (uint32_t)turn * a.splits);
  int e = turn;
  int64_t begin, end;
  if (a.longest_first) {
    // a lane per slice, which counts the slices that go before its own: keys are distinct, so that every slice has its turn
    const int off = lane < a.E ? a.offs[lane] : 0, size = lane < a.E ? a.sizes[lane] : 0;
    const uint32_t key = lane < a.E ? (uint32_t)(size < 0 ? 0 : size < 1 << 25 ? size : (1 << 25) - 1) << 6 | (uint32_t)(63 - lane) : 0u;
    int before = 0;
    for (int f0 = 0; f0 < a.E; f0 += 8)   // (a lane without a slice has a key of 0)
#pragma unroll
      for (int f = 0; f < 8; ++f) before += (uint32_t)__builtin_amdgcn_readlane((int)key, f0 + f) > key;
    e = __builtin_ctzll(__ballot(lane < a.E && before == turn));
    begin = __builtin_amdgcn_readlane(off, e), end = begin + __builtin_amdgcn_readlane(size, e);
  } else {
    begin = a.offs[e], end = begin + a.sizes[e];
  }
  const uint32_t g = t / (4u * a.tiles_m), tg = t - g * 4u * a.tiles_m;
  const uint32_t w = a.tiles_n - 4u * g < 4u ? a.tiles_n - 4u * g : 4u;
  const int m0 = (int)(tg / w) * BM, n0 = (int)(4u * g + tg % w) * BN;

  begin = begin < 0 ? 0 : begin;
  end = end > a.K ? a.K : end;
  const int64_t stages = end > begin ? (end - begin + kRaggedBK - 1) / kRaggedBK : 0;
  const int64_t first = stages * split / a.splits, last = stages * (split + 1) / a.splits;
  const int n_k = (int)(last - first);
  const int64_t r0 = begin + first * kRaggedBK;

  Operand<BM, WAVES> x(a.x, a.x_pitch, m0, a.x_cols, wave, lane);
  Operand<BN, WAVES> d(a.d, a.d_pitch, n0, a.d_cols, wave, lane);
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

  // The fragments of a step (16 rows) are requested while the instructions of the step before run: a wave's reads are then back in time,
  // and a stage needs one barrier, behind which its slot is free.
  s16x8_t xf[2][MF], df[2][NF];
  const auto fetch = [&](int into, uint32_t slot, int k) {
#pragma unroll
    for (int f = 0; f < NF; ++f) df[into][f] = fragment(d_at[f] + slot + k * 16 * 2 * BN, 2 * BN);
#pragma unroll
    for (int f = 0; f < MF; ++f) xf[into][f] = fragment(x_at[f] + slot + k * 16 * 2 * BM, 2 * BM);
  };
  // between(f) is called behind the f-th part of the instructions
  const auto multiply = [&](int from, auto between) {
#pragma unroll
    for (int f = 0; f < MF; ++f) {
#pragma unroll
      for (int h = 0; h < NF; ++h) acc[f][h] = mma<DT>(df[from][h], xf[from][f], acc[f][h]);
      between(f);
    }
    // two reads of the next step's fragments, one product: 1.97 ms in place of 2.06 with all reads in front (65536 rows over 32 slices, 2880 x 5760)
#pragma unroll
    for (int g = 0; g < MF * NF; ++g) {
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    }
  };
  struct Stage {
    s32x4_t x, d;
  };
  const auto stage = [&](int s) {
    const int64_t row = r0 + (int64_t)s * kRaggedBK, rows = s < n_k ? end - row : 0;
    return Stage{x.bounds(row, rows), d.bounds(row, rows)};
  };
  // (a copy holds its wave until the CU's address unit has taken it: dealt out among the products, the matrix units go on)
  constexpr int X_COPIES = Operand<BM, WAVES>::COPIES, COPIES = X_COPIES + Operand<BN, WAVES>::COPIES, FIRST = COPIES / 2;
  const auto copy = [&](const Stage &b, int c, uint32_t slot) {
    if (c < X_COPIES) x.copy(b.x, c, lds_base + slot);
    else d.copy(b.d, c - X_COPIES, lds_base + slot + BM * 2 * kRaggedBK);
  };

  if (n_k > 0) {
#pragma unroll
    for (int s = 0; s < RING; ++s) {
      const Stage b = stage(s);
#pragma unroll
      for (int c = 0; c < (s < RING - 1 ? COPIES : FIRST); ++c) copy(b, c, s * STAGE);
    }
    uint32_t slot = 0, next = STAGE, before = (RING - 1) * STAGE;
    wait_copies<(RING - 2) * COPIES + FIRST>();    // (copies complete in the order of their requests)
    sync_threads();
    fetch(0, 0, 0);
    Stage b = stage(RING - 1);
    for (int s = 0; s < n_k; ++s) {
      fetch(1, slot, 1);
      multiply(0, [&](int f) {   // the rest of the stage that the slot before takes
#pragma unroll
        for (int c = FIRST + f * (COPIES - FIRST) / MF; c < FIRST + (f + 1) * (COPIES - FIRST) / MF; ++c) copy(b, c, before);
      });
      wait_copies<(RING - 2) * COPIES>();
      sync_threads();   // stage s + 1 is visible; every wave has read stage s
      b = stage(s + RING);
      fetch(0, next, 0);
      multiply(1, [&](int f) {
#pragma unroll
        for (int c = f * FIRST / MF; c < (f + 1) * FIRST / MF; ++c) copy(b, c, slot);
      });
      before = slot;
      slot = next;
      next = next + STAGE == RING * STAGE ? 0 : next + STAGE;
    }
    wait_copies<0>();
  }
  sync_threads();

  // ---- results, through LDS
  const auto pack = [&](auto type, const f32x16_t &v, int q, uint8_t *to) {   // four neighbours of a row
    constexpr int YT = decltype(type)::value;
    const float c[4] = {v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
    if constexpr (YT == TAMD_F32) *(u32x4_t *)to = u32x4_t{f32_to_bits(c[0]), f32_to_bits(c[1]), f32_to_bits(c[2]), f32_to_bits(c[3])};
    else if constexpr (YT == TAMD_BF16) *(uint2 *)to = make_uint2(f32_to_bf16_bits(c[0]) | (f32_to_bf16_bits(c[1]) << 16), f32_to_bf16_bits(c[2]) | (f32_to_bf16_bits(c[3]) << 16));
    else *(uint2 *)to = make_uint2(f32_to_f16_bits(c[0]) | (f32_to_f16_bits(c[1]) << 16), f32_to_f16_bits(c[2]) | (f32_to_f16_bits(c[3]) << 16));
  };
  const auto last_piece = [&](auto type, u32x4_t v, uint8_t *to, int left) {  // of a row whose end is inside
    constexpr int YT = decltype(type)::value;
#pragma unroll
    for (int b = 0; b < 7; ++b) {
      if (b >= left) continue;
      if constexpr (YT == TAMD_F32) ((uint32_t *)to)[b] = v[b & 3];
      else ((uint16_t *)to)[b] = (uint16_t)(v[b / 2] >> (16 * (b & 1)));
    }
  };
  const auto store = [&](auto type) {
    constexpr int SIZE = decltype(type)::value == TAMD_F32 ? 4 : 2, PIECE = 16 / SIZE;
    uint8_t *const y = (uint8_t *)a.y + ((int64_t)e * a.y_stride_e + split * a.y_stride_split) * SIZE;
    if (a.whole_lines) {
      // Rows that begin on lines of 128 bytes: a wave's strip is whole lines of them, 32 rows at a time through LDS of its own, stored past
      // the caches (1332 rows over 32 slices, 2016 x 2112: 58 us, 76 with ordinary stores).
      constexpr int CHUNKS = NF * 32 / PIECE, PITCH = NF * 32 * SIZE + 16;
      uint8_t *const strip_lds = lds + wave * (32 * PITCH);
      const uint32_t from = wave_lds_offset((uint32_t)((lane / CHUNKS) * PITCH + (lane % CHUNKS) * 16));
      const int n = n0 + wn * NF * 32 + (lane % CHUNKS) * PIECE;
#pragma unroll
      for (int f = 0; f < MF; ++f) {
#pragma unroll
        for (int h = 0; h < NF; ++h)
#pragma unroll
          for (int q = 0; q < 4; ++q) pack(type, acc[f][h], q, strip_lds + (lane & 31) * PITCH + (h * 32 + q * 8 + (lane >> 5) * 4) * SIZE);
#pragma unroll
        for (int p = 0; p < CHUNKS / 2; ++p) {
          const u32x4_t v = *(const u32x4_t *)(strip_lds + from + p * (64 / CHUNKS) * PITCH);
          const int m = m0 + (wm * MF + f) * 32 + p * (64 / CHUNKS) + lane / CHUNKS;
          if (m >= a.M || n >= a.N) continue;
          uint8_t *const to = y + ((int64_t)m * a.y_stride_m + n) * SIZE;
          if (n + PIECE <= a.N) __builtin_nontemporal_store(v, (u32x4_t *)to);
          else last_piece(type, v, to, a.N - n);
        }
      }
      return;
    }
    // Others: the tile's rows (half of them at a time in float32) through all of LDS, so that a wave stores whole rows of the tile, of which it leaves
    // the fewest lines to others.  With few rows to a slice, where the stores are what takes the time, into the caches, which put these lines
    // together (760 rows over 60 slices, 237 x 2261: 26 us, 29 past them), else past them (20000 over 60, 700 x 720: 66, 70 into them).
    constexpr int TURNS = SIZE / 2, CHUNKS = BN / PIECE, PITCH = BN * SIZE + 16, FRAGMENTS = MF / TURNS, ROWS = BM / TURNS;
    static_assert(ROWS * PITCH <= S::LDS && ROWS * CHUNKS % (64 * WAVES) == 0, "a turn fits");
#pragma unroll
    for (int turn = 0; turn < TURNS; ++turn) {
      if (turn) sync_threads();
#pragma unroll
      for (int f = 0; f < FRAGMENTS; ++f)
#pragma unroll
        for (int h = 0; h < NF; ++h)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            pack(type, acc[turn * FRAGMENTS + f][h], q, lds + ((wm * FRAGMENTS + f) * 32 + (lane & 31)) * PITCH + ((wn * NF + h) * 32 + q * 8 + (lane >> 5) * 4) * SIZE);
      sync_threads();
#pragma unroll 4
      for (int p = 0; p < ROWS * CHUNKS / (64 * WAVES); ++p) {
        const int at = p * 64 * WAVES + (int)threadIdx.x, row = at / CHUNKS, chunk = at % CHUNKS;
        const u32x4_t v = *(const u32x4_t *)(lds + row * PITCH + chunk * 16);
        const int m = m0 + ((row / (FRAGMENTS * 32)) * MF + turn * FRAGMENTS) * 32 + row % (FRAGMENTS * 32), n = n0 + chunk * PIECE;
        if (m >= a.M || n >= a.N) continue;
        uint8_t *const to = y + ((int64_t)m * a.y_stride_m + n) * SIZE;
        if (n + PIECE > a.N) {
          last_piece(type, v, to, a.N - n);
        } else if (a.past_caches) {
          __builtin_nontemporal_store(v, (u32x4_by2_t *)to);
        } else {
          asm volatile("" ::: "memory");   // (else the compiler makes one store of the two, an ordinary one)
          *(u32x4_by2_t *)to = v;
          asm volatile("" ::: "memory");
        }
      }
    }
  };
  if (a.y_dtype == TAMD_F32) store(std::integral_constant<int, TAMD_F32>());
  else if (a.y_dtype == TAMD_BF16) store(std::integral_constant<int, TAMD_BF16>());
  else store(std::integral_constant<int, TAMD_F16>());
}

// The tiles that there are (BM x BN, stages in flight).  One of 128 x 256 or 256 x 128, two to a CU, for long slices of many tiles: 65536 rows over 32 slices,
// 2880 x 5760, 1.97 ms, and 2.27 with 128 x 128; 4096 over 8 of unequal lengths, 2048 x 4096, 91 and 104 us, 2048 over 8 55 and 57.  (256 x 256, one to a CU, gave 1.99
// ms, and with equal lengths 81 us where 128 x 256 gives 80.)
// 128 x 128 with two stages, four to a CU, where a slice has few of them: 1332 rows over 32 slices, 2016 x 2112, 58 us, 64 with three, which
// cost a CU its fourth workgroup; with 2500 rows to each of 64 slices, 64 x 64, the third stage gives 28 in place of 40.
enum RaggedTile { kTile128x256, kTile256x128, kTile128Short, kTile128 };

int ragged_k_bf16(const RaggedK &a, int tile, void *stream);
int ragged_k_f16(const RaggedK &a, int tile, void *stream);

template <int DT, int BM, int BN, int WM, int WN, int RING>
inline int ragged_k_launch(const RaggedK &a, hipStream_t st) {
  const auto kern = ragged_k_kernel<DT, BM, BN, WM, WN, RING>;
  if (int rc = raise_lds_limit_once((const void *)kern)) return rc;
  const uint64_t total = (uint64_t)a.tiles_m * a.tiles_n * a.E * a.splits;
  kern<<<(unsigned)((total + 255) / 256 * 256), 64 * WM * WN, RaggedShape<BM, BN, WM, WN, RING>::LDS, st>>>(a);
  return launch_status();
}
template <int DT>
inline int ragged_k_typed(const RaggedK &a, int tile, hipStream_t st) {
  if (tile == kTile128x256) return ragged_k_launch<DT, 128, 256, 1, 4, 3>(a, st);
  if (tile == kTile256x128) return ragged_k_launch<DT, 256, 128, 2, 2, 3>(a, st);
  return tile == kTile128 ? ragged_k_launch<DT, 128, 128, 2, 2, 3>(a, st) : ragged_k_launch<DT, 128, 128, 2, 2, 2>(a, st);
}

}  // namespace tamd
