// Rows of tokens to the rows of their experts and back, with gate weights, and the gradients of both.
//
// p[t, j] is the expert row of pick j of token t (anything outside [0, n_rows): none), g[t, j] its gate weight (1 without gates):
//   spread    dst[p[t,j], :] = g[t,j] src[t, :]           dots[t,j] = <src[t, :], other[p[t,j], :]>
//   collect   dst[t, :] = sum_j g[t,j] src[p[t,j], :]     dots[t,j] = <other[t, :], src[p[t,j], :]>
// `spread` is the dispatch and, with dots, the gradient of the sum; `collect` the sum over the picks and, with dots, the gradient of
// the dispatch.  Both go by token, so that a token's row is read (or written) once whatever k is, and its k expert rows are whole,
// contiguous pieces of memory.  What bounds it is memory: 16384 tokens of 2880 bf16, four picks, take 92 us for the dispatch (5.1 TB/s), 82 for the sum with gate
// weights (5.8), 173 and 108 for their gradients (4.9 and 5.2).  Sums are float32 in the order of j, a dot's partial sums are joined in a fixed order: no atomics.
#include "common.h"
#include <type_traits>

using namespace tamd;

namespace {

constexpr int64_t kMostThreads = 0xFFFFFF00ll;   // of a launch: whole workgroups, counted in 32 bits
constexpr int kPicks = 8;   // expert rows of a token that are handled together

// 16 bytes of a row: V elements.  ALIGNED: rows are made of such pieces on 16-byte boundaries; else pieces begin anywhere
template <int DT>
constexpr int kPiece = DT == TAMD_F32 ? 4 : 8;
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_by2_t __attribute__((ext_vector_type(4), aligned(2)));

template <bool ALIGNED>
using Piece = std::conditional_t<ALIGNED, u32x4_t, u32x4_by2_t>;
template <bool ALIGNED, bool ONCE = false>
TAMD_DEVICE u32x4_t load_raw(const void *row, int64_t byte) {
  const auto *const p = (const Piece<ALIGNED> *)((const char *)row + byte);
  if constexpr (ONCE) return __builtin_nontemporal_load(p);
  else return *p;
}
template <bool ALIGNED, bool ONCE>
TAMD_DEVICE void store_raw(void *row, int64_t byte, u32x4_t q) {
  auto *const p = (Piece<ALIGNED> *)((char *)row + byte);
  if constexpr (ONCE) __builtin_nontemporal_store((Piece<ALIGNED>)q, p);
  else *p = q;
}
// The last elements of a piece, without its first `again`
template <int DT>
TAMD_DEVICE void store_rest(void *row, int64_t byte, u32x4_t q, int again) {
#pragma unroll
  for (int e = 0; e < kPiece<DT>; ++e) {
    if (e < again) continue;
    if constexpr (DT == TAMD_F32) *(uint32_t *)((char *)row + byte + 4 * e) = q[e];
    else *(uint16_t *)((char *)row + byte + 2 * e) = (uint16_t)(q[e / 2] >> (16 * (e & 1)));
  }
}
// How a row of H elements is cut: into pieces of V, the last of which ends with the row and so may begin inside the one before (`again` of its elements
// are that one's too: both store the same, and the dots leave them out; where the result lies in the place of what the dots read, the last piece
// stores its own elements only, since another wave may still have to read the others: 36058 tokens of 730 bf16, four picks, 134 us, 131 elsewhere).  A tail by elements was one more wait for memory: 37125 tokens of 730 bf16, four
// picks, took 83 us for the dispatch, 85 for the sum, 150 and 110 for their gradients, and take 80, 64, 136 and 81 so.  Rows of less than a piece go by elements.
template <int DT, bool ALIGNED>
struct Cut {
  static constexpr int V = kPiece<DT>;
  int H, pieces, few;
  TAMD_DEVICE Cut(int H_) : H(H_), pieces(H_ < V ? 0 : H_ / V + (!ALIGNED && H_ % V != 0)), few(H_ < V ? H_ : 0) {}
  TAMD_DEVICE int first(int c) const { return ALIGNED || c * V <= H - V ? c * V : H - V; }
  TAMD_DEVICE int64_t byte(int c) const { return (int64_t)first(c) * (16 / V); }
  TAMD_DEVICE int again(int c) const { return ALIGNED ? 0 : c * V - first(c); }
};
// <x, y> of a piece, without its first `again` elements, added to a lane's sum.  A piece has a sum of its own, so that the lane's has a step per piece and not one
// per element: 5760 float32 by a wave are off by 33 half steps at most, in place of 96, in the same time.
template <int V>
TAMD_DEVICE float add_dot(const float (&x)[V], const float (&y)[V], int again, float dot) {
  float of_piece = 0.f;
#pragma unroll
  for (int e = 0; e < V; ++e) of_piece = e >= again ? __builtin_fmaf(x[e], y[e], of_piece) : of_piece;
  return dot + of_piece;
}
template <int DT>
TAMD_DEVICE void widen(u32x4_t q, float (&v)[kPiece<DT>]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (DT == TAMD_F32) {
      v[e] = bits_to_f32(q[e]);
    } else {
      v[2 * e] = DT == TAMD_BF16 ? bf16_bits_to_f32(q[e] & 0xFFFFu) : f16_bits_to_f32(q[e] & 0xFFFFu);
      v[2 * e + 1] = DT == TAMD_BF16 ? bf16_bits_to_f32(q[e] >> 16) : f16_bits_to_f32(q[e] >> 16);
    }
  }
}
template <int DT>
TAMD_DEVICE u32x4_t narrow(const float (&v)[kPiece<DT>]) {
  u32x4_t q;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (DT == TAMD_F32) q[e] = f32_to_bits(v[e]);
    else if constexpr (DT == TAMD_BF16) q[e] = f32_to_bf16_bits(v[2 * e]) | (f32_to_bf16_bits(v[2 * e + 1]) << 16);
    else q[e] = f32_to_f16_bits(v[2 * e]) | (f32_to_f16_bits(v[2 * e + 1]) << 16);
  }
  return q;
}

TAMD_DEVICE float load_gate(const void *p, int dt, int64_t i) {
  return dt == TAMD_F32 ? load_as_f32<TAMD_F32>(p, i) : dt == TAMD_BF16 ? load_as_f32<TAMD_BF16>(p, i) : load_as_f32<TAMD_F16>(p, i);
}
TAMD_DEVICE void store_gate(void *p, int dt, int64_t i, float v) {
  if (dt == TAMD_F32) store_from_f32<TAMD_F32>(p, i, v);
  else if (dt == TAMD_BF16) store_from_f32<TAMD_BF16>(p, i, v);
  else store_from_f32<TAMD_F16>(p, i, v);
}

template <int LANES>
TAMD_DEVICE float sum_over(float v) {
  return bits_to_f32(group_reduce<LANES>(f32_to_bits(v), [](uint32_t a, uint32_t b) { return f32_to_bits(bits_to_f32(a) + bits_to_f32(b)); }));
}

// What the LANES lanes of a token (16, a wave, or the workgroup's 256) know of it: up to kPicks of its expert rows and their weights, from 64 lanes on
// in scalar registers.
struct Picks {
  int32_t row[kPicks];
  float gate[kPicks];
};
template <int LANES>
TAMD_DEVICE void load_picks(const tamd_token_rows_args &a, int64_t t, int j0, Picks &p) {
#pragma unroll
  for (int j = 0; j < kPicks; ++j) {
    p.row[j] = -1;
    p.gate[j] = 1.0f;
    if (j0 + j < a.k) {
      int32_t r = a.row_indx[t * a.row_indx_stride + j0 + j];
      if constexpr (LANES >= 64) r = __builtin_amdgcn_readfirstlane(r);
      p.row[j] = (uint32_t)r < (uint32_t)a.n_rows ? r : -1;
      if (a.gates) p.gate[j] = load_gate(a.gates, a.gates_dtype, t * a.gates_stride + j0 + j);
    }
  }
}

template <int LANES>
TAMD_DEVICE int64_t token_of() {
  if constexpr (LANES == 256) return (int64_t)blockIdx.x;
  else if constexpr (LANES == 64) return (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  else return (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
}

// dots of the picks j0 ..: the lanes' sums joined, and the waves' in their order
template <int LANES>
TAMD_DEVICE void store_dots(const tamd_token_rows_args &a, int64_t t, int j0, const float (&dot)[kPicks], float *lds) {
  constexpr int WAVES = LANES / 64, OF_WAVE = LANES < 64 ? LANES : 64;
  const int lane = threadIdx.x & (OF_WAVE - 1), wave = threadIdx.x >> 6;
  float all[kPicks];
#pragma unroll
  for (int j = 0; j < kPicks; ++j) all[j] = j0 + j < a.k ? sum_over<OF_WAVE>(dot[j]) : 0.f;
  if constexpr (WAVES > 1) {
    sync_threads();
    if (lane == 0) {
#pragma unroll
      for (int j = 0; j < kPicks; ++j) lds[wave * kPicks + j] = all[j];
    }
    sync_threads();
#pragma unroll
    for (int j = 0; j < kPicks; ++j) {
      all[j] = lds[j];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) all[j] += lds[w * kPicks + j];
    }
    if (wave != 0) return;
  }
#pragma unroll
  for (int j = 0; j < kPicks; ++j)
    if (lane == j && j0 + j < a.k) store_gate(a.dots, a.gates_dtype, t * a.dots_stride + j0 + j, all[j]);
}

// Without gates (and without dots) rows are copied as bits.
template <int DT, bool ALIGNED, int LANES, bool DOTS, bool GATES, bool ONCE>
__global__ __launch_bounds__(256) void spread_kernel(tamd_token_rows_args a, bool in_place) {
  constexpr int V = kPiece<DT>, SIZE = 16 / V;
  __shared__ float lds[4 * kPicks];
  const int64_t t = token_of<LANES>();
  if (t >= a.T) return;
  const int at = threadIdx.x & (LANES - 1);
  const char *const src = (const char *)a.src + t * a.src_stride * SIZE;
  const Cut<DT, ALIGNED> cut(a.H);
  for (int j0 = 0; j0 < a.k; j0 += kPicks) {
    Picks p;
    load_picks<LANES>(a, t, j0, p);
    float dot[kPicks] = {};
    for (int c = at; c < cut.pieces; c += LANES) {
      const int64_t byte = cut.byte(c);
      const u32x4_t q = load_raw<ALIGNED, ONCE>(src, byte);
      float x[V];
      widen<DT>(q, x);
#pragma unroll
      for (int j = 0; j < kPicks; ++j) {
        if (p.row[j] < 0) continue;
        if constexpr (DOTS) {
          float y[V];
          widen<DT>(load_raw<ALIGNED, ONCE>((const char *)a.other + p.row[j] * a.other_stride * SIZE, byte), y);
          dot[j] = add_dot<V>(x, y, cut.again(c), dot[j]);
        }
        char *const row = (char *)a.dst + p.row[j] * a.dst_stride * SIZE;
        u32x4_t to = q;
        if constexpr (GATES) {
          float out[V];
#pragma unroll
          for (int e = 0; e < V; ++e) out[e] = x[e] * p.gate[j];
          to = narrow<DT>(out);
        }
        if (DOTS && !ALIGNED && in_place && cut.again(c) > 0) store_rest<DT>(row, byte, to, cut.again(c));
        else store_raw<ALIGNED, ONCE>(row, byte, to);
      }
    }
    if (!ALIGNED && at < cut.few) {
      const float x = load_as_f32<DT>(src, at);
#pragma unroll
      for (int j = 0; j < kPicks; ++j) {
        if (p.row[j] < 0) continue;
        if constexpr (DOTS) dot[j] = x * load_as_f32<DT>((const char *)a.other + p.row[j] * a.other_stride * SIZE, at);
        char *const row = (char *)a.dst + p.row[j] * a.dst_stride * SIZE;
        if constexpr (GATES) store_from_f32<DT>(row, at, x * p.gate[j]);
        else if constexpr (DT == TAMD_F32) ((uint32_t *)row)[at] = ((const uint32_t *)src)[at];
        else ((uint16_t *)row)[at] = ((const uint16_t *)src)[at];
      }
    }
    if constexpr (DOTS) store_dots<LANES>(a, t, j0, dot, lds);
  }
}

template <int DT, bool ALIGNED, int LANES, bool DOTS, bool ONCE>
__global__ __launch_bounds__(256) void collect_kernel(tamd_token_rows_args a) {
  constexpr int V = kPiece<DT>, SIZE = 16 / V;
  __shared__ float lds[4 * kPicks];
  const int64_t t = token_of<LANES>();
  if (t >= a.T) return;
  const int at = threadIdx.x & (LANES - 1);
  char *const dst = (char *)a.dst + t * a.dst_stride * SIZE;
  const char *const other = DOTS ? (const char *)a.other + t * a.other_stride * SIZE : nullptr;
  const Cut<DT, ALIGNED> cut(a.H);
  const bool few = a.k <= kPicks;    // all picks at once: their dots come with the sum
  Picks p;
  load_picks<LANES>(a, t, 0, p);
  float dot[kPicks] = {};
  for (int c = at; c < cut.pieces; c += LANES) {
    const int64_t byte = cut.byte(c);
    float sum[V] = {}, x[V];
    if constexpr (DOTS) widen<DT>(load_raw<ALIGNED, ONCE>(other, byte), x);
    for (int j0 = 0; j0 < a.k; j0 += kPicks) {
      if (j0) load_picks<LANES>(a, t, j0, p);
#pragma unroll
      for (int j = 0; j < kPicks; ++j) {
        if (p.row[j] < 0) continue;
        float y[V];
        widen<DT>(load_raw<ALIGNED, ONCE>((const char *)a.src + p.row[j] * a.src_stride * SIZE, byte), y);
#pragma unroll
        for (int e = 0; e < V; ++e) sum[e] = __builtin_fmaf(y[e], p.gate[j], sum[e]);
        if constexpr (DOTS) {
          if (few) dot[j] = add_dot<V>(x, y, cut.again(c), dot[j]);
        }
      }
    }
    if (!few) load_picks<LANES>(a, t, 0, p);
    store_raw<ALIGNED, ONCE>(dst, byte, narrow<DT>(sum));
  }
  if (!ALIGNED && at < cut.few) {
    float sum = 0.f;
    for (int j = 0; j < a.k; ++j) {
      const int32_t r = a.row_indx[t * a.row_indx_stride + j];
      if ((uint32_t)r >= (uint32_t)a.n_rows) continue;
      const float g = a.gates ? load_gate(a.gates, a.gates_dtype, t * a.gates_stride + j) : 1.0f;
      sum = __builtin_fmaf(load_as_f32<DT>((const char *)a.src + r * a.src_stride * SIZE, at), g, sum);
    }
    store_from_f32<DT>(dst, at, sum);
  }
  if constexpr (DOTS) {
    for (int j0 = 0; j0 < a.k; j0 += kPicks) {
      if (!few) {
        load_picks<LANES>(a, t, j0, p);
#pragma unroll
        for (int j = 0; j < kPicks; ++j) dot[j] = 0.f;
        for (int c = at; c < cut.pieces; c += LANES) {
          const int64_t byte = cut.byte(c);
          float x[V];
          widen<DT>(load_raw<ALIGNED>(other, byte), x);
#pragma unroll
          for (int j = 0; j < kPicks; ++j) {
            if (p.row[j] < 0) continue;
            float y[V];
            widen<DT>(load_raw<ALIGNED>((const char *)a.src + p.row[j] * a.src_stride * SIZE, byte), y);
            dot[j] = add_dot<V>(x, y, cut.again(c), dot[j]);
          }
        }
      }
      if (!ALIGNED && at < cut.few) {
        const float x = load_as_f32<DT>(other, at);
#pragma unroll
        for (int j = 0; j < kPicks; ++j)
          if (p.row[j] >= 0) dot[j] = x * load_as_f32<DT>((const char *)a.src + p.row[j] * a.src_stride * SIZE, at);
      }
      store_dots<LANES>(a, t, j0, dot, lds);
    }
  }
}

// The lanes of a token: 16 for short rows, the workgroup where a wave to a token would leave the chip's 8192 places for waves empty, or the row is long, else
// a wave (us, four picks unless said otherwise, rows that the caches do not hold):
//   dispatch of 20000 rows of 64 bf16, eight picks, 7.9 by 16 lanes and 17.8 by a wave; 7816 of 176, six picks, 8.8 and 10.6; 2386 of 352 6.0 and 4.4
//   dispatch of 64 rows of 2880 bf16 5.4 by a wave and 3.1 by 256 lanes; 1000 of 1440, eight picks, 10.7 and 7.7; 16384 of 2880 99 and 93
//   combine of 4099 rows of 1063 float32, two picks, 15.0 by a wave and 17.0 by 256 lanes; 1021 of 2016 bf16, six picks, 17.9 and 10.0
//   combine_backward of 4096 rows of 2880 bf16 45 by a wave and 50 by 256 lanes; 1021 of 2016, six picks, 25.7 and 16.3
inline int lanes_of(int T, int pieces, bool dots) {
  if (pieces <= 32 || (pieces <= 64 && T >= 8192)) return 16;
  if (pieces >= 128 && (T < (dots ? 2500 : 4096) || (!dots && pieces >= 320))) return 256;
  return 64;
}

template <int DT, bool ALIGNED, bool DOTS, bool GATES>
int launch(const tamd_token_rows_args &a, bool spread, hipStream_t st) {
  constexpr int SIZE = 16 / kPiece<DT>;
  const auto on_lines = [&](const void *p, int64_t stride) { return ((uintptr_t)p | (uintptr_t)(stride * SIZE)) % 128 == 0; };
  const bool whole_lines = ALIGNED && (int64_t)a.H * SIZE % 128 == 0 && on_lines(a.src, a.src_stride) && on_lines(a.dst, a.dst_stride) && (!DOTS || on_lines(a.other, a.other_stride));
  const int lanes = lanes_of(a.T, a.H / kPiece<DT>, DOTS);
  if ((int64_t)a.T * lanes > kMostThreads) return TAMD_E_TOO_LARGE;
  // Rows of more than the caches keep until they are used again go past them, read and written (us, four picks of 2880 bf16, 16384 tokens: dispatch 93 in place
  // of 96, sum 82 and 95, gradients 175 and 181, 108 and 121).  Below, what an operator leaves or finds in the caches is worth more: 1021 tokens of 2016,
  // six picks, whose rows the caches hold, sum 7.6 in place of 8.9.  Short rows whose ends share lines with others go through the caches, which put these
  // together (60000 tokens of 304, dispatch and gradients 66, 105, 66 in place of 75, 119, 70; 256, past the caches, 33, 59, 46 for 35, 62, 50); of long ones the
  // shared lines are few (12000 of 1500: 50, 83, 48 past them, 58, 85, 51 through them; 36058 of 736: 60, 111, 71 and 71, 119, 80).
  const double bytes = (double)a.T * ((double)a.k * (spread && DOTS ? 2 : 1) + 1) * a.H * (16 / kPiece<DT>);
  const bool once = bytes >= 64e6 && (whole_lines || a.H > 64 * kPiece<DT>);
  const auto end = [&](const void *p, int64_t stride) { return (uintptr_t)p + (uintptr_t)((int64_t)(a.n_rows - 1) * stride + a.H) * SIZE; };
  const bool in_place = spread && DOTS && a.n_rows > 0 && (uintptr_t)a.dst < end(a.other, a.other_stride) && (uintptr_t)a.other < end(a.dst, a.dst_stride);
  const auto go = [&](auto of) {
    constexpr int LANES = decltype(of)::value;
    const unsigned grid = (unsigned)(((int64_t)a.T * LANES + 255) / 256);
    if (spread && once) spread_kernel<DT, ALIGNED, LANES, DOTS, GATES, true><<<grid, 256, 0, st>>>(a, in_place);
    else if (spread) spread_kernel<DT, ALIGNED, LANES, DOTS, GATES, false><<<grid, 256, 0, st>>>(a, in_place);
    else if (once) collect_kernel<DT, ALIGNED, LANES, DOTS, true><<<grid, 256, 0, st>>>(a);
    else collect_kernel<DT, ALIGNED, LANES, DOTS, false><<<grid, 256, 0, st>>>(a);
  };
  if (lanes == 16) go(std::integral_constant<int, 16>());
  else if (lanes == 64) go(std::integral_constant<int, 64>());
  else go(std::integral_constant<int, 256>());
  return launch_status();
}
template <int DT, bool ALIGNED>
int launch(const tamd_token_rows_args &a, bool spread, hipStream_t st) {
  if (a.dots) return launch<DT, ALIGNED, true, true>(a, spread, st);   // (without gates by weights of 1, which load_picks gives)
  return a.gates ? launch<DT, ALIGNED, false, true>(a, spread, st) : launch<DT, ALIGNED, false, false>(a, spread, st);
}

template <int DT>
int launch(const tamd_token_rows_args &a, bool spread, hipStream_t st) {
  const int size = DT == TAMD_F32 ? 4 : 2;
  const auto whole = [&](const void *p, int64_t stride) { return ((uintptr_t)p | (uintptr_t)(stride * size)) % 16 == 0; };
  const bool aligned = a.H % kPiece<DT> == 0 && whole(a.src, a.src_stride) && whole(a.dst, a.dst_stride) && (!a.dots || whole(a.other, a.other_stride));
  return aligned ? launch<DT, true>(a, spread, st) : launch<DT, false>(a, spread, st);
}

int token_rows(const tamd_token_rows_args *args, size_t args_size, bool spread, void *stream) {
  if (!args || args_size != sizeof(tamd_token_rows_args)) return TAMD_E_INVALID;
  const tamd_token_rows_args &a = *args;
  const auto plain = [](int dt) { return dt == TAMD_F32 || dt == TAMD_BF16 || dt == TAMD_F16; };
  if (a.T < 0 || a.k < 0 || a.H < 0 || a.n_rows < 0) return TAMD_E_INVALID;
  if (!plain(a.dtype) || ((a.gates || a.dots) && !plain(a.gates_dtype))) return TAMD_E_UNSUPPORTED;
  if (a.src_stride < 0 || a.dst_stride < 0 || a.other_stride < 0 || a.row_indx_stride < 0 || a.gates_stride < 0 || a.dots_stride < 0) return TAMD_E_INVALID;
  if (a.T == 0 || (spread && a.k == 0)) return 0;
  if (a.k > 0 && !a.row_indx) return TAMD_E_INVALID;
  // (without expert rows there is nothing behind their pointers)
  const void *const by_row = spread ? a.dst : a.src, *const by_token = spread ? a.src : a.dst, *const kept_rows = spread ? a.other : nullptr;
  const void *const kept_tokens = spread ? nullptr : a.other;
  if (a.H > 0 && (!by_token || (a.n_rows > 0 && !by_row))) return TAMD_E_INVALID;
  if (a.H > 0 && a.dots && (spread ? a.n_rows > 0 && !kept_rows : !kept_tokens)) return TAMD_E_INVALID;
  if (a.H == 0 && !a.dots) return 0;
  const uintptr_t by = a.dtype == TAMD_F32 ? 4 : 2;
  if (((uintptr_t)a.src | (uintptr_t)a.dst | (uintptr_t)(a.dots ? a.other : nullptr)) % by != 0 || (uintptr_t)a.row_indx % 4 != 0) return TAMD_E_ALIGNMENT;
  if (((uintptr_t)a.gates | (uintptr_t)a.dots) % (a.gates_dtype == TAMD_F32 && (a.gates || a.dots) ? 4 : 2) != 0) return TAMD_E_ALIGNMENT;
  hipStream_t st = (hipStream_t)stream;
  return a.dtype == TAMD_F32 ? launch<TAMD_F32>(a, spread, st) : a.dtype == TAMD_BF16 ? launch<TAMD_BF16>(a, spread, st) : launch<TAMD_F16>(a, spread, st);
}

}  // namespace

extern "C" int tamd_dispatch(const tamd_token_rows_args *args, size_t args_size, void *stream) { return token_rows(args, args_size, true, stream); }
extern "C" int tamd_combine(const tamd_token_rows_args *args, size_t args_size, void *stream) { return token_rows(args, args_size, false, stream); }
