// SwiGLU for training: the forward pass keeps its input in 8 bits, the backward pass works from that.
//
//   g = min(a[2n], limit), l = clamp(a[2n + 1], -limit, limit), s = 1 / (1 + exp(-alpha g))
//   out[n]  = g s (l + 1)
//   da[2n]  = dout[n] (l + 1) s (1 + alpha g (1 - s))   where a[2n] <= limit, else 0
//   da[2n + 1] = dout[n] g s                            where |a[2n + 1]| <= limit, else 0
//
// What is kept is the MXFP8 form of a that tamd_downcast_mxfp makes of it (e4m3 values, one e8m0 scale per 32 along a row, rounded up):
// 1.03 bytes per value in place of the 2 of a itself.  The gradient is that of the function at the kept values.
//
// Four lanes share a group of 32, eight values (four pairs) each.  What bounds it is memory: 65536 x 2880 bf16 takes 242 us forward (6.3 TB/s) and 297
// backward with the activation again (6.4).  BIG, from 64 MB on: two groups per thread, everything past the caches, which do not keep that much until
// it is used (16384 x 2880: 62 us, 69 through them; ragged rows 40000 x 1002: 60 and 67, backward 57 and 64).  Below: one group per thread (1024 x 1056:
// 4.0 us, 4.4 with two), a and the results through the caches.  float32 takes the second form always: 16-byte pieces of its results are every other one
// of a line, which past the caches costs 6 % in place of gaining 4.  The kept values go past the caches in both: nothing reads them before the backward pass.
#include "mx_values.h"
#include <type_traits>

using namespace tamd;

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_by1_t __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t u32_by1_t __attribute__((aligned(1)));
typedef uint16_t u16_by1_t __attribute__((aligned(1)));
typedef uint32_t u32x2_by1_t __attribute__((ext_vector_type(2), aligned(1)));

template <bool ALIGNED, bool ONCE, typename T, typename BY1>
TAMD_DEVICE T load_piece(const void *p) {
  using Q = std::conditional_t<ALIGNED, T, BY1>;
  if constexpr (ONCE) return __builtin_nontemporal_load((const Q *)p);
  else return *(const Q *)p;
}
template <bool ALIGNED, bool ONCE, typename T, typename BY1>
TAMD_DEVICE void store_piece(void *p, T q) {
  using Q = std::conditional_t<ALIGNED, T, BY1>;
  if constexpr (ONCE) __builtin_nontemporal_store((Q)q, (Q *)p);
  else *(Q *)p = q;
}
template <bool ALIGNED, bool ONCE>
TAMD_DEVICE u32x4_t load16(const void *p) { return load_piece<ALIGNED, ONCE, u32x4_t, u32x4_by1_t>(p); }
template <bool ALIGNED, bool ONCE>
TAMD_DEVICE u32x2_t load8(const void *p) { return load_piece<ALIGNED, ONCE, u32x2_t, u32x2_by1_t>(p); }
template <bool ALIGNED, bool ONCE>
TAMD_DEVICE void store16(void *p, u32x4_t q) { store_piece<ALIGNED, ONCE, u32x4_t, u32x4_by1_t>(p, q); }
template <bool ALIGNED, bool ONCE>
TAMD_DEVICE void store8(void *p, u32x2_t q) { store_piece<ALIGNED, ONCE, u32x2_t, u32x2_by1_t>(p, q); }

constexpr float kMost = 3.40282346638528859812e38f;   // the greatest of float32

TAMD_DEVICE float widen16(uint32_t bits, int dt) { return dt == TAMD_BF16 ? bf16_bits_to_f32(bits) : f16_bits_to_f32(bits); }
template <int DT>
TAMD_DEVICE uint32_t pack2(float a, float b) {
  if constexpr (DT == TAMD_BF16) return f32_to_bf16_bits(a) | (f32_to_bf16_bits(b) << 16);
  return f32_to_f16_bits(a) | (f32_to_f16_bits(b) << 16);
}

// C (4 or 8) elements from element `at` of a row of L on, of which those behind the row are zeros.  The last piece of a ragged row is read with the
// elements before it, in one request as all others, and moved down when all requests are out (element by element 72359 x 98 bf16 took 23 us forward and 25
// backward, so 18 and 16; moved down as each comes, one request would wait for the next: 30 and 23).
template <int DT, int C>
struct Read {
  static constexpr int WORDS = C * (DT == TAMD_F32 ? 4 : 2) / 4;
  uint32_t q[WORDS];
  int by;                  // elements read before `at`
};
template <int DT, bool ALIGNED, bool ONCE, int C>
TAMD_DEVICE Read<DT, C> read(const void *row, int64_t at, int64_t L) {
  constexpr int SIZE = DT == TAMD_F32 ? 4 : 2, WORDS = Read<DT, C>::WORDS;
  Read<DT, C> r;
  const char *p = (const char *)row;
  const int64_t from = ALIGNED || at <= L - C ? at : (L < C ? 0 : L - C);
  r.by = ALIGNED ? 0 : (int)(at - from);
  p += from * SIZE;
  if (!ALIGNED && L < C) {
#pragma unroll
    for (int w = 0; w < WORDS; ++w) {
      if constexpr (DT == TAMD_F32) r.q[w] = w < L ? ((const uint32_t *)p)[w] : 0u;
      else r.q[w] = (2 * w < L ? (uint32_t)((const uint16_t *)p)[2 * w] : 0u) | (2 * w + 1 < L ? (uint32_t)((const uint16_t *)p)[2 * w + 1] << 16 : 0u);
    }
  } else if constexpr (WORDS == 2) {
    const u32x2_t q = load8<ALIGNED, ONCE>(p);
    r.q[0] = q[0], r.q[1] = q[1];
  } else {
#pragma unroll
    for (int i = 0; i < WORDS; i += 4) {
      const u32x4_t q = load16<ALIGNED, ONCE>(p + 4 * i);
#pragma unroll
      for (int e = 0; e < 4; ++e) r.q[i + e] = q[e];
    }
  }
  return r;
}
template <int DT, bool ALIGNED, int C>
TAMD_DEVICE void widen(const Read<DT, C> &r, float (&v)[C]) {
#pragma unroll
  for (int e = 0; e < C; ++e) v[e] = DT == TAMD_F32 ? bits_to_f32(r.q[e % Read<DT, C>::WORDS]) : widen16(e % 2 ? r.q[e / 2] >> 16 : r.q[e / 2] & 0xFFFFu, DT);
  if (!ALIGNED && r.by > 0) {
#pragma unroll
    for (int step = C / 2; step > 0; step /= 2) {
#pragma unroll
      for (int e = 0; e < C; ++e) v[e] = r.by & step ? (e + step < C ? v[e + step < C ? e + step : e] : 0.f) : v[e];
    }
#pragma unroll
    for (int e = 0; e < C; ++e) v[e] = r.by < C ? v[e] : 0.f;
  }
}
// `n` of them, an even number of C = 8, to p
template <int DT, bool ALIGNED, bool ONCE, int C>
TAMD_DEVICE void store_values(void *p, int n, float (&v)[C]) {
  if constexpr (DT == TAMD_F16) {   // (the last operation rounds to float32 and then to 16 bits, in every variant: the compiler would make one of them in some)
#pragma unroll
    for (int e = 0; e < C; ++e) asm volatile("" : "+v"(v[e]));
  }
  if (ALIGNED || n == C) {
    if constexpr (DT == TAMD_F32) {
#pragma unroll
      for (int i = 0; i < C; i += 4)
        store16<ALIGNED, ONCE>((float *)p + i, u32x4_t{f32_to_bits(v[i]), f32_to_bits(v[i + 1]), f32_to_bits(v[i + 2]), f32_to_bits(v[i + 3])});
    } else if constexpr (C == 8) {
      store16<ALIGNED, ONCE>(p, u32x4_t{pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]), pack2<DT>(v[4], v[5]), pack2<DT>(v[6], v[7])});
    } else {
      store8<ALIGNED, ONCE>(p, u32x2_t{pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3])});
    }
  } else if constexpr (C == 8 && DT != TAMD_F32) {
#pragma unroll
    for (int e = 0; e < C; e += 2)
      if (e < n) *(u32_by1_t *)((uint16_t *)p + e) = pack2<DT>(v[e], v[e + 1]);
  } else {
#pragma unroll
    for (int e = 0; e < C; ++e)
      if (e < n) store_from_f32<DT>(p, e, v[e]);
  }
}

struct GluShape {
  GroupDiv div;            // rows and groups of a row
  int64_t L;               // values of a row: 2 N
  float alpha, limit;      // (limit: the greatest number without one)
  int has_limit;
};

// The clamped pair and the gate's sigmoid, by exp2 and a reciprocal of 1 ulp each.  Comparisons, so that a NaN stays one.
struct Pair {
  float g, l, s;
  bool g_free, l_free;     // not beyond the limit
};
// KEPT: a type's lowest value may have been kept as -2^128.  It counts as the lowest of float32, so that the zero of its sigmoid makes zeros, and so that it
// has a sigmoid where alpha is 0.
template <bool KEPT>
TAMD_DEVICE Pair pair_of(float g, float l, const GluShape &sh) {
  Pair p;
  const bool g_in = !(g > sh.limit), l_in = !(__builtin_fabsf(l) > sh.limit);
  p.g_free = g_in || !sh.has_limit;
  p.l_free = l_in || !sh.has_limit;
  p.g = (KEPT ? g_in : p.g_free) ? g : sh.limit;
  p.l = (KEPT ? l_in : p.l_free) ? l : __builtin_copysignf(sh.limit, l);
  if constexpr (KEPT) p.g = p.g < -kMost ? -kMost : p.g;
  p.s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504088896340736f * sh.alpha * p.g));
  return p;
}

template <int DT, bool ALIGNED, bool BIG>
__global__ __launch_bounds__(256) void checkpoint_kernel(const void *__restrict__ a, int64_t a_stride, void *__restrict__ out, int64_t out_stride,
                                                         uint8_t *__restrict__ values, int64_t v_stride, uint8_t *__restrict__ scales, int64_t s_stride,
                                                         GluShape sh) {
  constexpr int SIZE = DT == TAMD_F32 ? 4 : 2, U = BIG ? 2 : 1;
  const int sub = threadIdx.x & 3;
  const int64_t gid0 = (int64_t)blockIdx.x * (64 * U) + (threadIdx.x >> 2);
  int64_t r[U], g[U];
  int n[U];
  Read<DT, 8> in[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t gid = gid0 + u * 64;
    int64_t b;
    place_group(sh.div, gid < sh.div.total ? gid : 0, b, r[u], g[u]);
    const int64_t left = sh.L - g[u] * 32 - sub * 8;
    n[u] = gid >= sh.div.total || left <= 0 ? 0 : (left < 8 ? (int)left : 8);
    if (!ALIGNED || n[u]) in[u] = read<DT, ALIGNED, BIG, 8>((const char *)a + r[u] * a_stride * SIZE, g[u] * 32 + sub * 8, sh.L);
    else in[u] = {};
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float v[8];
    widen<DT, ALIGNED, 8>(in[u], v);
    float m = 0.f;
    bool any_nan = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      m = __builtin_fmaxf(m, __builtin_fabsf(v[j]));
      any_nan |= v[j] != v[j];
    }
    // (the group's four lanes are a quad: swaps inside it are moves in the register file)
    m = __builtin_fmaxf(m, bits_to_f32((uint32_t)__builtin_amdgcn_update_dpp(0, (int)f32_to_bits(m), 0xB1, 0xF, 0xF, true)));
    m = __builtin_fmaxf(m, bits_to_f32((uint32_t)__builtin_amdgcn_update_dpp(0, (int)f32_to_bits(m), 0x4E, 0xF, 0xF, true)));
    uint32_t byte, code[2] = {0, 0};
    const float by = group_scale<QK_E4M3>(m, TAMD_ROUND_UP, byte);
    if (!any_nan && byte < 0xFEu) {
      float c[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) c[j] = __builtin_amdgcn_fmed3f(v[j] * by, -448.0f, 448.0f);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        code[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c[4 * h + 2], c[4 * h + 3], __builtin_amdgcn_cvt_pk_fp8_f32(c[4 * h], c[4 * h + 1], 0, false), true);
    } else {   // (an infinite magnitude times a multiplier of zero is a NaN too)
#pragma unroll
      for (int j = 0; j < 8; ++j) code[j >> 2] |= fp8_code<QK_E4M3>(v[j] * by) << (8 * (j & 3));
    }
    float o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const Pair p = pair_of<false>(v[2 * j], v[2 * j + 1], sh);
      const float gs = p.g * p.s;
      o[j] = __builtin_fmaf(gs, p.l, gs);
    }
    if (n[u] == 0) continue;
    store_values<DT, ALIGNED, BIG, 4>((char *)out + (r[u] * out_stride + g[u] * 16 + sub * 4) * SIZE, n[u] / 2, o);
    uint8_t *const vp = values + r[u] * v_stride + g[u] * 32 + sub * 8;
    if (ALIGNED || n[u] == 8) {
      store8<ALIGNED, true>(vp, u32x2_t{code[0], code[1]});
    } else {
#pragma unroll
      for (int j = 0; j < 8; j += 2)
        if (j < n[u]) *(u16_by1_t *)(vp + j) = (uint16_t)(code[j >> 2] >> (8 * (j & 3)));
    }
    if (sub == 0) scales[r[u] * s_stride + g[u]] = (uint8_t)byte;
  }
}

template <int DT, bool ALIGNED, bool AGAIN, bool BIG>
__global__ __launch_bounds__(256) void backward_kernel(const void *__restrict__ dout, int64_t d_stride, const uint8_t *__restrict__ values, int64_t v_stride,
                                                       const uint8_t *__restrict__ scales, int64_t s_stride, void *__restrict__ da, int64_t da_stride,
                                                       void *__restrict__ out, int64_t out_stride, GluShape sh) {
  constexpr int SIZE = DT == TAMD_F32 ? 4 : 2, U = BIG ? 2 : 1;
  const int sub = threadIdx.x & 3;
  const int64_t gid0 = (int64_t)blockIdx.x * (64 * U) + (threadIdx.x >> 2);
  int64_t r[U], g[U];
  int n[U];
  uint32_t code[U][2], byte[U];
  int by[U];
  Read<DT, 4> in[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t gid = gid0 + u * 64;
    int64_t b;
    place_group(sh.div, gid < sh.div.total ? gid : 0, b, r[u], g[u]);
    const int64_t left = sh.L - g[u] * 32 - sub * 8;
    n[u] = gid >= sh.div.total || left <= 0 ? 0 : (left < 8 ? (int)left : 8);
    const uint8_t *const vp = values + r[u] * v_stride;
    const int64_t at = g[u] * 32 + sub * 8;
    const int64_t from = ALIGNED || at <= sh.L - 8 ? at : (sh.L < 8 ? 0 : sh.L - 8);
    by[u] = (int)(at - from);
    code[u][0] = code[u][1] = byte[u] = 0;
    in[u] = {};
    if (ALIGNED && n[u] == 0) continue;
    if (!ALIGNED && sh.L < 8) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < sh.L) code[u][j >> 2] |= (uint32_t)vp[j] << (8 * (j & 3));
    } else {
      const u32x2_t q = load8<ALIGNED, BIG>(vp + from);
      code[u][0] = q[0], code[u][1] = q[1];
    }
    byte[u] = scales[r[u] * s_stride + g[u]];
    in[u] = read<DT, ALIGNED, BIG, 4>((const char *)dout + r[u] * d_stride * SIZE, at / 2, sh.L / 2);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (n[u] == 0) continue;
    if (!ALIGNED && by[u] > 0) {   // (less than 8: something is there)
      const uint64_t moved = ((uint64_t)code[u][1] << 32 | code[u][0]) >> (8 * by[u]);
      code[u][0] = (uint32_t)moved, code[u][1] = (uint32_t)(moved >> 32);
    }
    float d[4];
    widen<DT, ALIGNED, 4>(in[u], d);
    // 2^(byte - 127); 0 for 0, as tamd_upcast_mxfp has it, NaN for 255
    const float scale = bits_to_f32(byte[u] == 255u ? 0x7FC00000u : byte[u] << 23);
    typedef float f32x2_t __attribute__((ext_vector_type(2)));
    float v[8], o[4], dv[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)code[u][h], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)code[u][h], true);
      v[4 * h] = lo.x * scale, v[4 * h + 1] = lo.y * scale, v[4 * h + 2] = hi.x * scale, v[4 * h + 3] = hi.y * scale;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const Pair p = pair_of<true>(v[2 * j], v[2 * j + 1], sh);
      const float gs = p.g * p.s;
      o[j] = __builtin_fmaf(gs, p.l, gs);
      // s (1 + alpha g (1 - s)) as s + alpha (g s - (g s) s), of which nothing overflows where s is 0 or 1
      const float slope = d[j] * __builtin_fmaf(sh.alpha, __builtin_fmaf(-gs, p.s, gs), p.s);
      dv[2 * j] = p.g_free ? __builtin_fmaf(slope, p.l, slope) : 0.f;
      dv[2 * j + 1] = p.l_free ? d[j] * gs : 0.f;
    }
    store_values<DT, ALIGNED, BIG, 8>((char *)da + (r[u] * da_stride + g[u] * 32 + sub * 8) * SIZE, n[u], dv);
    if constexpr (AGAIN) store_values<DT, ALIGNED, BIG, 4>((char *)out + (r[u] * out_stride + g[u] * 16 + sub * 4) * SIZE, n[u] / 2, o);
  }
}

bool shape(GluShape &sh, int64_t M, int64_t N, float alpha, float limit, int has_limit, bool big, unsigned &blocks) {
  const int64_t G = (2 * N + 31) / 32, per = big ? 128 : 64;
  sh.div = group_div(1, M, G);
  // (an infinite limit cuts nothing off: it is none, so that a value that is kept as 2^128 counts as the greatest here too)
  const bool cuts = has_limit && limit <= kMost;
  sh.L = 2 * N, sh.alpha = alpha, sh.limit = cuts ? limit : kMost, sh.has_limit = cuts;
  const int64_t n = (sh.div.total + per - 1) / per;
  blocks = (unsigned)n;
  return n < 1 << 24;    // (a launch counts its threads in 32 bits)
}
bool is_big(int dtype, int64_t M, int64_t N) { return dtype != TAMD_F32 && (double)M * N * 8 >= 64e6; }
bool whole(const void *p, int64_t stride_bytes, int by) { return ((uintptr_t)p | (uintptr_t)stride_bytes) % by == 0; }
bool plain(int dt) { return dt == TAMD_F32 || dt == TAMD_BF16 || dt == TAMD_F16; }

}  // namespace

extern "C" int tamd_swiglu_checkpoint(const void *a, int dtype, int64_t M, int64_t N, int64_t a_stride, void *out, int64_t out_stride, uint8_t *values,
                                      int64_t values_stride, uint8_t *scales, int64_t scales_stride, float alpha, float limit, int has_limit, void *stream) {
  if (M < 0 || N < 0 || a_stride < 0 || out_stride < 0 || values_stride < 0 || scales_stride < 0 || (has_limit && !(limit >= 0.f))) return TAMD_E_INVALID;
  if (!plain(dtype)) return TAMD_E_UNSUPPORTED;
  if (M == 0 || N == 0) return 0;
  if (!a || !out || !values || !scales) return TAMD_E_INVALID;
  const int size = dtype == TAMD_F32 ? 4 : 2;
  if (!whole(a, 0, size) || !whole(out, 0, size)) return TAMD_E_ALIGNMENT;
  if (M >= ((int64_t)1 << 31) || N >= ((int64_t)1 << 30)) return TAMD_E_TOO_LARGE;
  const bool aligned = N % 4 == 0 && whole(a, a_stride * size, 16) && whole(out, out_stride * size, 4 * size) && whole(values, values_stride, 8);
  const bool big = is_big(dtype, M, N);
  GluShape sh;
  unsigned blocks;
  if (!shape(sh, M, N, alpha, limit, has_limit, big, blocks)) return TAMD_E_TOO_LARGE;
  hipStream_t st = (hipStream_t)stream;
  const auto go = [&](auto dt, auto al, auto large) {
    constexpr int DT = decltype(dt)::value;
    checkpoint_kernel<DT, decltype(al)::value, DT != TAMD_F32 && decltype(large)::value>
        <<<blocks, 256, 0, st>>>(a, a_stride, out, out_stride, values, values_stride, scales, scales_stride, sh);
  };
  const auto with = [&](auto dt) {
    const std::true_type yes;
    const std::false_type no;
    if (big) aligned ? go(dt, yes, yes) : go(dt, no, yes);
    else aligned ? go(dt, yes, no) : go(dt, no, no);
  };
  if (dtype == TAMD_F32) with(std::integral_constant<int, TAMD_F32>());
  else if (dtype == TAMD_BF16) with(std::integral_constant<int, TAMD_BF16>());
  else with(std::integral_constant<int, TAMD_F16>());
  return launch_status();
}

extern "C" int tamd_swiglu_backward(const void *dout, int dtype, int64_t M, int64_t N, int64_t dout_stride, const uint8_t *values, int64_t values_stride,
                                    const uint8_t *scales, int64_t scales_stride, void *da, int64_t da_stride, void *out, int64_t out_stride, float alpha,
                                    float limit, int has_limit, void *stream) {
  if (M < 0 || N < 0 || dout_stride < 0 || values_stride < 0 || scales_stride < 0 || da_stride < 0 || out_stride < 0 || (has_limit && !(limit >= 0.f)))
    return TAMD_E_INVALID;
  if (!plain(dtype)) return TAMD_E_UNSUPPORTED;
  if (M == 0 || N == 0) return 0;
  if (!dout || !values || !scales || !da) return TAMD_E_INVALID;
  const int size = dtype == TAMD_F32 ? 4 : 2;
  if (!whole(dout, 0, size) || !whole(da, 0, size) || !whole(out, 0, size)) return TAMD_E_ALIGNMENT;
  if (M >= ((int64_t)1 << 31) || N >= ((int64_t)1 << 30)) return TAMD_E_TOO_LARGE;
  const bool aligned = N % 4 == 0 && whole(dout, dout_stride * size, 4 * size) && whole(da, da_stride * size, 16) && whole(values, values_stride, 8) &&
                       (!out || whole(out, out_stride * size, 4 * size));
  const bool big = is_big(dtype, M, N);
  GluShape sh;
  unsigned blocks;
  if (!shape(sh, M, N, alpha, limit, has_limit, big, blocks)) return TAMD_E_TOO_LARGE;
  hipStream_t st = (hipStream_t)stream;
  const auto go = [&](auto dt, auto al, auto again, auto large) {
    constexpr int DT = decltype(dt)::value;
    backward_kernel<DT, decltype(al)::value, decltype(again)::value, DT != TAMD_F32 && decltype(large)::value>
        <<<blocks, 256, 0, st>>>(dout, dout_stride, values, values_stride, scales, scales_stride, da, da_stride, out, out_stride, sh);
  };
  const auto with = [&](auto dt) {
    const std::true_type yes;
    const std::false_type no;
    if (big && aligned) out ? go(dt, yes, yes, yes) : go(dt, yes, no, yes);
    else if (big) out ? go(dt, no, yes, yes) : go(dt, no, no, yes);
    else if (aligned) out ? go(dt, yes, yes, no) : go(dt, yes, no, no);
    else out ? go(dt, no, yes, no) : go(dt, no, no, no);
  };
  if (dtype == TAMD_F32) with(std::integral_constant<int, TAMD_F32>());
  else if (dtype == TAMD_BF16) with(std::integral_constant<int, TAMD_BF16>());
  else with(std::integral_constant<int, TAMD_F16>());
  return launch_status();
}
