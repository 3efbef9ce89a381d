// A whole mixture-of-experts layer for a few tokens in two launches: 16-bit activations x MXFP4 weights.
//
//   y[t] = sum_j g[t,j] * (W2[e]^T h[t,j] + b2[e]),   h[t,j] = swiglu(W1[e]^T x[t] + b1[e]),   e = pick j of token t,
//
// g the softmax over a token's k largest logits.  Every picked expert's weights are read once (more than 16 tokens on one
// expert: its up projection once per 16), so with a handful of rows per expert the layer is bound by HBM; what counts next
// to the bytes are launches and the latencies in front of the first weight.
//
//   moe_up_kernel    every workgroup picks the experts by itself (a few hundred logits, no launch for them), then walks
//                    over (picked expert, strip of 32 columns = 16 gate / linear pairs).  Its eight waves split K; the partial
//                    sums meet in LDS; h times its gate weight goes to memory.
//   moe_down_kernel  a workgroup owns 16 columns of y.  Its sixteen waves cut the list of (picked expert, 128 K) into equal
//                    parts; a row of the matrix cores' tile is a token, so the sum over the experts is the sum in the
//                    accumulators: no partial results in memory, no atomics, one rounding.
//
// h is kept as two 16-bit planes, its rounding and what that leaves (16 bits more), each a row of its own in the tile of the
// down projection: with up to eight tokens these rows are there anyhow, and the layer's error is that of its one rounding
// at the end.  The gate weights enter h in float32 before that.
//
// v_mfma_f32_16x16x32: lane (c = lane % 16, h = lane / 16) is row c of A and column c of B.  A block of 128 K is read as
// 16 bytes (32 codes, one scale) per lane: lane (c, h) takes group h of column c, consumed 8 K at a time by four MFMAs.
// Both value layouts serve it: in 4 KB blocks a wave's load is one run of 1 KB, with strided columns 16 runs of 64 bytes.
#pragma once
#include "moe_matmul_stream.h"

namespace tamd {

constexpr int kMoeTokens = 64;     // a token is a bit of a 64-bit mask per expert
constexpr int kMoeExperts = 512;   // one thread each
constexpr int kMoePicks = 16;
constexpr int kMoeSlots = 512;     // picks of all tokens
constexpr uint32_t kMoeOob = 0x7FFFFFF0u;   // past the end of every buffer: such a load gives zeros

// What the first launch hands to the second, at the start of the workspace.
struct MoeTables {
  int32_t n_active;
  int32_t pad[3];
  uint64_t mask[kMoeExperts];       // of the picked experts in ascending order: their tokens
  uint16_t expert[kMoeExperts];
  uint16_t start[kMoeExperts];      // first row of the expert's tokens in h
  float gate[kMoeSlots];            // [T, k]
  uint16_t pick[kMoeSlots];
};
constexpr int64_t kMoeTableBytes = (sizeof(MoeTables) + 255) / 256 * 256;

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

// Loads through a buffer descriptor: an offset past `bytes` gives zeros, so that masks cost no branch.
struct Buffer {
  __amdgpu_buffer_rsrc_t r;
  TAMD_DEVICE Buffer(const void *base, int64_t bytes)
      : r(__builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), 0, (uint32_t)(bytes < 0x7FFFFFF0 ? bytes : 0x7FFFFFF0), 0x00020000)) {}
  template <int NT = 0>
  TAMD_DEVICE u32x4_t load16(uint32_t off, uint32_t uniform = 0) const { return __builtin_amdgcn_raw_buffer_load_b128(r, off, uniform, NT); }
  TAMD_DEVICE u32x2_t load8(uint32_t off, uint32_t uniform = 0) const { return __builtin_amdgcn_raw_buffer_load_b64(r, off, uniform, 0); }
  TAMD_DEVICE uint32_t load4(uint32_t off, uint32_t uniform = 0) const { return __builtin_amdgcn_raw_buffer_load_b32(r, off, uniform, 0); }
  TAMD_DEVICE uint32_t load2(uint32_t off, uint32_t uniform = 0) const { return (uint32_t)__builtin_amdgcn_raw_buffer_load_b16(r, off, uniform, 0); }
  TAMD_DEVICE uint32_t load1(uint32_t off, uint32_t uniform = 0) const { return (uint32_t)__builtin_amdgcn_raw_buffer_load_b8(r, off, uniform, 0); }
};

TAMD_DEVICE uint64_t uniform64(uint64_t v) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)v) | (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(v >> 32)) << 32;
}

template <int XDT>
TAMD_DEVICE typename Mma<XDT>::frag_t as_frag(u32x4_t v) { return __builtin_bit_cast(typename Mma<XDT>::frag_t, v); }

// One expert's weights of one product as the lanes of a wave read them.  BLOCKS / SHUFFLED: values in 4 KB blocks, scales in the
// CDNA4 pre-shuffle; else both contiguous along K, column by column.
template <bool BLOCKS, bool SHUFFLED>
struct ExpertWeights {
  Buffer w, sc;
  uint32_t groups, n_kb, col_bytes, sc_col;
  TAMD_DEVICE ExpertWeights(const tamd_moe_weights &p, int e, int K, int N)
      : w((const uint8_t *)p.w + e * p.w_stride_e, BLOCKS ? (int64_t)((N + 63) / 64) * ((K + 127) / 128) * 4096 : (int64_t)(N - 1) * p.w_stride_n + K / 2),
        sc(p.scale + e * p.scale_stride_e, SHUFFLED ? (int64_t)(N / 32) * ((K + 255) / 256) * 256 : (int64_t)(N - 1) * p.scale_stride_n + K / 32),
        groups((uint32_t)K / 32u), n_kb((uint32_t)(K + 127) / 128u), col_bytes((uint32_t)p.w_stride_n), sc_col((uint32_t)p.scale_stride_n) {}

  // 32 codes of column 32 * strip + 2 c + f, K 128 kb + 32 h ..; zeros past K
  TAMD_DEVICE u32x4_t codes(uint32_t strip, uint32_t f, uint32_t kb, uint32_t c, uint32_t h) const {
    if constexpr (BLOCKS) {
      const uint32_t slot = h ^ ((c >> 2) & 3u) ^ (2u * f);
      return w.template load16<2>((c + 32u * f + 16u * (strip & 1u)) * 64u + slot * 16u, ((strip >> 1) * n_kb + kb) * 4096u);
    } else {
      return w.template load16<2>(4u * kb + h < groups ? (32u * strip + 2u * c + f) * col_bytes + 64u * kb + 16u * h : kMoeOob);
    }
  }
  // their scale, as a dword whose byte `scale_shift` is it
  TAMD_DEVICE void scales2(uint32_t strip, uint32_t kb, uint32_t c, uint32_t h, uint32_t &s0, uint32_t &s1) const {
    if constexpr (SHUFFLED) {
      const u32x2_t v = sc.load8(64u * h + 4u * ((2u * c) & 15u), (strip * ((groups + 7u) / 8u) + (kb >> 1)) * 256u);
      s0 = v.x, s1 = v.y;
    } else {
      const uint32_t g = 4u * kb + h, at = (32u * strip + 2u * c) * sc_col + g;
      s0 = sc.load1(g < groups ? at : kMoeOob);
      s1 = sc.load1(g < groups ? at + sc_col : kMoeOob);
    }
  }
  TAMD_DEVICE uint32_t scale1(uint32_t strip, uint32_t f, uint32_t kb, uint32_t c, uint32_t h) const {
    if constexpr (SHUFFLED) {
      const uint32_t n = 2u * c + f;
      return sc.load1(64u * h + 4u * (n & 15u) + 2u * (kb & 1u) + (n >> 4), (strip * ((groups + 7u) / 8u) + (kb >> 1)) * 256u);
    } else {
      const uint32_t g = 4u * kb + h;
      return sc.load1(g < groups ? (32u * strip + 2u * c + f) * sc_col + g : kMoeOob);
    }
  }
  // the scale as the conversion takes it: a float32 of which only the exponent counts
  TAMD_DEVICE static float factor2(uint32_t word, uint32_t kb, uint32_t c) {
    if constexpr (SHUFFLED) return bits_to_f32((word >> (16u * (kb & 1u) + 8u * (c >> 3)) & 0xFFu) << 23);
    else return bits_to_f32(word << 23);
  }
};

struct MoeRouting {
  uint64_t by_expert[kMoeExperts];   // tokens of an expert
  uint64_t mask[kMoeExperts];        // the picked ones packed
  uint16_t expert[kMoeExperts], start[kMoeExperts], first[kMoeExperts];
  uint16_t pick[kMoeSlots];
  float gate[kMoeSlots], row_gate[kMoeSlots];
  int32_t wave_sum[8];
  int32_t n_active;
};

// Picks of all tokens, by a workgroup of 512 threads.  A wave takes a row at a time, its logits in the lanes' registers; ties go to the
// lower column, order and softmax are those of tamd_topk_forward, the gate weights stay float32.
TAMD_DEVICE void moe_route(const tamd_moe_layer_args &a, MoeRouting &r) {
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  const int E = a.n_experts, k = a.n_picks;
  r.by_expert[tid] = 0;
  sync_threads();
  for (int t = wave; t < a.n_tokens; t += 8) {
    uint32_t key[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int col = j * kWave + lane;
      key[j] = 0;
      if (j * kWave < E) {   // (key 0 stands for no column: the lowest NaN shares the second lowest key)
        const float v = load_any_f32(a.logits, a.logits_dtype, t * a.logits_stride + (col < E ? col : E - 1));
        const uint32_t u = ordered_bits(v);
        key[j] = col < E ? (u > 1u ? u : 1u) : 0u;
      }
    }
    uint32_t top = 0, mine = 0;
    int my_col = 0;
    for (int p = 0; p < k; ++p) {
      uint32_t m = key[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) m = key[j] > m ? key[j] : m;
      m = group_max_u32<kWave>(m);
      int col = 0;
#pragma unroll
      for (int j = 7; j >= 0; --j) {
        const uint64_t at = __ballot(key[j] == m);
        if (at) col = j * kWave + __builtin_ctzll(at);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j * kWave + lane == col) key[j] = 0;
      if (p == 0) top = m;
      if (lane == p) mine = m, my_col = col;
    }
    const float e = lane < k ? expf(logit_of(mine) - logit_of(top)) : 0.f;
    const uint32_t sum = group_reduce<kWave>(f32_to_bits(e), [](uint32_t x, uint32_t y) { return f32_to_bits(bits_to_f32(x) + bits_to_f32(y)); });
    if (lane < k) {
      r.pick[t * k + lane] = (uint16_t)my_col;
      r.gate[t * k + lane] = e / bits_to_f32(sum);
      atomicOr((unsigned long long *)&r.by_expert[my_col], 1ull << t);
    }
  }
  sync_threads();
  // the picked experts in ascending order, and where their rows begin: one scan of both counts
  const uint64_t m = r.by_expert[tid];
  const int both = __popcll(m) + (m ? 1 << 16 : 0), incl = wave_incl_scan(both);
  if (lane == kWave - 1) r.wave_sum[wave] = incl;
  sync_threads();
  int before = incl - both;
#pragma unroll
  for (int w = 0; w < 8; ++w) before += w < wave ? r.wave_sum[w] : 0;
  if (m) {
    const int at = before >> 16;
    r.mask[at] = m;
    r.expert[at] = (uint16_t)tid;
    r.start[at] = (uint16_t)(before & 0xFFFF);
    r.first[tid] = (uint16_t)(before & 0xFFFF);
  }
  if (tid == 511) r.n_active = (before + both) >> 16;
  sync_threads();
  if (tid < a.n_tokens * k) {
    const int e = r.pick[tid], t = tid / k;
    r.row_gate[r.first[e] + __popcll(r.by_expert[e] & ((1ull << t) - 1ull))] = r.gate[tid];
  }
  sync_threads();
}

// swiglu_fast with clamps that leave a NaN as it is.
TAMD_DEVICE float swiglu_keeping_nan(const tamd_moe_layer_args &a, float g, float l) {
  if (a.act_has_limit) {
    g = g > a.act_limit ? a.act_limit : g;
    l = l > a.act_limit ? a.act_limit : l < -a.act_limit ? -a.act_limit : l;
  }
  return swiglu_fast(g, l, a.act_alpha, 0.f, false);
}

// NB blocks of 128 K per wave at a time.
template <int XDT, bool BLOCKS, bool SHUFFLED, int NB>
__global__ __launch_bounds__(512, NB >= 3 ? 2 : 4) void moe_up_kernel(tamd_moe_layer_args a) {
  typedef Mma<XDT> M;
  __shared__ MoeRouting r;
  __shared__ f32x4_t red[8][2][kWave];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  const uint32_t c = lane & 15, h = lane >> 4;
  const int K = a.hidden, I = a.inter;
  moe_route(a, r);
  const int n_active = __builtin_amdgcn_readfirstlane(r.n_active);
  MoeTables *tab = (MoeTables *)a.workspace;
  uint16_t *planes = (uint16_t *)((uint8_t *)a.workspace + kMoeTableBytes);
  if (blockIdx.x == 0) {
    if (tid == 0) tab->n_active = n_active;
    if (tid < n_active) tab->mask[tid] = r.mask[tid], tab->expert[tid] = r.expert[tid], tab->start[tid] = r.start[tid];
    if (tid < a.n_tokens * a.n_picks) tab->gate[tid] = r.gate[tid], tab->pick[tid] = r.pick[tid];
  }
  const uint32_t strips = (uint32_t)I / 16u, n_kb = (uint32_t)(K + 127) / 128u;
  const Buffer x(a.x, (int64_t)(a.n_tokens - 1) * a.x_stride_m * 2 + 2 * K);
  for (uint32_t u = blockIdx.x; u < (uint32_t)n_active * strips; u += gridDim.x) {
    const uint32_t at = u / strips, strip = u % strips;
    const int e = __builtin_amdgcn_readfirstlane((int)r.expert[at]);
    const uint64_t mask = uniform64(r.mask[at]);
    const int rows = __popcll(mask), start = __builtin_amdgcn_readfirstlane((int)r.start[at]);
    const ExpertWeights<BLOCKS, SHUFFLED> w(a.up, e, K, 2 * I);
    // lane m: the m-th token of the expert (each token's lane sends itself there)
    const int rank = __popcll(mask & ((1ull << lane) - 1ull));
    const int token_at = __builtin_amdgcn_ds_permute(4 * ((mask >> lane & 1) ? rank : 63 - (lane - rank)), lane);
    for (int m0 = 0; m0 < rows; m0 += 16) {
      const int token = __builtin_amdgcn_ds_bpermute(4 * (m0 + (int)c), token_at);
      const uint32_t x_row = m0 + (int)c < rows ? (uint32_t)(token * a.x_stride_m * 2) + 64u * h : kMoeOob;
      f32x4_t acc0 = {0.f, 0.f, 0.f, 0.f}, acc1 = acc0;
      for (uint32_t k0 = 0; k0 < n_kb; k0 += 8 * NB) {
        const uint32_t kb0 = k0 + (uint32_t)wave * NB;
        u32x4_t q0[NB], q1[NB], xr[NB][4];
        uint32_t s0[NB], s1[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i)
          if (kb0 + i < n_kb) {
            q0[i] = w.codes(strip, 0, kb0 + i, c, h);
            q1[i] = w.codes(strip, 1, kb0 + i, c, h);
            w.scales2(strip, kb0 + i, c, h, s0[i], s1[i]);
#pragma unroll
            for (int j = 0; j < 4; ++j) xr[i][j] = x.load16(4u * (kb0 + i) + h < w.groups ? x_row + 256u * (kb0 + i) + 16u * j : kMoeOob);
          }
#pragma unroll
        for (int i = 0; i < NB; ++i)
          if (kb0 + i < n_kb) {
            const float f0 = w.factor2(s0[i], kb0 + i, c), f1 = w.factor2(s1[i], kb0 + i, c);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              acc0 = Mma16<XDT>::mma(as_frag<XDT>(xr[i][j]), M::expand(q0[i][j], f0), acc0);
              acc1 = Mma16<XDT>::mma(as_frag<XDT>(xr[i][j]), M::expand(q1[i][j], f1), acc1);
            }
          }
      }
      red[wave][0][lane] = acc0;
      red[wave][1][lane] = acc1;
      sync_threads();
      // row m of the tile, pair c of the strip: element (4 h + i) of lanes (c, h)
      const int m = tid >> 4, pair = tid & 15;
      if (m < 16 && m0 + m < rows) {
        const int from = (m >> 2) * 16 + pair;
        float g = 0.f, l = 0.f;
#pragma unroll
        for (int v = 0; v < 8; ++v) g += ((const float *)&red[v][0][from])[m & 3], l += ((const float *)&red[v][1][from])[m & 3];
        if (a.up.bias) {
          const int64_t b = e * a.up.bias_stride_e + 32 * (int64_t)strip + 2 * pair;
          g += load_any_f32(a.up.bias, a.up.bias_dtype, b);
          l += load_any_f32(a.up.bias, a.up.bias_dtype, b + 1);
        }
        const int row = start + m0 + m;
        const float v = r.row_gate[row] * swiglu_keeping_nan(a, g, l);
        const uint32_t hi = XDT == TAMD_BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v);
        const float rest = v - (XDT == TAMD_BF16 ? bf16_bits_to_f32(hi) : f16_bits_to_f32(hi));
        const float lo = rest - rest == 0.f ? rest : 0.f;   // (infinities leave nothing)
        uint16_t *p = planes + (int64_t)row * 2 * I + 16 * strip + pair;
        p[0] = (uint16_t)hi;
        p[I] = (uint16_t)(XDT == TAMD_BF16 ? f32_to_bf16_bits(lo) : f32_to_f16_bits(lo));
      }
      sync_threads();
    }
  }
}

// MT tiles of 16 rows, which are eight tokens with two planes each.  W waves, U blocks of 128 K requested together.
template <int XDT, bool BLOCKS, bool SHUFFLED, int MT, int U, int W>
__global__ __launch_bounds__(64 * W, W / 4) void moe_down_kernel(tamd_moe_layer_args a) {
  typedef Mma<XDT> M;
  __shared__ uint64_t s_mask[kMoeExperts];
  __shared__ uint16_t s_expert[kMoeExperts], s_start[kMoeExperts], s_pick[kMoeSlots];
  __shared__ float s_gate[kMoeSlots];
  __shared__ f32x4_t red[W][kWave];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  const uint32_t c = lane & 15, h = lane >> 4;
  const int K = a.inter, N = a.hidden;
  const MoeTables *tab = (const MoeTables *)a.workspace;
  const int slots = a.n_tokens * a.n_picks;
  if (tid < slots) {   // (no more experts than slots, no more slots than threads)
    s_mask[tid] = tab->mask[tid], s_expert[tid] = tab->expert[tid], s_start[tid] = tab->start[tid];
    s_gate[tid] = tab->gate[tid], s_pick[tid] = tab->pick[tid];
  }
  const uint32_t n_active = (uint32_t)__builtin_amdgcn_readfirstlane(tab->n_active);
  sync_threads();
  const Buffer planes((const uint8_t *)a.workspace + kMoeTableBytes, (int64_t)slots * 4 * K);
  const uint32_t strip = blockIdx.x >> 1, f = blockIdx.x & 1u, n_kb = (uint32_t)(K + 127) / 128u, total = n_active * n_kb;
  uint32_t item = (uint32_t)((uint64_t)total * (uint32_t)wave / (uint32_t)W);
  const uint32_t end = (uint32_t)((uint64_t)total * (uint32_t)(wave + 1) / (uint32_t)W);
  f32x4_t sum[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) sum[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  while (item < end) {
    const uint32_t at = item / n_kb;
    uint32_t kb = item - at * n_kb;
    const uint32_t kb_end = n_kb - kb < end - item ? n_kb : kb + (end - item);
    item += kb_end - kb;
    const uint64_t mask = uniform64(s_mask[at]);
    const ExpertWeights<BLOCKS, SHUFFLED> w(a.down, __builtin_amdgcn_readfirstlane((int)s_expert[at]), K, N);
    const uint32_t start = s_start[at];
    // row 2 i + p of tile t is plane p of token 8 t + i, if that token picked the expert
    uint32_t row[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int token = 8 * t + (int)(c >> 1);
      const uint32_t at_row = start + (uint32_t)__popcll(mask & ((1ull << token) - 1ull));
      row[t] = (mask >> token & 1) ? (at_row * 2u + (c & 1u)) * (uint32_t)(2 * K) + 64u * h : kMoeOob;
    }
    f32x4_t acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (; kb < kb_end; kb += U) {
      u32x4_t q[U];
      uint32_t s[U];
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (kb + i < kb_end) {
          q[i] = w.codes(strip, f, kb + i, c, h);
          s[i] = w.scale1(strip, f, kb + i, c, h);
        }
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        if (MT > 1 && !((uint32_t)(mask >> (8 * t)) & 0xFFu)) continue;
        u32x4_t xr[U][4];
#pragma unroll
        for (int i = 0; i < U; ++i)
          if (kb + i < kb_end) {
#pragma unroll
            for (int j = 0; j < 4; ++j) xr[i][j] = planes.load16(4u * (kb + i) + h < w.groups ? row[t] + 256u * (kb + i) + 16u * j : kMoeOob);
          }
#pragma unroll
        for (int i = 0; i < U; ++i)
          if (kb + i < kb_end) {
            const float factor = bits_to_f32(s[i] << 23);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[t] = Mma16<XDT>::mma(as_frag<XDT>(xr[i][j]), M::expand(q[i][j], factor), acc[t]);
          }
      }
    }
    // only the rows of the expert's own tokens: its NaN or infinite weights are no other token's
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (mask >> (8 * t + 2 * h + (i >> 1)) & 1) sum[t][i] += acc[t][i];
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    red[wave][lane] = sum[t];
    sync_threads();
    const int i = tid >> 4, col = tid & 15, token = 8 * t + i;   // token i of the tile: elements 2 (i % 2) and the next of lanes (col, i / 2)
    if (i < 8 && token < a.n_tokens) {
      float v = 0.f;
#pragma unroll
      for (int s = 0; s < W; ++s) {
        const float *p = (const float *)&red[s][(i >> 1) * 16 + col] + 2 * (i & 1);
        v += p[0] + p[1];
      }
      const int64_t n = 32 * (int64_t)strip + 2 * col + f;
      if (a.down.bias)
        for (int j = 0; j < a.n_picks; ++j) {
          const int slot = token * a.n_picks + j;
          v = __builtin_fmaf(s_gate[slot], load_any_f32(a.down.bias, a.down.bias_dtype, s_pick[slot] * a.down.bias_stride_e + n), v);
        }
      store_any(a.y, XDT, token * a.y_stride_m + n, v);
    }
    sync_threads();
  }
}

// NB of the up projection: rounds of 8 NB blocks; the fewest blocks' time, then the fewest rounds.
inline int moe_up_nb(int hidden) {
  const int n_kb = (hidden + 127) / 128;
  int best = 1, least = 1 << 30;
  for (int nb = 4; nb >= 1; --nb) {
    const int cost = (n_kb + 8 * nb - 1) / (8 * nb) * nb;
    if (cost < least) least = cost, best = nb;
  }
  return best;
}

template <int XDT, bool BLOCKS, bool SHUFFLED>
int launch_moe_up(const tamd_moe_layer_args &a, hipStream_t st) {
  int cus = 0;
  if (int rc = cu_count(cus)) return rc;
  const int64_t slots = (int64_t)a.n_tokens * a.n_picks, most = (slots < a.n_experts ? slots : a.n_experts) * (a.inter / 16);
  const dim3 grid((unsigned)(most < 2 * cus ? most : 2 * cus));
  switch (moe_up_nb(a.hidden)) {
    case 1: moe_up_kernel<XDT, BLOCKS, SHUFFLED, 1><<<grid, 512, 0, st>>>(a); break;
    case 2: moe_up_kernel<XDT, BLOCKS, SHUFFLED, 2><<<grid, 512, 0, st>>>(a); break;
    case 3: moe_up_kernel<XDT, BLOCKS, SHUFFLED, 3><<<grid, 512, 0, st>>>(a); break;
    default: moe_up_kernel<XDT, BLOCKS, SHUFFLED, 4><<<grid, 512, 0, st>>>(a); break;
  }
  return launch_status();
}

template <int XDT, bool BLOCKS, bool SHUFFLED>
int launch_moe_down(const tamd_moe_layer_args &a, hipStream_t st) {
  const dim3 grid((unsigned)(a.hidden / 16));
  if (a.n_tokens <= 8) moe_down_kernel<XDT, BLOCKS, SHUFFLED, 1, 3, 16><<<grid, 1024, 0, st>>>(a);
  else if (a.n_tokens <= 16) moe_down_kernel<XDT, BLOCKS, SHUFFLED, 2, 2, 16><<<grid, 1024, 0, st>>>(a);
  else if (a.n_tokens <= 32) moe_down_kernel<XDT, BLOCKS, SHUFFLED, 4, 4, 8><<<grid, 512, 0, st>>>(a);
  else moe_down_kernel<XDT, BLOCKS, SHUFFLED, 8, 2, 8><<<grid, 512, 0, st>>>(a);
  return launch_status();
}

template <int XDT>
int moe_layer_of(const tamd_moe_layer_args &a, hipStream_t st) {
  const auto of = [](const tamd_moe_weights &w) { return 2 * (w.w_layout == TAMD_W_CDNA4_BLOCKS) + (w.scale_layout == TAMD_SCALE_CDNA4); };
  int (*const up[4])(const tamd_moe_layer_args &, hipStream_t) = {launch_moe_up<XDT, false, false>, launch_moe_up<XDT, false, true>,
                                                                  launch_moe_up<XDT, true, false>, launch_moe_up<XDT, true, true>};
  int (*const down[4])(const tamd_moe_layer_args &, hipStream_t) = {launch_moe_down<XDT, false, false>, launch_moe_down<XDT, false, true>,
                                                                    launch_moe_down<XDT, true, false>, launch_moe_down<XDT, true, true>};
  if (int rc = up[of(a.up)](a, st)) return rc;
  return down[of(a.down)](a, st);
}

int moe_layer_bf16(const tamd_moe_layer_args &a, hipStream_t st);
int moe_layer_f16(const tamd_moe_layer_args &a, hipStream_t st);

}  // namespace tamd
