// A whole mixture-of-experts layer for a few tokens in two or three launches: 16-bit activations x MXFP4 weights.
//
//   y[t] = sum_j g[t,j] * (W2[e]^T h[t,j] + b2[e]),   h[t,j] = swiglu(W1[e]^T x[t] + b1[e]),   e = pick j of token t,
//
// g the softmax over a token's k largest logits.  Every picked expert's weights are read once (more than 16 tokens on one
// expert: its up projection once per 16), so with a handful of rows per expert the layer is bound by HBM; what counts next
// to the bytes are launches and the latencies in front of the first weight.
//
//   moe_up_kernel    every workgroup picks the experts by itself (a few hundred logits, no launch for them), then walks
//                    over its part of the (picked expert, strip of 32 columns = 16 gate / linear pairs).  Its eight waves split K; the
//                    partial sums meet in LDS; h times its gate weight goes to memory.
//   moe_down_kernel  a workgroup owns 16 columns of y and walks over the picked experts, its eight waves splitting K; the
//                    tokens' sums stay in LDS.  Where that leaves CUs without work the experts of all strips are dealt out evenly.
//   moe_join_kernel  then adds up what several workgroups have of a strip, in a fixed order.
//
// h is kept as two 16-bit planes, its rounding and what that leaves (16 bits more), each a row of its own in the tile of the
// down projection: with up to eight tokens these rows are there anyhow, and the layer's error is that of its one rounding
// at the end.  The gate weights enter h in float32 before that.  With float16 the second plane is 2^11 times as large, which its sums are
// divided by: what a rounding leaves is at most half of the value then, and not lost below float16's smallest step.
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
template <int XDT>
constexpr float kMoeRest = XDT == TAMD_F16 ? 0x1p11f : 1.f;   // of the second plane of h
constexpr uint32_t kMoeOob = 0x7FFFFFF0u;   // past the end of every buffer: such a load gives zeros

// What the first launch hands to the second, at the start of the workspace.
struct MoeTables {
  int32_t n_active;
  int32_t pad[3];
  uint16_t expert[kMoeExperts];     // the picked ones in ascending order
  uint16_t start[kMoeExperts];      // first row of the expert's tokens in h
  float gate[kMoeSlots];            // [T, k]
  uint16_t pick[kMoeSlots];
  uint8_t token[kMoeSlots];         // of a row of h
};
constexpr int64_t kMoeTableBytes = (sizeof(MoeTables) + 255) / 256 * 256;
constexpr int kMoeShares = 256;   // workgroups between which the down projection is dealt out; two partial sums of 16 columns each, behind h

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

template <int XDT>
TAMD_DEVICE typename Mma<XDT>::frag_t as_frag(u32x4_t v) { return __builtin_bit_cast(typename Mma<XDT>::frag_t, v); }

// What is added to an offset: nothing, or what takes it past the end.  Hidden from the compiler, which otherwise branches around the
// loads; behind a branch it no longer knows how many requests are outstanding and waits for all of them.
TAMD_DEVICE uint32_t dead_unless(bool there) {
  uint32_t d = there ? 0u : kMoeOob;
  asm volatile("" : "+s"(d));
  return d;
}

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

  // 32 codes of column 32 * strip + 2 c + f, K 128 kb + 32 h ..; zeros past K.  `dead` is added to every offset: kMoeOob for what is not there
  // (see dead_unless).
  TAMD_DEVICE u32x4_t codes(uint32_t strip, uint32_t f, uint32_t kb, uint32_t c, uint32_t h, uint32_t dead) const {
    if constexpr (BLOCKS) {
      const uint32_t slot = h ^ ((c >> 2) & 3u) ^ (2u * f);
      return w.template load16<2>(dead + (c + 32u * f + 16u * (strip & 1u)) * 64u + slot * 16u, ((strip >> 1) * n_kb + kb) * 4096u);
    } else {
      return w.template load16<2>(4u * kb + h < groups ? dead + (32u * strip + 2u * c + f) * col_bytes + 64u * kb + 16u * h : kMoeOob);
    }
  }
  // the scales of columns 2 c and 2 c + 1 of a strip, each as a dword that `factor2` takes it from
  TAMD_DEVICE void scales2(uint32_t strip, uint32_t kb, uint32_t c, uint32_t h, uint32_t dead, uint32_t &s0, uint32_t &s1) const {
    if constexpr (SHUFFLED) {
      const u32x2_t v = sc.load8(dead + 64u * h + 4u * ((2u * c) & 15u), (strip * ((groups + 7u) / 8u) + (kb >> 1)) * 256u);
      s0 = v.x, s1 = v.y;
    } else {
      const uint32_t g = 4u * kb + h, at = dead + (32u * strip + 2u * c) * sc_col + g;
      s0 = sc.load1(g < groups ? at : kMoeOob);
      s1 = sc.load1(g < groups ? at + sc_col : kMoeOob);
    }
  }
  // the same of one column (f) in parts: what depends on the lane, and the scalar offset of a block; nothing is masked
  TAMD_DEVICE uint32_t code_offset(uint32_t strip, uint32_t f, uint32_t c, uint32_t h) const {
    return BLOCKS ? (c + 32u * f + 16u * (strip & 1u)) * 64u + (h ^ ((c >> 2) & 3u) ^ (2u * f)) * 16u : (32u * strip + 2u * c + f) * col_bytes + 16u * h;
  }
  TAMD_DEVICE uint32_t code_block(uint32_t strip, uint32_t kb) const { return BLOCKS ? ((strip >> 1) * n_kb + kb) * 4096u : 64u * kb; }
  TAMD_DEVICE uint32_t scale_offset(uint32_t strip, uint32_t f, uint32_t c, uint32_t h) const {
    const uint32_t n = 2u * c + f;
    return SHUFFLED ? 64u * h + 4u * (n & 15u) + (n >> 4) : (32u * strip + n) * sc_col + h;
  }
  TAMD_DEVICE uint32_t scale_block(uint32_t strip, uint32_t kb) const {
    return SHUFFLED ? (strip * ((groups + 7u) / 8u) + (kb >> 1)) * 256u + 2u * (kb & 1u) : 4u * kb;
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
  uint8_t row_token[kMoeSlots];
  int32_t wave_sum[8];
  int32_t n_active;
};

// Picks of a wave's tokens, a row's logits EPL per lane; ties go to the lower column, order and softmax are those of
// tamd_topk_forward, the gate weights stay float32.
template <int EPL>
TAMD_DEVICE void moe_pick(const tamd_moe_layer_args &a, MoeRouting &r, int wave, int lane) {
  const int E = a.n_experts, k = a.n_picks;
  for (int t = wave; t < a.n_tokens; t += 8) {
    uint32_t key[EPL];
#pragma unroll
    for (int j = 0; j < EPL; ++j) {   // (key 0 stands for no column: the lowest NaN shares the second lowest key)
      const int col = j * kWave + lane;
      const uint32_t u = ordered_bits(load_any_f32(a.logits, a.logits_dtype, t * a.logits_stride + (col < E ? col : E - 1)));
      key[j] = col < E ? (u > 1u ? u : 1u) : 0u;
    }
    uint32_t top = 0, mine = 0;
    int my_col = 0;
    for (int p = 0; p < k; ++p) {
      uint32_t m = key[0];
#pragma unroll
      for (int j = 1; j < EPL; ++j) m = key[j] > m ? key[j] : m;
      m = group_max_u32<kWave>(m);
      int col = 0;
#pragma unroll
      for (int j = EPL - 1; j >= 0; --j) {
        const uint64_t at = __ballot(key[j] == m);
        if (at) col = j * kWave + __builtin_ctzll(at);
      }
#pragma unroll
      for (int j = 0; j < EPL; ++j)
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
}

// Routing of all tokens, by a workgroup of 512 threads, a wave per row.
TAMD_DEVICE void moe_route(const tamd_moe_layer_args &a, MoeRouting &r) {
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  const int E = a.n_experts, k = a.n_picks;
  r.by_expert[tid] = 0;
  sync_threads();
  if (E <= kWave) moe_pick<1>(a, r, wave, lane);
  else if (E <= 2 * kWave) moe_pick<2>(a, r, wave, lane);
  else moe_pick<8>(a, r, wave, lane);
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
    const int row = r.first[e] + __popcll(r.by_expert[e] & ((1ull << t) - 1ull));
    r.row_gate[row] = r.gate[tid];
    r.row_token[row] = (uint8_t)t;
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

// A workgroup per CU takes a contiguous part of the units (picked expert, strip of 32 columns): consecutive strips of an expert, whose
// rows of x then stay in registers.  Its eight waves split K, NB blocks of 128 each; the weights of two units are in flight
// (48 KB per CU with NB = 3), their partial sums meet in LDS, a barrier per unit.  A stage is a unit, 16 of its rows and 8 * NB
// blocks of K; with ROUNDS (long K, many rows per expert) a unit may have several of K and x travels with the weights.
// As a loop without requests ahead, two workgroups per CU, 16 tokens of 128 experts of 2880 x 5760 took 154 us, 76 so: 5.9 TB/s.
template <int XDT, bool BLOCKS, bool SHUFFLED, int NB, bool ROUNDS>
__global__ __launch_bounds__(512, 2) void moe_up_kernel(tamd_moe_layer_args a) {
  typedef Mma<XDT> M;
  __shared__ MoeRouting r;
  __shared__ f32x4_t red[2][8][2][kWave];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  const uint32_t c = lane & 15, h = lane >> 4;
  const int K = a.hidden, I = a.inter;
  moe_route(a, r);
  const int n_active = __builtin_amdgcn_readfirstlane(r.n_active);
  MoeTables *tab = (MoeTables *)a.workspace;
  uint16_t *planes = (uint16_t *)((uint8_t *)a.workspace + kMoeTableBytes);
  if (blockIdx.x == 0) {
    if (tid == 0) tab->n_active = n_active;
    if (tid < n_active) tab->expert[tid] = r.expert[tid], tab->start[tid] = r.start[tid];
    if (tid < a.n_tokens * a.n_picks) tab->gate[tid] = r.gate[tid], tab->pick[tid] = r.pick[tid], tab->token[tid] = r.row_token[tid];
  }
  const uint32_t strips = (uint32_t)I / 16u, n_kb = (uint32_t)(K + 127) / 128u, units = (uint32_t)n_active * strips;
  const uint32_t unit0 = (uint32_t)((uint64_t)units * blockIdx.x / gridDim.x), unit1 = (uint32_t)((uint64_t)units * (blockIdx.x + 1) / gridDim.x);
  if (unit0 == unit1) return;
  const Buffer x(a.x, (int64_t)(a.n_tokens - 1) * a.x_stride_m * 2 + 2 * K);
  const int total_rows = a.n_tokens * a.n_picks;
  const auto first_row = [&](uint32_t at) { return (int)r.start[at]; };
  const auto end_row = [&](uint32_t at) { return (int)at + 1 < n_active ? (int)r.start[at + 1] : total_rows; };

  struct Cursor {
    uint32_t unit, at, strip, k0;
    int m0;
  };
  // With ROUNDS a unit's stages follow each other; else all strips of an expert come before its next 16 rows: x stays.
  const auto advance = [&](Cursor &p) {
    if constexpr (ROUNDS) {
      p.k0 += 8 * NB;
      if (p.k0 < n_kb) return;
      p.k0 = 0;
      p.m0 += 16;
      if (p.m0 < __builtin_amdgcn_readfirstlane(end_row(p.at) - first_row(p.at))) return;
      p.m0 = 0;
    }
    ++p.unit, ++p.strip;
    if (!ROUNDS && (p.strip == strips || p.unit == unit1) && p.m0 + 16 < __builtin_amdgcn_readfirstlane(end_row(p.at) - first_row(p.at))) {
      const uint32_t first = p.at * strips > unit0 ? p.at * strips : unit0;
      p.m0 += 16, p.strip -= p.unit - first, p.unit = first;
    } else if (p.strip == strips) {
      p.strip = 0, p.m0 = 0, ++p.at;
    }
  };
  struct Stage {
    u32x4_t q0[NB], q1[NB], x[ROUNDS ? NB : 1][4];
    uint32_t s0[NB], s1[NB];
    u32x2_t bias;   // of the pair tid % 16 of the strip: two float32, or two 16-bit numbers in the first dword
  };
  const bool bias_f32 = a.up.bias_dtype == TAMD_F32;
  const int bias_bytes = a.up.bias ? (bias_f32 ? 4 : 2) : 0;
  const auto request_x = [&](u32x4_t (&to)[ROUNDS ? NB : 1][4], int i, const Cursor &p, uint32_t x_row, uint32_t dead) {
    const uint32_t kb = p.k0 + (uint32_t)wave * NB + i;
#pragma unroll
    for (int j = 0; j < 4; ++j) to[i][j] = x.load16(4u * kb + h < (uint32_t)K / 32u ? dead + x_row + 256u * kb + 16u * j : kMoeOob);
  };
  const auto x_row_of = [&](const Cursor &p) {   // row c of the tile: the byte offset of its token's x
    const int row = __builtin_amdgcn_readfirstlane(first_row(p.at)) + p.m0 + (int)c;
    return row < __builtin_amdgcn_readfirstlane(end_row(p.at)) ? (uint32_t)r.row_token[row] * (uint32_t)(2 * a.x_stride_m) + 64u * h : kMoeOob;
  };
  const auto request = [&](Stage &s, Cursor &p) {
    const bool live = p.unit < unit1;
    const uint32_t at = live ? p.at : 0u;
    const int e = __builtin_amdgcn_readfirstlane((int)r.expert[at]);
    const ExpertWeights<BLOCKS, SHUFFLED> w(a.up, e, K, 2 * I);
    uint32_t x_row = 0;
    if constexpr (ROUNDS) x_row = x_row_of(Cursor{p.unit, at, p.strip, p.k0, p.m0});
    const Buffer bias((const uint8_t *)a.up.bias + e * a.up.bias_stride_e * bias_bytes, 2 * (int64_t)I * bias_bytes);
    s.bias = bias.load8((16u * p.strip + (uint32_t)(tid & 15)) * 2u * (uint32_t)bias_bytes);
    __builtin_amdgcn_sched_barrier(0);   // (one order wherever this is expanded: the waits are counted from it)
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const uint32_t kb = p.k0 + (uint32_t)wave * NB + i, dead = dead_unless(live && kb < n_kb);
      s.q0[i] = w.codes(p.strip, 0, kb, c, h, dead);
      __builtin_amdgcn_sched_barrier(0);
      s.q1[i] = w.codes(p.strip, 1, kb, c, h, dead);
      __builtin_amdgcn_sched_barrier(0);
      w.scales2(p.strip, kb, c, h, dead, s.s0[i], s.s1[i]);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (ROUNDS) {
        request_x(s.x, i, p, x_row, dead);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (live) advance(p);
  };

  Cursor ask, now;
  ask.unit = unit0, ask.at = unit0 / strips, ask.strip = unit0 % strips, ask.k0 = 0, ask.m0 = 0;
  now = ask;
  u32x4_t xr[ROUNDS ? 1 : NB][4];
  uint32_t x_at = 0xFFFFFFFFu;
  int x_m0 = 0;
  f32x4_t acc0 = {0.f, 0.f, 0.f, 0.f}, acc1 = acc0;
  uint32_t turn = 0;
  const auto load_x = [&]() {
    if constexpr (!ROUNDS) {
      const uint32_t x_row = x_row_of(now);
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const uint32_t kb = (uint32_t)wave * NB + i;
#pragma unroll
        for (int j = 0; j < 4; ++j) xr[i][j] = x.load16(4u * kb + h < (uint32_t)K / 32u ? x_row + 256u * kb + 16u * j : kMoeOob);
      }
      // awaited here: behind the branch the compiler would have to await everything in every stage
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) asm volatile("" : "+v"(xr[i][j]));
      x_at = now.at, x_m0 = now.m0;
    }
  };
  const auto multiply = [&](const Stage &s) {
    const bool live = now.unit < unit1;
    if constexpr (!ROUNDS)
      if (live && (x_at != now.at || x_m0 != now.m0)) load_x();
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const uint32_t kb = now.k0 + (uint32_t)wave * NB + i;
      const float f0 = ExpertWeights<BLOCKS, SHUFFLED>::factor2(s.s0[i], kb, c), f1 = ExpertWeights<BLOCKS, SHUFFLED>::factor2(s.s1[i], kb, c);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u32x4_t xv;
        if constexpr (ROUNDS) xv = s.x[i][j];
        else xv = xr[i][j];
        acc0 = Mma16<XDT>::mma(as_frag<XDT>(xv), M::expand(s.q0[i][j], f0), acc0);
        acc1 = Mma16<XDT>::mma(as_frag<XDT>(xv), M::expand(s.q1[i][j], f1), acc1);
      }
    }
    const Cursor done = now;
    if (live) advance(now);
    if (ROUNDS && now.k0 != 0) return;   // (more of this unit's K)
    red[turn][wave][0][lane] = acc0;
    red[turn][wave][1][lane] = acc1;
    acc0 = acc1 = f32x4_t{0.f, 0.f, 0.f, 0.f};
    sync_threads();
    // row m of the tile, pair of the strip: element m % 4 of lanes (pair, m / 4)
    const uint32_t done_at = live ? done.at : 0u;
    const int m = tid >> 4, pair = tid & 15, row = first_row(done_at) + done.m0 + m;
    if (live && m < 16 && row < end_row(done_at)) {
      const int from = (m >> 2) * 16 + pair;
      float g = 0.f, l = 0.f;
#pragma unroll
      for (int v = 0; v < 8; ++v) g += ((const float *)&red[turn][v][0][from])[m & 3], l += ((const float *)&red[turn][v][1][from])[m & 3];
      g += bias_f32 ? bits_to_f32(s.bias.x) : a.up.bias_dtype == TAMD_BF16 ? bf16_bits_to_f32(s.bias.x & 0xFFFFu) : f16_bits_to_f32(s.bias.x & 0xFFFFu);
      l += bias_f32 ? bits_to_f32(s.bias.y) : a.up.bias_dtype == TAMD_BF16 ? bf16_bits_to_f32(s.bias.x >> 16) : f16_bits_to_f32(s.bias.x >> 16);
      const float v = r.row_gate[row] * swiglu_keeping_nan(a, g, l);
      const uint32_t hi = XDT == TAMD_BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v);
      const float rest = v - (XDT == TAMD_BF16 ? bf16_bits_to_f32(hi) : f16_bits_to_f32(hi));
      const float lo = rest - rest == 0.f ? kMoeRest<XDT> * rest : 0.f;   // (infinities leave nothing)
      uint16_t *p = planes + (int64_t)row * 2 * I + 16 * done.strip + pair;
      p[0] = (uint16_t)hi;
      p[I] = (uint16_t)(XDT == TAMD_BF16 ? f32_to_bf16_bits(lo) : f32_to_f16_bits(lo));
    }
    turn ^= 1;   // (the next stage's sums go to the other half: one barrier between two uses of either)
  };

  load_x();
  Stage s0, s1;
  request(s0, ask);
  request(s1, ask);
  while (now.unit < unit1) {
    multiply(s0);
    request(s0, ask);
    multiply(s1);   // (possibly of nothing: with a way out in between the compiler would await all requests of a round)
    request(s1, ask);
  }
}

struct MoeDownLds {
  float gate[kMoeSlots];
  uint16_t expert[kMoeExperts], start[kMoeExperts + 8], pick[kMoeSlots];
  uint8_t token[kMoeSlots];
};
static_assert(sizeof(MoeDownLds) % 16 == 0);
// The experts of all strips of 16 columns, strip by strip, are dealt out evenly to up to `shares` workgroups, none of which has none:
// where one begins, and whose an expert of a strip is.  (Less than 2^24 of them, so that 32 bits do.  Divisions of 64 take as long: 5 tokens of 32
// experts of 2016 x 1056 15.2 us for the down projection and 3.9 for the join either way.)
constexpr int64_t kMoeDealt = 1 << 24;
struct MoeDeal {
  uint32_t items, shares;
  TAMD_DEVICE MoeDeal(uint32_t n_active, int N, uint32_t shares_) : items(n_active * ((uint32_t)N / 16u)), shares(shares_ < items ? shares_ : items) {}
  TAMD_DEVICE uint32_t begin(uint32_t w) const { return items * w / shares; }
  TAMD_DEVICE uint32_t owner(uint32_t at) const { return ((at + 1u) * shares - 1u) / items; }
};
__host__ __device__ inline int64_t moe_partial_at(int64_t slots, int64_t inter) { return kMoeTableBytes + (slots * inter * 4 + 15) / 16 * 16; }

template <int NB, int RC>
constexpr int kMoeDownPitch = 256 * NB + 16;   // bytes of a row of h in a wave's buffer (rows 16 bytes apart on the banks)

// A workgroup has 16 columns of y at a time, all of the picked experts or (DEALT) some of them; its eight waves split K, NB blocks of 128 each, and walk over
// the experts with the weights of D of them in flight.  A row of a tile is a plane of one of the expert's tokens, RC tokens at a time; when these are multiplied
// a wave adds the tokens' sums to its own copy of the output in LDS, where the copies are added up at last: no atomics, and
// NaN or infinite weights stay with the tokens that picked them.
//
// h comes as a few dense requests and goes through LDS, a buffer per wave, to where the MFMAs want it: requested in their layout
// it takes four requests per block, most lanes of which bring nothing, and a request costs the CU about 20 cycles whatever it
// brings (16 tokens of 128 experts of 2880 x 2880: 90 us, 53 so, and 49 dealt out, 4.6 TB/s).
template <int XDT, bool BLOCKS, bool SHUFFLED, int NB, int RC, int D, bool ROUNDS, bool DEALT>
__global__ __launch_bounds__(512, 2) void moe_down_kernel(tamd_moe_layer_args a) {
  typedef Mma<XDT> M;
  typedef ExpertWeights<BLOCKS, SHUFFLED> Weights;
  constexpr int W = 8, PITCH = kMoeDownPitch<NB, RC>, XR = NB * RC / 2 > 0 ? (NB * RC + 1) / 2 : 1;   // dense requests of 2 RC rows
  constexpr int NS = SHUFFLED ? NB / 2 + 1 : NB;   // scale requests: a dword of the pre-shuffle serves blocks 2 i and 2 i + 1
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  MoeDownLds &s = *(MoeDownLds *)lds;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  uint8_t *const rows_lds = lds + sizeof(MoeDownLds) + wave * (2 * RC * PITCH);
  float *const sums = (float *)(lds + sizeof(MoeDownLds) + W * (2 * RC * PITCH));   // [W, n_tokens, 16]
  const uint32_t c = lane & 15, h = lane >> 4;
  const int K = a.inter, N = a.hidden, T = a.n_tokens;
  const MoeTables *tab = (const MoeTables *)a.workspace;
  const int slots = T * a.n_picks;
  const uint32_t n_active = (uint32_t)__builtin_amdgcn_readfirstlane(tab->n_active);
  uint32_t strip = blockIdx.x, ask_at = 0, left = n_active;   // from this expert of this strip on, so many experts of strips
  if constexpr (DEALT) {
    const MoeDeal deal(n_active, N, gridDim.x);
    if (blockIdx.x >= deal.shares) return;
    const uint32_t begin = deal.begin(blockIdx.x);
    strip = begin / n_active, ask_at = begin - strip * n_active, left = deal.begin(blockIdx.x + 1) - begin;
  }
  if (tid < slots) {   // (no more experts than slots)
    s.expert[tid] = tab->expert[tid], s.start[tid] = (uint32_t)tid < n_active ? tab->start[tid] : (uint16_t)slots;
    s.gate[tid] = tab->gate[tid], s.pick[tid] = tab->pick[tid], s.token[tid] = tab->token[tid];
  }
  if (tid == 0) s.start[slots] = (uint16_t)slots;
  for (int i = tid; i < W * T * 16; i += 64 * W) sums[i] = 0.f;
  sync_threads();
  const Buffer planes((const uint8_t *)a.workspace + kMoeTableBytes, (int64_t)slots * 4 * K);
  const uint32_t n_kb = (uint32_t)(K + 127) / 128u, groups = (uint32_t)K / 32u;

  // ---- a stage is an expert of a strip and, with ROUNDS, 8 NB blocks of K from k0 on; these are cut evenly.  What a lane adds to the offsets
  // depends on the place in K alone: made once, or once per stage with ROUNDS.
  const auto rows_at = [&](uint32_t at, uint32_t &row, uint32_t &rows) {
    row = (uint32_t)__builtin_amdgcn_readfirstlane((int)s.start[at]);
    rows = (uint32_t)__builtin_amdgcn_readfirstlane((int)s.start[at + 1]) - row;
  };
  struct Place {
    uint32_t kb0, code_off[NB], scale_off[NS], x_off[XR];
  };
  const Weights form(a.down, 0, K, N);
  const auto place_at = [&](uint32_t of_16, uint32_t k0) {
    const uint32_t strip = of_16 >> 1, f = of_16 & 1u;
    Place p;
    const uint32_t here = n_kb - k0 < 8u * NB ? n_kb - k0 : 8u * NB, from = here * (uint32_t)wave / W, n = here * (uint32_t)(wave + 1) / W - from;
    p.kb0 = k0 + from;
    const uint32_t code = form.code_offset(strip, f, c, h), scale = form.scale_offset(strip, f, c, h);
#pragma unroll
    for (int i = 0; i < NB; ++i) p.code_off[i] = (uint32_t)i < n && (BLOCKS || 4u * (p.kb0 + i) + h < groups) ? code : kMoeOob;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      if constexpr (SHUFFLED) p.scale_off[i] = 2u * ((p.kb0 >> 1) + i) < n_kb ? scale & ~3u : kMoeOob;   // blocks 2 (kb0 / 2 + i) and the next
      else p.scale_off[i] = (uint32_t)i < n && 4u * (p.kb0 + i) + h < groups ? scale : kMoeOob;
    }
    // 16-byte chunk i * 64 + lane of the rows: row by row, 16 NB chunks each; zeros past K and past this wave's blocks (an infinite h
    // times the zeros in place of another wave's codes would be NaN)
#pragma unroll
    for (int i = 0; i < XR; ++i) {
      const uint32_t chunk = (uint32_t)(i * kWave + lane), of = chunk / (16u * NB), at = chunk % (16u * NB), k = 128u * p.kb0 + 8u * at;
      p.x_off[i] = of < 2u * RC && at < 16u * n && k < (uint32_t)K ? of * (uint32_t)(2 * K) + 2u * k : kMoeOob;
    }
    return p;
  };
  struct Stage {
    u32x4_t q[NB], x[XR];
    uint32_t s[NS];
  };
  const auto request_x = [&](u32x4_t (&to)[XR], const Place &p, uint32_t row, uint32_t rows) {
#pragma unroll
    for (int i = 0; i < XR; ++i) {
      const uint32_t of = (uint32_t)(i * kWave + lane) / (16u * NB);
      uint32_t off = of < 2u * rows ? p.x_off[i] : kMoeOob;
      asm volatile("" : "+v"(off));   // (as in dead_unless)
      to[i] = planes.load16(off, row * (uint32_t)(4 * K));
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // where the next request and the next product are
  uint32_t asked = strip, now_at = ask_at, ask_k0 = 0, now_k0 = 0, to_ask = left, to_do = left;
  Place fixed = place_at(asked, 0);
  const auto request = [&](Stage &st) {
    const bool live = to_ask > 0;
    const uint32_t at = live ? ask_at : 0u;
    Weights w(a.down, __builtin_amdgcn_readfirstlane((int)s.expert[at]), K, N);
    if (!live) w.w = w.sc = Buffer(a.down.w, 0);   // (empty buffers: zeros)
    uint32_t row, rows;
    rows_at(at, row, rows);
    const Place p = ROUNDS ? place_at(asked, ask_k0) : fixed;
    request_x(st.x, p, row, live ? rows : 0u);
    const uint32_t code_s = form.code_block(asked >> 1, p.kb0);
#pragma unroll
    for (int i = 0; i < NB; ++i) {   // (one order wherever this is expanded: the waits are counted from it)
      st.q[i] = w.w.template load16<2>(p.code_off[i], code_s + (BLOCKS ? 4096u : 64u) * i);
      __builtin_amdgcn_sched_barrier(0);
    }
    const uint32_t scale_s = SHUFFLED ? form.scale_block(asked >> 1, p.kb0 & ~1u) : form.scale_block(asked >> 1, p.kb0);
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      if constexpr (SHUFFLED) st.s[i] = w.sc.load4(p.scale_off[i], scale_s + 256u * i);
      else st.s[i] = w.sc.load1(p.scale_off[i], scale_s + 4u * i);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (ROUNDS) {
      ask_k0 += 8 * NB;
      if (ask_k0 < n_kb) return;
      ask_k0 = 0;
    }
    ++ask_at;
    if (live) --to_ask;
    if constexpr (DEALT) {
      if (ask_at >= n_active) {
        ask_at = 0, ++asked;
        if (!ROUNDS) fixed = place_at(asked, 0);
      }
    }
  };
  const uint32_t a_row = wave_lds_offset((c & (2u * RC - 1u)) * PITCH + 64u * h);   // (rows past the buffer's repeat: no one reads their sums)
  const auto multiply = [&](const Stage &st) {
    const bool live = to_do > 0;
    const uint32_t f = strip & 1u;
    uint32_t row, rows;
    rows_at(live ? now_at : 0u, row, rows);
    const Place p = ROUNDS ? place_at(strip, now_k0) : fixed;   // (of `fixed` what lies along K is used: the same for all strips)
    const auto tile = [&](const u32x4_t (&x)[XR], uint32_t t0) {
#pragma unroll
      for (int i = 0; i < XR; ++i) {
        const uint32_t chunk = (uint32_t)(i * kWave + lane), of = chunk / (16u * NB), at = chunk % (16u * NB);
        if (XR * kWave == 2 * RC * 16 * NB || of < 2u * RC) *(u32x4_t *)(rows_lds + of * PITCH + 16u * at) = x[i];
      }
      f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        uint32_t scale;
        if constexpr (SHUFFLED) {
          const uint32_t odd = p.kb0 & 1u, word0 = st.s[i / 2], word1 = st.s[i & 1 ? (i / 2 + 1 < NS ? i / 2 + 1 : i / 2) : i / 2];
          scale = (odd ? word1 : word0) >> (8u * ((2u * c + f) >> 4) + 16u * ((odd + i) & 1u)) & 0xFFu;
        } else {
          scale = st.s[i];
        }
        const float factor = bits_to_f32(scale << 23);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc = Mma16<XDT>::mma(as_frag<XDT>(*(const u32x4_t *)(rows_lds + a_row + 256u * i + 16u * j)), M::expand(st.q[i][j], factor), acc);
      }
      // elements 2 p and 2 p + 1 of lane (c, h) are the planes of token 2 h + p of the tile
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t of = 2u * h + e;
        if (live && of < RC && t0 + of < rows) sums[(wave * T + s.token[row + t0 + of]) * 16 + (int)c] += acc[2 * e] + 1.f / kMoeRest<XDT> * acc[2 * e + 1];
      }
    };
    tile(st.x, 0);
    if (live) {
      for (uint32_t t0 = RC; t0 < rows; t0 += RC) {   // more tokens than are requested ahead
        u32x4_t x[XR];
        request_x(x, p, row + t0, rows - t0);
#pragma unroll
        for (int i = 0; i < XR; ++i) asm volatile("" : "+v"(x[i]));   // awaited here, not behind the branch
        tile(x, t0);
      }
    }
  };

  // ---- the biases of this thread's outputs by their gate weights, eight picks requested at a time
  const auto bias_of = [&](int i) {
    float v = 0.f;
    const int64_t n = 32 * (int64_t)(strip >> 1) + 2 * (i & 15) + (strip & 1u);
    for (int j0 = 0; j0 < a.n_picks; j0 += 8) {
      float b[8], g[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int slot = (i >> 4) * a.n_picks + (j0 + j < a.n_picks ? j0 + j : a.n_picks - 1);
        g[j] = s.gate[slot];
        b[j] = load_any_f32(a.down.bias, a.down.bias_dtype, s.pick[slot] * a.down.bias_stride_e + n);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) v = j0 + j < a.n_picks ? __builtin_fmaf(g[j], b[j], v) : v;
    }
    return v;
  };
  static_assert(kMoeTokens * 16 <= 2 * 64 * W);   // two outputs per thread at most
  bool from_start = !DEALT || now_at == 0;   // the strip's first expert is this workgroup's
  float from_bias[2] = {0.f, 0.f};
  if (a.down.bias && from_start) {
#pragma unroll
    for (int m = 0; m < 2; ++m)
      if (tid + m * 64 * W < T * 16) from_bias[m] = bias_of(tid + m * 64 * W);
  }
  // Behind the strip's last expert here: the waves' sums go to y, or, where other workgroups have experts of it, to the workspace.
  float *const partial = (float *)((uint8_t *)a.workspace + moe_partial_at(slots, K)) + (int64_t)blockIdx.x * 2 * (T * 16);
  const auto finish = [&](bool last) {
    sync_threads();
    const bool whole = !DEALT || (from_start && now_at == n_active);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int i = tid + m * 64 * W;
      if (i < T * 16) {
        float v = from_bias[m];
#pragma unroll
        for (int w = 0; w < W; ++w) v += sums[w * T * 16 + i];
        if (whole) store_any(a.y, XDT, (i >> 4) * a.y_stride_m + 32 * (int64_t)(strip >> 1) + 2 * (i & 15) + (strip & 1u), v);
        else partial[(from_start ? T * 16 : 0) + i] = v;
        if (!last) {
#pragma unroll
          for (int w = 0; w < W; ++w) sums[w * T * 16 + i] = 0.f;
        }
      }
    }
    if (!last) {
      ++strip, now_at = 0, from_start = true;
      if (a.down.bias) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
          if (tid + m * 64 * W < T * 16) from_bias[m] = bias_of(tid + m * 64 * W);
      }
      sync_threads();
    }
  };

  Stage st[D];
#pragma unroll
  for (int d = 0; d < D; ++d) request(st[d]);
  while (to_do > 0) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      multiply(st[d]);
      request(st[d]);
      if (to_do > 0) {
        if (ROUNDS) now_k0 += 8 * NB;
        if (!ROUNDS || now_k0 >= n_kb) {
          now_k0 = 0, ++now_at, --to_do;
          if constexpr (DEALT)
            if (to_do > 0 && now_at == n_active) finish(false);
        }
      }
    }
  }
  finish(true);
}

// Adds up what several workgroups have of 16 columns; those that one has alone are in y already.
template <int XDT>
__global__ __launch_bounds__(256) void moe_join_kernel(tamd_moe_layer_args a, uint32_t shares) {
  const MoeTables *tab = (const MoeTables *)a.workspace;
  const uint32_t n_active = (uint32_t)__builtin_amdgcn_readfirstlane(tab->n_active), strip = blockIdx.x;
  const MoeDeal deal(n_active, a.hidden, shares);
  const uint32_t from = deal.owner(strip * n_active), to = deal.owner(strip * n_active + n_active - 1u);
  if (from == to) return;
  const int outs = a.n_tokens * 16;
  const float *const partial = (const float *)((const uint8_t *)a.workspace + moe_partial_at(a.n_tokens * a.n_picks, a.inter));
  for (int i = threadIdx.x; i < outs; i += 256) {
    float v = partial[(int64_t)(2 * from + 1) * outs + i];
    for (uint32_t w = from + 1; w <= to; ++w) v += partial[(int64_t)(2 * w) * outs + i];
    store_any(a.y, XDT, (i >> 4) * a.y_stride_m + 32 * (int64_t)(strip >> 1) + 2 * (i & 15) + (strip & 1u), v);
  }
}

// Blocks of 128 K per wave: rounds of 8 NB blocks; the fewest blocks' time, then the fewest rounds.
inline int moe_nb(int K) {
  const int n_kb = (K + 127) / 128;
  int best = 1, least = 1 << 30;
  for (int nb = 3; nb >= 1; --nb) {
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
  const dim3 grid((unsigned)(most < cus ? most : cus));
  const int nb = moe_nb(a.hidden);
  if ((int64_t)a.n_tokens * a.n_picks > 8 * (int64_t)a.n_experts || 8 * nb < (a.hidden + 127) / 128) {
    switch (nb) {
      case 1: moe_up_kernel<XDT, BLOCKS, SHUFFLED, 1, true><<<grid, 512, 0, st>>>(a); break;
      case 2: moe_up_kernel<XDT, BLOCKS, SHUFFLED, 2, true><<<grid, 512, 0, st>>>(a); break;
      default: moe_up_kernel<XDT, BLOCKS, SHUFFLED, 3, true><<<grid, 512, 0, st>>>(a); break;
    }
  } else {
    switch (nb) {
      case 1: moe_up_kernel<XDT, BLOCKS, SHUFFLED, 1, false><<<grid, 512, 0, st>>>(a); break;
      case 2: moe_up_kernel<XDT, BLOCKS, SHUFFLED, 2, false><<<grid, 512, 0, st>>>(a); break;
      default: moe_up_kernel<XDT, BLOCKS, SHUFFLED, 3, false><<<grid, 512, 0, st>>>(a); break;
    }
  }
  return launch_status();
}

template <int XDT, bool BLOCKS, bool SHUFFLED, int NB, int RC, int D>
int launch_moe_down_of(const tamd_moe_layer_args &a, hipStream_t st) {
  int cus = 0;
  if (int rc = cu_count(cus)) return rc;
  // One strip per workgroup, or the experts of all strips dealt out: where nine experts or more of a strip that no CU has to do meanwhile are
  // saved the join costs less.  16 tokens of 128 experts of 2880 x 2880 (19 saved) take 129 us and 126, 32 of 32 (10; eight tokens ahead) 138 and 122,
  // 64 of 128 of 512 x 1024 (96) 129 and 74, but 2 of 64 of 1024 x 2048 (8) 23 and 26, one of 2880 x 2880 (1) 22 and 27.
  const int64_t strips = a.hidden / 16, slots = (int64_t)a.n_tokens * a.n_picks, most = slots < a.n_experts ? slots : a.n_experts;
  const int64_t shares = cus < kMoeShares ? cus : kMoeShares;
  const bool rounds = 8 * NB < (a.inter + 127) / 128, dealt = ((strips + shares - 1) / shares * shares - strips) * most >= 9 * shares && strips * most < kMoeDealt;
  const auto kernel = dealt ? (rounds ? moe_down_kernel<XDT, BLOCKS, SHUFFLED, NB, RC, D, true, true> : moe_down_kernel<XDT, BLOCKS, SHUFFLED, NB, RC, D, false, true>)
                            : (rounds ? moe_down_kernel<XDT, BLOCKS, SHUFFLED, NB, RC, D, true, false> : moe_down_kernel<XDT, BLOCKS, SHUFFLED, NB, RC, D, false, false>);
  const size_t lds = sizeof(MoeDownLds) + 8 * 2 * RC * kMoeDownPitch<NB, RC> + (size_t)a.n_tokens * 8 * 16 * 4;
  if (lds > 64 * 1024)
    if (int rc = raise_lds_limit_once((const void *)kernel)) return rc;
  kernel<<<(unsigned)(dealt ? shares : strips), 512, lds, st>>>(a);
  if (dealt) moe_join_kernel<XDT><<<(unsigned)strips, 256, 0, st>>>(a, (uint32_t)shares);
  return launch_status();
}

// Tokens of an expert that are requested ahead: two where more are rare, four, or eight.  Eight of three blocks do not fit the
// registers, and two blocks are two rounds of K for as many columns: there four serve up to six rows on average (32 tokens of 32
// experts of 2880 x 2880: 114 us, 132 with eight; with two blocks or one eight are better from 2.5 on, 64 of 128 of 2048 x 768: 110 and 119).
template <int XDT, bool BLOCKS, bool SHUFFLED, int NB>
int launch_moe_down_nb(const tamd_moe_layer_args &a, hipStream_t st) {
  const float rows = (float)(a.n_tokens * a.n_picks) / (float)a.n_experts;
  if (a.n_tokens <= 2 || rows <= 0.75f) return launch_moe_down_of<XDT, BLOCKS, SHUFFLED, NB, 2, 4>(a, st);
  if (a.n_tokens <= 4 || rows <= (NB == 3 ? 6.f : 2.5f)) return launch_moe_down_of<XDT, BLOCKS, SHUFFLED, NB, 4, 3>(a, st);
  return launch_moe_down_of<XDT, BLOCKS, SHUFFLED, NB < 3 ? NB : 2, 8, 2>(a, st);
}

template <int XDT, bool BLOCKS, bool SHUFFLED>
int launch_moe_down(const tamd_moe_layer_args &a, hipStream_t st) {
  switch (moe_nb(a.inter)) {
    case 1: return launch_moe_down_nb<XDT, BLOCKS, SHUFFLED, 1>(a, st);
    case 2: return launch_moe_down_nb<XDT, BLOCKS, SHUFFLED, 2>(a, st);
    default: return launch_moe_down_nb<XDT, BLOCKS, SHUFFLED, 3>(a, st);
  }
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
