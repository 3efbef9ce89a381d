// One token per row of logits: temperature, top-k, top-p, min-p, by a given uniform number.
//
// A row's order is by logit, the largest first, equal ones by index; w = exp((x - max) / temperature).  What top-k, top-p and min-p keep is
// a prefix of that order, and the token is the first of it whose running sum of w exceeds u times the sum of all kept: nothing
// has to be sorted, every question is "where does the running count or sum reach this".
//
// w is taken in 64 bits and held as a whole number of units of 2^-(62 - log2 V): sums of whole numbers do not depend on their order, so
// the same row gives the same token however the work is cut, and they are off by less than 2^-37 of the row's mass.
#include "common.h"

namespace tamd {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / kWave;

struct RowSettings {
  double t;
  double top_p, min_p, u;
  int top_k;         // 0: all
  bool greedy;
};

TAMD_DEVICE RowSettings settings_of(const tamd_sample_args &a, int row) {
  RowSettings s;
  const float t = a.temperature ? a.temperature[row] : a.temperature_value;
  s.greedy = !(t > 0.f);
  s.t = (double)t;
  s.top_p = a.top_p ? a.top_p[row] : a.top_p_value;
  const float min_p = a.min_p ? a.min_p[row] : a.min_p_value;
  s.min_p = min_p < 1.f ? (double)min_p : min_p >= 1.f ? 1.0 : 0.0;   // (NaN: 0)
  const int k = a.top_k ? a.top_k[row] : a.top_k_value;
  s.top_k = k > 0 && k < a.V ? k : 0;
  const float u = a.u[row];
  s.u = u > 0.f ? (double)(u < 1.f ? u : 0.99999994f) : 0.0;   // (NaN: 0)
  return s;
}

// A logit's place in the order; NaN counts as -inf.
template <int DT>
TAMD_DEVICE uint32_t key_at(const void *logits, int64_t i) {
  const float v = load_as_f32<DT>(logits, i);
  return ordered_bits(v != v ? -__builtin_inff() : v);
}
constexpr uint32_t kNothing = 0x007FFFFFu;   // key of -inf

// Weight of a logit in a row whose largest is `top` (> -inf): with infinite ones, all of these alike and nothing else.
TAMD_DEVICE double weight_of(uint32_t key, double top, double t) {
  const double v = logit_of(key);
  if (v == top) return 1.0;
  return key <= kNothing || top == __builtin_inf() ? 0.0 : exp((v - top) / t);
}

struct Found {
  uint32_t key;      // of the element
  int64_t count;     // elements before that key
  uint64_t mass;     // their mass
};

template <typename T>
TAMD_DEVICE T block_sum(T v, T *tmp) {
#pragma unroll
  for (int o = 1; o < kWave; o *= 2) v += __shfl_xor(v, o);
  if (threadIdx.x % kWave == 0) tmp[threadIdx.x / kWave] = v;
  sync_threads();
  T s = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) s += tmp[w];
  sync_threads();
  return s;
}

// The element of a whole row at which the running count (by_mass: mass) reaches `target` >= 1, three bits of its key at a time.
template <int DT>
TAMD_DEVICE Found find_in_row(const void *logits, int64_t row, int V, double top, double t, double unit, bool by_mass, uint64_t target, uint64_t *tmp) {
  Found f{0, 0, 0};
  for (int shift = 30; shift >= 0; shift -= 3) {
    const int bits = shift == 30 ? 2 : 3;
    uint32_t count[8] = {};
    uint64_t mass[8] = {};
    for (int i = threadIdx.x; i < V; i += kThreads) {
      const uint32_t key = key_at<DT>(logits, row + i);
      if (shift + bits < 32 && key >> (shift + bits) != f.key >> (shift + bits)) continue;
      const uint32_t d = key >> shift & ((1u << bits) - 1u);
      const uint64_t w = (uint64_t)(weight_of(key, top, t) * unit + 0.5);
#pragma unroll
      for (int j = 0; j < 8; ++j) count[j] += d == j, mass[j] += d == j ? w : 0;
    }
    int at = 0;
    bool found = false;
#pragma unroll
    for (int j = 7; j >= 0; --j) {
      const uint64_t n = block_sum<uint64_t>(count[j], tmp), m = block_sum<uint64_t>(mass[j], tmp);
      const uint64_t upto = by_mass ? f.mass + m : f.count + n;
      if (!found && (upto >= target || j == 0)) found = true, at = j;
      else if (!found) f.count += n, f.mass += m;
    }
    f.key |= (uint32_t)at << shift;
  }
  return f;
}

template <int DT>
TAMD_DEVICE int sample_row(const tamd_sample_args &a, int r, uint64_t *tmp) {
  const int tid = threadIdx.x, V = a.V;
  const int64_t row = r * a.logits_stride;
  const RowSettings s = settings_of(a, r);
  // the first of the largest
  uint64_t best = 0;
  for (int i = tid; i < V; i += kThreads) {
    const uint64_t v = (uint64_t)key_at<DT>(a.logits, row + i) << 32 | (0xFFFFFFFFu - (uint32_t)i);
    best = v > best ? v : best;
  }
#pragma unroll
  for (int o = 1; o < kWave; o *= 2) {
    const uint64_t v = __shfl_xor(best, o);
    best = v > best ? v : best;
  }
  if (tid % kWave == 0) tmp[tid / kWave] = best;
  sync_threads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) best = tmp[w] > best ? tmp[w] : best;
  sync_threads();
  const uint32_t top_key = (uint32_t)(best >> 32);
  if (top_key <= kNothing) return -1;
  if (s.greedy) return (int)(0xFFFFFFFFu - (uint32_t)best);
  const double top = logit_of(top_key), t = s.t, unit = (double)(1ull << (62 - (32 - __builtin_clz((uint32_t)V))));
  const auto fixed = [&](uint32_t key) { return (uint64_t)(weight_of(key, top, t) * unit + 0.5); };
  // the kept prefix: what has a larger key than `last`, and `ties` elements of it
  uint32_t last = 0;
  int64_t ties = V;
  uint64_t sum;
  if (s.top_k) {
    const Found f = find_in_row<DT>(a.logits, row, V, top, t, unit, false, (uint64_t)s.top_k, tmp);
    last = f.key, ties = s.top_k - f.count;
    sum = f.mass + (uint64_t)ties * fixed(last);
  } else {
    uint64_t mine = 0;
    for (int i = tid; i < V; i += kThreads) mine += fixed(key_at<DT>(a.logits, row + i));
    sum = block_sum<uint64_t>(mine, tmp);
  }
  if (s.top_p < 1.0) {
    const double want = ceil(s.top_p * (double)sum);
    const uint64_t target = want >= 1.0 ? (want < (double)sum ? (uint64_t)want : sum) : 1;
    const Found f = find_in_row<DT>(a.logits, row, V, top, t, unit, true, target, tmp);
    const uint64_t w = fixed(f.key);
    const int64_t n = w ? (int64_t)((target - f.mass + w - 1) / w) : 1;
    if (f.key > last || (f.key == last && n < ties)) last = f.key, ties = n, sum = f.mass + (uint64_t)n * w;
  }
  if (s.min_p > 0.0 && weight_of(last, top, t) < s.min_p) {
    uint64_t mine = 0;
    for (int i = tid; i < V; i += kThreads) {
      const uint32_t key = key_at<DT>(a.logits, row + i);
      if (key > last && (key == top_key || weight_of(key, top, t) >= s.min_p)) mine += fixed(key);
    }
    sum = block_sum<uint64_t>(mine, tmp);
  }
  const uint64_t at = (uint64_t)(s.u * (double)sum) + 1, target = at < sum ? at : sum;
  const Found f = find_in_row<DT>(a.logits, row, V, top, t, unit, true, target, tmp);
  // which of the equal ones
  int64_t skip = (int64_t)((target - f.mass - 1) / fixed(f.key));
  for (int i0 = 0; i0 < V; i0 += kThreads) {
    const int i = i0 + tid;
    const uint64_t mask = __ballot(i < V && key_at<DT>(a.logits, row + (i < V ? i : 0)) == f.key);
    if (tid % kWave == 0) tmp[tid / kWave] = mask;
    sync_threads();
    int64_t n = 0;
    int token = -1;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      uint64_t m = tmp[w];
      const int here = __popcll(m);
      if (token < 0 && n + here > skip) {
        for (int64_t j = n; j < skip; ++j) m &= m - 1;
        token = i0 + w * kWave + __builtin_ctzll(m);
      }
      n += here;
    }
    sync_threads();
    if (token >= 0) return token;
    skip -= n;
  }
  return -1;   // (not reached)
}

template <int DT>
__global__ __launch_bounds__(kThreads, 4) void sample_kernel(tamd_sample_args a) {
  __shared__ uint64_t tmp[kWaves];
  const int token = sample_row<DT>(a, blockIdx.x, tmp);
  if (threadIdx.x == 0) a.tokens[blockIdx.x] = token;
}

}  // namespace
}  // namespace tamd

using namespace tamd;

extern "C" int64_t tamd_sample_workspace(int R, int V) { return R < 0 || V < 0 ? TAMD_E_INVALID : 16; }

extern "C" int tamd_sample(const tamd_sample_args *args, size_t args_size, void *stream) {
  if (!args || args_size != sizeof(tamd_sample_args)) return TAMD_E_INVALID;
  const tamd_sample_args &a = *args;
  if (a.R < 0 || a.V < 1) return TAMD_E_INVALID;
  if (a.logits_dtype != TAMD_F32 && a.logits_dtype != TAMD_BF16 && a.logits_dtype != TAMD_F16) return TAMD_E_UNSUPPORTED;
  if (a.V > (1 << 20) || a.R > (1 << 20)) return TAMD_E_TOO_LARGE;
  if (a.R == 0) return 0;
  if (!a.logits || !a.u || !a.tokens || !a.workspace || a.logits_stride < 0) return TAMD_E_INVALID;
  hipStream_t st = (hipStream_t)stream;
  if (a.logits_dtype == TAMD_F32) sample_kernel<TAMD_F32><<<a.R, kThreads, 0, st>>>(a);
  else if (a.logits_dtype == TAMD_BF16) sample_kernel<TAMD_BF16><<<a.R, kThreads, 0, st>>>(a);
  else sample_kernel<TAMD_F16><<<a.R, kThreads, 0, st>>>(a);
  return launch_status();
}
