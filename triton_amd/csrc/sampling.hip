// One token per row of logits: temperature, top-k, top-p, min-p, by a given uniform number.
//
// A row's order is by logit, the largest first, equal ones by index; w = exp((x - max) / temperature).  What top-k, top-p and min-p keep is
// a prefix of that order, and the token is the first of it whose running sum of w exceeds u times the sum of all kept: nothing
// has to be sorted, every question is "where does the running count or sum reach this".
//
// w is taken in 64 bits and held as a whole number of units of 2^-fraction (sample_weights.h, with what that leaves of the sums): sums of whole
// numbers do not depend on their order, so the same row gives the same token however the work is cut.  What rounds to zero is
// not there at all: it cannot be drawn, and adds nothing to what top-k keeps.  Where min-p ends is decided by the logits, in 64 bits.
//
// Five launches, three of them over (chunk of a row, row):
//   extremes   the largest logit (of greedy rows with its index) and the smallest;
//   histogram  mass (and for top-k count) of the logits in 2048 bins of equal width between the two, or down to where w is zero;
//   bounds     a workgroup per row finds in the histogram the few bins in which the ends of top-k, top-p and min-p and the token
//              can lie;
//   collect    gathers the logits of those, a few hundred of the whole vocabulary;
//   finish     a workgroup per row sorts them and answers the questions exactly.
// Where that is faster a workgroup goes through all of it for a row, in one launch (sample_whole).  A row that has more than 4096 logits in those
// bins -- many equal or nearly equal ones -- is searched by the bits of its keys (search_row): slower, but right for any row.
#include "common.h"
#include "sample_weights.h"

namespace tamd {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / kWave;
constexpr int kBins = 2048, kMost = 4096;   // candidates that are sorted
constexpr int kChunk = 8192, kMaxChunks = 64;
constexpr int kShort = 24000;
constexpr int kRowsAtOnce = 4096;           // of one round of launches (the workspace holds as many)

// Whether a workgroup does a row alone.  That takes about 9 us and one for every 2000 logits, as often as there are rows for a CU; the
// five launches take 24 and one for every 1600 logits of a CU's share.  Measured: 1 row of 8192 13.7 and 24.0, of 32000 25.0 and 25.0,
// of 65536 41 and 26; 256 rows of 65536 48 and 63.  (By the 256 CUs of a whole MI355X on any device: the size of the workspace goes by it.)
inline bool sample_whole(int R, int V) {
  constexpr int cus = 256;
  return V <= kShort || (int64_t)((R + cus - 1) / cus) * (18000 + V) <= 48000 + (int64_t)R * V / cus * 5 / 4;
}

struct RowSettings {
  double t;          // temperature
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

// 2^(fraction - j / 256) by the threads of a workgroup.
TAMD_DEVICE void make_powers(double *powers, int V) {
  if (threadIdx.x < 256) powers[threadIdx.x] = exp2(fraction_bits(V) - (double)threadIdx.x * 0.00390625);
}

// Weights of a row whose largest logit is `top` (> -inf).  y = log2(1 / w).  An infinite logit is kHuge here: such ones weigh alike, and
// nothing else does (y in steps of one, from kHuge).
constexpr double kHuge = 1e300;
struct RowScale {
  double top, to_y, to_bin;
  int fraction;
  const double *powers;
  TAMD_DEVICE RowScale(double top_, double to_y_, double to_bin_, int V, const double *powers_)
      : top(top_), to_y(to_y_), to_bin(to_bin_), fraction(fraction_bits(V)), powers(powers_) {}
  TAMD_DEVICE RowScale(uint32_t top_key, uint32_t least_key, double t, int V, const double *powers_)
      : top(__builtin_fmin((double)logit_of(top_key), kHuge)), to_y(top == kHuge ? 1.0 : 1.4426950408889634 / t), fraction(fraction_bits(V)), powers(powers_) {
    const double most = y_of(logit_of(least_key)), range = counts(most) ? most : fraction + 1;
    to_bin = range > 0.0 ? kBins / range : 0.0;
  }
  // (of -inf: infinite, or NaN at an infinite temperature; neither counts)
  TAMD_DEVICE double y_of(float v) const {
#pragma clang fp contract(off)
    return (top - __builtin_fmin((double)v, kHuge)) * to_y;
  }
  TAMD_DEVICE bool counts(double y) const { return y < fraction + 1; }   // half a unit or more
  TAMD_DEVICE int bin_of(double y) const { return (int)__builtin_fmin(y * to_bin, (double)(kBins - 1)); }
  TAMD_DEVICE uint64_t units_of(double y) const { return weight_units(y, powers); }
  TAMD_DEVICE uint64_t units(uint32_t key) const {
    const double y = y_of(logit_of(key));
    return counts(y) ? units_of(y) : 0;
  }
};

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

// Inclusive scan over the workgroup of one value per thread; `tmp` has a place per wave.
template <typename T>
TAMD_DEVICE T block_scan(T v, T *tmp) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
#pragma unroll
  for (int o = 1; o < kWave; o *= 2) {
    const T x = __shfl_up(v, o);
    v += lane >= o ? x : 0;
  }
  if (lane == kWave - 1) tmp[wave] = v;
  sync_threads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) v += w < wave ? tmp[w] : 0;
  sync_threads();
  return v;
}

// What one thread finds and the others wait for.
struct Shared {
  uint64_t tmp[kWaves];
  uint64_t sum;
  uint64_t found_mass, found_count;
  int digit;
  int at[2];
  int token;
  uint32_t n, base;
};

// The element of a whole row at which the running count (by_mass: mass) reaches `target` >= 1, eleven bits of its key at a time: a
// histogram of the next bits of the keys that share the bits so far.  hist: room for kBins 12-byte entries.
template <int DT>
TAMD_DEVICE Found find_in_row(const void *logits, int64_t row, int V, const RowScale &scale, bool by_mass, uint64_t target, uint64_t *hist, Shared &sh) {
  const int tid = threadIdx.x;
  uint64_t *mass = hist;
  uint32_t *count = (uint32_t *)(hist + kBins);
  Found f{0, 0, 0};
#pragma clang loop unroll(disable)
  for (int shift = 21; shift >= 0; shift = shift == 21 ? 10 : shift == 10 ? 0 : -1) {
    const int bits = shift ? 11 : 10;
    for (int b = tid; b < kBins; b += kThreads) mass[b] = 0, count[b] = 0;
    sync_threads();
    for (int i0 = 0; i0 < V; i0 += kThreads) {
      const int i = i0 + tid;
      const uint32_t key = key_at<DT>(logits, row + (i < V ? i : 0));
      bool on = i < V && (shift == 21 || key >> (shift + bits) == f.key >> (shift + bits));
      const uint32_t d = key >> shift & ((1u << bits) - 1u);
      const uint64_t units = scale.units(key);
      // (the two first keys of a wave once for all lanes that share them: rows that come here have few different ones, and additions to
      // one place take turns; 131072 equal logits took 789 us, 340 so)
      for (int j = 0; j < 2; ++j) {
        const uint64_t left = __ballot(on);
        if (left == 0) break;
        const int first = __builtin_ctzll(left);
        const uint32_t same = (uint32_t)__builtin_amdgcn_readlane((int)key, first);
        const uint32_t n = (uint32_t)__popcll(__ballot(on && key == same));
        if (tid % kWave == first) {
          atomicAdd((unsigned long long *)&mass[d], (unsigned long long)(units * n));
          atomicAdd(&count[d], n);
        }
        on = on && key != same;
      }
      if (on) {
        atomicAdd((unsigned long long *)&mass[d], (unsigned long long)units);
        atomicAdd(&count[d], 1u);
      }
    }
    sync_threads();
    // from the largest digit down: thread t has the digits kBins - 1 - 2 t and the one below
    const int d = kBins - 1 - 2 * tid;
    const uint64_t m0 = mass[d], m1 = mass[d - 1], n0 = count[d], n1 = count[d - 1];
    const uint64_t ms = block_scan<uint64_t>(m0 + m1, sh.tmp) - m0 - m1 + f.mass, ns = block_scan<uint64_t>(n0 + n1, sh.tmp) - n0 - n1 + (uint64_t)f.count;
    const uint64_t c0 = by_mass ? ms : ns, c1 = c0 + (by_mass ? m0 : n0), c2 = c1 + (by_mass ? m1 : n1);
    if (c0 < target && target <= c1) sh.digit = d, sh.found_mass = ms, sh.found_count = ns;
    if (c1 < target && target <= c2) sh.digit = d - 1, sh.found_mass = ms + m0, sh.found_count = ns + n0;
    sync_threads();
    f.key |= (uint32_t)sh.digit << shift, f.mass = sh.found_mass, f.count = (int64_t)sh.found_count;
    sync_threads();
  }
  return f;
}

// Where the kept prefix ends, from the row's sums.
TAMD_DEVICE uint64_t top_p_target(double top_p, uint64_t sum) {   // the prefix ends where the sum reaches it
  const double want = ceil(top_p * (double)sum);
  return want >= 1.0 ? (want < (double)sum ? (uint64_t)want : sum) : 1;
}
TAMD_DEVICE uint64_t token_target(double u, uint64_t sum) {       // the token is where the sum reaches it
  const uint64_t at = (uint64_t)(u * (double)sum) + 1;
  return at < sum ? at : sum;
}

// The token of a row whose largest logit is known, by the bits of the keys.  min_p_y as in Bounds.
template <int DT>
TAMD_DEVICE int search_row(const tamd_sample_args &a, int r, const RowSettings &s, const RowScale &scale, double min_p_y, uint64_t *hist, Shared &sh) {
  const int tid = threadIdx.x, V = a.V;
  uint64_t *tmp = sh.tmp;
  const int64_t row = r * a.logits_stride;
  const auto sum_of = [&](uint32_t above, double most) {   // of larger keys with no larger y
    uint64_t mine = 0;
    for (int i = tid; i < V; i += kThreads) {
      const uint32_t key = key_at<DT>(a.logits, row + i);
      mine += key > above && scale.y_of(logit_of(key)) <= most ? scale.units(key) : 0;
    }
    return block_sum<uint64_t>(mine, tmp);
  };
  // the kept prefix: what has a larger key than `last`, and `ties` elements of it
  uint32_t last = kNothing + 1;
  int64_t ties = V;
  uint64_t sum = s.top_k ? 0 : sum_of(kNothing, (double)__builtin_inff()), target = 0;
  Found f{0, 0, 0};
  // where top-k ends, where top-p ends, the token
#pragma clang loop unroll(disable)
  for (int ask = s.top_k ? 0 : s.top_p < 1.0 ? 1 : 2; ask < 3; ask = ask == 0 && s.top_p < 1.0 ? 1 : ask == 2 ? 3 : 2) {
    // (of -inf y may be NaN)
    if (ask == 2 && s.min_p > 0.0 && !(scale.y_of(logit_of(last)) <= min_p_y)) sum = sum_of(last, min_p_y);
    target = ask == 0 ? (uint64_t)s.top_k : ask == 1 ? top_p_target(s.top_p, sum) : token_target(s.u, sum);
    f = find_in_row<DT>(a.logits, row, V, scale, ask != 0, target, hist, sh);
    const uint64_t w = scale.units(f.key);
    if (ask == 0) {
      last = f.key, ties = s.top_k - f.count;
      sum = f.mass + (uint64_t)ties * w;
    } else if (ask == 1) {
      const int64_t n = w ? (int64_t)((target - f.mass + w - 1) / w) : 1;
      if (f.key > last || (f.key == last && n < ties)) last = f.key, ties = n, sum = f.mass + (uint64_t)n * w;
    }
  }
  // which of the equal ones
  int64_t skip = (int64_t)((target - f.mass - 1) / scale.units(f.key));
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

// A chunk's logits, NaN as -inf, eight per thread at a time in two vectors whatever the row's alignment; what is past the end is
// -inf.  The next eight are requested before the last are used, the first eight as soon as this is made: each launch has a
// trip to memory or two in front of its first use, and with one vector in flight the largest logit of 64 rows of 131072 took 9.6 us.
template <int DT>
struct Chunk {
  static constexpr int kStep = 8 * kThreads;
  const tamd_sample_args &a;
  int64_t row;
  int at, end;
  float v[8];
  TAMD_DEVICE Chunk(const tamd_sample_args &a_, int r, int c, int chunk)
      : a(a_), row(r * a_.logits_stride), at(c * chunk), end(at + chunk < a_.V ? at + chunk : a_.V) { request(); }
  TAMD_DEVICE void request() {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int i = at + 4 * (q * kThreads + (int)threadIdx.x);
      float *to = v + 4 * q;
      if (i + 4 <= end) {
        if constexpr (DT == TAMD_F32) {
          __builtin_memcpy(to, (const float *)a.logits + row + i, 16);
        } else {
          uint16_t b[4];
          __builtin_memcpy(b, (const uint16_t *)a.logits + row + i, 8);
#pragma unroll
          for (int j = 0; j < 4; ++j) to[j] = DT == TAMD_BF16 ? bf16_bits_to_f32(b[j]) : f16_bits_to_f32(b[j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) to[j] = i + j < end ? load_as_f32<DT>(a.logits, row + i + j) : -__builtin_inff();
      }
    }
  }
  // use(v, index): four logits of consecutive indexes
  template <typename F>
  TAMD_DEVICE void each(F use) {
    while (at < end) {
      float now[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) now[j] = v[j];
      const int from = at + 4 * (int)threadIdx.x;
      at += kStep;
      if (at < end) request();
#pragma unroll
      for (int j = 0; j < 8; ++j) now[j] = now[j] != now[j] ? -__builtin_inff() : now[j];
      use(now, from);
      use(now + 4, from + 4 * kThreads);
    }
  }
};

// Element of the order as one number: the larger, the earlier.
TAMD_DEVICE uint64_t element_of(uint32_t key, int i) { return (uint64_t)key << 32 | (0xFFFFFFFFu - (uint32_t)i); }
TAMD_DEVICE uint32_t key_of(uint64_t e) { return (uint32_t)(e >> 32); }
TAMD_DEVICE int index_of(uint64_t e) { return (int)(0xFFFFFFFFu - (uint32_t)e); }

struct Workspace {
  uint64_t *first;        // [rows, chunks] largest element
  uint32_t *least;        // [rows, chunks] smallest key above -inf (0xFFFFFFFF: none)
  uint64_t *mass;         // [rows, bins]
  uint32_t *count;        // [rows, bins]
  uint32_t *collected;    // [rows] candidates
  uint64_t *candidates;   // [rows, kMost]
  void *bounds;           // [rows] Bounds
};
constexpr int64_t kRowBytes = kMaxChunks * 12 + kBins * 12 + 4 + kMost * 8 + 96;

inline Workspace workspace_of(void *p, int rows) {
  uint8_t *at = (uint8_t *)p;
  const auto take = [&](int64_t bytes) { uint8_t *q = at; at += bytes * rows; return q; };
  Workspace w;
  w.candidates = (uint64_t *)take(kMost * 8), w.bounds = take(96), w.mass = (uint64_t *)take(kBins * 8), w.first = (uint64_t *)take(kMaxChunks * 8);
  w.count = (uint32_t *)take(kBins * 4), w.least = (uint32_t *)take(kMaxChunks * 4), w.collected = (uint32_t *)take(4);
  return w;
}

// Largest element (its index for greedy rows only: that takes four times the instructions) and smallest key above -inf of a
// workgroup's part of a row; every thread gets them.
template <int DT>
TAMD_DEVICE void extremes_of(Chunk<DT> &logits, bool greedy, uint64_t &first, uint32_t &least, uint64_t *s_first, uint32_t *s_least) {
  const int tid = threadIdx.x;
  first = 0, least = 0xFFFFFFFFu;
  if (greedy) {
    logits.each([&](const float *v, int i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint64_t e = element_of(ordered_bits(v[j]), i + j);
        first = e > first ? e : first;
      }
    });
  } else {
    float most = -__builtin_inff(), fewest = __builtin_inff();
    logits.each([&](const float *v, int) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        most = __builtin_fmaxf(most, v[j]);
        fewest = __builtin_fminf(fewest, v[j] > -__builtin_inff() ? v[j] : __builtin_inff());
      }
    });
    first = element_of(ordered_bits(most), 0), least = ordered_bits(fewest);
  }
#pragma unroll
  for (int o = 1; o < kWave; o *= 2) {
    const uint64_t e = __shfl_xor(first, o);
    const uint32_t l = __shfl_xor(least, o);
    first = e > first ? e : first;
    least = l < least ? l : least;
  }
  if (tid % kWave == 0) s_first[tid / kWave] = first, s_least[tid / kWave] = least;
  sync_threads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    first = s_first[w] > first ? s_first[w] : first;
    least = s_least[w] < least ? s_least[w] : least;
  }
}

template <int DT>
__global__ __launch_bounds__(kThreads) void extremes_kernel(tamd_sample_args a, Workspace ws, int chunk) {
  __shared__ uint64_t s_first[kWaves];
  __shared__ uint32_t s_least[kWaves];
  const int c = blockIdx.x, r = blockIdx.y, tid = threadIdx.x;
  Chunk<DT> logits(a, r, c, chunk);
  for (int b = c * kThreads + tid; b < kBins; b += gridDim.x * kThreads) ws.mass[(int64_t)r * kBins + b] = 0, ws.count[(int64_t)r * kBins + b] = 0;
  if (c == 0 && tid == 0) ws.collected[r] = 0;
  uint64_t first;
  uint32_t least;
  extremes_of<DT>(logits, settings_of(a, r).greedy, first, least, s_first, s_least);
  if (tid == 0) ws.first[r * kMaxChunks + c] = first, ws.least[r * kMaxChunks + c] = least;
}

// A row's extremes from its chunks', by every thread.
TAMD_DEVICE void row_extremes(const Workspace &ws, int r, int chunks, uint64_t &first, uint32_t &least) {
  const int lane = threadIdx.x % kWave;
  first = lane < chunks ? ws.first[r * kMaxChunks + lane] : 0;
  least = lane < chunks ? ws.least[r * kMaxChunks + lane] : 0xFFFFFFFFu;
#pragma unroll
  for (int o = 1; o < kWave; o *= 2) {
    const uint64_t e = __shfl_xor(first, o);
    const uint32_t l = __shfl_xor(least, o);
    first = e > first ? e : first;
    least = l < least ? l : least;
  }
}

// Adds a workgroup's part of a row to a histogram in LDS.
template <int DT>
TAMD_DEVICE void add_to_histogram(Chunk<DT> &logits, const RowScale &scale, bool counting, uint64_t *mass, uint32_t *count) {
  // (no branch but around the additions: a logit at a time, each waiting for its power, 64 rows of 131072 took 14.7 us and 256 of 100000
  // 31.0, so 14.4 and 30.5: the additions in LDS and the logits are what is left)
  logits.each([&](const float *v, int) {
    double y[4];
    uint64_t units[4];
    int bin[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = scale.y_of(v[j]), bin[j] = scale.bin_of(y[j]), units[j] = scale.units_of(y[j]);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (scale.counts(y[j])) atomicAdd((unsigned long long *)&mass[bin[j]], (unsigned long long)units[j]);
    if (counting) {   // (only top-k asks for counts)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (scale.counts(y[j])) atomicAdd(&count[bin[j]], 1u);
    }
  });
}

template <int DT>
__global__ __launch_bounds__(kThreads) void histogram_kernel(tamd_sample_args a, Workspace ws, int chunk) {
  __shared__ uint64_t mass[kBins];
  __shared__ uint32_t count[kBins];
  __shared__ double powers[256];
  const int c = blockIdx.x, r = blockIdx.y, tid = threadIdx.x;
  Chunk<DT> logits(a, r, c, chunk);
  uint64_t first;
  uint32_t least;
  row_extremes(ws, r, gridDim.x, first, least);
  const RowSettings s = settings_of(a, r);
  if (s.greedy || key_of(first) <= kNothing) return;
  make_powers(powers, a.V);
  for (int b = tid; b < kBins; b += kThreads) mass[b] = 0, count[b] = 0;
  const RowScale scale(key_of(first), least, s.t, a.V, powers);
  sync_threads();
  add_to_histogram<DT>(logits, scale, s.top_k != 0, mass, count);
  sync_threads();
  for (int b = tid; b < kBins; b += kThreads)
    if (mass[b]) {
      atomicAdd((unsigned long long *)&ws.mass[(int64_t)r * kBins + b], (unsigned long long)mass[b]);
      if (s.top_k) atomicAdd(&ws.count[(int64_t)r * kBins + b], count[b]);
    }
}

// n <= kMost elements of `list` (room for the next power of two), largest first afterwards.  Up to kCounted by counting the larger ones of
// each, all threads sharing the comparisons.  Up to kThreads every wave sorts 64 in its registers, and an element's place is how many
// of every wave's are larger, which seven steps of halving tell.  The last launch takes 6.7 us with the first and 8.2 with the second
// for one row of some hundred candidates, 16.4 and 9.9 for 64 rows of some 600.  Else steps of the bitonic network.
constexpr int kCounted = 256;
TAMD_DEVICE void sort_elements(uint64_t *list, int n, uint32_t *rank) {
  const int tid = threadIdx.x, lane = tid % kWave;
  if (n <= kCounted) {
    int wide = kWave;
    while (wide < n) wide *= 2;
    const int i = tid % wide, part = tid / wide, parts = kThreads / wide;
    if (tid < kCounted) rank[tid] = 0;
    sync_threads();
    const uint64_t e = i < n ? list[i] : 0;
    uint32_t larger = 0;
    for (int j = n * part / parts; j < n * (part + 1) / parts; ++j) larger += list[j] > e;
    if (i < n && larger) atomicAdd(&rank[i], larger);
    sync_threads();
    if (tid < n) list[rank[tid]] = e;   // (wide >= n: thread tid holds element tid; all are different)
    sync_threads();
    return;
  }
  if (n <= kThreads) {
    const int runs = (n + kWave - 1) / kWave;
    uint64_t e = tid < n ? list[tid] : 0;   // (0: smaller than any element; the list's own are all different)
    if (tid < runs * kWave) {
#pragma unroll
      for (int k = 2; k <= kWave; k *= 2)
#pragma unroll
        for (int j = k / 2; j > 0; j /= 2) {
          const uint64_t other = __shfl_xor(e, j);
          const bool larger = ((lane & k) == 0) == ((lane & j) == 0);   // (k = 64: the largest come first)
          e = (other > e) == larger ? other : e;
        }
      list[tid] = e;
    }
    sync_threads();
    int place = lane;
    if (tid < n) {   // (zeros are last of their run, behind all that count)
      for (int g = 0; g < runs; g += 4) {
        int at[4] = {0, 0, 0, 0};
#pragma unroll
        for (int step = kWave / 2; step > 0; step /= 2)
#pragma unroll
          for (int q = 0; q < 4; ++q) at[q] += g + q < runs && list[(g + q) * kWave + at[q] + step - 1] > e ? step : 0;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (g + q < runs && g + q != tid / kWave) place += at[q] + (list[(g + q) * kWave + at[q]] > e);
      }
    }
    sync_threads();
    if (e) list[place] = e;
    sync_threads();
    return;
  }
  int size = 2;
  while (size < n) size *= 2;
  for (int i = n + tid; i < size; i += kThreads) list[i] = 0;
  sync_threads();
  for (int k = 2; k <= size; k *= 2)
    for (int j = k / 2; j > 0; j /= 2) {
      for (int p = tid; p < size / 2; p += kThreads) {
        const int i = 2 * j * (p / j) + p % j;
        const uint64_t x = list[i], y = list[i + j];
        if ((x < y) == ((i & k) == 0)) list[i] = y, list[i + j] = x;
      }
      sync_threads();
    }
}

// What is known of a row in front of the gathering.
struct Bounds {
  int from[4], to[4];      // bins of the candidates: the ends of top-k, top-p and min-p, and the token
  uint64_t mass, min_mass; // of the row; in front of the bins in which min-p ends
  double top, to_y, to_bin;
  double min_p_y;          // min-p keeps what has no larger y: w >= min_p is y <= log2(1 / min_p)
  uint32_t count;
  int done;                // the token is known
};
static_assert(sizeof(Bounds) <= 96);

// The token, from n <= kMost sorted candidates.  before_mass / before_rank: what lies in front of every bin; bin_mass / bin_rank: room for as
// many, or the same.
TAMD_DEVICE int pick_among(const RowSettings &s, const RowScale &scale, const Bounds &b, const uint64_t *list, int n, const uint64_t *before_mass,
                           const uint32_t *before_rank, uint64_t *bin_mass, uint32_t *bin_rank, Shared &sh) {
  constexpr int PER = kMost / kThreads;
  const int tid = threadIdx.x;
  uint64_t units[PER], before[PER], run = 0, enough = 0;
  uint32_t rank[PER];
  int bin[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = PER * tid + j;
    const double y = i < n ? scale.y_of(logit_of(key_of(list[i]))) : 1e9;
    units[j] = scale.counts(y) ? scale.units_of(y) : 0;
    bin[j] = scale.counts(y) ? scale.bin_of(y) : -1;
    before[j] = run;
    run += units[j];
    enough += bin[j] >= b.from[2] && bin[j] <= b.to[2] && y <= b.min_p_y ? units[j] : 0;
  }
  const uint64_t start = block_scan<uint64_t>(run, sh.tmp) - run;
  // the first candidate of a bin leaves what the running sums of the bin's candidates lack
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = PER * tid + j;
    if (bin[j] >= 0 && (i == 0 || scale.bin_of(scale.y_of(logit_of(key_of(list[i - 1])))) != bin[j])) {
      bin_mass[bin[j]] = before_mass[bin[j]] - (start + before[j]);
      if (s.top_k) bin_rank[bin[j]] = before_rank[bin[j]] - (uint32_t)i;
    }
  }
  if (tid == 0) sh.sum = b.mass, sh.token = -1;
  sync_threads();
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    before[j] += start + (bin[j] >= 0 ? bin_mass[bin[j]] : 0);
    rank[j] = (uint32_t)(PER * tid + j) + (bin[j] >= 0 && s.top_k ? bin_rank[bin[j]] : 0u);
  }
  if (s.top_k && (uint32_t)s.top_k < b.count) {
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (bin[j] >= 0 && rank[j] == (uint32_t)s.top_k - 1) sh.sum = before[j] + units[j];
    sync_threads();
  }
  if (s.top_p < 1.0) {
    const uint64_t target = top_p_target(s.top_p, sh.sum);
    sync_threads();
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (bin[j] >= 0 && before[j] < target && target <= before[j] + units[j]) sh.sum = before[j] + units[j];
    sync_threads();
  }
  uint64_t sum = sh.sum;
  if (s.min_p > 0.0) {
    const uint64_t has = b.min_mass + block_sum<uint64_t>(enough, sh.tmp);
    sum = has < sum ? has : sum;
  }
  const uint64_t target = token_target(s.u, sum);
#pragma unroll
  for (int j = 0; j < PER; ++j)
    if (bin[j] >= 0 && before[j] < target && target <= before[j] + units[j]) sh.token = index_of(list[PER * tid + j]);
  sync_threads();
  return sh.token;
}

// The bin in which the running count or sum reaches `target`, from the prefix sums in front of the bins; every thread gets it.
template <typename T>
TAMD_DEVICE int bin_reaching(const T *before, T target, int &slot) {
  target = target < 1 ? 1 : target > before[kBins] ? before[kBins] : target;
#pragma unroll
  for (int j = 0; j < kBins / kThreads; ++j) {
    const int b = threadIdx.x * (kBins / kThreads) + j;
    if (before[b] < target && target <= before[b + 1]) slot = b;
  }
  sync_threads();
  const int found = slot;
  sync_threads();
  return found;
}

// The bins in which the ends of what is kept and the token can lie: lo and hi enclose the sum of what is kept.  A thread brings two bins of
// the row's histogram; mass and rank become what lies in front of every bin.
TAMD_DEVICE Bounds find_bounds(const RowSettings &s, const RowScale &scale, uint64_t m0, uint64_t m1, uint32_t n0, uint32_t n1, uint64_t *mass, uint32_t *rank,
                               Shared &sh) {
  static_assert(kBins == 2 * kThreads);
  const int tid = threadIdx.x;
  const uint64_t upto = block_scan<uint64_t>(m0 + m1, sh.tmp);
  mass[2 * tid] = upto - m0 - m1, mass[2 * tid + 1] = upto - m1;
  if (tid == kThreads - 1) mass[kBins] = upto;
  if (s.top_k) {
    const uint32_t n = block_scan<uint32_t>(n0 + n1, (uint32_t *)sh.tmp);
    rank[2 * tid] = n - n0 - n1, rank[2 * tid + 1] = n - n1;
    if (tid == kThreads - 1) rank[kBins] = n;
  }
  sync_threads();
  Bounds b;
#pragma unroll
  for (int j = 0; j < 4; ++j) b.from[j] = kBins, b.to[j] = -1;
  b.mass = mass[kBins], b.count = s.top_k ? rank[kBins] : 0u, b.min_mass = 0, b.min_p_y = 0.0, b.done = 0;
  b.top = scale.top, b.to_y = scale.to_y, b.to_bin = scale.to_bin;
  uint64_t lo = b.mass, hi = lo;
  if (s.top_k && (uint32_t)s.top_k < b.count) {
    b.from[0] = b.to[0] = bin_reaching<uint32_t>(rank, (uint32_t)s.top_k, sh.at[0]);
    lo = mass[b.from[0]], hi = mass[b.to[0] + 1];
  }
  if (s.top_p < 1.0) {
    b.from[1] = bin_reaching<uint64_t>(mass, top_p_target(s.top_p, lo), sh.at[0]);
    b.to[1] = lo == hi ? b.from[1] : bin_reaching<uint64_t>(mass, top_p_target(s.top_p, hi), sh.at[1]);
    lo = mass[b.from[1]];
    hi = mass[b.to[1] + 1] < hi ? mass[b.to[1] + 1] : hi;
  }
  if (s.min_p > 0.0) {
    b.min_p_y = -log2(s.min_p);
    const int at = scale.counts(b.min_p_y) ? scale.bin_of(b.min_p_y) : kBins - 1;
    b.from[2] = at > 0 ? at - 1 : 0, b.to[2] = at < kBins - 1 ? at + 1 : kBins - 1;
    b.min_mass = mass[b.from[2]];
    lo = b.min_mass < lo ? b.min_mass : lo;
    hi = mass[b.to[2] + 1] < hi ? mass[b.to[2] + 1] : hi;
  }
  b.from[3] = bin_reaching<uint64_t>(mass, token_target(s.u, lo), sh.at[0]);
  b.to[3] = lo == hi ? b.from[3] : bin_reaching<uint64_t>(mass, token_target(s.u, hi), sh.at[1]);
  return b;
}

// (In a launch of its own: done by every workgroup of the next two, as at first, these took 40 us for 64 rows of 131072; the three
// now take 26, for one row 18 instead of 21.)
__global__ __launch_bounds__(kThreads) void bounds_kernel(tamd_sample_args a, Workspace ws, int chunks) {
  __shared__ uint64_t mass[kBins + 1];
  __shared__ uint32_t rank[kBins + 1];
  __shared__ Shared sh;
  const int r = blockIdx.x, tid = threadIdx.x;
  const int64_t h = (int64_t)r * kBins + 2 * tid;
  const uint64_t m0 = ws.mass[h], m1 = ws.mass[h + 1];
  const uint32_t n0 = ws.count[h], n1 = ws.count[h + 1];
  uint64_t first;
  uint32_t least;
  row_extremes(ws, r, chunks, first, least);
  const RowSettings s = settings_of(a, r);
  Bounds *out = (Bounds *)ws.bounds + r;
  if (s.greedy || key_of(first) <= kNothing) {
    if (tid == 0) out->done = 1, a.tokens[r] = key_of(first) <= kNothing ? -1 : index_of(first);
    return;
  }
  const RowScale scale(key_of(first), least, s.t, a.V, nullptr);
  const Bounds b = find_bounds(s, scale, m0, m1, n0, n1, mass, rank, sh);
  ws.mass[h] = mass[2 * tid], ws.mass[h + 1] = mass[2 * tid + 1];
  if (s.top_k) ws.count[h] = rank[2 * tid], ws.count[h + 1] = rank[2 * tid + 1];
  if (tid == 0) *out = b;
}

// Gathers the candidates of a workgroup's part of a row in LDS; more than kMost are only counted.
template <int DT>
TAMD_DEVICE void gather(Chunk<DT> &logits, const Bounds &b, const RowScale &scale, uint64_t *list, Shared &sh) {
  uint32_t from[4], more[4];   // (an empty range: from = kBins, and nothing is as large)
#pragma unroll
  for (int q = 0; q < 4; ++q) from[q] = (uint32_t)b.from[q], more[q] = b.to[q] > b.from[q] ? (uint32_t)(b.to[q] - b.from[q]) : 0u;
  logits.each([&](const float *v, int i) {
    bool is[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double y = scale.y_of(v[j]);
      const uint32_t bin = (uint32_t)scale.bin_of(y);
      is[j] = false;
#pragma unroll
      for (int q = 0; q < 4; ++q) is[j] |= bin - from[q] <= more[q];
      is[j] &= scale.counts(y);
    }
    if (is[0] | is[1] | is[2] | is[3]) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (is[j]) {
          const uint32_t at = atomicAdd(&sh.n, 1u);
          if (at < kMost) list[at] = element_of(ordered_bits(v[j]), i + j);
        }
    }
  });
}

// (In LDS first: an atomic on the row's counter takes a trip to memory, and they take turns; one per candidate took 282 us for 64 rows
// of 131072.)
template <int DT>
__global__ __launch_bounds__(kThreads) void collect_kernel(tamd_sample_args a, Workspace ws, int chunk) {
  __shared__ uint64_t list[kMost];
  __shared__ Shared sh;
  const int c = blockIdx.x, r = blockIdx.y, tid = threadIdx.x;
  Chunk<DT> logits(a, r, c, chunk);
  const Bounds b = ((const Bounds *)ws.bounds)[r];
  if (b.done) return;
  const RowScale scale(b.top, b.to_y, b.to_bin, a.V, nullptr);
  if (tid == 0) sh.n = 0;
  sync_threads();
  gather<DT>(logits, b, scale, list, sh);
  sync_threads();
  const uint32_t n = sh.n, stored = n < kMost ? n : kMost;
  if (n == 0) return;
  if (tid == 0) sh.base = atomicAdd(&ws.collected[r], n);
  sync_threads();
  for (uint32_t i = tid; i < stored; i += kThreads)
    if (sh.base + i < kMost) ws.candidates[(int64_t)r * kMost + sh.base + i] = list[i];
}

// The token of a row.  (As the last workgroup of the row in the launch before, found by a ticket, this cost a write-back of the L2 per
// workgroup: 61 us for the two together, 64 rows of 131072.)
template <int DT>
__global__ __launch_bounds__(kThreads) void finish_kernel(tamd_sample_args a, Workspace ws) {
  __shared__ uint64_t list[kMost];
  __shared__ uint64_t bin_mass[kBins];
  __shared__ uint32_t bin_rank[kBins];
  __shared__ double powers[256];
  __shared__ Shared sh;
  const int r = blockIdx.x, tid = threadIdx.x;
  const Bounds b = ((const Bounds *)ws.bounds)[r];
  if (b.done) return;
  const uint32_t collected = ws.collected[r];
  const RowSettings s = settings_of(a, r);
  make_powers(powers, a.V);
  const RowScale scale(b.top, b.to_y, b.to_bin, a.V, powers);
  int token;
  if (collected > kMost) {
    sync_threads();
    token = search_row<DT>(a, r, s, scale, b.min_p_y, list, sh);
  } else {
    const int n = (int)collected;
    for (int i = tid; i < n; i += kThreads) list[i] = ws.candidates[(int64_t)r * kMost + i];
    sort_elements(list, n, bin_rank);
    token = pick_among(s, scale, b, list, n, ws.mass + (int64_t)r * kBins, ws.count + (int64_t)r * kBins, bin_mass, bin_rank, sh);
  }
  if (tid == 0) a.tokens[r] = token;
}

// All of it for a row, in LDS: three reads of the row, and what bounds it is their arithmetic, 75 instructions a logit (13, 38 and 25).
template <int DT>
__global__ __launch_bounds__(kThreads) void whole_row_kernel(tamd_sample_args a) {
  __shared__ uint64_t list[kMost], mass[kBins + 1];
  __shared__ uint32_t rank[kBins + 1], places[kCounted];
  __shared__ double powers[256];
  __shared__ Shared sh;
  static_assert(kCounted >= kWaves);
  const int r = blockIdx.x, tid = threadIdx.x;
  const RowSettings s = settings_of(a, r);
  uint64_t first;
  uint32_t least;
  {
    Chunk<DT> logits(a, r, 0, a.V);
    mass[2 * tid] = mass[2 * tid + 1] = 0, rank[2 * tid] = rank[2 * tid + 1] = 0;
    if (tid == 0) sh.n = 0;
    make_powers(powers, a.V);
    extremes_of<DT>(logits, s.greedy, first, least, sh.tmp, places);
  }
  if (s.greedy || key_of(first) <= kNothing) {
    if (tid == 0) a.tokens[r] = key_of(first) <= kNothing ? -1 : index_of(first);
    return;
  }
  const RowScale scale(key_of(first), least, s.t, a.V, powers);
  {
    Chunk<DT> logits(a, r, 0, a.V);
    add_to_histogram<DT>(logits, scale, s.top_k != 0, mass, rank);
  }
  Chunk<DT> logits(a, r, 0, a.V);
  sync_threads();
  const uint64_t m0 = mass[2 * tid], m1 = mass[2 * tid + 1];
  const uint32_t n0 = rank[2 * tid], n1 = rank[2 * tid + 1];
  const Bounds b = find_bounds(s, scale, m0, m1, n0, n1, mass, rank, sh);   // (a barrier before either is written)
  gather<DT>(logits, b, scale, list, sh);
  sync_threads();
  int token;
  if (sh.n > kMost) {
    token = search_row<DT>(a, r, s, scale, b.min_p_y, list, sh);
  } else {
    const int n = (int)sh.n;
    sort_elements(list, n, places);
    token = pick_among(s, scale, b, list, n, mass, rank, mass, rank, sh);
  }
  if (tid == 0) a.tokens[r] = token;
}

template <int DT>
int launch_sample(const tamd_sample_args &args, hipStream_t st) {
  if (sample_whole(args.R, args.V)) {
    whole_row_kernel<DT><<<args.R, kThreads, 0, st>>>(args);
    return launch_status();
  }
  int cus = 0;
  if (int rc = cu_count(cus)) return rc;
  for (int r = 0; r < args.R; r += kRowsAtOnce) {
    tamd_sample_args a = args;
    a.R = args.R - r < kRowsAtOnce ? args.R - r : kRowsAtOnce;
    a.logits = (const uint8_t *)a.logits + r * a.logits_stride * dtype_size(a.logits_dtype);
    a.u += r, a.tokens += r;
    if (a.temperature) a.temperature += r;
    if (a.top_k) a.top_k += r;
    if (a.top_p) a.top_p += r;
    if (a.min_p) a.min_p += r;
    // chunks of 8192, longer ones where these are more than two workgroups per CU (each scans the row's histogram) or more than a wave reads
    int chunk = kChunk;
    while ((int64_t)((a.V + chunk - 1) / chunk) * a.R > 2 * cus && chunk < 8 * kChunk) chunk *= 2;
    while ((a.V + chunk - 1) / chunk > kMaxChunks) chunk *= 2;
    const Workspace ws = workspace_of(a.workspace, a.R);
    const dim3 grid((unsigned)((a.V + chunk - 1) / chunk), (unsigned)a.R);
    chunk = ((a.V + (int)grid.x - 1) / (int)grid.x + 255) / 256 * 256;   // all of them alike (grid.x of these are V or more)
    extremes_kernel<DT><<<grid, kThreads, 0, st>>>(a, ws, chunk);
    histogram_kernel<DT><<<grid, kThreads, 0, st>>>(a, ws, chunk);
    bounds_kernel<<<a.R, kThreads, 0, st>>>(a, ws, (int)grid.x);
    collect_kernel<DT><<<grid, kThreads, 0, st>>>(a, ws, chunk);
    finish_kernel<DT><<<a.R, kThreads, 0, st>>>(a, ws);
    if (int rc = launch_status()) return rc;
  }
  return 0;
}

}  // namespace
}  // namespace tamd

using namespace tamd;

extern "C" int64_t tamd_sample_workspace(int R, int V) {
  if (R < 0 || V < 0) return TAMD_E_INVALID;
  return V <= kShort ? 16 : (R < kRowsAtOnce ? R : kRowsAtOnce) * kRowBytes + 16;
}

extern "C" int64_t tamd_sample_workspace_exact(int R, int V) {
  if (R < 0 || V < 0) return TAMD_E_INVALID;
  return sample_whole(R, V) ? 16 : tamd_sample_workspace(R, V);
}

extern "C" int tamd_sample(const tamd_sample_args *args, size_t args_size, void *stream) {
  if (!args || args_size != sizeof(tamd_sample_args)) return TAMD_E_INVALID;
  const tamd_sample_args &a = *args;
  if (a.R < 0 || a.V < 1) return TAMD_E_INVALID;
  if (a.logits_dtype != TAMD_F32 && a.logits_dtype != TAMD_BF16 && a.logits_dtype != TAMD_F16) return TAMD_E_UNSUPPORTED;
  if (a.V > (1 << 20) || a.R > (1 << 20)) return TAMD_E_TOO_LARGE;
  if (a.R == 0) return 0;
  if (!a.logits || !a.u || !a.tokens || !a.workspace || a.logits_stride < 0) return TAMD_E_INVALID;
  if ((uintptr_t)a.workspace % 16 != 0) return TAMD_E_ALIGNMENT;
  hipStream_t st = (hipStream_t)stream;
  return a.logits_dtype == TAMD_F32 ? launch_sample<TAMD_F32>(a, st) : a.logits_dtype == TAMD_BF16 ? launch_sample<TAMD_BF16>(a, st) : launch_sample<TAMD_F16>(a, st);
}
