// Gradient of the picked gate weights brought back to the logits.  With the picks i_1 .. i_k of a row, z_j its logits there and d_j the
// gradient of pick j's weight:
//   softmax    p = softmax(z over the picks),  dx[i_j] = p_j (d_j - sum_m p_m d_m)
//   plain      dx[i_j] = d_j
// and 0 in every other column.  p is computed again from the logits in float32: the weights that the forward pass stored may have been
// rounded to 16 bits.  LANES lanes share a row: the picks sit in the first of them, every lane writes 16 bytes of the row at a
// time and asks the others which of its columns were picked; equal picks of a row add up, in their order.
#include "common.h"
#include <type_traits>

using namespace tamd;

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

struct TopkBackward {
  const void *x;
  int64_t x_stride;
  const int16_t *indx;
  int64_t indx_stride;
  const void *d;
  int64_t d_stride;
  void *dx;
  int64_t dx_stride;
  int64_t rows, live;     // rows, and those of them that were routed
  int E, k, softmax, d_dtype;
};

template <int L, typename OP>
TAMD_DEVICE float over_lanes(float v, OP op) {
  return bits_to_f32(group_reduce<L>(f32_to_bits(v), [&](uint32_t a, uint32_t b) { return f32_to_bits(op(bits_to_f32(a), bits_to_f32(b))); }));
}

// A row's picks in its lanes' registers: k <= LANES.
template <int DT, int LANES, bool ALIGNED>
__global__ __launch_bounds__(256) void topk_backward_kernel(TopkBackward a) {
  constexpr int V = DT == TAMD_F32 ? 4 : 8;
  const int lane = threadIdx.x & (LANES - 1);
  const int64_t row = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  if (row >= a.rows) return;    // (a whole group of lanes)
  int col = -1;
  float g = 0.f;
  if (lane < a.k && row < a.live) {
    const int c = a.indx[row * a.indx_stride + lane];
    if (c >= 0 && c < a.E) {
      const int64_t at = row * a.d_stride + lane;
      col = c;
      g = a.d_dtype == TAMD_F32 ? load_as_f32<TAMD_F32>(a.d, at) : a.d_dtype == TAMD_BF16 ? load_as_f32<TAMD_BF16>(a.d, at) : load_as_f32<TAMD_F16>(a.d, at);
    }
  }
  if (a.softmax) {
    const auto larger = [](float x, float y) { return __builtin_fmaxf(x, y); };
    const auto added = [](float x, float y) { return x + y; };
    const float z = col >= 0 ? load_as_f32<DT>(a.x, row * a.x_stride + col) : -__builtin_inff();
    const float most = over_lanes<LANES>(z, larger);
    const float e = col >= 0 ? expf(z - most) : 0.f;
    const float p = e / over_lanes<LANES>(e, added);
    const float dot = over_lanes<LANES>(col >= 0 ? p * g : 0.f, added);
    g = p * (g - dot);
  }
  for (int c0 = lane * V; c0 - lane * V < a.E; c0 += LANES * V) {
    float v[V] = {};
    for (int j = 0; j < a.k; ++j) {
      const int at = __shfl(col, j, LANES) - c0;
      const float of = __shfl(g, j, LANES);
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] += at == e ? of : 0.f;
    }
    if (ALIGNED && c0 + V <= a.E) {
      u32x4_t out;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (DT == TAMD_F32) out[e] = f32_to_bits(v[e]);
        else if constexpr (DT == TAMD_BF16) out[e] = f32_to_bf16_bits(v[2 * e]) | (f32_to_bf16_bits(v[2 * e + 1]) << 16);
        else out[e] = f32_to_f16_bits(v[2 * e]) | (f32_to_f16_bits(v[2 * e + 1]) << 16);
      }
      *(u32x4_t *)((char *)a.dx + (row * a.dx_stride + c0) * (16 / V)) = out;
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (c0 + e < a.E) store_from_f32<DT>(a.dx, row * a.dx_stride + c0 + e, v[e]);
    }
  }
}

}  // namespace

extern "C" int tamd_topk_backward(const void *x, int dtype, int64_t x_stride, int64_t n_rows, int64_t n_live, int n_cols, int k, int apply_softmax,
                                  const int16_t *indx, int64_t indx_stride, const void *dvals, int dvals_dtype, int64_t dvals_stride, void *dx,
                                  int64_t dx_stride, void *stream) {
  if (n_rows < 0 || n_live < 0 || n_cols < 0 || k < 0 || x_stride < 0 || indx_stride < 0 || dvals_stride < 0 || dx_stride < 0) return TAMD_E_INVALID;
  const auto plain = [](int dt) { return dt == TAMD_F32 || dt == TAMD_BF16 || dt == TAMD_F16; };
  if (!plain(dtype) || !plain(dvals_dtype)) return TAMD_E_UNSUPPORTED;
  if (n_cols >= 32768 || k > 64 || n_rows >= ((int64_t)1 << 32)) return TAMD_E_TOO_LARGE;
  if (n_rows == 0 || n_cols == 0) return 0;
  if (!dx || (k > 0 && n_live > 0 && (!indx || !dvals || (apply_softmax && !x)))) return TAMD_E_INVALID;
  const int size = dtype == TAMD_F32 ? 4 : 2;
  if ((uintptr_t)x % size || (uintptr_t)dvals % (dvals_dtype == TAMD_F32 ? 4 : 2) || (uintptr_t)dx % size || (uintptr_t)indx % 2) return TAMD_E_ALIGNMENT;
  const TopkBackward a{x, x_stride, indx, indx_stride, dvals, dvals_stride, dx, dx_stride, n_rows, n_live, n_cols, k, apply_softmax != 0, dvals_dtype};
  hipStream_t st = (hipStream_t)stream;
  const bool aligned = ((uintptr_t)dx | (uintptr_t)(dx_stride * size)) % 16 == 0;
  // 16 lanes to a row where they hold its picks and write it in few turns, else a wave
  const bool narrow = k <= 16 && n_cols <= 512;
  if (n_rows * (narrow ? 16 : 64) > 0xFFFFFF00ll) return TAMD_E_TOO_LARGE;   // (a launch counts its threads in 32 bits)
  const auto go = [&](auto dt, auto lanes) {
    constexpr int DT = decltype(dt)::value, L = decltype(lanes)::value;
    const unsigned blocks = (unsigned)((n_rows + 256 / L - 1) / (256 / L));
    if (aligned) topk_backward_kernel<DT, L, true><<<blocks, 256, 0, st>>>(a);
    else topk_backward_kernel<DT, L, false><<<blocks, 256, 0, st>>>(a);
  };
  const auto with = [&](auto dt) {
    if (narrow) go(dt, std::integral_constant<int, 16>());
    else go(dt, std::integral_constant<int, 64>());
  };
  if (dtype == TAMD_F32) with(std::integral_constant<int, TAMD_F32>());
  else if (dtype == TAMD_BF16) with(std::integral_constant<int, TAMD_BF16>());
  else with(std::integral_constant<int, TAMD_F16>());
  return launch_status();
}
