// Entry points of the products over ragged rows: checks, the choice of the tile and of the splits of long slices, and the sum of these.
#include "ragged_k.h"

using namespace tamd;

namespace {

struct Plan {
  int tile, tiles_m, tiles_n, splits;
  int64_t pitch, bytes;      // of the partial sums: elements of a row, bytes of all
};

// Tiles of 256 x 256 where they fill the chip and slices are long, else of 128 x 128; slices cut where tiles alone leave CUs idle.
Plan make_plan(int M, int N, int E, int64_t K) {
  Plan p;
  const auto tiles = [&](int b) { return (int64_t)((M + b - 1) / b) * ((N + b - 1) / b) * E; };
  const int64_t rows = K / E;     // in the mean
  p.tile = rows >= 256 && tiles(256) >= 256 ? 256 : 128;
  p.tiles_m = (M + p.tile - 1) / p.tile, p.tiles_n = (N + p.tile - 1) / p.tile;
  const int64_t n = tiles(p.tile);
  int64_t s = n >= 256 ? 1 : 512 / n;
  if (s > rows / 256) s = rows / 256;
  p.splits = (int)(s < 1 ? 1 : s);
  p.pitch = ((int64_t)N + 3) / 4 * 4;
  p.bytes = p.splits > 1 ? p.splits * (int64_t)E * M * p.pitch * 4 : 0;
  return p;
}

__global__ __launch_bounds__(256) void ragged_k_join_kernel(const float *__restrict__ part, int64_t rows, int N, int64_t pitch, int splits, void *__restrict__ y,
                                                            int64_t y_stride_e, int64_t y_stride_m, int M, int y_dtype) {
  const int64_t per = pitch / 4, at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= rows * per) return;
  const int64_t row = at / per, e = row / M, m = row - e * M;
  const int n = (int)(at - row * per) * 4;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = 0; s < splits; ++s) {   // (columns past N hold what the memory held; they go nowhere)
    const float4 v = *(const float4 *)(part + (s * rows + row) * pitch + n);
    sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
  }
  const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (n + j >= N) continue;
    const int64_t to = e * y_stride_e + m * y_stride_m + n + j;
    if (y_dtype == TAMD_F32) store_from_f32<TAMD_F32>(y, to, v[j]);
    else if (y_dtype == TAMD_BF16) store_from_f32<TAMD_BF16>(y, to, v[j]);
    else store_from_f32<TAMD_F16>(y, to, v[j]);
  }
}

bool sizes_ok(int M, int N, int E, int64_t K) { return M >= 0 && N >= 0 && E >= 0 && K >= 0; }
bool too_large(int M, int N, int E, int64_t K) {
  return K >= ((int64_t)1 << 31) || (double)((M + 127) / 128) * ((N + 127) / 128) * E > 8e6 || (double)E * M * N > 2e12;
}

}  // namespace

extern "C" int64_t tamd_ragged_k_matmul_workspace(int M, int N, int E, int64_t K) {
  if (!sizes_ok(M, N, E, K)) return TAMD_E_INVALID;
  if (M == 0 || N == 0 || E == 0) return 0;
  if (too_large(M, N, E, K)) return TAMD_E_TOO_LARGE;
  return make_plan(M, N, E, K).bytes;
}

extern "C" int tamd_ragged_k_matmul(const tamd_ragged_k_args *args, size_t args_size, void *stream) {
  if (!args || args_size != sizeof(tamd_ragged_k_args)) return TAMD_E_INVALID;
  const tamd_ragged_k_args &a = *args;
  if (!sizes_ok(a.M, a.N, a.E, a.K)) return TAMD_E_INVALID;
  if (a.dtype != TAMD_BF16 && a.dtype != TAMD_F16) return TAMD_E_UNSUPPORTED;
  if (a.y_dtype != TAMD_F32 && a.y_dtype != TAMD_BF16 && a.y_dtype != TAMD_F16) return TAMD_E_UNSUPPORTED;
  if (a.x_stride < 0 || a.d_stride < 0 || a.y_stride_e < 0 || a.y_stride_m < 0) return TAMD_E_INVALID;
  if (a.M == 0 || a.N == 0 || a.E == 0) return 0;
  if (too_large(a.M, a.N, a.E, a.K)) return TAMD_E_TOO_LARGE;
  if (!a.y || !a.slice_offs || (a.K > 0 && (!a.x || !a.d))) return TAMD_E_INVALID;
  const int size = a.y_dtype == TAMD_F32 ? 4 : 2;
  if ((uintptr_t)a.x % 2 || (uintptr_t)a.d % 2 || (uintptr_t)a.y % size) return TAMD_E_ALIGNMENT;
  const Plan p = make_plan(a.M, a.N, a.E, a.K);
  if (p.splits > 1 && (!a.workspace || (uintptr_t)a.workspace % 16)) return a.workspace ? TAMD_E_ALIGNMENT : TAMD_E_INVALID;
  // rows that copies of 16 bytes take whole, and a stage's of which 31 bits count
  const auto whole = [](const void *q, int64_t pitch, int cols) { return (uintptr_t)q % 16 == 0 && pitch % 8 == 0 && cols % 8 == 0 && pitch < 1 << 24; };
  const bool dma = whole(a.x, a.x_stride, a.M) && whole(a.d, a.d_stride, a.N);
  RaggedK k{a.x, a.d, a.x_stride, a.d_stride, a.slice_offs, a.y, a.y_stride_e, a.y_stride_m, 0, a.K, a.M, a.N, a.E, a.y_dtype, 0, p.tiles_m, p.tiles_n, p.splits};
  if (p.splits > 1) {
    k.y = a.workspace, k.y_dtype = TAMD_F32, k.y_stride_m = p.pitch, k.y_stride_e = a.M * p.pitch, k.y_stride_split = (int64_t)a.E * a.M * p.pitch, k.whole_stores = 1;
  } else {
    k.whole_stores = (uintptr_t)a.y % 16 == 0 && (a.N * size) % 16 == 0 && (a.y_stride_m * size) % 16 == 0 && (a.y_stride_e * size) % 16 == 0;
  }
  const int rc = a.dtype == TAMD_BF16 ? ragged_k_bf16(k, p.tile, dma, stream) : ragged_k_f16(k, p.tile, dma, stream);
  if (rc != 0 || p.splits == 1) return rc;
  const int64_t rows = (int64_t)a.E * a.M, threads = rows * (p.pitch / 4);
  ragged_k_join_kernel<<<(unsigned)((threads + 255) / 256), 256, 0, (hipStream_t)stream>>>((const float *)a.workspace, rows, a.N, p.pitch, p.splits, a.y, a.y_stride_e,
                                                                                             a.y_stride_m, a.M, a.y_dtype);
  return launch_status();
}
