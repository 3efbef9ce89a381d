// Entry points of the products over ragged rows: checks, the choice of the tile and of the splits of long slices, and the sum of these; rows laid out
// for the kernels' copies.
#include "mx_values.h"
#include "ragged_k.h"

using namespace tamd;

namespace {

struct Plan {
  int tile, tiles_m, tiles_n, splits;   // tile: a RaggedTile
  int64_t pitch;                        // elements of a row of partial sums
  bool longest_first;
  bool lay_x, lay_d;                    // operands that the copies cannot take as they are
  int64_t x_at, d_at, part_at, bytes;   // where these and the partial sums lie in the workspace
};

int filled_up(int cols) { return (cols + 7) / 8 * 8; }

// Rows that copies of 16 bytes take whole, and a stage's of which 31 bits count.  Rows that overlap (an expanded operand's have a pitch of 0) are
// none: the copies' bounds end a slice by the bytes up to its last row's end, which keep the next row out only if that begins behind them.
bool whole(const void *q, int64_t pitch, int cols) { return (uintptr_t)q % 16 == 0 && pitch % 8 == 0 && cols % 8 == 0 && pitch >= cols && pitch < 1 << 24; }
// Rows that can be laid out by one launch, whose threads are counted in 32 bits
bool few_enough(int64_t K, int cols) { return K * (filled_up(cols) / 8) <= 0xFFFFFF00ll; }

// The tile by the rows of a slice in the mean and the tiles that there are (figures beside RaggedTile), and the splits of long slices of few
// tiles: a stage of 32 rows takes 0.57 us in a workgroup of its own; the partial sums cost a launch of 5 us, and 8 bytes each at the caches' rate.
Plan make_plan(const tamd_ragged_k_args &a) {
  const int M = a.M, N = a.N, E = a.E;
  const int64_t K = a.K;
  Plan p;
  const auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  const int64_t rows = K / E, flat = up(M, 128) * up(N, 256), tall = up(M, 256) * up(N, 128), n = up(M, 128) * up(N, 128) * E;
  const int64_t few = (flat <= tall ? flat : tall) * E;
  const bool large = rows >= 256 && few >= 1024 && rows * few >= 393216;
  p.tile = large ? (flat <= tall ? kTile128x256 : kTile256x128) : (rows <= 128 ? kTile128Short : kTile128);
  p.tiles_m = (int)up(M, p.tile == kTile256x128 ? 256 : 128), p.tiles_n = (int)up(N, p.tile == kTile128x256 ? 256 : 128);
  p.splits = 1;
  const double stages = (double)up(rows, 32);
  double best = 0.57 * stages;
  for (int s = 2; !large && s <= 64 && s * n <= 512; s *= 2) {
    const double t = 0.57 * up((int64_t)stages, s) + 5.0 + (double)s * E * M * N * 8 / 4e6;
    if (t < best) best = t, p.splits = s;
  }
  // The longest slices first, so that the last round of workgroups is of short ones, where a slice has rows enough to pay for the order (8 comparisons to
  // eight slices in every workgroup): 30966 rows over 8 slices of 1200 to 7800, 2152 x 424, 123 us in place of 154; 6448 over 8, 1152 x 4736, 86 and 95; 43728
  // over 32, 640 x 4608, 287 and 295; 17056 over 60, 936 x 4040, 254 and 252 (not so, with 284 rows).  Slices of one length lose up to 1 %.
  p.longest_first = E > 1 && E <= 64 && rows > 128 && rows >= 16 * E;
  p.pitch = ((int64_t)N + 3) / 4 * 4;
  p.lay_x = K > 0 && !whole(a.x, a.x_stride, M), p.lay_d = K > 0 && !whole(a.d, a.d_stride, N);
  p.x_at = 0;
  p.d_at = p.x_at + (p.lay_x ? K * filled_up(M) * 2 : 0);
  p.part_at = p.d_at + (p.lay_d ? K * filled_up(N) * 2 : 0);
  p.bytes = p.part_at + (p.splits > 1 ? p.splits * (int64_t)E * M * p.pitch * 4 : 0);
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

// Rows of C elements to rows of whole 16-byte pieces, the last one filled up with zeros: a thread per piece, read with what alignment it has.
// One launch for both operands (blockIdx.y).
struct Laid {
  const uint16_t *src;
  uint16_t *dst;
  int64_t pitch, pieces, per;
  FastDiv by;
  int C;
};
struct LaidBoth {
  Laid of[2];
};
__global__ __launch_bounds__(256) void lay_rows_kernel(LaidBoth both) {
  const Laid &l = both.of[blockIdx.y];
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= l.pieces) return;
  const int64_t row = l.pieces < ((int64_t)1 << 31) ? (int64_t)div_by((uint32_t)at, l.by) : at / l.per, col = (at - row * l.per) * 8;
  const uint16_t *const p = l.src + row * l.pitch + col;
  u32x4_t q = {0, 0, 0, 0};
  if (col + 8 <= l.C) {
    q = *(const u32x4_by2_t *)p;
  } else {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (col + e < l.C) q[e / 2] |= (uint32_t)p[e] << (16 * (e & 1));
  }
  *(u32x4_t *)(l.dst + at * 8) = q;
}
Laid laid(const void *src, int64_t pitch, int C, int64_t K, void *dst) {
  const int64_t per = filled_up(C) / 8;
  return Laid{(const uint16_t *)src, (uint16_t *)dst, pitch, K * per, per, fast_div(per), C};
}

bool sizes_ok(int M, int N, int E, int64_t K) { return M >= 0 && N >= 0 && E >= 0 && K >= 0; }
bool too_large(int M, int N, int E, int64_t K) {
  return K >= ((int64_t)1 << 31) || M >= 1 << 24 || N >= 1 << 24 || (double)K * (M > N ? M : N) > 2e12 || (double)((M + 127) / 128) * ((N + 127) / 128) * E > 8e6 || (double)E * M * N > 2e12;
}

// 0 and `ok` for a call that computes something, 0 for one that need not, or an error
int check(const tamd_ragged_k_args *args, size_t args_size, bool &ok) {
  ok = false;
  if (!args || args_size != sizeof(tamd_ragged_k_args)) return TAMD_E_INVALID;
  const tamd_ragged_k_args &a = *args;
  if (!sizes_ok(a.M, a.N, a.E, a.K)) return TAMD_E_INVALID;
  if (a.dtype != TAMD_BF16 && a.dtype != TAMD_F16) return TAMD_E_UNSUPPORTED;
  if (a.y_dtype != TAMD_F32 && a.y_dtype != TAMD_BF16 && a.y_dtype != TAMD_F16) return TAMD_E_UNSUPPORTED;
  if (a.x_stride < 0 || a.d_stride < 0 || a.y_stride_e < 0 || a.y_stride_m < 0) return TAMD_E_INVALID;
  if (a.M == 0 || a.N == 0 || a.E == 0) return 0;
  if (too_large(a.M, a.N, a.E, a.K)) return TAMD_E_TOO_LARGE;
  if ((!whole(a.x, a.x_stride, a.M) && !few_enough(a.K, a.M)) || (!whole(a.d, a.d_stride, a.N) && !few_enough(a.K, a.N))) return TAMD_E_TOO_LARGE;
  if (!a.y || !a.slice_offs || !a.slice_sizes || (a.K > 0 && (!a.x || !a.d))) return TAMD_E_INVALID;
  if ((uintptr_t)a.slice_offs % 4 || (uintptr_t)a.slice_sizes % 4 || (uintptr_t)a.x % 2 || (uintptr_t)a.d % 2 || (uintptr_t)a.y % (a.y_dtype == TAMD_F32 ? 4 : 2)) return TAMD_E_ALIGNMENT;
  ok = true;
  return 0;
}

}  // namespace

extern "C" int64_t tamd_ragged_k_matmul_workspace(const tamd_ragged_k_args *args, size_t args_size) {
  bool ok;
  const int rc = check(args, args_size, ok);
  return ok ? make_plan(*args).bytes : rc;
}

extern "C" int tamd_ragged_k_matmul(const tamd_ragged_k_args *args, size_t args_size, void *stream) {
  bool ok;
  if (const int rc = check(args, args_size, ok)) return rc;
  if (!ok) return 0;
  const tamd_ragged_k_args &a = *args;
  const Plan p = make_plan(a);
  if (p.bytes > 0 && !a.workspace) return TAMD_E_INVALID;
  if (p.bytes > 0 && (uintptr_t)a.workspace % 16) return TAMD_E_ALIGNMENT;
  hipStream_t st = (hipStream_t)stream;
  uint8_t *const room = (uint8_t *)a.workspace;
  const int size = a.y_dtype == TAMD_F32 ? 4 : 2;
  RaggedK k{a.x, a.d, a.x_stride, a.d_stride, a.M, a.N, a.slice_offs, a.slice_sizes, a.y, a.y_stride_e, a.y_stride_m, 0, a.K, a.M, a.N, a.E, a.y_dtype, 0, 0, p.tiles_m, p.tiles_n, p.splits, p.longest_first};
  LaidBoth both;
  int n = 0;
  if (p.lay_x) {
    k.x = room + p.x_at, k.x_cols = filled_up(a.M), k.x_pitch = k.x_cols;
    both.of[n++] = laid(a.x, a.x_stride, a.M, a.K, room + p.x_at);
  }
  if (p.lay_d) {
    k.d = room + p.d_at, k.d_cols = filled_up(a.N), k.d_pitch = k.d_cols;
    both.of[n++] = laid(a.d, a.d_stride, a.N, a.K, room + p.d_at);
  }
  if (n > 0) {
    const int64_t most = n > 1 && both.of[1].pieces > both.of[0].pieces ? both.of[1].pieces : both.of[0].pieces;
    lay_rows_kernel<<<dim3((unsigned)((most + 255) / 256), n), 256, 0, st>>>(both);
    if (const int rc = launch_status()) return rc;
  }
  if (p.splits > 1) {
    k.y = room + p.part_at, k.y_dtype = TAMD_F32, k.y_stride_m = p.pitch, k.y_stride_e = a.M * p.pitch, k.y_stride_split = (int64_t)a.E * a.M * p.pitch;
  } else {
    k.whole_lines = ((uintptr_t)a.y | (uintptr_t)(a.y_stride_m * size) | (uintptr_t)(a.y_stride_e * size)) % 128 == 0;
    k.past_caches = a.K / a.E >= 64;
  }
  const int rc = a.dtype == TAMD_BF16 ? ragged_k_bf16(k, p.tile, stream) : ragged_k_f16(k, p.tile, stream);
  if (rc != 0 || p.splits == 1) return rc;
  const int64_t rows = (int64_t)a.E * a.M, threads = rows * (p.pitch / 4);
  ragged_k_join_kernel<<<(unsigned)((threads + 255) / 256), 256, 0, st>>>((const float *)(room + p.part_at), rows, a.N, p.pitch, p.splits, a.y, a.y_stride_e, a.y_stride_m,
                                                                         a.M, a.y_dtype);
  return launch_status();
}
