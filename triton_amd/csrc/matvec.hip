// Entry point of the product with 4-bit weights: checks, then the launch of the rows' type.
#include "matvec.h"

using namespace tamd;

extern "C" int tamd_matvec(const tamd_matvec_args *args, size_t args_size, void *stream) {
  if (!args || args_size != sizeof(tamd_matvec_args)) return TAMD_E_INVALID;
  const tamd_matvec_args &a = *args;
  const auto plain = [](int dt) { return dt == TAMD_F32 || dt == TAMD_BF16 || dt == TAMD_F16; };
  if (a.M < 0 || a.N < 0 || a.K < 32) return TAMD_E_INVALID;
  if (a.group != 32 && a.group != 64 && a.group != 128) return TAMD_E_UNSUPPORTED;
  if (a.K % a.group != 0) return TAMD_E_INVALID;
  if (a.x_dtype != TAMD_BF16 && a.x_dtype != TAMD_F16) return TAMD_E_UNSUPPORTED;
  if (a.scale_dtype != TAMD_BF16 && a.scale_dtype != TAMD_F16) return TAMD_E_UNSUPPORTED;
  if (!plain(a.y_dtype) || (a.bias && !plain(a.bias_dtype))) return TAMD_E_INVALID;
  if (a.M == 0 || a.N == 0) return 0;
  if (!a.x || !a.codes || !a.scales || !a.y || a.x_stride_m < 0 || a.y_stride_m < 0) return TAMD_E_INVALID;
  if (!aligned(a.x, 16) || a.x_stride_m % 8 != 0 || !aligned(a.codes, 16) || !aligned(a.scales, 16) || !aligned(a.zeros, 16)) return TAMD_E_ALIGNMENT;
  if (a.K > (1 << 20) || a.M > 32 * 65535 || a.N > (1 << 30)) return TAMD_E_UNSUPPORTED;   // (a strip and the grid stay in 31 bits)
  if (a.x_stride_m >= ((int64_t)kMoeOob - 2 * a.K) / (2 * kMatvecRows)) return TAMD_E_UNSUPPORTED;  // 64 rows are addressed with 32 bits
  hipStream_t st = (hipStream_t)stream;
  return a.x_dtype == TAMD_BF16 ? matvec_bf16(a, st) : matvec_f16(a, st);
}
