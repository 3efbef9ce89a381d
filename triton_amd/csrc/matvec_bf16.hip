// bfloat16 rows of the product with 4-bit weights.
#include "matvec.h"

namespace tamd {
int matvec_bf16(const tamd_matvec_args &a, hipStream_t st) { return matvec_of<TAMD_BF16>(a, st); }
}  // namespace tamd
