// float16 rows of the product with 4-bit weights.
#include "matvec.h"

namespace tamd {
int matvec_f16(const tamd_matvec_args &a, hipStream_t st) { return matvec_of<TAMD_F16>(a, st); }
}  // namespace tamd
