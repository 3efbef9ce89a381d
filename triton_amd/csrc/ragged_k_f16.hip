// Products over ragged rows: f16 operands.
#include "ragged_k.h"

namespace tamd {
int ragged_k_f16(const RaggedK &a, int tile, void *stream) { return ragged_k_typed<TAMD_F16>(a, tile, (hipStream_t)stream); }
}  // namespace tamd
