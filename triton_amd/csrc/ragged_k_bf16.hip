// Products over ragged rows: bf16 operands.
#include "ragged_k.h"

namespace tamd {
int ragged_k_bf16(const RaggedK &a, int tile, void *stream) { return ragged_k_typed<TAMD_BF16>(a, tile, (hipStream_t)stream); }
}  // namespace tamd
