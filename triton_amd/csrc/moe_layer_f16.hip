// float16 activations of the whole expert layer.
#include "moe_layer.h"

namespace tamd {
int moe_layer_f16(const tamd_moe_layer_args &a, hipStream_t st) { return moe_layer_of<TAMD_F16>(a, st); }
}  // namespace tamd
