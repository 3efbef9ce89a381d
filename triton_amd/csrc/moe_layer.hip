// Entry point of the whole expert layer: checks, then the launches of the activations' type.
#include "moe_layer.h"

namespace tamd {
namespace {

int check_moe_weights(const tamd_moe_weights &p, int64_t K, int64_t N) {
  if (!p.w || !p.scale) return TAMD_E_INVALID;
  if (p.bias && p.bias_dtype != TAMD_F32 && p.bias_dtype != TAMD_F16 && p.bias_dtype != TAMD_BF16) return TAMD_E_INVALID;
  if (p.w_layout != TAMD_W_STRIDED && p.w_layout != TAMD_W_CDNA4_BLOCKS) return TAMD_E_INVALID;
  if (p.scale_layout != TAMD_SCALE_STRIDED && p.scale_layout != TAMD_SCALE_CDNA4) return TAMD_E_INVALID;
  const bool blocks = p.w_layout == TAMD_W_CDNA4_BLOCKS, shuffled = p.scale_layout == TAMD_SCALE_CDNA4;
  if (p.w_stride_e < 0 || p.scale_stride_e < 0 || (!blocks && p.w_stride_n < 0) || (!shuffled && p.scale_stride_n < 0)) return TAMD_E_INVALID;
  if (!aligned(p.w, 16) || p.w_stride_e % 16 != 0 || (!blocks && p.w_stride_n % 16 != 0)) return TAMD_E_ALIGNMENT;
  if (shuffled && (!aligned(p.scale, 16) || p.scale_stride_e % 16 != 0)) return TAMD_E_ALIGNMENT;
  if (p.bias && (!aligned(p.bias, 4) || (p.bias_dtype != TAMD_F32 && p.bias_stride_e % 2 != 0))) return TAMD_E_ALIGNMENT;   // pairs of 16-bit numbers
  // one expert is addressed with 32 bits
  const int64_t most = kMoeOob, w_bytes = blocks ? (N + 63) / 64 * ((K + 127) / 128) * 4096 : K / 2;
  if (w_bytes >= most || (!blocks && p.w_stride_n >= (most - w_bytes) / N)) return TAMD_E_UNSUPPORTED;
  if (!shuffled && p.scale_stride_n >= (most - K / 32) / N) return TAMD_E_UNSUPPORTED;
  return 0;
}

}  // namespace
}  // namespace tamd

using namespace tamd;

extern "C" int64_t tamd_moe_layer_workspace(int n_tokens, int n_picks, int inter) {
  if (n_tokens < 0 || n_picks < 0 || inter < 0) return TAMD_E_INVALID;
  return moe_partial_at((int64_t)n_tokens * n_picks, inter) + (int64_t)kMoeShares * 2 * n_tokens * 16 * 4;
}

extern "C" int tamd_moe_layer(const tamd_moe_layer_args *args, size_t args_size, void *stream) {
  if (!args || args_size != sizeof(tamd_moe_layer_args)) return TAMD_E_INVALID;
  const tamd_moe_layer_args &a = *args;
  if (a.n_tokens < 0 || a.n_experts < 1 || a.n_picks < 1 || a.n_picks > a.n_experts) return TAMD_E_INVALID;
  if (a.hidden < 32 || a.hidden % 32 != 0 || a.inter < 32 || a.inter % 32 != 0) return TAMD_E_INVALID;
  if (a.x_dtype != TAMD_BF16 && a.x_dtype != TAMD_F16) return TAMD_E_UNSUPPORTED;
  if (a.logits_dtype != TAMD_F32 && a.logits_dtype != TAMD_BF16 && a.logits_dtype != TAMD_F16) return TAMD_E_INVALID;
  if (a.n_tokens > kMoeTokens || a.n_experts > kMoeExperts || a.n_picks > kMoePicks || (int64_t)a.n_tokens * a.n_picks > kMoeSlots)
    return TAMD_E_TOO_LARGE;
  if (a.n_tokens == 0) return 0;
  if (!a.x || !a.logits || !a.y || !a.workspace || a.x_stride_m < 0 || a.logits_stride < 0 || a.y_stride_m < 0) return TAMD_E_INVALID;
  if (a.hidden > (1 << 20) || a.inter > (1 << 20)) return TAMD_E_UNSUPPORTED;   // (products of sizes below stay in 64 bits, grids in 31)
  if (!aligned(a.x, 16) || a.x_stride_m % 8 != 0 || !aligned(a.workspace, 16)) return TAMD_E_ALIGNMENT;
  if (a.x_stride_m >= ((int64_t)kMoeOob - 2 * a.hidden) / (2 * kMoeTokens)) return TAMD_E_UNSUPPORTED;   // rows are addressed with 32 bits
  if ((int64_t)a.n_tokens * a.n_picks * a.inter * 4 >= (int64_t)kMoeOob) return TAMD_E_UNSUPPORTED;
  if (int rc = check_moe_weights(a.up, a.hidden, 2 * (int64_t)a.inter)) return rc;
  if (int rc = check_moe_weights(a.down, a.inter, a.hidden)) return rc;
  hipStream_t st = (hipStream_t)stream;
  return a.x_dtype == TAMD_BF16 ? moe_layer_bf16(a, st) : moe_layer_f16(a, st);
}
