// Instantiations of the drafted-token attention kernel (one translation unit per cache and product type, so
// that they compile side by side).
#include "draft_attention_kernel.hpp"

namespace pa {

int launch_draft_bf16_as_f16(const DraftParams& p, int head_dim, int rows, unsigned grid, hipStream_t st) {
  return launch_draft<KV_BF16, CT_F16>(p, head_dim, rows, grid, st);
}

}  // namespace pa
