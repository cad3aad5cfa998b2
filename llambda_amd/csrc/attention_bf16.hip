// attention_bf16.hip -- the attention kernels of caches in bf16 (attention_tile.h).
#include "attention_tile.h"

namespace llhip {

hipError_t attn_attend_bf16(const AttnPlan& p, const AttnCall& c, const AttnCut& cut, uint32_t grid, hipStream_t s) {
  if (p.row_type == kAttnBF16) return attn_attend_width<kAttnBF16, __bf16>(p, c, cut, grid, s);
  return attn_attend_width<kAttnBF16, float>(p, c, cut, grid, s);
}

}  // namespace llhip
