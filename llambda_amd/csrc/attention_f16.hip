// attention_f16.hip -- the attention kernels of caches in f16 (attention_tile.h).
#include "attention_tile.h"

namespace llhip {

hipError_t attn_attend_f16(const AttnPlan& p, const AttnCall& c, const AttnCut& cut, uint32_t grid, hipStream_t s) {
  if (p.row_type == kAttnF16) return attn_attend_width<kAttnF16, _Float16>(p, c, cut, grid, s);
  return attn_attend_width<kAttnF16, float>(p, c, cut, grid, s);
}

}  // namespace llhip
