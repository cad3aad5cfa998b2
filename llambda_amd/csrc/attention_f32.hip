// attention_f32.hip -- the attention kernels of caches in f32 (attention_tile.h).
#include "attention_tile.h"

namespace llhip {

hipError_t attn_attend_f32(const AttnPlan& p, const AttnCall& c, const AttnCut& cut, uint32_t grid, hipStream_t s) {
  return attn_attend_width<kAttnF32, float>(p, c, cut, grid, s);
}

}  // namespace llhip
