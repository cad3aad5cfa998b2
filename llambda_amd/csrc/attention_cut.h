// attention_cut.h -- how a call is cut into items, and where a position lies, for the kernels of attention.hip and
// attention_tile.h alike.
#pragma once

#include "attention.h"

namespace llhip {

// Positions that the rows m0 .. m0 + cut.rows - 1 of a sequence see.
__device__ __forceinline__ int attn_seen_keys(const AttnPlan& p, const AttnCall& c, const AttnCut& cut, int m0,
                                              int length, int context) {
  if (c.parents) return context + length;
  return context + min(length, (m0 + cut.rows - 1) / p.group + 1);
}

// Positions of a part, whole tiles: about the work of a kv head's rows (`keys`, over all tiles) over the workgroups
// that the device holds.
__device__ __forceinline__ int attn_chunk(const AttnPlan& p, const AttnCut& cut, int64_t keys) {
  const int64_t share = ((keys * p.kv_heads - 1) >> cut.slots_log2) + 1;
  return ((int)min(max(share, (int64_t)cut.min_keys), (int64_t)1 << 30) + 63) & ~63;
}

// Parts of the positions that a tile sees, no longer than `chunk`.
__device__ __forceinline__ int attn_parts_of(int seen, int chunk) {
  return seen <= chunk ? 1 : (int)(((uint32_t)seen + chunk - 1) / (uint32_t)chunk);
}
// Part k of the n equal ones, of whole tiles.  (None is empty: they are no longer than the chunk that n came from.)
__device__ __forceinline__ void attn_part(AttnItem& it, int seen, int n, int k, int part) {
  const uint32_t size = n > 1 ? (((uint32_t)seen + n - 1) / n + 63) & ~63u : seen;
  it.key0 = k * size;
  it.key1 = min((k + 1) * size, (uint32_t)seen);
  it.part = n > 1 ? part + k : -1;
}

// Element 0 of position `pos` of kv head 0 (heads are 1 << page_shift rows apart).
__device__ __forceinline__ size_t attn_cell(const AttnPlan& p, int layer, int page, int pos) {
  return ((((size_t)layer * p.pages + page) * p.kv_heads << p.page_shift) + (pos & ((1 << p.page_shift) - 1))) *
         p.head_dim;
}

// Eight elements in the cache's type, to the nearest; what is beyond it becomes an infinity.
template <typename To, typename From>
__device__ __forceinline__ void attn_put8(To* to, const From* from) {
  typedef From From8 __attribute__((ext_vector_type(8)));
  typedef To To8 __attribute__((ext_vector_type(8)));
  const From8 v = *reinterpret_cast<const From8*>(from);
  if constexpr (sizeof(From) == sizeof(To)) *reinterpret_cast<To8*>(to) = __builtin_bit_cast(To8, v);
  else *reinterpret_cast<To8*>(to) = __builtin_convertvector(v, To8);
}

}  // namespace llhip
