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

__device__ __forceinline__ int attn_units(const AttnCut& cut, int seen) { return ((seen - 1) >> cut.unit_log2) + 1; }

// Units of a share, so that cut.shares of them hold `units`.
__device__ __forceinline__ int64_t attn_share(const AttnCut& cut, int64_t units) {
  return units <= cut.shares ? 1 : (int64_t)((double)units * cut.each) + 1;
}
// The share that unit `at` is in.
__device__ __forceinline__ int attn_share_of(int64_t at, int64_t share) {
  int64_t n = (int64_t)((double)at / (double)share);
  while (n * share > at) --n;
  while ((n + 1) * share <= at) ++n;
  return (int)n;
}

// How far an end of a share of `share` units may move to spare a tile a part; in a tile of `units`, less than half of
// them, so that an end behind the tile stays behind it.
__device__ __forceinline__ int attn_slack(int64_t share) { return (int)min(share / 16, (int64_t)1 << 20); }
__device__ __forceinline__ int attn_slack_in(int slack, int units) { return min(slack, (units - 1) / 2); }

// The item that share `index` has of a tile of `seen` positions, whose units begin at `start`; false if none.  A share
// has two places among the partial results: for the tile that it begins within, and for the one that it ends within.
__device__ __forceinline__ bool attn_item(const AttnCut& cut, const AttnWorker& w, int index, int seen, int64_t start,
                                          AttnItem& it) {
  const int units = attn_units(cut, seen), slack = attn_slack_in(w.slack, units);
  const int64_t end = start + units;
  auto near = [&](int64_t at) { return at <= start + slack ? start : at >= end - slack ? end : at; };
  const int64_t lo = near(w.from), hi = near(w.to);
  if (lo >= hi) return false;
  it.key0 = (int)(lo - start) << cut.unit_log2;
  it.key1 = (int)min((hi - start) << cut.unit_log2, (int64_t)seen);
  it.part = lo == start && hi == end ? -1 : 2 * index + (lo == start && w.from < start - cut.overhead);
  return true;
}
// The join of a tile of which share `index` has the first units but not the last.
__device__ __forceinline__ AttnJoin attn_join(const AttnCut& cut, const AttnItem& it, int seen, int64_t start,
                                              int64_t share, int index) {
  const int units = attn_units(cut, seen);
  const int64_t last = start + units - attn_slack_in(attn_slack(share), units) - 1;  // the last part begins by here
  return AttnJoin{it.begin, it.length, it.m0, attn_share_of(last, share) - index + 1, it.part, 2 * (index + 1),
                  it.sequence};
}

// Element 0 of position `pos` of kv head 0 (heads are 1 << page_shift rows apart).
__device__ __forceinline__ size_t attn_cell(const AttnPlan& p, int layer, int page, int pos) {
  return ((((size_t)layer * p.pages + page) * p.kv_heads << p.page_shift) + (pos & ((1 << p.page_shift) - 1))) *
         p.head_dim;
}

// Eight elements in the cache's type, to the nearest; what is beyond it becomes an infinity.
template <typename T>
using attn_eight = T __attribute__((ext_vector_type(8)));
template <typename To, typename From>
__device__ __forceinline__ void attn_put8(To* to, const attn_eight<From>& v) {
  typedef attn_eight<To> To8;
  if constexpr (sizeof(From) == sizeof(To)) *reinterpret_cast<To8*>(to) = __builtin_bit_cast(To8, v);
  else *reinterpret_cast<To8*>(to) = __builtin_convertvector(v, To8);
}

}  // namespace llhip
