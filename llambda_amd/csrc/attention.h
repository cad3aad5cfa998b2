// attention.h -- attention of new rows of several sequences over a paged cache
// (attention.hip, attention_tile.h).
//
// Sequence i has c cached tokens and n new rows.  The rows' keys and values are
// rounded to the cache's type and put at positions c .. c + n - 1; then, per row
// r and head h (of kv head h / group), over the positions j that the row sees,
//   s_j = scale q . K_j,   p = softmax(s),   y = sum_j p_j V_j
// A row sees j <= c + r, or, as a node of a tree, j < c, itself and its ancestors.
// Position j of a sequence is row j % page of page table[i][j / page] of the pool
// [layers][pages][kv_heads][page][head_dim].
#pragma once

#include "common.h"

namespace llhip {

constexpr int kAttnMaxHeadDim = 256;
constexpr int kAttnTreeNodes = 256;                    // nodes of a tree, at most
constexpr int kAttnFewSequences = 256;  // of a call that needs no launch before the attend kernel
constexpr int kAttnFewTokens = 256;
constexpr int kAttnTreeWords = kAttnTreeNodes / 32;

enum AttnType : int { kAttnF32 = 0, kAttnF16 = 1, kAttnBF16 = 30 };  // GGML's tags

enum AttnError : int {
  kAttnErrOffsets = 1,  // offsets not ascending within the call's tokens
  kAttnErrContext = 2,  // more tokens than the session's context, or fewer than none
  kAttnErrPage = 4,     // a page outside the pool
  kAttnErrTree = 8,     // a parent that is no earlier node, or too many nodes
  kAttnErrPath = 16,    // an accepted path that does not ascend
};

// A call's work: rows of a sequence and kv head in tiles (row m is token m / group, head m % group of the group), each
// with the positions that it sees in units of 2^AttnCut::unit_log2.  All kv heads' tiles are alike.
struct AttnTile {
  int sequence, begin, length, context;  // the sequence's first row in the call, its rows, cached tokens
  int m0, seen;
  int64_t start;                         // its first unit among all, behind its overhead
};
// A workgroup's share, for each kv head: units from .. to - 1, of tile `tile` and those that follow.  An end of it that lies
// no further than `slack` from an end of a tile is taken to be there.
struct AttnWorker {
  int64_t from, to;
  int tile, slack;
};
// What a workgroup does at a time: positions of a tile.
struct AttnItem {
  int sequence, begin, length, context;
  int m0, key0, key1;
  int part;  // -1: all that the tile sees; else where in the partial results it goes
};
// A tile that begins in a workgroup's share and ends in another's: its first part, and the place of the second, from
// which on every other one is its.  parts 0: there is none.
struct AttnJoin {
  int begin, length, m0, parts, part0, part1;
  int sequence;
};

// Quotients by a divisor of whole numbers below 2^31.
struct AttnDivisor {
  uint32_t divisor, factor, shift;
};
inline AttnDivisor attn_divisor(uint32_t d) {
  uint32_t l = 0;
  while ((1ull << l) < d) ++l;
  return AttnDivisor{d, (uint32_t)((((1ull << l) - d) << 32) / d + 1), l};
}
__host__ __device__ __forceinline__ int operator/(int n, const AttnDivisor& d) {
  const uint32_t high = (uint32_t)(((uint64_t)d.factor * (uint32_t)n) >> 32);
  return (int)((high + (uint32_t)n) >> d.shift);
}
__host__ __device__ __forceinline__ int operator%(int n, const AttnDivisor& d) { return n - n / d * (int)d.divisor; }

struct AttnPlan {
  int heads, kv_heads, head_dim;
  AttnDivisor group;       // heads to a kv head
  int row_type, cache_type;
  float scale;
  int layers, pages, page_shift;
  int max_context, max_tokens, max_sequences;
  void* keys;
  void* values;
  int* error;  // [2]: AttnErrors of the calls since they were last taken, those taken
  // workspace of a call
  int* run;             // [max_sequences]: 0: refused, nothing of it is read or written
  AttnTile* tiles;      // [AttnSizes::tiles]
  AttnWorker* workers;  // [AttnSizes::workers]
  AttnJoin* joins;      // [AttnSizes::shares]
  int* counts;          // workers, joins
  uint32_t* tree;       // [max_tokens][kAttnTreeWords]: a row's ancestors and itself
  float* part_y;        // [part][kv_heads][tile rows][padded head_dim]
  float2* part_ml;      // [part][kv_heads][tile rows]: reference exponent and sum
};

struct AttnCall {
  const void* q;
  const void* k;
  const void* v;
  void* y;
  int64_t q_stride, k_stride, v_stride, y_stride;  // elements from row to row
  int layer, tokens, sequences;
  const int* offsets;   // [sequences + 1], null: one row each
  const int* context;   // [sequences]
  const int* table;     // [sequences][table_stride]
  int64_t table_stride;
  const int* parents;   // [tokens], null: causal
};

struct AttnAccept {
  const int* context;
  const int* table;
  int64_t table_stride;
  const int* paths;     // [sequences][path_stride]
  int64_t path_stride;
  const int* counts;    // [sequences]
  int sequences;
};

// Workspace for calls of at most max_tokens and max_sequences.
struct AttnSizes {
  int64_t tiles, workers, shares, part_rows;  // part_rows: rows of part_ml; part_y has attn_padded(head_dim) floats each
};
AttnSizes attn_sizes(const AttnPlan& p);
// Keys of a tile that wavefronts share: what registers hold of their scores.  (Rows of 16 bits.  16 trees of 61 nodes, heads
// of 256: 32 keys 127 us, 64 118.  Heads of 64, 28 over 4: 3 prompts of 600 tokens behind 2000 64 keys 101 us, 128 89, one of
// 5000 161 and 153, 16 of 500 77 and 80.  Heads of 128: the same kind 160 and 153, 270 and 273, 120 and 137.)
constexpr int attn_shared_keys(int padded, int row_bytes) {
  return row_bytes == 2 && padded == 64 ? 128 : row_bytes == 4 && padded == 256 ? 32 : 64;
}
// Wavefronts that share a tile of keys: eight, two to a SIMD, where rows, sums and probabilities fit 256 registers.  A tile has
// 32 rows for each, so that the plan and the kernels have to agree.
constexpr int attn_shared_waves(int cache_type, int row_bytes, int padded) {
  return padded == 256 || (cache_type == kAttnBF16 && row_bytes == 4 && padded == 128) ? 4 : 8;
}
inline int attn_padded(int head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }
inline int attn_table_width(const AttnPlan& p) { return (p.max_context + (1 << p.page_shift) - 1) >> p.page_shift; }

// Whether a call's launches have grids that exist.
bool attn_call_fits(const AttnPlan& p, const AttnCall& c);
hipError_t attn_run_launch(const AttnPlan& p, const AttnCall& c, hipStream_t stream);
hipError_t attn_accept_launch(const AttnPlan& p, const AttnAccept& a, hipStream_t stream);
hipError_t attn_take_error_launch(const AttnPlan& p, hipStream_t stream);

// How a call is cut.
struct AttnCut {
  bool shared;      // the waves of a workgroup share a tile of keys (and have rows of their own), or the reverse
  bool few;         // the attend kernel makes the plan and puts the new rows into the cache
  int rows;         // of a tile
  int unit_log2;    // positions of a unit, whole tiles of keys
  int overhead;     // units that a tile costs beside its own
  int shares;       // for each kv head, of equal size, where tiles are divided
  double each;      // 1 / shares
};
// The kernels of one cache type (attention_f16.hip, attention_bf16.hip, attention_f32.hip).
hipError_t attn_attend_f16(const AttnPlan& p, const AttnCall& c, const AttnCut& cut, uint32_t grid, hipStream_t s);
hipError_t attn_attend_bf16(const AttnPlan& p, const AttnCall& c, const AttnCut& cut, uint32_t grid, hipStream_t s);
hipError_t attn_attend_f32(const AttnPlan& p, const AttnCall& c, const AttnCut& cut, uint32_t grid, hipStream_t s);

}  // namespace llhip
