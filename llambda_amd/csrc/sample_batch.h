// sample_batch.h -- the next token of each row of a batch of logits
// (sample_batch.hip): temperature, top-k, top-p, min-p and the draw, from
// given random numbers.
//
// For a row l with x = l / T, in 64 bits: w = exp(x - max x).  Rank order is by
// logit, higher first, lower index first among equals.  Kept are, one filter
// after the other: the first k ranks; the shortest run of ranks whose weights
// reach p of what top-k kept; weights >= min_p (the largest is 1).  The token
// is the first, by index, at which the sum of kept weights exceeds r times
// their total.  T = 0 takes the first rank.  A row gets -1 where a logit is
// NaN, no logit lies above -inf, or its parameters are out of range.
#pragma once

#include "common.h"
#include "sample_weight.h"

namespace llhip {

// Workspace: at most 61 KB a row.
constexpr int kBatchChunk = 256;  // logits whose maximum the first launch records
constexpr int kBatchMaxVocab = 262144;
constexpr int kBatchMaxChunks = kBatchMaxVocab / kBatchChunk;
constexpr int kBatchCounter = 64;  // ints from a row's counter to the next: additions to one line wait for each other
constexpr int kBatchList = 4096;  // logits of the bin that a cut falls into, or candidates

struct SampleRows {
  const float* logits;  // [rows][n]
  int n, rows;
  // [rows] each, null: 1, 0 (off), 1 (off), 0 (off)
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  const float* random;  // [rows], in [0, 1)
  int* tokens;          // [rows]
  // workspace, per row
  float* chunk_max;      // [chunks]
  uint64_t* chunk_mass;  // [chunks]: weights kept above the cut
  uint64_t* bins;        // [kBatchBins]
  uint64_t* list;        // [kBatchList]
  int* listed;           // [kBatchCounter], the first counts
  float* filled;         // [4]: a row of fewer logits
  int spread;            // set by the launch: few rows, each with many workgroups
};

inline int sample_chunks(int n) { return (n + kBatchChunk - 1) / kBatchChunk; }
hipError_t sample_rows_launch(SampleRows s, hipStream_t stream);

}  // namespace llhip
