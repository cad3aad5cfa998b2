// score.h -- log probabilities of given tokens, entropy and top alternatives of
// rows of logits (score.hip).
//
// Per row, with m = max x and S = sum exp(x - m):
//   log p_t = x_t - m - log S,   H = log S + (sum exp(x - m) (m - x)) / S
// and the `top` tokens of the highest logits, the lower index first among equals.
#pragma once

#include "common.h"

namespace llhip {

constexpr int kScoreMaxVocab = 262144;
constexpr int kScoreMaxTop = 64;
constexpr int kScoreChunk = 2048;  // logits of a wavefront
constexpr int kScoreMaxChunks = kScoreMaxVocab / kScoreChunk;

// What a wavefront found in its chunk: sums relative to the chunk's largest logit (NaN: no such row has a
// distribution), candidates for the top tokens.
struct ScorePart {
  double sum, weighted;
  float top;
  int candidates;
};
struct ScoreCandidate {
  float logit;
  int token;
};

struct ScoreRows {
  const float* logits;
  int64_t stride;      // from row to row
  int count, rows;
  const int* given;    // [rows][givens]
  int givens, top;
  float* log_probs;    // [rows][givens], or null
  float* entropy;      // [rows], or null
  int* top_tokens;     // [rows][top], or null
  float* top_log_probs;
  // workspace
  ScorePart* parts;            // [rows][chunks]
  ScoreCandidate* candidates;  // [rows][chunks][kScoreMaxTop]
};

inline int score_chunks(int64_t count) { return (int)((count + kScoreChunk - 1) / kScoreChunk); }
hipError_t score_rows_launch(const ScoreRows& r, hipStream_t stream);

}  // namespace llhip
