// ssm.h -- the Mamba-2 mixer between ssm_in's rows and ssm_out's (ssm.hip):
// short causal convolution, selective state space scan, gated group norm.
//
// A row of the input holds [z: HP | x: HP | B: GN | C: GN | dt: H] (H heads of
// P channels, G groups of heads that share B and C of N).  For token t of a
// sequence, per channel c of x | B | C and head h of group g:
//   u_c  = silu(b_c + sum_k w_ck raw_{t-W+1+k, c})       (W taps, oldest first)
//   dt   = softplus(dt_t + dt_bias_h),  a = exp(dt A_h)
//   s    = a s + dt x B^T                                 [P][N], fp32
//   y    = s C + D_h x
//   out  = v / sqrt(mean_group(v^2) + eps) * norm,  v = y silu(z)
// A sequence's state between calls is its last W - 1 raw rows of x | B | C,
// oldest first, and s of every head: slot i of the pools conv_states
// [slots][W - 1][HP + 2 GN] and ssm_states [slots][H][P][N].
#pragma once

#include "common.h"

namespace llhip {

constexpr int kSsmChunk = 32;        // tokens per chunk of the scan
constexpr int kSsmMaxConv = 4;       // taps (2 at least)
constexpr int kSsmMaxHeadDim = 128;
constexpr int kSsmMaxState = 256;
constexpr int kSsmMaxNormWidth = 16384;  // channels of a norm group

enum SsmError : int {
  kSsmErrOffsets = 1,   // offsets not ascending within the call's tokens
  kSsmErrSlot = 2,      // a slot outside the pool
  kSsmErrConflict = 4,  // a slot that one sequence writes and another reads or writes
};

// A sequence of a call, as the plan kernel found it.
struct SsmSequence {
  int begin, length;  // rows of the call
  int from, to;       // slots (-1: zeros / not kept)
  int chunk0;         // its first chunk in the workspace
  int segments;
  int state0;         // of several segments: its first entry of seg_states
  int run;            // 0: refused, nothing of it is read or written
};

struct SsmLayerPlan {
  int heads, head_dim, groups, state, conv;
  int slots, max_tokens, max_sequences;
  float epsilon;
  const float* conv_weight;  // [W][HP + 2 GN]
  const float* conv_bias;    // [HP + 2 GN]
  const float* dt_bias;      // [H]
  const float* a;            // [H]
  const float* d;            // [H]
  const float* norm;         // [HP]
  float* conv_states;
  float* ssm_states;
  int* error;  // [2]: SsmErrors of the calls since they were last taken, those taken
  // workspace of calls with offsets, for max_tokens and max_sequences
  SsmSequence* sequences;  // [max_sequences]
  int2* segments;          // [max_segments]: sequence, index within it
  int2* chunks;            // [max_chunks]: sequence, index within it
  int* counts;             // segments, chunks
  uint8_t* images;         // [chunk][G][ssm_image_bytes]: B, C after the convolution, C B^T
  float* scales;           // [chunk][G][2][kSsmChunk]: 2^14 over the scales of B's and C's images
  float* decay;            // [chunk][H][3][kSsmChunk]: dt, log2 of the decay since the chunk's start (hi, lo)
  // segments of the sequences that have several, max_states in all
  float* seg_states;       // [H][P][N] each: the state that enters it
  float* seg_decay;        // [H] each: log2 of its decay
};

struct SsmCall {
  const float* x;
  float* y;
  int tokens, sequences;
  const int* offsets;  // [sequences + 1], null: one token each
  const int* from;     // [sequences], null: slot i
  const int* to;
};

inline int ssm_row(const SsmLayerPlan& p) {
  return 2 * p.heads * p.head_dim + 2 * p.groups * p.state + p.heads;
}
// Bounds of the tables and buffers of a call of at most so many.
int64_t ssm_max_chunks(int64_t tokens, int64_t sequences);
int64_t ssm_max_segments(const SsmLayerPlan& p, int64_t tokens, int64_t sequences);
size_t ssm_image_bytes(int state);
int64_t ssm_max_states(const SsmLayerPlan& p, int64_t tokens);

// Whether a call's launches have grids that exist.
bool ssm_call_fits(const SsmLayerPlan& p, const SsmCall& c);
// Enqueue a call (one that fits) on `stream`: one token of each sequence where offsets is
// null, else sequences of any lengths.
hipError_t ssm_step_launch(const SsmLayerPlan& p, const SsmCall& c, hipStream_t stream);
hipError_t ssm_run_launch(const SsmLayerPlan& p, const SsmCall& c, hipStream_t stream);
hipError_t ssm_take_error_launch(const SsmLayerPlan& p, hipStream_t stream);

}  // namespace llhip
