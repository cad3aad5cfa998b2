// score.hip -- log probabilities, entropy and top alternatives (score.h).
//
// Two launches.  score_chunk_kernel reads each logit once: a wavefront takes 2048
// of a row into registers, finds their maximum, the sums of exp(x - m) and of exp(x
// - m) (m - x) and what of them can be among the row's top tokens: those at or
// above a bound that at least `top` lanes reach with their largest (a lane's
// largest are distinct logits).  The bound comes from a few bisections; where it
// leaves more than 64 (equal logits, or neighbours in one lane), the exact `top`
// first are chosen instead.  score_row_kernel joins a row's chunks in 64 bits.
// The first kernel is bound by the logits' traffic, one row by latency.
#include "score.h"

#include <cfloat>

#include "mfma.h"

namespace llhip {

constexpr int kScoreWaves = 4;
constexpr int kScorePer = kScoreChunk / 64;  // logits of a lane
typedef float f32x4a4 __attribute__((ext_vector_type(4), aligned(4)));

// Integers in the order of floats (no NaN).
__device__ __forceinline__ int ordered(float v) {
  const int b = __builtin_bit_cast(int, v);
  return b ^ ((b >> 31) & 0x7FFFFFFF);
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// Lane l's logit 4 k + j is the chunk's 4 (l + 64 k) + j.
struct ChunkOrder {
  int lane;
  __device__ __forceinline__ int index(int i) const { return 4 * (lane + 64 * (i / 4)) + i % 4; }
};

__global__ __launch_bounds__(64 * kScoreWaves) void score_chunk_kernel(ScoreRows r, int chunks) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t id = (int64_t)blockIdx.x * kScoreWaves + wave;
  const int row = (int)(id / chunks), chunk = (int)(id % chunks);
  if (row >= r.rows) return;
  const int first = chunk * kScoreChunk, n = min(kScoreChunk, r.count - first);
  const float* x = r.logits + row * r.stride + first;
  const ChunkOrder order{lane};
  float v[kScorePer];
  if (n == kScoreChunk) {
#pragma unroll
    for (int k = 0; k < kScorePer / 4; ++k) {
      const f32x4a4 q = __builtin_nontemporal_load(reinterpret_cast<const f32x4a4*>(x + 4 * (lane + 64 * k)));
#pragma unroll
      for (int j = 0; j < 4; ++j) v[4 * k + j] = q[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < kScorePer; ++i) v[i] = order.index(i) < n ? x[order.index(i)] : -__builtin_inff();
  }
#pragma unroll
  for (int i = 0; i < kScorePer; ++i) v[i] += 0.f;  // -0 ranks as 0
  float mine = v[0];
  bool bad = false;
#pragma unroll
  for (int i = 0; i < kScorePer; ++i) {
    mine = fmaxf(mine, v[i]);
    bad = bad || !(v[i] < __builtin_inff());  // NaN and +inf
  }
  const float top = wave_max(mine);
  ScorePart* part = r.parts + (int64_t)row * chunks + chunk;
  if (__ballot(bad)) {
    if (lane == 0) *part = ScorePart{0, 0, __builtin_nanf(""), 0};
    return;
  }
  // exp(x - m) in single precision is right to 1e-7 of the largest; the sum keeps terms next to 1, whose loss would
  // show in the log probability of a token that is nearly certain
  const float reference = top == -__builtin_inff() ? 0.f : top;
  double sum = 0;
  float weighted = 0.f;
#pragma unroll
  for (int i = 0; i < kScorePer; ++i) {
    const float d = v[i] - reference;
    const float e = __builtin_amdgcn_exp2f(d * 1.44269504088896340736f);
    sum += (double)e;
    weighted -= e > 0.f ? e * d : 0.f;
  }
  sum = wave_sum(sum);
  const double all_weighted = wave_sum((double)weighted);
  int found = 0;
  if (r.top > 0 && top > -__builtin_inff()) {
    const int need = r.top;
    ScoreCandidate* list = r.candidates + ((int64_t)row * chunks + chunk) * kScoreMaxTop;
    // a bound that at least `need` lanes' largest reach, -inf's place if there are not so many
    const int none = ordered(-__builtin_inff());
    const int key = ordered(mine);
    int lo = none + 1, hi = ordered(top);
    if (need == 1) lo = hi;
    if (__popcll(__ballot(key >= lo)) <= need) hi = lo;
    while (hi > lo) {
      const int mid = lo + (int)(((uint32_t)hi - (uint32_t)lo + 1) / 2);
      const int reach = __popcll(__ballot(key >= mid));
      if (reach >= need) lo = mid;
      else hi = mid - 1;
      if (reach >= need && reach <= need + 4) break;
    }
    int total = 0;
#pragma unroll
    for (int i = 0; i < kScorePer; ++i) total += __popcll(__ballot(ordered(v[i]) >= lo));
    int above = lo, equal = 0;  // taken: keys >= above, and the first `equal` of key above - 1
    if (total > kScoreMaxTop) {
      // the largest key that at least `need` logits reach
      hi = ordered(top);
      while (hi > lo) {
        const int mid = lo + (int)(((uint32_t)hi - (uint32_t)lo + 1) / 2);
        int reach = 0;
#pragma unroll
        for (int i = 0; i < kScorePer; ++i) reach += __popcll(__ballot(ordered(v[i]) >= mid));
        if (reach >= need) lo = mid;
        else hi = mid - 1;
      }
      above = lo + 1;
      equal = need;
#pragma unroll
      for (int i = 0; i < kScorePer; ++i) equal -= __popcll(__ballot(ordered(v[i]) >= above));
    }
#pragma unroll
    for (int i = 0; i < kScorePer; ++i) {
      const bool take = ordered(v[i]) >= above;
      const uint64_t takes = __ballot(take);
      if (take) list[found + __popcll(takes & ((1ull << lane) - 1))] = ScoreCandidate{v[i], first + order.index(i)};
      found += __popcll(takes);
    }
    if (equal > 0) {
      // in the order of their indices: by k, then by lane, then by j
#pragma unroll
      for (int k = 0; k < kScorePer / 4; ++k) {
        uint64_t same[4];
        int before = 0, all = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          same[j] = __ballot(ordered(v[4 * k + j]) == above - 1);
          before += __popcll(same[j] & ((1ull << lane) - 1));
          all += __popcll(same[j]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (same[j] >> lane & 1) {
            if (before < equal) list[found + before] = ScoreCandidate{v[4 * k + j], first + order.index(4 * k + j)};
            ++before;
          }
        const int taken = min(all, equal);
        found += taken;
        equal -= taken;
      }
    }
  }
  if (lane == 0) *part = ScorePart{sum, all_weighted, top, found};
}

// A row's chunks.  Keys rank candidates by logit, then by index, and are distinct; 0 is none.
constexpr int kRowThreads = 256;
constexpr int kRowSlots = kScoreMaxChunks * kScoreMaxTop / kRowThreads;

__global__ __launch_bounds__(kRowThreads) void score_row_kernel(ScoreRows r, int chunks) {
  __shared__ float tops[kRowThreads / 64];
  __shared__ double sums[kRowThreads / 64][2];
  __shared__ uint64_t keys[kRowThreads];
  __shared__ uint64_t chosen[kScoreMaxTop * kRowSlots];
  __shared__ uint64_t bound;
  __shared__ int chosen_count;
  const int row = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
  static_assert(kScoreMaxChunks <= kRowThreads, "a thread for each chunk");
  ScorePart part{0, 0, -__builtin_inff(), 0};
  if (t < chunks) part = r.parts[(int64_t)row * chunks + t];
  const bool nan = __syncthreads_or(part.top != part.top);
  const float wave_top = wave_max(part.top);
  if (lane == 0) tops[wave] = wave_top;
  if (t == 0) {
    bound = 0;
    chosen_count = 0;
  }
  __syncthreads();
  float top = tops[0];
#pragma unroll
  for (int w = 1; w < kRowThreads / 64; ++w) top = fmaxf(top, tops[w]);
  const bool empty = nan || top == -__builtin_inff();  // no distribution
  const double lead = empty || part.top == -__builtin_inff() ? 0.0 : (double)top - (double)part.top;
  const double scale = part.sum > 0 ? exp(-lead) : 0.0;
  const double sum = wave_sum(scale * part.sum);
  const double weighted = wave_sum(part.sum > 0 ? scale * (part.weighted + lead * part.sum) : 0.0);
  if (lane == 0) sums[wave][0] = sum, sums[wave][1] = weighted;
  __syncthreads();
  double s = 0, w = 0;
#pragma unroll
  for (int i = 0; i < kRowThreads / 64; ++i) s += sums[i][0], w += sums[i][1];
  const double log_sum = log(s);
  const float* x = r.logits + row * r.stride;
  auto log_prob = [&](float logit) {
    return empty ? __builtin_nanf("") : (float)((double)logit - (double)top - log_sum);
  };
  if (t == 0 && r.entropy) r.entropy[row] = empty ? __builtin_nanf("") : (float)(log_sum + w / s);
  if (r.log_probs)
    for (int g = t; g < r.givens; g += kRowThreads) {
      const int token = r.given[(int64_t)row * r.givens + g];
      r.log_probs[(int64_t)row * r.givens + g] =
          token >= 0 && token < r.count ? log_prob(x[token]) : __builtin_nanf("");
    }
  if (r.top == 0) return;
  int filled = 0;
  if (!empty) {
    uint64_t best = 0, own[kRowSlots];
#pragma unroll
    for (int k = 0; k < kRowSlots; ++k) {
      own[k] = 0;
      const int slot = t + kRowThreads * k, c = slot / kScoreMaxTop;
      if (c < chunks && slot % kScoreMaxTop < r.parts[(int64_t)row * chunks + c].candidates) {
        const ScoreCandidate v = r.candidates[(int64_t)row * chunks * kScoreMaxTop + slot];
        own[k] = (uint64_t)((uint32_t)ordered(v.logit) ^ 0x80000000u) << 32 | (uint32_t)~v.token;
      }
      best = own[k] > best ? own[k] : best;
    }
    keys[t] = best;
    __syncthreads();
    // the key that `top` threads' best reach
    int rank = 0;
    for (int i = 0; i < kRowThreads; ++i) rank += keys[i] > best;
    if (best && rank == r.top - 1) bound = best;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kRowSlots; ++k)
      if (own[k] && own[k] >= bound) chosen[atomicAdd(&chosen_count, 1)] = own[k];
    __syncthreads();
    const int n = chosen_count;
    filled = min(n, r.top);
    for (int i = t; i < n; i += kRowThreads) {
      const uint64_t key = chosen[i];
      int place = 0;
      for (int j = 0; j < n; ++j) place += chosen[j] > key;
      if (place < r.top) {
        const int token = (int)~(uint32_t)key;
        if (r.top_tokens) r.top_tokens[(int64_t)row * r.top + place] = token;
        if (r.top_log_probs) r.top_log_probs[(int64_t)row * r.top + place] = log_prob(x[token]);
      }
    }
  }
  // places without a token
  for (int i = filled + t; i < r.top; i += kRowThreads) {
    if (r.top_tokens) r.top_tokens[(int64_t)row * r.top + i] = -1;
    if (r.top_log_probs) r.top_log_probs[(int64_t)row * r.top + i] = empty ? __builtin_nanf("") : -__builtin_inff();
  }
}

hipError_t score_rows_launch(const ScoreRows& r, hipStream_t s) {
  const int chunks = score_chunks(r.count);
  const int64_t blocks = ((int64_t)r.rows * chunks + kScoreWaves - 1) / kScoreWaves;
  hipLaunchKernelGGL(score_chunk_kernel, dim3((uint32_t)blocks), dim3(64 * kScoreWaves), 0, s, r, chunks);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(score_row_kernel, dim3(r.rows), dim3(kRowThreads), 0, s, r, chunks);
  return hipGetLastError();
}

}  // namespace llhip
