// score.hip -- log probabilities, entropy and top alternatives (score.h).
//
// Two launches.  score_chunk_kernel reads each logit once: a wavefront takes 2048
// of a row into registers, finds their maximum, the sums of exp(x - m) and of exp(x
// - m) (m - x) and what of them can be among the row's top tokens: those at or
// above a bound that at least `top` lanes reach with their largest (a lane's
// largest are distinct logits).  The bound comes from a few bisections; where it
// leaves more than 64 (equal logits, or neighbours in one lane), the exact `top`
// first are chosen instead.  score_row_kernel joins a row's chunks in 64 bits.
// The first kernel is bound by the logits' traffic: 2048 rows of 128256, 1.05 GB, in
// 193 us, 5.4 TB/s, or 225 after a pause (the second 6.5); one row by latency, 6 + 8 us.  A wavefront joins a
// row: 16 of them with a barrier between took 15 us for one row and 43 for 2048.
#include "score.h"

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

// LDS accesses of this wavefront so far are done before those that follow.
__device__ __forceinline__ void lds_order() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

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

// A row's chunks, by one wavefront: lane l takes chunks l and l + 64.  Keys rank candidates by logit, then by index, and
// are distinct; 0 is none.
constexpr int kRowChosen = 512;
constexpr int kRowKeys = 4096;  // candidates of a row that are kept in LDS
static_assert(kScoreMaxChunks <= 128, "two chunks to a lane");

__device__ __forceinline__ uint64_t candidate_key(const ScoreCandidate& v) {
  return (uint64_t)((uint32_t)ordered(v.logit) ^ 0x80000000u) << 32 | (uint32_t)~v.token;
}
__device__ __forceinline__ float key_logit(uint64_t key) {
  const int o = (int)((uint32_t)(key >> 32) ^ 0x80000000u);
  return __builtin_bit_cast(float, o ^ ((o >> 31) & 0x7FFFFFFF));
}
__device__ __forceinline__ uint64_t wave_max_key(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t u = __shfl_xor(v, o, 64);
    v = u > v ? u : v;
  }
  return v;
}
// use(key) for each candidate of a lane's two lists of n[0] and n[1], BATCH of which are on their way at once.
template <int BATCH, typename Use>
__device__ __forceinline__ void each_candidate(const ScoreCandidate* list, const int (&n)[2], Use&& use) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const ScoreCandidate* at = list + 64 * h * kScoreMaxTop;
    for (int i = 0; i < n[h]; i += BATCH) {
      ScoreCandidate v[BATCH];
#pragma unroll
      for (int k = 0; k < BATCH; ++k) v[k] = at[min(i + k, n[h] - 1)];
#pragma unroll
      for (int k = 0; k < BATCH; ++k)
        if (i + k < n[h]) use(candidate_key(v[k]));
    }
  }
}

// RANKED: more than one top token (a wavefront to a workgroup then, for the LDS's sake).
template <bool RANKED>
__global__ __launch_bounds__(RANKED ? 64 : 256) void score_row_kernel(ScoreRows r, int chunks) {
  __shared__ uint64_t kept[RANKED ? kRowKeys : 1], chosen[RANKED ? kRowChosen : 1];
  __shared__ int chosen_count;
  const int lane = threadIdx.x & 63, row = blockIdx.x * (RANKED ? 1 : 4) + (threadIdx.x >> 6);
  if (row >= r.rows) return;
  const float* x = r.logits + row * r.stride;
  const int* given = r.given + (int64_t)row * r.givens;
  auto given_logit = [&](int g) {
    const int token = given[g];
    return token >= 0 && token < r.count ? x[token] : __builtin_nanf("");
  };
  const float first_given = lane < r.givens ? given_logit(lane) : 0.f;  // on its way beside the sums
  ScorePart part[2] = {{0, 0, -__builtin_inff(), 0}, {0, 0, -__builtin_inff(), 0}};
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (lane + 64 * h < chunks) part[h] = r.parts[(int64_t)row * chunks + lane + 64 * h];
  const bool nan = __ballot(part[0].top != part[0].top || part[1].top != part[1].top) != 0;
  const float top = wave_max(fmaxf(part[0].top, part[1].top));
  const bool empty = nan || top == -__builtin_inff();  // no distribution
  double s = 0, w = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (part[h].sum > 0) {
      const double lead = (double)top - (double)part[h].top, scale = exp(-lead);
      s += scale * part[h].sum;
      w += scale * (part[h].weighted + lead * part[h].sum);
    }
  s = wave_sum(s);
  w = wave_sum(w);
  const double log_sum = log(s);
  auto log_prob = [&](float logit) {
    return empty ? __builtin_nanf("") : (float)((double)logit - (double)top - log_sum);
  };
  if (lane == 0 && r.entropy) r.entropy[row] = empty ? __builtin_nanf("") : (float)(log_sum + w / s);
  if (r.log_probs)
    for (int g = lane; g < r.givens; g += 64)
      r.log_probs[(int64_t)row * r.givens + g] = log_prob(g == lane ? first_given : given_logit(g));
  if (r.top == 0) return;
  auto place_token = [&](int place, uint64_t key) {
    const int token = (int)~(uint32_t)key;
    if (r.top_tokens) r.top_tokens[(int64_t)row * r.top + place] = token;
    if (r.top_log_probs) r.top_log_probs[(int64_t)row * r.top + place] = log_prob(key_logit(key));
  };
  int filled = 0;
  if (!empty) {
    const ScoreCandidate* list = r.candidates + ((int64_t)row * chunks + lane) * kScoreMaxTop;
    const int n[2] = {part[0].candidates, part[1].candidates};
    uint64_t best = 0;
    if constexpr (!RANKED) {
      each_candidate<2>(list, n, [&](uint64_t key) { best = key > best ? key : best; });
      best = wave_max_key(best);
      if (lane == 0) place_token(0, best);
      filled = 1;
    } else {
      int end = n[0] + n[1];
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(end, o, 64);
        if (lane >= o) end += u;
      }
      const int total = __builtin_amdgcn_readlane(end, 63);
      const bool keep = total <= kRowKeys;
      int at = end - n[0] - n[1];
      each_candidate<16>(list, n, [&](uint64_t key) {
        best = key > best ? key : best;
        if (keep) kept[at++] = key;
      });
      if (lane == 0) chosen_count = 0;
      chosen[lane] = best;
      lds_order();
      auto each = [&](auto&& use) {
        if (keep) {
#pragma unroll 8
          for (int i = lane; i < total; i += 64) use(kept[i]);
        } else {
          each_candidate<16>(list, n, use);
        }
      };
      // the key that `top` lanes' best reach; if there are not so many lanes, or more keys reach it than there is room
      // for, one that enough keys reach
      int rank = 0;
#pragma unroll 8
      for (int i = 0; i < 64; ++i) rank += chosen[i] > best;
      const uint64_t bests = __ballot(best && rank == r.top - 1);
      uint64_t bound = 1;
      if (bests) bound = __shfl(best, __ffsll((unsigned long long)bests) - 1, 64);
      auto reach = [&](uint64_t least) {
        int count = 0;
        each([&](uint64_t key) { count += key >= least; });
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) count += __shfl_xor(count, o, 64);
        return count;
      };
      filled = reach(bound);
      if (filled > kRowChosen) {
        uint64_t hi = wave_max_key(best);
        while (hi > bound && filled > kRowChosen) {
          const uint64_t mid = bound + (hi - bound + 1) / 2;
          const int count = reach(mid);
          if (count >= r.top) bound = mid, filled = count;
          else hi = mid - 1;
        }
      }
      lds_order();
      each([&](uint64_t key) {
        if (key >= bound) chosen[atomicAdd(&chosen_count, 1)] = key;
      });
      lds_order();
      for (int i = lane; i < filled; i += 64) {
        const uint64_t key = chosen[i];
        int place = 0;
#pragma unroll 4
        for (int j = 0; j < filled; ++j) place += chosen[j] > key;
        if (place < r.top) place_token(place, key);
      }
      filled = min(filled, r.top);
    }
  }
  // places without a token
  for (int i = filled + lane; i < r.top; i += 64) {
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
  if (r.top > 1) hipLaunchKernelGGL(score_row_kernel<true>, dim3(r.rows), dim3(64), 0, s, r, chunks);
  else hipLaunchKernelGGL(score_row_kernel<false>, dim3((r.rows + 3) / 4), dim3(256), 0, s, r, chunks);
  return hipGetLastError();
}

}  // namespace llhip
