// route_token.h -- one token's routing (route.h) by one wavefront.
//
// Order is decided in 64 bits, where two scores that single precision rounds
// together still differ.  Without a bias and groups the scores' order is the
// logits', which need no exponentials but those of the taken experts.
#pragma once

#include "moe_gate.h"
#include "route.h"

namespace llhip {

// LDS of one wavefront's routing.
template <int JPL>
struct RouteScratch {
  int64_t sel[kSelectScratch];
  double score[kWave * JPL];   // s by expert
  int64_t choice[kWave * JPL]; // key of c by expert
  int cand[kWave + 1];
  double group[kRouteMaxGroups];
};

struct RouteRank {
  int idx;  // -1: unfilled
  float w;
  int error;  // on every lane: 1 = unfilled places, 2 = the sum to divide by is not positive
};

// Order-preserving key of a double that is no NaN.
__device__ __forceinline__ int64_t key_of(double v) {
  const int64_t b = __builtin_bit_cast(int64_t, v == 0.0 ? 0.0 : v);
  return b >= 0 ? b : b ^ 0x7FFFFFFFFFFFFFFFll;
}
__device__ __forceinline__ double of_key(int64_t k) {
  return __builtin_bit_cast(double, k >= 0 ? k : k ^ 0x7FFFFFFFFFFFFFFFll);
}
constexpr int64_t kNoKey = INT64_MIN;

__device__ __forceinline__ double wave_sum_f64(double v) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
  return v;
}

// The K highest of the lanes' keys (expert lane + 64 j in c[j]), lower expert
// first among equals: lane r < K receives rank r's expert (-1: fewer).  As
// wave_select: the K-th highest of the lanes' maxima bounds the candidates,
// which are compacted into LDS and ranked by counting.
template <int JPL>
__device__ __forceinline__ int select_keys(int64_t (&c)[JPL], int K, int lane, RouteScratch<JPL>& s) {
  int64_t h = c[0];
#pragma unroll
  for (int j = 1; j < JPL; ++j) h = c[j] > h ? c[j] : h;
  s.sel[lane] = h;
  __builtin_amdgcn_wave_barrier();
  int rank = 0;
#pragma unroll
  for (int i = 0; i < kWave; ++i) rank += (s.sel[i] > h || (s.sel[i] == h && i < lane)) ? 1 : 0;
  const int64_t t = readlane64(h, (int)__builtin_ctzll(__ballot(rank == K - 1)));
  bool take[JPL];
  int cnt = 0;
#pragma unroll
  for (int j = 0; j < JPL; ++j) {
    take[j] = c[j] >= t && c[j] != kNoKey;
    cnt += take[j] ? 1 : 0;
  }
  int pre = 0, total = 0;
#pragma unroll
  for (int b = 0; b < 5; ++b) {
    const uint64_t m = __ballot((cnt >> b) & 1);
    pre += (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32),
                                          __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u)) << b;
    total += __popcll(m) << b;
  }
  int mine = -1;
  if (total > kWave) {
    // round by round (equal keys, or many of a lane's above the bound)
    for (int r = 0; r < K; ++r) {
      int64_t best = kNoKey;
      int at = INT_MAX;
#pragma unroll
      for (int j = JPL - 1; j >= 0; --j)
        if (c[j] >= best && c[j] != kNoKey) {
          best = c[j];
          at = lane + kWave * j;
        }
      for (int o = 32; o > 0; o >>= 1) {
        const int64_t k2 = __shfl_xor(best, o, kWave);
        const int a2 = __shfl_xor(at, o, kWave);
        if (k2 > best || (k2 == best && a2 < at)) {
          best = k2;
          at = a2;
        }
      }
      if (best == kNoKey) break;
      if (lane == r) mine = at;
#pragma unroll
      for (int j = 0; j < JPL; ++j)
        if (at == lane + kWave * j) c[j] = kNoKey;
    }
    return mine;
  }
  int at = pre;
  int64_t* keys = s.sel + kWave;
#pragma unroll
  for (int j = 0; j < JPL; ++j) {
    keys[take[j] ? at : kWave] = c[j];
    s.cand[take[j] ? at : kWave] = lane + kWave * j;
    at += take[j] ? 1 : 0;
  }
  __builtin_amdgcn_wave_barrier();
  const int64_t k = keys[min(lane, kWave - 1)];
  const int e = s.cand[lane];
  __builtin_amdgcn_wave_barrier();
  int r = 0;
  for (int i = 0; i < total; ++i) r += (keys[i] > k || (keys[i] == k && s.cand[i] < e)) ? 1 : 0;
  __builtin_amdgcn_wave_barrier();
  int* out = reinterpret_cast<int*>(s.sel);  // the maxima are no longer needed
  if (lane < total) out[r] = e;
  __builtin_amdgcn_wave_barrier();
  if (lane < min(K, total)) mine = out[lane];
  return mine;
}

// raw[j]: the logit of expert lane + 64 j (any value past the last expert).
template <int JPL>
__device__ __forceinline__ RouteRank route_token(const RouteSpec& p, const float (&raw)[JPL],
                                                 int lane, RouteScratch<JPL>& s) {
  const int E = p.experts, K = p.top_k;
  float vals[JPL];
  float best = -INFINITY;
#pragma unroll
  for (int j = 0; j < JPL; ++j) {
    vals[j] = lane + kWave * j < E ? selectable(raw[j]) : -INFINITY;
    best = fmaxf(best, vals[j]);
  }
  // exp(l - max), 1 for the maxima themselves (which may be infinite)
  auto power = [&](float v) { return v == best ? 1.0 : exp((double)v - (double)best); };
  auto sigmoid = [](float v) { return 1.0 / (1.0 + exp(-(double)v)); };
  if (!p.sigmoid) best = wave_max(best);
  int mine;
  double w = 0.0;
  if (!p.bias && p.groups == 1) {
    float v;
    wave_select<JPL>(vals, K, lane, s.sel, mine, v);
    const bool has = lane < K && mine >= 0;
    if (!has) mine = -1;
    if (p.sigmoid) {
      w = has ? sigmoid(v) : 0.0;
    } else {
      w = has ? power(v) : 0.0;
      if (!p.norm) {
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < JPL; ++j) sum += vals[j] > -INFINITY ? power(vals[j]) : 0.0;
        sum = wave_sum_f64(sum);
        w = has ? w / sum : 0.0;
      }
    }
  } else {
    double sc[JPL];
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < JPL; ++j) {
      const bool in = vals[j] > -INFINITY;
      sc[j] = !in ? 0.0 : p.sigmoid ? sigmoid(vals[j]) : power(vals[j]);
      sum += sc[j];
    }
    if (!p.sigmoid) {
      sum = wave_sum_f64(sum);
#pragma unroll
      for (int j = 0; j < JPL; ++j) sc[j] = sc[j] / sum;
    }
    int64_t c[JPL];
#pragma unroll
    for (int j = 0; j < JPL; ++j) {
      const int e = lane + kWave * j;
      const double v = sc[j] + (p.bias ? (double)p.bias[min(e, E - 1)] : 0.0);
      c[j] = vals[j] > -INFINITY && v == v ? key_of(v) : kNoKey;
      s.score[e] = sc[j];
      s.choice[e] = c[j];
    }
    if (p.groups > 1) {
      __builtin_amdgcn_wave_barrier();
      // 64 / groups lanes (a power of two) per group find its two highest
      const int size = E / p.groups;
      int lanes = kWave / p.groups;
      lanes = 1 << (31 - __builtin_clz(lanes));
      const int g = lane / lanes;
      int64_t a = kNoKey, b = kNoKey;
      if (g < p.groups)
        for (int i = lane - g * lanes; i < size; i += lanes) {
          const int64_t k = s.choice[g * size + i];
          if (k > a) {
            b = a;
            a = k;
          } else if (k > b) {
            b = k;
          }
        }
      for (int o = 1; o < lanes; o <<= 1) {
        const int64_t a2 = __shfl_xor(a, o, kWave), b2 = __shfl_xor(b, o, kWave);
        const int64_t low = a < a2 ? a : a2, high = b > b2 ? b : b2;
        a = a > a2 ? a : a2;
        b = low > high ? low : high;
      }
      double score = -INFINITY;
      if (a != kNoKey) score = of_key(a);
      // (beside -inf, +inf stays: their sum would be NaN, which ranks nowhere)
      if (p.group_rank > 1 && a != kNoKey && b != kNoKey && score < INFINITY) score += of_key(b);
      const bool leader = g < p.groups && lane == g * lanes;
      if (leader) s.group[g] = score;
      __builtin_amdgcn_wave_barrier();
      int rank = 0;
      if (leader)
        for (int i = 0; i < p.groups; ++i) {
          const double v = s.group[i];
          rank += (v > score || (v == score && i < g)) ? 1 : 0;
        }
      const uint64_t open = __ballot(leader && a != kNoKey && rank < p.top_groups);
#pragma unroll
      for (int j = 0; j < JPL; ++j) {
        const int e = min(lane + kWave * j, E - 1);
        if (!((open >> (e / size * lanes)) & 1)) c[j] = kNoKey;
      }
    }
    mine = select_keys<JPL>(c, K, lane, s);
    w = mine >= 0 ? s.score[mine] : 0.0;
  }
  int error = __ballot(lane < K && mine < 0) ? 1 : 0;
  if (p.norm) {
    const double sum = wave_sum_f64(w);
    if (!(sum > 0.0)) error |= 2;
    else w = w / sum;
  }
  return RouteRank{mine, (float)(w * (double)p.scale), error};
}

}  // namespace llhip
