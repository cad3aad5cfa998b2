// route.hip -- routing to experts from logits (route.h), a wavefront per token.
//
// One launch, nothing but the logits read and the chosen experts written.  One
// token of 128 experts 4.6 us, 301 of 256 in groups 7.6 (both a launch and one
// token's chain of reductions); 8192 of 512 experts 10.8 us, 1.6 TB/s: bound by
// the vector unit, 69% of whose issue cycles 563 instructions a token take, most
// of them the selection's, which counts the ranks of 64-bit entries (64 lanes'
// maxima, then the candidates).  Where weights are normalised and there is
// neither bias nor group, a wavefront takes one exponential, its experts'.
#include "route.h"

#include "route_token.h"

namespace llhip {

// Tokens of a workgroup: four, two where a token's scores take 16 KB of LDS.
template <int JPL>
constexpr int kRouteTokens = JPL > 8 ? 2 : 4;

template <int JPL>
__global__ void __launch_bounds__(64 * kRouteTokens<JPL>) route_kernel(RouteSpec p, const float* __restrict__ logits,
                                                    int tokens, int* __restrict__ indices,
                                                    float* __restrict__ weights) {
  __shared__ RouteScratch<JPL> scratch[kRouteTokens<JPL>];
  const int t = blockIdx.x * kRouteTokens<JPL> + (threadIdx.x >> 6);
  if (t >= tokens) return;
  const int lane = threadIdx.x & 63;
  const float* row = logits + (int64_t)t * p.experts;
  float raw[JPL];
#pragma unroll
  for (int j = 0; j < JPL; ++j) raw[j] = row[min(lane + kWave * j, p.experts - 1)];
  const RouteRank r = route_token<JPL>(p, raw, lane, scratch[threadIdx.x >> 6]);
  if (lane >= p.top_k) return;
  indices[(int64_t)t * p.top_k + lane] = r.idx;
  weights[(int64_t)t * p.top_k + lane] = r.w;
}

template <int JPL>
static hipError_t launch(const RouteSpec& p, const float* logits, int tokens, int* indices,
                         float* weights, hipStream_t s) {
  constexpr int n = kRouteTokens<JPL>;
  hipLaunchKernelGGL(route_kernel<JPL>, dim3((tokens + n - 1) / n), dim3(64 * n), 0, s, p, logits, tokens,
                     indices, weights);
  return hipGetLastError();
}

hipError_t route_launch(const RouteSpec& p, const float* logits, int tokens, int* indices,
                        float* weights, hipStream_t s) {
  if (p.experts <= 64) return launch<1>(p, logits, tokens, indices, weights, s);
  if (p.experts <= 128) return launch<2>(p, logits, tokens, indices, weights, s);
  if (p.experts <= 256) return launch<4>(p, logits, tokens, indices, weights, s);
  if (p.experts <= 512) return launch<8>(p, logits, tokens, indices, weights, s);
  if (p.experts <= 1024) return launch<16>(p, logits, tokens, indices, weights, s);
  return hipErrorInvalidValue;
}

}  // namespace llhip
