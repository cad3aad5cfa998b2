// sample_weight.h -- a logit's weight in the sampling of a batch
// (sample_batch.hip) as an integer in steps of 2^-44, and its bin.
//
// Several kernels form the weight of one logit anew, and one of them draws by
// the sums that another made of them: it must be the same integer wherever it
// is formed.  So every fused multiply-add is written out, and the compiler
// contracts no other product and sum, whatever stands around them.
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

namespace llhip {

constexpr int kBatchBins = 2048;               // of (max - l) / T, 64 to one
constexpr double kMassOne = 17592186044416.0;  // 2^44

// A logit's bin, ascending as the logit falls (the last takes the rest, whose weights round to
// nothing), and its weight as an integer: the bin's power times e^-f, f < 1 / 64.
struct Weighed {
  int bin;
  uint64_t weight;
};

// powers: [kBatchBins], e^(-b / 64) times 2^44.  sharpness: 1 / temperature.
__host__ __device__ __forceinline__ Weighed weigh(const double* powers, float v, float top, double sharpness) {
#pragma clang fp contract(off)
  const double below = (double)top - (double)v, rate = 64.0 * sharpness;
  const double t = v == top ? 0.0 : below * rate;
  if (!(t < (double)(kBatchBins - 1))) return Weighed{kBatchBins - 1, 0};
  const int b = (int)t;
  const float f = (float)(t - (double)b) * (1.f / 64);
  // 1 - e^-f by its series to f^5 (the next term is below f^6 / 720 < 2^-45)
  float g = fmaf(-f, 1.f / 120, 1.f / 24);
  g = fmaf(-f, g, 1.f / 6);
  g = fmaf(-f, g, 0.5f);
  g = fmaf(-f, g, 1.f);
  g = f * g;
  const double w = powers[b];
  // (the integer is the low bits of the sum with 2^52)
  const uint64_t bits = __builtin_bit_cast(uint64_t, fma(w, -(double)g, w) + 4503599627370496.0);
  return Weighed{b, bits & 0xFFFFFFFFFFFFFull};
}

}  // namespace llhip
