// sample_batch.hip -- the next token of each row (sample_batch.h).
//
// sample_chunks_kernel reads the logits once and records the maximum of each
// 256 of them (a chunk).  What follows reads only what a row has to:
//   top-k of at most as many ranks as there are chunks: at least k logits are
//     at or above the k-th highest chunk maximum, and few more.  The row's
//     workgroup (sample_finish_kernel) reads the chunks that reach it and lists
//     those logits in LDS: up to 32 ranks are settled by one wavefront.  Of few
//     rows with more ranks several workgroups list them, in the launch before
//   no top-k: the row is shared by as many workgroups as fit.  With top-p
//     (sample_mass_kernel) its weights are summed by bins of (max - l) / T, 64 to
//     one; then (sample_cut_kernel) every chunk's weight above the bin that the
//     cut falls into is summed, and that bin's logits are listed; without, every
//     chunk's weights of at least min-p
//   more ranks than chunks: the same bins hold counts, and all logits down to
//     the bin of the k-th are listed
//   lists that outgrow their 4096 entries (equal logits, more ranks): passes of
//     the row's workgroup over all of it, resolving the cut digit by digit
// At the end there is a lowest kept logit and each chunk's kept weight; the
// draw finds its chunk by their sums and reads that.  Weights of whole rows are
// integers in steps of 2^-44, so that sums do not depend on the atomics' order;
// with the bins' powers in a table one takes 5 operations in 64 bits and a
// short series in 32 (off by 1.4e-9 of it at most), a fourth of an exponential in
// 64 bits, which bound these passes.
// Rows of 128256 logits (us), launch by launch: maxima 14 for 160 rows (5.9 TB/s),
// 3.5 for one; bins 32 and 6, weights above the cut 44 and 10 where all rows have
// top-p, 25 where all have min-p alone; the finish 25 with 200 ranks (of one row 8.5
// in the launch before and 11), 18 and 15 with top-p, 7 with min-p.
#include "sample_batch.h"

#include <climits>

#include "moe_gate.h"

namespace llhip {

typedef float f32x4a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));

constexpr int kRowThreads = 1024;

// The parameters of a row.
struct RowParams {
  double sharpness, top_p, min_p, random;  // sharpness: 1 / temperature
  int top_k;                               // 0: off
  bool bad;
};

__device__ __forceinline__ RowParams row_params(const SampleRows& s, int row) {
  RowParams p;
  const float t = s.temperature ? s.temperature[row] : 1.f;
  const float tp = s.top_p ? s.top_p[row] : 1.f, mp = s.min_p ? s.min_p[row] : 0.f;
  const float r = s.random[row];
  const int k = s.top_k ? s.top_k[row] : 0;
  p.bad = !(t >= 0.f && t <= 3.402823466e38f) || !(tp > 0.f && tp <= 1.f) || !(mp >= 0.f && mp <= 1.f) ||
          !(r >= 0.f && r < 1.f) || k < 0;
  p.sharpness = t > 0.f ? 1.0 / (double)t : 1.0;
  p.top_k = t > 0.f ? (k >= s.n ? 0 : k) : 1;
  p.top_p = tp;
  p.min_p = mp;
  p.random = r;
  return p;
}

// exp(x) for x <= 0 in 64 bits: 2^n e^r with |r| <= ln 2 / 2, e^r by its Taylor
// series to r^12 (what follows is below 2e-16).  r by Cody and Waite's reduction: ln 2
// as the sum of its first 32 bits, whose products with n are exact, and the rest.
__device__ __forceinline__ double exp_below(double x) {
  const double n = rint(x * 1.44269504088896340736);
  double r = fma(n, -6.93147180369123816490e-01, x);
  r = fma(n, -1.90821492927058770002e-10, r);
  double e = 1.0 / 479001600.0;
  e = fma(e, r, 1.0 / 39916800.0);
  e = fma(e, r, 1.0 / 3628800.0);
  e = fma(e, r, 1.0 / 362880.0);
  e = fma(e, r, 1.0 / 40320.0);
  e = fma(e, r, 1.0 / 5040.0);
  e = fma(e, r, 1.0 / 720.0);
  e = fma(e, r, 1.0 / 120.0);
  e = fma(e, r, 1.0 / 24.0);
  e = fma(e, r, 1.0 / 6.0);
  e = fma(e, r, 0.5);
  e = fma(e, r, 1.0);
  e = fma(e, r, 1.0);
  return x < -700.0 ? 0.0 : ldexp(e, (int)n);
}

// exp((l - max) / T), r = 1 / T; 1 for the maximum itself, which may be infinite.
__device__ __forceinline__ double weight(float l, float top, double r) {
  return l == top ? 1.0 : exp_below(((double)l - (double)top) * r);
}

// Order-preserving key of a float that is no NaN; -0 and +0 are equal.
__device__ __forceinline__ uint32_t order_of(float f) {
  const uint32_t u = __builtin_bit_cast(uint32_t, f == 0.f ? 0.f : f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float of_order(uint32_t k) {
  return __builtin_bit_cast(float, (k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}
// Rank order as one integer: higher logit, then lower index.
__device__ __forceinline__ uint64_t entry_of(float l, int i) {
  return (uint64_t)order_of(l) << 32 | (0xFFFFFFFFu - (uint32_t)i);
}
__device__ __forceinline__ float entry_logit(uint64_t e) { return of_order((uint32_t)(e >> 32)); }
__device__ __forceinline__ int entry_index(uint64_t e) { return (int)(0xFFFFFFFFu - (uint32_t)e); }

// The chunk's four logits of this lane.  Rows have four at least; a lane whose
// four pass the row's end reads its last four, and takes its own from them, with
// -inf past the row, when they are used: a branch at the load would have it wait
// for the one before.
__device__ __forceinline__ f32x4a4 request_chunk(const float* row, int n, int chunk, int lane) {
  return *reinterpret_cast<const f32x4a4*>(row + min(chunk * kBatchChunk + 4 * lane, n - 4));
}
__device__ __forceinline__ void take_chunk(const f32x4a4& q, int n, int chunk, int lane, float (&v)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = q[e];
  if ((chunk + 1) * kBatchChunk <= n) return;
  const int i = chunk * kBatchChunk + 4 * lane, past = i - min(i, n - 4);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float own = -INFINITY;
#pragma unroll
    for (int f = e; f < 4; ++f) own = f - e == past ? q[f] : own;
    v[e] = own;
  }
}
__device__ __forceinline__ void load_chunk(const float* row, int n, int chunk, int lane, float (&v)[4]) {
  take_chunk(request_chunk(row, n, chunk, lane), n, chunk, lane, v);
}

// Rows of fewer than four logits, filled up with -inf.
__global__ void __launch_bounds__(256) sample_fill_kernel(SampleRows s) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= 4 * s.rows) return;
  s.filled[i] = (i & 3) < s.n ? s.logits[(int64_t)(i >> 2) * s.n + (i & 3)] : -INFINITY;
}

constexpr int kChunksPerWave = 4;

__global__ void __launch_bounds__(256) sample_chunks_kernel(SampleRows s) {
  const int row = blockIdx.y, lane = threadIdx.x & 63;
  const int chunks = (s.n + kBatchChunk - 1) / kBatchChunk;
  for (int i = blockIdx.x * 256 + threadIdx.x; i < kBatchBins; i += gridDim.x * 256)
    s.bins[(int64_t)row * kBatchBins + i] = 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) s.listed[row * kBatchCounter] = 0;
  const int first = (blockIdx.x * 4 + (threadIdx.x >> 6)) * kChunksPerWave;
  if (first >= chunks) return;
  const float* logits = s.logits + (int64_t)row * s.n;
  f32x4a4 q[kChunksPerWave];
#pragma unroll
  for (int c = 0; c < kChunksPerWave; ++c) q[c] = request_chunk(logits, s.n, min(first + c, chunks - 1), lane);
#pragma unroll
  for (int c = 0; c < kChunksPerWave; ++c) {
    float v[4];
    take_chunk(q[c], s.n, min(first + c, chunks - 1), lane, v);
    bool nan = false;
    float m = -INFINITY;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      nan |= v[e] != v[e];
      m = fmaxf(m, v[e]);
    }
    m = wave_max(m);
    nan = __ballot(nan) != 0;
    if (lane == 0 && first + c < chunks) s.chunk_max[(int64_t)row * chunks + first + c] = nan ? NAN : m;
  }
}

// ------------------------------------------------------------------ a workgroup on a row

struct RowLds {
  uint64_t list[kBatchList];
  uint64_t bins[kBatchBins];
  double powers[kBatchBins];  // e^(-b / 64), times 2^44
  uint64_t mass[kBatchMaxChunks];
  float chunk_max[kBatchMaxChunks];
  uint64_t wave[kRowThreads / 64];
  uint64_t result[4];
  int count;
};

// Every thread of the block calls the functions below, but for draw_by_wave.

// Inclusive prefix sums of T over the block in thread order; *total gets the sum.
template <typename T>
__device__ __forceinline__ T block_scan(T v, RowLds& l, T* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  T* part = reinterpret_cast<T*>(l.wave);
  for (int o = 1; o < 64; o <<= 1) {
    const T u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  if (lane == 63) part[wave] = v;
  __syncthreads();
  T before = 0, all = 0;
  for (int w = 0; w < kRowThreads / 64; ++w) {
    const T u = part[w];
    before += w < wave ? u : (T)0;
    all += u;
  }
  __syncthreads();
  *total = all;
  return before + v;
}

// The row's highest logit, its chunks' in LDS; false where it has none or a NaN (a chunk with one
// carries it).
__device__ __forceinline__ bool row_top(RowLds& l, const SampleRows& s, int row, bool bad, float& top) {
  const int tid = threadIdx.x, chunks = (s.n + kBatchChunk - 1) / kBatchChunk;
  const float m = tid < chunks ? s.chunk_max[(int64_t)row * chunks + tid] : -INFINITY;
  const bool nan = m != m;
  if (tid < chunks) l.chunk_max[tid] = m;
  top = wave_max(nan ? -INFINITY : m);
  float* tops = reinterpret_cast<float*>(l.wave);
  if ((tid & 63) == 0) tops[tid >> 6] = top;
  const int any = __syncthreads_or(nan || bad);
  for (int w = 0; w < kRowThreads / 64; ++w) top = fmaxf(top, tops[w]);
  __syncthreads();
  return !any && top > -INFINITY;
}

__device__ __forceinline__ void make_powers(RowLds& l) {
  for (int b = threadIdx.x; b < kBatchBins; b += kRowThreads) l.powers[b] = kMassOne * exp_below(-(double)b / 64);
  __syncthreads();
}

// Sort list[0, n) in descending order.  Up to one entry a thread: by counting the larger ones (no two
// are equal), the threads of an entry sharing the count; else by a bitonic network.
__device__ __forceinline__ void sort_list(RowLds& l, int n) {
  if (n <= kRowThreads) {
    int log2g = 0;
    while (log2g < 4 && n <= (kRowThreads >> (log2g + 1))) ++log2g;
    const int g = 1 << log2g, item = threadIdx.x >> log2g, part = threadIdx.x & (g - 1);
    if (threadIdx.x == 0) l.list[n] = 0;  // entries are read in pairs
    __syncthreads();
    const uint64_t mine = item < n ? l.list[item] : 0;
    int rank = 0;
    if (item < n) {
#pragma unroll 4
      for (int i = 2 * part; i < n; i += 2 * g) {
        const u64x2 pair = *reinterpret_cast<const u64x2*>(&l.list[i]);
        rank += (pair.x > mine ? 1 : 0) + (pair.y > mine ? 1 : 0);
      }
    }
    for (int o = 1; o < g; o <<= 1) rank += __shfl_xor(rank, o, 64);
    __syncthreads();
    if (item < n && part == 0) l.list[rank] = mine;
    __syncthreads();
    return;
  }
  int size = 2 * kRowThreads;
  while (size < n) size <<= 1;
  for (int i = threadIdx.x; i < size; i += kRowThreads)
    if (i >= n) l.list[i] = 0;
  __syncthreads();
  for (int k = 2; k <= size; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int i = threadIdx.x; i < size / 2; i += kRowThreads) {
        const int a = ((i & ~(j - 1)) << 1) | (i & (j - 1)), b = a + j;
        const bool descending = (a & k) == 0;
        const uint64_t x = l.list[a], y = l.list[b];
        if (descending ? x < y : x > y) {
          l.list[a] = y;
          l.list[b] = x;
        }
      }
      __syncthreads();
    }
}

// A chunk's logits where `take` to a list of `count` entries (those past its end are counted only), by
// every lane of a wavefront.
template <typename Counter>
__device__ __forceinline__ void append(uint64_t* list, Counter* count, const bool (&take)[4], const float (&v)[4],
                                       int chunk) {
  const int lane = threadIdx.x & 63;
  const uint64_t below = (1ull << lane) - 1ull;
  int all = 0, ahead = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint64_t m = __ballot(take[e]);
    all += __popcll(m);
    ahead += __popcll(m & below);
  }
  if (!all) return;
  int at = 0;
  if (lane == 0) at = atomicAdd(count, all);
  at = __builtin_amdgcn_readfirstlane(at) + ahead;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (take[e]) {
      if (at < kBatchList) list[at] = entry_of(v[e], chunk * kBatchChunk + 4 * lane + e);
      ++at;
    }
}

// The chunks [first, last) of a row by the block's wavefronts, four of each in flight: f(chunk, logits)
// for those that `wanted` names.
template <typename Wanted, typename F>
__device__ __forceinline__ void each_chunk(const float* row, int n, int first, int last, Wanted&& wanted, F&& f) {
  constexpr int kStep = kRowThreads / 64, kAhead = 4;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // 64 of this wavefront's chunks at a time
  for (int c0 = first + wave; c0 < last; c0 += kStep * 64) {
    const int mine = c0 + kStep * lane;
    uint64_t todo = __ballot(mine < last && wanted(min(mine, last - 1)));
    while (todo) {
      f32x4a4 q[kAhead];
      int c[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        c[k] = todo ? c0 + kStep * __builtin_ctzll(todo) : -1;
        todo &= todo - 1;
        q[k] = request_chunk(row, n, c[k] >= 0 ? c[k] : c[0], lane);
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (c[k] >= 0) {
          float v[4];
          take_chunk(q[k], n, c[k], lane, v);
          f(c[k], v);
        }
    }
  }
}

template <int CTRL>
__device__ __forceinline__ uint64_t dpp_u64(uint64_t v) {
  return (uint64_t)(uint32_t)dpp_i<CTRL>((int)(v >> 32)) << 32 | (uint32_t)dpp_i<CTRL>((int)v);
}
__device__ __forceinline__ uint64_t readlane_u64(uint64_t v, int lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v) {
  v += dpp_u64<kDppXor1>(v);
  v += dpp_u64<kDppXor2>(v);
  v += dpp_u64<kDppHalfMirror>(v);
  v += dpp_u64<kDppMirror>(v);
  return readlane_u64(v, 0) + readlane_u64(v, 16) + readlane_u64(v, 32) + readlane_u64(v, 48);
}

// A min-p as an integer weight: weights of at least it are kept.
__device__ __forceinline__ uint64_t least_weight(RowParams p) { return (uint64_t)ceil(p.min_p * kMassOne); }

// ------------------------------------------------------------------ rows without top-k

// The row's chunks to this workgroup of those on it.
__device__ __forceinline__ void share_of(int chunks, int& first, int& last) {
  const int shares = gridDim.x, per = (chunks + shares - 1) / shares;
  first = blockIdx.x * per;
  last = min(chunks, first + per);
}

__global__ void __launch_bounds__(kRowThreads) sample_mass_kernel(SampleRows s) {
  extern __shared__ __align__(16) uint8_t raw[];
  RowLds& l = *reinterpret_cast<RowLds*>(raw);
  const int row = blockIdx.y;
  const RowParams p = row_params(s, row);
  const int chunks = (s.n + kBatchChunk - 1) / kBatchChunk;
  if (p.bad || (p.top_k ? p.top_k <= chunks : p.top_p >= 1.0)) return;
  float top;
  if (!row_top(l, s, row, false, top)) return;
  for (int b = threadIdx.x; b < kBatchBins; b += kRowThreads) l.bins[b] = 0;
  make_powers(l);
  int first, last;
  share_of(chunks, first, last);
  each_chunk(s.logits + (int64_t)row * s.n, s.n, first, last, [&](int c) { return l.chunk_max[c] > -INFINITY; },
             [&](int, const float (&v)[4]) {
#pragma unroll
               for (int e = 0; e < 4; ++e) {
                 const Weighed w = weigh(l.powers, v[e], top, p.sharpness);
                 const uint64_t count = p.top_k ? (v[e] > -INFINITY ? 1 : 0) : w.weight;
                 if (count) atomicAdd((unsigned long long*)&l.bins[w.bin], (unsigned long long)count);
               }
             });
  __syncthreads();
  for (int b = threadIdx.x; b < kBatchBins; b += kRowThreads)
    if (l.bins[b])
      atomicAdd((unsigned long long*)&s.bins[(int64_t)row * kBatchBins + b], (unsigned long long)l.bins[b]);
}

// The bin that the row's cut falls into and how much lies above it, from its bins: counts with top-k,
// weights without.
__device__ __forceinline__ void cut_bin(RowLds& l, const SampleRows& s, int row, RowParams p, int& bin, uint64_t& above,
                          uint64_t& need) {
  constexpr int kPer = kBatchBins / kRowThreads;
  const uint64_t* bins = s.bins + (int64_t)row * kBatchBins + threadIdx.x * kPer;
  uint64_t own[kPer], sum = 0, total;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    own[k] = bins[k];
    sum += own[k];
  }
  const uint64_t incl = block_scan(sum, l, &total);
  need = p.top_k ? (uint64_t)p.top_k : (uint64_t)ceil(p.top_p * (double)total);
  need = need > total ? total : need > 0 ? need : 1;
  if (incl >= need && incl - sum < need) {
    uint64_t run = incl - sum;
    int at = 0;
#pragma unroll
    for (int k = 0; k + 1 < kPer; ++k)
      if (at == k && run + own[k] < need) {
        run += own[k];
        ++at;
      }
    l.result[0] = (uint64_t)(threadIdx.x * kPer + at);
    l.result[1] = run;
  }
  __syncthreads();
  bin = (int)l.result[0];
  above = l.result[1];
  __syncthreads();
}

// Rows of at most so many ranks have their bound found by one wavefront, which draws the token too if no
// more logits than kWaveList reach it.  160 rows, 16 ranks 10.6 us for the last launch (15.8 by the whole
// workgroup), 32 13.1 (16.8), 40 23.2 (17.7: the bound's selection leaves its fast path).
constexpr int kWaveRanks = 32, kWaveList = 256;

// Whether the candidates of a row with more ranks are listed by the row's workgroups before the last launch.
__device__ __forceinline__ bool listed_ahead(const SampleRows& s, RowParams p) { return s.spread && p.top_k > kWaveRanks; }

// A bound that at least `ranks` chunks reach, and few more: the highest chunk maxima by their keys' upper
// bits, eight at a time.
__device__ __forceinline__ float ranks_bound(RowLds& l, int chunks, int ranks) {
  const int tid = threadIdx.x, lane = tid & 63;
  uint32_t prefix = 0;
  int above = 0;
  uint32_t* hist = reinterpret_cast<uint32_t*>(l.bins);
  const uint32_t key = tid < chunks ? order_of(l.chunk_max[tid]) : 0;
  for (int shift = 24; shift >= 8; shift -= 8) {
    for (int i = tid; i < 256; i += kRowThreads) hist[i] = 0;
    __syncthreads();
    if (tid < chunks && (shift == 24 || key >> (shift + 8) == prefix)) atomicAdd(&hist[(key >> shift) & 255], 1u);
    __syncthreads();
    if (tid < 64) {
      // four bins a lane, from the top
      int c[4], sum = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) sum += c[j] = (int)hist[255 - 4 * lane - j];
      int incl = sum;
      for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(incl, o, 64);
        if (lane >= o) incl += u;
      }
      int run = above + incl - sum;
      if (run < ranks && run + sum >= ranks) {
        int at = 0;
#pragma unroll
        for (int j = 0; j < 3; ++j)
          if (at == j && run + c[j] < ranks) {
            run += c[j];
            ++at;
          }
        l.result[0] = (uint64_t)(255 - 4 * lane - at);
        l.result[1] = (uint64_t)run;
      }
    }
    __syncthreads();
    prefix = prefix << 8 | (uint32_t)l.result[0];
    above = (int)l.result[1];
    __syncthreads();
  }
  const float bound = of_order(prefix << 8);
  return bound == bound ? bound : -INFINITY;  // (the keys below -inf's)
}

// The row's logits of at least `bound` in the chunks [first, last) to a list.
template <typename Counter>
__device__ __forceinline__ void list_from(const RowLds& l, const float* row, int n, int first, int last, float bound,
                                          uint64_t* list, Counter* count) {
  each_chunk(row, n, first, last, [&](int c) { return l.chunk_max[c] >= bound && l.chunk_max[c] > -INFINITY; },
             [&](int c, const float (&v)[4]) {
               bool take[4];
#pragma unroll
               for (int e = 0; e < 4; ++e) take[e] = v[e] >= bound && v[e] > -INFINITY;
               append(list, count, take, v, c);
             });
}

__global__ void __launch_bounds__(kRowThreads) sample_cut_kernel(SampleRows s) {
  extern __shared__ __align__(16) uint8_t raw[];
  RowLds& l = *reinterpret_cast<RowLds*>(raw);
  const int row = blockIdx.y, lane = threadIdx.x & 63;
  const RowParams p = row_params(s, row);
  const int chunks = (s.n + kBatchChunk - 1) / kBatchChunk;
  if (p.bad || (p.top_k && p.top_k <= chunks && !listed_ahead(s, p))) return;
  float top;
  if (!row_top(l, s, row, false, top)) return;
  if (p.top_k && p.top_k <= chunks) {
    const float bound = ranks_bound(l, chunks, p.top_k);
    int first, last;
    share_of(chunks, first, last);
    list_from(l, s.logits + (int64_t)row * s.n, s.n, first, last, bound, s.list + (int64_t)row * kBatchList,
              s.listed + row * kBatchCounter);
    return;
  }
  make_powers(l);
  int bin = kBatchBins;  // without top-p all weights lie above the cut
  uint64_t above, need;
  if (p.top_k || p.top_p < 1.0) cut_bin(l, s, row, p, bin, above, need);
  // (top-k keeps by rank first: all down to the cut's bin are listed, and no weights summed)
  const uint64_t least = p.top_k ? 0 : least_weight(p);
  int first, last;
  share_of(chunks, first, last);
  uint64_t* mass = s.chunk_mass + (int64_t)row * chunks;
  // chunks that hold nothing above the cut or in its bin, or nothing that min-p keeps
  auto wanted = [&](int c) {
    const Weighed w = weigh(l.powers, l.chunk_max[c], top, p.sharpness);
    return l.chunk_max[c] > -INFINITY && w.bin <= bin && w.weight >= least;
  };
  for (int c = first + threadIdx.x; c < last; c += kRowThreads)
    if (!p.top_k && !wanted(c)) mass[c] = 0;
  each_chunk(s.logits + (int64_t)row * s.n, s.n, first, last, wanted, [&](int c, const float (&v)[4]) {
    uint64_t held = 0;
    bool take[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const Weighed w = weigh(l.powers, v[e], top, p.sharpness);
      take[e] = (p.top_k ? w.bin <= bin : w.bin == bin) && v[e] > -INFINITY;
      if (w.bin < bin && w.weight >= least) held += w.weight;
    }
    append(s.list + (int64_t)row * kBatchList, s.listed + row * kBatchCounter, take, v, c);
    if (p.top_k) return;
    held = wave_sum_u64(held);
    if (lane == 0) mass[c] = held;
  });
}

// ------------------------------------------------------------------ the token

// The token of a list by the first wavefront: ranks by counting, then a rank a lane.
__device__ __forceinline__ void draw_by_wave(RowLds& l, int n, RowParams p, float top, int* token) {
  const int lane = threadIdx.x & 63;
  const int ranks = min(n, p.top_k);
  uint64_t mine[kWaveList / 64];
  int rank[kWaveList / 64];
#pragma unroll
  for (int j = 0; j < kWaveList / 64; ++j) {
    mine[j] = lane + 64 * j < n ? l.list[lane + 64 * j] : 0;
    rank[j] = 0;
  }
  for (int i = 0; i < n; ++i) {
    const uint64_t e = l.list[i];
#pragma unroll
    for (int j = 0; j < kWaveList / 64; ++j)
      if (64 * j < n) rank[j] += e > mine[j] ? 1 : 0;
  }
  uint64_t* sorted = l.bins;
#pragma unroll
  for (int j = 0; j < kWaveList / 64; ++j)
    if (lane + 64 * j < n && rank[j] < ranks) sorted[rank[j]] = mine[j];
  __builtin_amdgcn_wave_barrier();
  const uint64_t e = sorted[min(lane, ranks - 1)];
  __builtin_amdgcn_wave_barrier();
  double w = lane < ranks ? weight(entry_logit(e), top, p.sharpness) : 0.0;
  double upto = w;
  for (int o = 1; o < 64; o <<= 1) {
    const double u = __shfl_up(upto, o, 64);
    if (lane >= o) upto += u;
  }
  const double all = __shfl(upto, 63, 64);
  // the filters keep a run from the first rank on
  const bool keep = lane < ranks && (lane == 0 || p.top_p >= 1.0 || upto - w < p.top_p * all) && w >= p.min_p;
  const int kept = __popcll(__ballot(keep));
  if (lane >= kept) w = 0.0;
  const int index = lane < kept ? entry_index(e) : INT_MAX;
  // the sum up to each one's index
  double run = 0.0, total = 0.0;
  for (int i = 0; i < kept; ++i) {
    const double wi = __builtin_bit_cast(double, readlane_u64(__builtin_bit_cast(uint64_t, w), i));
    total += wi;
    run += __builtin_amdgcn_readlane(index, i) <= index ? wi : 0.0;
  }
  const bool past = lane < kept && run > p.random * total;
  const int found = wave_min(past ? index : INT_MAX), last = wave_max_i(lane < kept ? index : -1);
  if (lane == 0) *token = found < INT_MAX ? found : last;
}

// The token by the chunks' kept weights and the lowest entry kept.
__device__ __forceinline__ int draw_from_chunks(RowLds& l, const float* row, int n, RowParams p, float top,
                                                uint64_t cut) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int chunks = (n + kBatchChunk - 1) / kBatchChunk;
  const uint64_t least = least_weight(p);
  uint64_t total;
  const uint64_t mine = tid < chunks ? l.mass[tid] : 0;
  const uint64_t upto = block_scan(mine, l, &total);
  const double at = p.random * (double)total;
  if (tid == 0) {
    l.result[0] = ~0ull;
    l.count = INT_MAX;
  }
  __syncthreads();
  // the chunk at which the sum passes the mark, then the logit
  if (tid < chunks && (double)upto > at && !((double)(upto - mine) > at)) {
    l.result[0] = (uint64_t)tid;
    l.result[1] = upto - mine;
  }
  __syncthreads();
  const int chunk = (int)l.result[0];
  if (chunk < 0) return -1;
  if (wave == 0) {
    float v[4];
    load_chunk(row, n, chunk, lane, v);
    uint64_t own[4], sum = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      own[e] = 0;
      if (v[e] > -INFINITY && entry_of(v[e], chunk * kBatchChunk + 4 * lane + e) >= cut) {
        const uint64_t w = weigh(l.powers, v[e], top, p.sharpness).weight;
        own[e] = w >= least ? w : 0;
      }
      sum += own[e];
    }
    uint64_t incl = sum;
    for (int o = 1; o < 64; o <<= 1) {
      const uint64_t u = __shfl_up(incl, o, 64);
      if (lane >= o) incl += u;
    }
    uint64_t run = l.result[1] + incl - sum;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      run += own[e];
      if (own[e] && (double)run > at) atomicMin(&l.count, chunk * kBatchChunk + 4 * lane + e);
    }
  }
  __syncthreads();
  return l.count;
}

// What of a sorted list is kept, into the chunks' weights: the first whose weights ahead of them do not
// reach `need` (0: top-p of the list's total), of at least min-p.  Returns the lowest entry kept by need.
constexpr int kOwn = kBatchList / kRowThreads;
__device__ __forceinline__ uint64_t keep_from_list(RowLds& l, int n, RowParams p, float top, uint64_t above,
                                                   uint64_t need) {
  const int tid = threadIdx.x;
  const uint64_t least = least_weight(p);
  uint64_t own = 0, values[kOwn], total;
#pragma unroll
  for (int k = 0; k < kOwn; ++k) {
    const int i = tid * kOwn + k;
    values[k] = i < n ? weigh(l.powers, entry_logit(l.list[i]), top, p.sharpness).weight : 0;
    own += values[k];
  }
  uint64_t run = above + block_scan(own, l, &total) - own;
  if (need == 0) need = p.top_p < 1.0 ? max((uint64_t)ceil(p.top_p * (double)total), (uint64_t)1) : ~0ull;
  if (tid == 0) l.result[2] = 0;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kOwn; ++k) {
    const int i = tid * kOwn + k;
    if (i < n && run < need) {
      if (values[k] >= least)
        atomicAdd((unsigned long long*)&l.mass[entry_index(l.list[i]) / kBatchChunk], (unsigned long long)values[k]);
      // the last of them
      if (run + values[k] >= need || i == n - 1) l.result[2] = l.list[i];
    }
    run += values[k];
  }
  __syncthreads();
  const uint64_t cut = l.result[2];
  __syncthreads();
  return cut;
}

// The highest entry e such that the entries >= e reach `need` (their number, or their weight where
// `by_mass`), of the row's entries >= floor_entry; floor_entry where all of those do not.
__device__ __forceinline__ uint64_t row_cut(RowLds& l, const float* row, int n, float top, double t, bool by_mass,
                            uint64_t need, uint64_t floor_entry) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int chunks = (n + kBatchChunk - 1) / kBatchChunk;
  uint64_t* bins = l.bins;
  for (int i = tid; i < kBatchBins; i += kRowThreads) bins[i] = 0;
  __syncthreads();
  auto value = [&](const Weighed& w) -> uint64_t { return by_mass ? w.weight : 1; };
  for (int c = wave; c < chunks; c += kRowThreads / 64) {
    float v[4];
    load_chunk(row, n, c, lane, v);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (v[e] > -INFINITY && entry_of(v[e], c * kBatchChunk + 4 * lane + e) >= floor_entry) {
        const Weighed w = weigh(l.powers, v[e], top, t);
        atomicAdd((unsigned long long*)&bins[w.bin], (unsigned long long)value(w));
      }
  }
  __syncthreads();
  // the bin that reaches it
  constexpr int kPer = kBatchBins / kRowThreads;
  uint64_t sum = 0;
  for (int k = 0; k < kPer; ++k) sum += bins[tid * kPer + k];
  uint64_t total;
  const uint64_t incl = block_scan(sum, l, &total);
  if (total < need) return floor_entry;
  if (incl >= need && incl - sum < need) {
    uint64_t above = incl - sum;
    int b = tid * kPer;
    while (above + bins[b] < need) above += bins[b++];
    l.result[0] = (uint64_t)b;
    l.result[1] = above;
  }
  if (tid == 0) l.count = 0;
  __syncthreads();
  const int bin = (int)l.result[0];
  uint64_t above = l.result[1];
  __syncthreads();
  for (int c = wave; c < chunks; c += kRowThreads / 64) {
    float v[4];
    load_chunk(row, n, c, lane, v);
    bool take[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      take[e] = v[e] > -INFINITY && entry_of(v[e], c * kBatchChunk + 4 * lane + e) >= floor_entry &&
                weigh(l.powers, v[e], top, t).bin == bin;
    append(l.list, &l.count, take, v, c);
  }
  __syncthreads();
  const int listed = l.count;
  __syncthreads();
  if (listed <= kBatchList) {
    sort_list(l, listed);
    uint64_t own = 0, values[kOwn];
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
      const int i = tid * kOwn + k;
      values[k] = i < listed ? value(weigh(l.powers, entry_logit(l.list[i]), top, t)) : 0;
      own += values[k];
    }
    uint64_t run = above + block_scan(own, l, &total) - own;
    if (tid == 0) l.result[2] = floor_entry;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
      if (run < need && run + values[k] >= need) l.result[2] = l.list[tid * kOwn + k];
      run += values[k];
    }
    __syncthreads();
    const uint64_t cut = l.result[2];
    __syncthreads();
    return cut;
  }
  // too many for the list: eight bits of the entries at a time
  uint64_t prefix = 0;
  for (int shift = 56; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kRowThreads) bins[i] = 0;
    __syncthreads();
    for (int c = wave; c < chunks; c += kRowThreads / 64) {
      float v[4];
      load_chunk(row, n, c, lane, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint64_t x = entry_of(v[e], c * kBatchChunk + 4 * lane + e);
        const Weighed w = weigh(l.powers, v[e], top, t);
        if (v[e] > -INFINITY && x >= floor_entry && w.bin == bin && (shift == 56 || x >> (shift + 8) == prefix))
          atomicAdd((unsigned long long*)&bins[(x >> shift) & 255], (unsigned long long)value(w));
      }
    }
    __syncthreads();
    const uint64_t mine = tid < 256 ? bins[255 - tid] : 0;
    const uint64_t upto = block_scan(mine, l, &total) + above;
    if (tid < 256 && upto >= need && upto - mine < need) {
      l.result[2] = (uint64_t)(255 - tid);
      l.result[3] = upto - mine;
    }
    __syncthreads();
    prefix = prefix << 8 | l.result[2];
    above = l.result[3];
    __syncthreads();
  }
  return prefix;
}

// The token of a row by passes over all of it.
__device__ __forceinline__ int draw_from_row(RowLds& l, const float* row, int n, RowParams p, float top) {
  const int lane = threadIdx.x & 63, chunks = (n + kBatchChunk - 1) / kBatchChunk;
  const double t = p.sharpness;
  uint64_t cut = 0, total;
  auto kept_of = [&](const float (&v)[4], int c, uint64_t least) {
    uint64_t sum = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (v[e] > -INFINITY && entry_of(v[e], c * kBatchChunk + 4 * lane + e) >= cut) {
        const uint64_t w = weigh(l.powers, v[e], top, t).weight;
        sum += w >= least ? w : 0;
      }
    return sum;
  };
  auto all = [](int) { return true; };
  if (p.top_k) cut = row_cut(l, row, n, top, t, false, (uint64_t)p.top_k, 0);
  if (p.top_p < 1.0) {
    // of what top-k kept
    uint64_t sum = 0;
    each_chunk(row, n, 0, chunks, all, [&](int c, const float (&v)[4]) { sum += kept_of(v, c, 0); });
    block_scan(sum, l, &total);
    const uint64_t need = (uint64_t)ceil(p.top_p * (double)total);
    cut = row_cut(l, row, n, top, t, true, need > 0 ? need : 1, cut);
  }
  const uint64_t least = least_weight(p);
  each_chunk(row, n, 0, chunks, all, [&](int c, const float (&v)[4]) {
    const uint64_t sum = wave_sum_u64(kept_of(v, c, least));
    if (lane == 0) l.mass[c] = sum;
  });
  __syncthreads();
  return draw_from_chunks(l, row, n, p, top, cut);
}

// Rows with top-k: the candidates to the list; their number (beyond the list's end: too many).
__device__ __forceinline__ int list_candidates(RowLds& l, const float* row, int n, RowParams p, float top) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int chunks = (n + kBatchChunk - 1) / kBatchChunk;
  float bound = -INFINITY;
  if (p.top_k <= kWaveRanks) {
    if (wave == 0) {
      constexpr int kPer = kBatchMaxChunks / 64;
      float v[kPer];
#pragma unroll
      for (int j = 0; j < kPer; ++j) v[j] = lane + 64 * j < chunks ? l.chunk_max[lane + 64 * j] : -INFINITY;
      int at;
      float kth;
      wave_select<kPer>(v, p.top_k, lane, reinterpret_cast<int64_t*>(l.bins), at, kth);
      // (fewer chunks with a logit: every logit is a candidate)
      if (lane == p.top_k - 1) l.result[0] = __builtin_bit_cast(uint32_t, at >= 0 ? kth : -INFINITY);
    }
    __syncthreads();
    bound = __builtin_bit_cast(float, (uint32_t)l.result[0]);
  } else {
    bound = ranks_bound(l, chunks, p.top_k);
  }
  if (tid == 0) l.count = 0;
  __syncthreads();
  list_from(l, row, n, 0, chunks, bound, l.list, &l.count);
  __syncthreads();
  return l.count;
}

__global__ void __launch_bounds__(kRowThreads) sample_finish_kernel(SampleRows s) {
  extern __shared__ __align__(16) uint8_t raw[];
  RowLds& l = *reinterpret_cast<RowLds*>(raw);
  const int row = blockIdx.x, tid = threadIdx.x;
  const int chunks = (s.n + kBatchChunk - 1) / kBatchChunk;
  const float* logits = s.logits + (int64_t)row * s.n;
  const RowParams p = row_params(s, row);
  float top;
  if (!row_top(l, s, row, p.bad, top)) {
    if (tid == 0) s.tokens[row] = -1;
    return;
  }
  int token;
  if (p.top_k) {
    int n;
    if (p.top_k <= chunks && !listed_ahead(s, p)) {
      n = list_candidates(l, logits, s.n, p, top);
    } else {
      n = s.listed[row * kBatchCounter];
      for (int i = tid; i < min(n, kBatchList); i += kRowThreads) l.list[i] = s.list[(int64_t)row * kBatchList + i];
      __syncthreads();
    }
    if (p.top_k <= kWaveRanks && n <= kWaveList) {
      if (tid < 64) draw_by_wave(l, n, p, top, s.tokens + row);
      return;
    }
    __syncthreads();
    make_powers(l);
    if (n <= kBatchList) {
      sort_list(l, n);
      const int ranks = min(n, p.top_k);
      for (int c = tid; c < chunks; c += kRowThreads) l.mass[c] = 0;
      __syncthreads();
      const uint64_t cut = keep_from_list(l, ranks, p, top, 0, 0);
      token = draw_from_chunks(l, logits, s.n, p, top, cut);
    } else {
      token = draw_from_row(l, logits, s.n, p, top);
    }
  } else {
    make_powers(l);
    int bin;
    uint64_t above = 0, need = 0;
    if (p.top_p < 1.0) cut_bin(l, s, row, p, bin, above, need);
    const int n = p.top_p < 1.0 ? s.listed[row * kBatchCounter] : 0;
    if (n > kBatchList) {
      token = draw_from_row(l, logits, s.n, p, top);
    } else {
      for (int c = tid; c < chunks; c += kRowThreads) l.mass[c] = s.chunk_mass[(int64_t)row * chunks + c];
      for (int i = tid; i < n; i += kRowThreads) l.list[i] = s.list[(int64_t)row * kBatchList + i];
      __syncthreads();
      uint64_t cut = 0;
      if (n) {
        sort_list(l, n);
        cut = keep_from_list(l, n, p, top, above, need);
      }
      token = draw_from_chunks(l, logits, s.n, p, top, cut);
    }
  }
  if (tid == 0) s.tokens[row] = token;
}

template <typename Kernel>
static hipError_t launch_rows(Kernel k, dim3 grid, const SampleRows& s, hipStream_t stream) {
  hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)sizeof(RowLds));
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(k, grid, dim3(kRowThreads), sizeof(RowLds), stream, s);
  return hipGetLastError();
}

// Rows up to which their workgroups list the candidates of a top-k above kWaveRanks: a CU alone gets 20 GB/s
// from beyond its L2.  A call with 200 ranks of 128256: one row 23.4 us (29.0 by the row's workgroup), 16
// rows 27.3 (30.9), 32 36.6 (34.0), 160 52.6 (46.2).
constexpr int kSpreadRows = 16;

hipError_t sample_rows_launch(SampleRows s, hipStream_t stream) {
  if (s.n < 4) {
    hipLaunchKernelGGL(sample_fill_kernel, dim3((4 * s.rows + 255) / 256), dim3(256), 0, stream, s);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    s.logits = s.filled;
    s.n = 4;
  }
  const int chunks = sample_chunks(s.n);
  hipLaunchKernelGGL(sample_chunks_kernel, dim3((chunks + 4 * kChunksPerWave - 1) / (4 * kChunksPerWave), s.rows),
                     dim3(256), 0, stream, s);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  // Workgroups to a row: twice what fills the device, for rows with top-k leave theirs idle.  160 rows,
  // a third of them without top-k, 16 + 25 us for these passes, with half as many 23 + 32; but where all
  // have top-p 33 + 44 and 27 + 39 (each workgroup reads the maxima and makes the powers anew).
  const int shares = max(1, min(1024 / s.rows, (chunks + 15) / 16));
  s.spread = s.rows <= kSpreadRows;
  // (which rows have a top-k or top-p is known on the device only; no array: none has)
  if (s.top_p || s.top_k) e = launch_rows(sample_mass_kernel, dim3(shares, s.rows), s, stream);
  if (e != hipSuccess) return e;
  e = launch_rows(sample_cut_kernel, dim3(shares, s.rows), s, stream);
  if (e != hipSuccess) return e;
  return launch_rows(sample_finish_kernel, dim3(s.rows), s, stream);
}

}  // namespace llhip
