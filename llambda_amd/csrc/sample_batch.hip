// sample_batch.hip -- the next token of each row (sample_batch.h).
//
// sample_chunks_kernel reads the logits once, a wavefront per 256 of them, and
// records each chunk's maximum (and its mass exp((l - max) / T) where the row
// needs its total).  sample_finish_kernel, a workgroup per row, then reads only
// what it has to:
//   top-k of at most as many ranks as there are chunks: at least k logits are
//     at or above the k-th highest chunk maximum, and few more; the chunks that
//     reach it are read again and those logits listed in LDS
//   min-p: the logits whose weight reaches it, likewise
//   neither, and no top-p: the draw goes by the chunks' masses and reads one
//     chunk
//   else, and where a list outgrows LDS: the whole row, binned by
//     (max - l) / T in steps of 1/64, the bin that the cut falls into listed or,
//     if it is too large (equal logits), resolved digit by digit
// A list is sorted by (logit, index), cut by top-k, top-p and min-p, sorted by
// index and drawn from.  Masses of whole rows are 64-bit integers in steps of
// 2^-44, so that sums do not depend on the order of the atomics.
#include "sample_batch.h"

#include <climits>

namespace llhip {

typedef float f32x4a4 __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kFinishThreads = 1024;
constexpr int kListMax = 4096;
constexpr int kBins = 2048;         // of (max - l) / T, 64 to one; the last takes the rest
constexpr double kMassOne = 17592186044416.0;  // 2^44

// The parameters of a row, and what follows from them.
struct RowParams {
  double temperature, top_p, min_p, random;
  int top_k;      // 0: off
  bool bad;
  bool mass;      // the row needs its total before it is cut
};

__device__ __forceinline__ RowParams row_params(const SampleRows& s, int row) {
  RowParams p;
  const float t = s.temperature ? s.temperature[row] : 1.f;
  const float tp = s.top_p ? s.top_p[row] : 1.f, mp = s.min_p ? s.min_p[row] : 0.f;
  const float r = s.random[row];
  const int k = s.top_k ? s.top_k[row] : 0;
  p.bad = !(t >= 0.f && t <= 3.402823466e38f) || !(tp > 0.f && tp <= 1.f) || !(mp >= 0.f && mp <= 1.f) ||
          !(r >= 0.f && r < 1.f) || k < 0;
  p.temperature = t > 0.f ? t : 1.0;
  p.top_k = t > 0.f ? (k >= s.n ? 0 : k) : 1;
  p.top_p = tp;
  p.min_p = mp;
  p.random = r;
  p.mass = p.top_k == 0 && (tp < 1.f || !(mp > 0.f));
  return p;
}

// exp(l / T - max / T); 1 for the maximum itself, which may be infinite.
__device__ __forceinline__ double weight(float l, float top, double t) {
  return l == top ? 1.0 : exp((double)l / t - (double)top / t);
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

// The chunk's four logits of this lane, -inf past the row.
__device__ __forceinline__ void load_chunk(const float* row, int n, int chunk, int lane, float (&v)[4]) {
  const int i = chunk * kBatchChunk + 4 * lane;
  if (i + 4 <= n) {
    const f32x4a4 q = *reinterpret_cast<const f32x4a4*>(row + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = q[e];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = i + e < n ? row[i + e] : -INFINITY;
  }
}

constexpr int kChunksPerWave = 4;

__global__ void __launch_bounds__(256) sample_chunks_kernel(SampleRows s) {
  const int row = blockIdx.y, lane = threadIdx.x & 63;
  const int chunks = (s.n + kBatchChunk - 1) / kBatchChunk;
  const int first = (blockIdx.x * 4 + (threadIdx.x >> 6)) * kChunksPerWave;
  if (first >= chunks) return;
  const float* logits = s.logits + (int64_t)row * s.n;
  float v[kChunksPerWave][4];
#pragma unroll
  for (int c = 0; c < kChunksPerWave; ++c)
    load_chunk(logits, s.n, min(first + c, chunks - 1), lane, v[c]);
  const RowParams p = row_params(s, row);
#pragma unroll
  for (int c = 0; c < kChunksPerWave; ++c) {
    bool nan = false;
    float m = -INFINITY;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      nan |= v[c][e] != v[c][e];
      m = fmaxf(m, v[c][e]);
    }
    m = wave_max(m);
    double mass = 0.0;
    if (p.mass) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        mass += v[c][e] > -INFINITY ? weight(v[c][e], m, p.temperature) : 0.0;
      for (int o = 32; o > 0; o >>= 1) mass += __shfl_xor(mass, o, 64);
    }
    nan = __ballot(nan) != 0;
    if (lane == 0 && first + c < chunks) {
      s.chunk_max[(int64_t)row * chunks + first + c] = nan ? NAN : m;
      s.chunk_mass[(int64_t)row * chunks + first + c] = mass;
    }
  }
}

// ------------------------------------------------------------------ the row's workgroup

struct FinishLds {
  uint64_t list[kListMax];
  double weights[kListMax];       // of the list; the bins' masses
  uint32_t counts[kBins];
  double chunk_mass[kBatchMaxChunks];
  float chunk_max[kBatchMaxChunks];
  uint64_t wave[kFinishThreads / 64];
  uint64_t result[4];
  int count;
};

// Every thread of the block calls the functions below.

// Inclusive prefix sums of T over the block in thread order; *total gets the sum.
template <typename T>
__device__ T block_scan(T v, FinishLds& l, T* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  T* part = reinterpret_cast<T*>(l.wave);
  for (int o = 1; o < 64; o <<= 1) {
    const T u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  if (lane == 63) part[wave] = v;
  __syncthreads();
  T before = 0, all = 0;
  for (int w = 0; w < kFinishThreads / 64; ++w) {
    const T u = part[w];
    before += w < wave ? u : (T)0;
    all += u;
  }
  __syncthreads();
  *total = all;
  return before + v;
}

// Sort list[0, n) in descending order (n <= kListMax; zeros pad it).
__device__ void sort_list(FinishLds& l, int n) {
  int size = 64;
  while (size < n) size <<= 1;
  for (int i = threadIdx.x; i < size; i += kFinishThreads)
    if (i >= n) l.list[i] = 0;
  __syncthreads();
  for (int k = 2; k <= size; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int i = threadIdx.x; i < size / 2; i += kFinishThreads) {
        const int a = (i / j) * 2 * j + i % j, b = a + j;
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

// Append where `take`, by every lane of a wavefront; entries past the list's end are counted only.
__device__ __forceinline__ void append(FinishLds& l, bool take, uint64_t e) {
  const uint64_t m = __ballot(take);
  if (!m) return;
  const int lane = threadIdx.x & 63;
  int at = 0;
  if (lane == 0) at = atomicAdd(&l.count, __popcll(m));
  at = __builtin_amdgcn_readfirstlane(at) + __popcll(m & ((1ull << lane) - 1ull));
  if (take && at < kListMax) l.list[at] = e;
}

// Weights of list[0, n) and their running sums in list order, kListMax / kFinishThreads entries a
// thread: before[k] is the sum ahead of entry threadIdx.x * 4 + k.
constexpr int kOwn = kListMax / kFinishThreads;
__device__ double list_sums(FinishLds& l, int n, float top, double t, bool by_index, double (&w)[kOwn],
                            double (&before)[kOwn]) {
  double sum = 0.0;
#pragma unroll
  for (int k = 0; k < kOwn; ++k) {
    const int i = threadIdx.x * kOwn + k;
    w[k] = 0.0;
    if (i < n) {
      const uint64_t e = l.list[i];
      w[k] = weight(of_order((uint32_t)(by_index ? e : e >> 32)), top, t);
    }
    before[k] = sum;
    sum += w[k];
  }
  double total;
  const double mine = block_scan(sum, l, &total) - sum;
#pragma unroll
  for (int k = 0; k < kOwn; ++k) before[k] += mine;
  return total;
}

// The token of the list of `n` candidates, which holds all that top-k or min-p keep.  `row_mass`:
// the row's total weight, for rows without top-k.
__device__ int draw_from_list(FinishLds& l, int n, const RowParams& p, float top, double row_mass) {
  sort_list(l, n);
  if (p.top_k) n = min(n, p.top_k);
  double w[kOwn], before[kOwn];
  double total = list_sums(l, n, top, p.temperature, false, w, before);
  const double reach = p.top_p * (p.top_k ? total : row_mass);
  int kept = 0;
#pragma unroll
  for (int k = 0; k < kOwn; ++k) {
    const int i = threadIdx.x * kOwn + k;
    // the filters keep a run from the first rank on
    kept += i < n && (p.top_p >= 1.0 || before[k] < reach || i == 0) && w[k] >= p.min_p ? 1 : 0;
  }
  int all;
  block_scan(kept, l, &all);
  n = all;
  for (int i = threadIdx.x; i < n; i += kFinishThreads) l.list[i] = l.list[i] << 32 | l.list[i] >> 32;
  __syncthreads();
  sort_list(l, n);
  total = list_sums(l, n, top, p.temperature, true, w, before);
  if (threadIdx.x == 0) l.count = INT_MAX;
  __syncthreads();
  const double at = p.random * total;
#pragma unroll
  for (int k = 0; k < kOwn; ++k) {
    const int i = threadIdx.x * kOwn + k;
    if (i < n && before[k] + w[k] > at) {
      atomicMin(&l.count, i);
      break;
    }
  }
  __syncthreads();
  const int i = l.count < n ? l.count : n - 1;
  return (int)(0xFFFFFFFFu - (uint32_t)(l.list[i] >> 32));
}

// 64-bit fixed-point weights of whole rows.
__device__ __forceinline__ uint64_t fixed_weight(float v, float top, double t) {
  return (uint64_t)(weight(v, top, t) * kMassOne + 0.5);
}

// Bin of a logit: ascends as the logit falls.
__device__ __forceinline__ int bin_of(float v, float top, float scale) {
  const float b = v == top ? 0.f : (top - v) * scale;
  return b < (float)(kBins - 1) ? (int)b : kBins - 1;
}

// The highest entry e such that the entries >= e reach `need` (their number, or their mass where
// `by_mass`), among the entries <= limit of the row.  0 where all of them do not.  `reached`: what the
// entries above e hold.
__device__ uint64_t row_cut(FinishLds& l, const float* row, int n, float top, double t, bool by_mass,
                            uint64_t need, uint64_t floor_entry) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int chunks = (n + kBatchChunk - 1) / kBatchChunk;
  const float scale = (float)(64.0 / t);
  uint64_t* bins = reinterpret_cast<uint64_t*>(l.weights);
  for (int i = tid; i < kBins; i += kFinishThreads) bins[i] = 0;
  __syncthreads();
  auto value = [&](float v) { return by_mass ? fixed_weight(v, top, t) : 1ull; };
  for (int c = wave; c < chunks; c += kFinishThreads / 64) {
    float v[4];
    load_chunk(row, n, c, lane, v);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (v[e] > -INFINITY && entry_of(v[e], c * kBatchChunk + 4 * lane + e) >= floor_entry)
        atomicAdd((unsigned long long*)&bins[bin_of(v[e], top, scale)], (unsigned long long)value(v[e]));
  }
  __syncthreads();
  // the bin that reaches it
  constexpr int kPer = kBins / kFinishThreads;
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
  for (int c = wave; c < chunks; c += kFinishThreads / 64) {
    float v[4];
    load_chunk(row, n, c, lane, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint64_t x = entry_of(v[e], c * kBatchChunk + 4 * lane + e);
      append(l, v[e] > -INFINITY && x >= floor_entry && bin_of(v[e], top, scale) == bin, x);
    }
  }
  __syncthreads();
  const int listed = l.count;
  __syncthreads();
  if (listed <= kListMax) {
    sort_list(l, listed);
    uint64_t own = 0, values[kOwn];
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
      const int i = tid * kOwn + k;
      values[k] = i < listed ? value(entry_logit(l.list[i])) : 0;
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
    for (int i = tid; i < 256; i += kFinishThreads) bins[i] = 0;
    __syncthreads();
    for (int c = wave; c < chunks; c += kFinishThreads / 64) {
      float v[4];
      load_chunk(row, n, c, lane, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint64_t x = entry_of(v[e], c * kBatchChunk + 4 * lane + e);
        if (v[e] > -INFINITY && x >= floor_entry && bin_of(v[e], top, scale) == bin &&
            (shift == 56 || x >> (shift + 8) == prefix))
          atomicAdd((unsigned long long*)&bins[(x >> shift) & 255], (unsigned long long)value(v[e]));
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
__device__ int draw_from_row(FinishLds& l, const float* row, int n, const RowParams& p, float top) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int chunks = (n + kBatchChunk - 1) / kBatchChunk;
  const double t = p.temperature;
  uint64_t cut = 0;
  if (p.top_k) cut = row_cut(l, row, n, top, t, false, (uint64_t)p.top_k, 0);
  uint64_t* mass = reinterpret_cast<uint64_t*>(l.chunk_mass);
  uint64_t total;
  auto chunk_masses = [&] {
    for (int c = wave; c < chunks; c += kFinishThreads / 64) {
      float v[4];
      load_chunk(row, n, c, lane, v);
      uint64_t sum = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (v[e] > -INFINITY && entry_of(v[e], c * kBatchChunk + 4 * lane + e) >= cut) {
          const double w = weight(v[e], top, t);
          sum += w >= p.min_p ? (uint64_t)(w * kMassOne + 0.5) : 0;
        }
      for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
      if (lane == 0) mass[c] = sum;
    }
    __syncthreads();
  };
  if (p.top_p < 1.0) {
    // what top-k kept, without min-p
    uint64_t sum = 0;
    for (int c = wave; c < chunks; c += kFinishThreads / 64) {
      float v[4];
      load_chunk(row, n, c, lane, v);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (v[e] > -INFINITY && entry_of(v[e], c * kBatchChunk + 4 * lane + e) >= cut)
          sum += fixed_weight(v[e], top, t);
    }
    block_scan(sum, l, &total);
    const double reach = p.top_p * (double)total;
    uint64_t need = (uint64_t)reach;
    need += (double)need < reach ? 1 : 0;
    cut = row_cut(l, row, n, top, t, true, need > 0 ? need : 1, cut);
  }
  chunk_masses();
  const uint64_t mine = tid < chunks ? mass[tid] : 0;
  const uint64_t upto = block_scan(mine, l, &total);
  const double at = p.random * (double)total;
  if (tid == 0) l.result[0] = ~0ull;
  __syncthreads();
  // the chunk at which the sum passes the mark, then the logit
  if (tid < chunks && (double)upto > at && !((double)(upto - mine) > at)) {
    l.result[0] = (uint64_t)tid;
    l.result[1] = upto - mine;
  }
  __syncthreads();
  const int chunk = (int)l.result[0];
  if (chunk < 0) return -1;
  uint64_t run = l.result[1];
  if (tid == 0) l.count = INT_MAX;
  __syncthreads();
  if (wave == 0) {
    float v[4];
    load_chunk(row, n, chunk, lane, v);
    uint64_t own[4], sum = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      own[e] = 0;
      if (v[e] > -INFINITY && entry_of(v[e], chunk * kBatchChunk + 4 * lane + e) >= cut) {
        const double w = weight(v[e], top, t);
        own[e] = w >= p.min_p ? (uint64_t)(w * kMassOne + 0.5) : 0;
      }
      sum += own[e];
    }
    uint64_t incl = sum;
    for (int o = 1; o < 64; o <<= 1) {
      const uint64_t u = __shfl_up(incl, o, 64);
      if (lane >= o) incl += u;
    }
    run += incl - sum;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      run += own[e];
      if (own[e] && (double)run > at) atomicMin(&l.count, chunk * kBatchChunk + 4 * lane + e);
    }
  }
  __syncthreads();
  return l.count;
}

__global__ void __launch_bounds__(kFinishThreads) sample_finish_kernel(SampleRows s) {
  extern __shared__ __align__(16) uint8_t raw[];
  FinishLds& l = *reinterpret_cast<FinishLds*>(raw);
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int chunks = (s.n + kBatchChunk - 1) / kBatchChunk;
  const float* logits = s.logits + (int64_t)row * s.n;
  const RowParams p = row_params(s, row);
  const float* cmax = s.chunk_max + (int64_t)row * chunks;
  // the row's maximum; a chunk with a NaN carries it
  float m = tid < chunks ? cmax[tid] : -INFINITY;
  const bool nan = m != m;
  if (tid < chunks) l.chunk_max[tid] = m;
  if (tid == 0) l.count = 0;
  float top = wave_max(nan ? -INFINITY : m);
  float* tops = reinterpret_cast<float*>(l.wave);
  if (lane == 0) tops[wave] = top;
  const int bad = __syncthreads_or(nan || p.bad);
  for (int w = 0; w < kFinishThreads / 64; ++w) top = fmaxf(top, tops[w]);
  __syncthreads();
  if (bad || !(top > -INFINITY)) {
    if (tid == 0) s.tokens[row] = -1;
    return;
  }
  const double t = p.temperature;
  double row_mass = 0.0;
  if (p.mass) {
    const double mine = tid < chunks && m > -INFINITY
                            ? s.chunk_mass[(int64_t)row * chunks + tid] * weight(m, top, t) : 0.0;
    const double upto = block_scan(mine, l, &row_mass);
    if (p.top_p >= 1.0) {
      // no filter: the chunk at which the sum passes the mark, then the logit
      const double at = p.random * row_mass;
      if (tid == 0) l.count = INT_MAX;
      __syncthreads();
      if (mine > 0.0 && upto > at) atomicMin(&l.count, tid);
      __syncthreads();
      int chunk = l.count;
      __syncthreads();
      if (chunk == INT_MAX) {  // the mark lies past the last sum's rounding: the last chunk with mass
        if (tid == 0) l.count = -1;
        __syncthreads();
        if (mine > 0.0) atomicMax(&l.count, tid);
        __syncthreads();
        chunk = l.count;
        __syncthreads();
      }
      if (tid == chunk) l.weights[0] = upto - mine;
      __syncthreads();
      if (wave == 0) {
        float v[4];
        load_chunk(logits, s.n, chunk, lane, v);
        double w[4], sum = 0.0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e] = v[e] > -INFINITY ? weight(v[e], top, t) : 0.0;
          sum += w[e];
        }
        double incl = sum;
        for (int o = 1; o < 64; o <<= 1) {
          const double u = __shfl_up(incl, o, 64);
          if (lane >= o) incl += u;
        }
        double run = l.weights[0] + (incl - sum);
        int found = INT_MAX, last = -1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          run += w[e];
          const int i = chunk * kBatchChunk + 4 * lane + e;
          if (w[e] > 0.0) {
            if (run > at) found = min(found, i);
            last = i;
          }
        }
        for (int o = 32; o > 0; o >>= 1) {
          found = min(found, __shfl_xor(found, o, 64));
          last = max(last, __shfl_xor(last, o, 64));
        }
        if (lane == 0) s.tokens[row] = found == INT_MAX ? last : found;
      }
      return;
    }
  }
  bool list = p.top_k ? p.top_k <= chunks : p.min_p > 0.0;
  if (list) {
    // the chunks that hold candidates, and the candidates
    uint32_t bound = 0;
    if (p.top_k) {
      if (tid < chunks) l.list[tid] = (uint64_t)order_of(m) << 32 | (uint32_t)tid;
      __syncthreads();
      sort_list(l, chunks);
      bound = (uint32_t)(l.list[p.top_k - 1] >> 32);
      __syncthreads();
    }
    for (int c = wave; c < chunks; c += kFinishThreads / 64) {
      const float cm = l.chunk_max[c];
      if (!(cm > -INFINITY) || (p.top_k ? order_of(cm) < bound : weight(cm, top, t) < p.min_p)) continue;
      float v[4];
      load_chunk(logits, s.n, c, lane, v);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        append(l, v[e] > -INFINITY && (p.top_k ? order_of(v[e]) >= bound : weight(v[e], top, t) >= p.min_p),
               entry_of(v[e], c * kBatchChunk + 4 * lane + e));
    }
    __syncthreads();
    list = l.count <= kListMax;
  }
  const int n = l.count;
  __syncthreads();
  const int token = list ? draw_from_list(l, n, p, top, row_mass) : draw_from_row(l, logits, s.n, p, top);
  if (tid == 0) s.tokens[row] = token;
}

hipError_t sample_rows_launch(const SampleRows& s, hipStream_t stream) {
  const int chunks = sample_chunks(s.n);
  hipLaunchKernelGGL(sample_chunks_kernel, dim3((chunks + 4 * kChunksPerWave - 1) / (4 * kChunksPerWave), s.rows),
                     dim3(256), 0, stream, s);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  e = hipFuncSetAttribute(reinterpret_cast<const void*>(sample_finish_kernel),
                          hipFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(FinishLds));
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(sample_finish_kernel, dim3(s.rows), dim3(kFinishThreads), sizeof(FinishLds), stream, s);
  return hipGetLastError();
}

}  // namespace llhip
