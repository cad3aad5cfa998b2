// attention.hip -- attention over a paged cache: what comes before and after the
// products (attention_tile.h).
//
// A call is up to three launches.  attn_prepare_kernel checks the sequences, rounds the
// new rows' keys and values into their pages and notes each tree row's ancestors,
// while one workgroup cuts the call into shares: the rows of a sequence and kv head
// are taken in tiles (row m is token m / group, head m % group, so that the heads of
// a group share what is read of the cache), and what all tiles see is dealt out
// evenly, where tiles are few, over as many workgroups as the device has CUs.  The
// attend kernel does the shares; the join adds up the parts of tiles that lie in
// several.  A call of few rows has no first launch (attention_tile.h), and so a step
// of one sequence is two: 13 + 5 us behind 4096 tokens, bound by latency.  Around the
// 97 us of attending 2311 tokens of prompts lie 9 of preparing and 10 of joining;
// moving the accepted nodes of 16 trees takes 4.5.  (Averages; the least are a few percent below.)
#include "attention_cut.h"

#include <algorithm>
#include <cstdint>

#include "mfma.h"

namespace llhip {

constexpr int kPlanThreads = 256;

static __host__ __device__ __forceinline__ int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// ------------------------------------------------------------------- checks
struct Sequence {
  int begin, length, context;
};

__device__ __forceinline__ Sequence sequence_of(const AttnCall& c, int i) {
  Sequence s;
  s.begin = c.offsets ? c.offsets[i] : i;
  s.length = c.offsets ? c.offsets[i + 1] - s.begin : 1;
  s.context = c.context[i];
  return s;
}

// Whether the offsets ascend within the call's tokens (by a whole workgroup).
__device__ bool offsets_hold(const AttnCall& c) {
  if (!c.offsets) return true;
  bool ok = true;
  for (int i = threadIdx.x; i <= c.sequences; i += blockDim.x) {
    const int v = c.offsets[i];
    ok = ok && v >= 0 && v <= c.tokens && (i == 0 || c.offsets[i - 1] <= v);
  }
  return __syncthreads_and(ok);
}

// Whether a sequence's context, pages or tree are wrong, which is noted (by a whole workgroup).
__device__ bool sequence_refused(const AttnPlan& p, const AttnCall& c, int i, const Sequence& s) {
  int bad = 0;
  if (s.context < 0 || (int64_t)s.context + s.length > p.max_context) {
    bad = kAttnErrContext;
  } else {
    const int pages = ceil_div(s.context + s.length, 1 << p.page_shift);
    for (int e = threadIdx.x; e < pages; e += blockDim.x)
      if ((uint32_t)c.table[i * c.table_stride + e] >= (uint32_t)p.pages) bad = kAttnErrPage;
  }
  if (c.parents) {
    if (s.length > kAttnTreeNodes) {
      bad |= kAttnErrTree;
    } else {
      for (int j = threadIdx.x; j < s.length; j += blockDim.x) {
        const int parent = c.parents[s.begin + j];
        if (parent < -1 || parent >= j) bad |= kAttnErrTree;
      }
    }
  }
  if (bad) atomicOr(p.error, bad);
  return __syncthreads_or(bad);
}

// ------------------------------------------------------------------- the cut
// Inclusive sum over the workgroup; `total` receives all of it.
template <typename T>
__device__ T block_scan(T v, T* lds, T& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const T u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  if (lane == 63) lds[wave] = v;
  __syncthreads();
  total = 0;
  T before = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    if (w < wave) before += lds[w];
    total += lds[w];
  }
  __syncthreads();
  return v + before;
}

// Tiles and shares.  Where tiles are few, or one is long, equal shares of all units (a tile that lies in several of
// them has as many parts); where they are many, each tile is a share and the long ones come first, so that the short
// ones fill what they leave.  (Tiles of like length are then in the order of a counter: no result depends on it.)
constexpr int kLengths = 32;
constexpr int kManyTiles = 2;  // for each share

__device__ void plan(const AttnPlan& p, const AttnCall& c, const AttnCut& cut) {
  __shared__ int scan[kPlanThreads / 64], ends[kPlanThreads], lengths[kPlanThreads], contexts[kPlanThreads],
      begins[kPlanThreads], places[kLengths], longest;
  __shared__ int64_t scan_units[kPlanThreads / 64];
  if (!offsets_hold(c)) {
    if (threadIdx.x == 0) {
      atomicOr(p.error, kAttnErrOffsets);
      p.counts[0] = p.counts[1] = 0;
    }
    return;
  }
  if (threadIdx.x == 0) longest = 0;
  if (threadIdx.x < kLengths) places[threadIdx.x] = 0;
  int before = 0;
  int64_t units = 0;
  for (int i0 = 0; i0 < c.sequences; i0 += kPlanThreads) {
    const int i = i0 + threadIdx.x;
    Sequence s{0, 0, 0};
    if (i < c.sequences) s = sequence_of(c, i);
    // a refused sequence's tiles do nothing; they only have to be few
    if (s.context < 0 || (int64_t)s.context + s.length > p.max_context) s.context = s.length = 0;
    int tiles;
    ends[threadIdx.x] = block_scan((s.length * (int)p.group.divisor + cut.rows - 1) / cut.rows, scan, tiles);
    lengths[threadIdx.x] = s.length;
    contexts[threadIdx.x] = s.context;
    begins[threadIdx.x] = s.begin;
    __syncthreads();
    for (int t0 = 0; t0 < tiles; t0 += kPlanThreads) {
      const int t = t0 + threadIdx.x;
      AttnTile tile{};
      if (t < tiles) {
        int which = 0;
        for (int hi = kPlanThreads - 1; which < hi;) {  // the first sequence whose tiles end behind t
          const int mid = (which + hi) / 2;
          if (ends[mid] > t) hi = mid;
          else which = mid + 1;
        }
        const int m0 = (ends[which] - 1 - t) * cut.rows;
        tile = AttnTile{i0 + which, begins[which], lengths[which], contexts[which], m0,
                        attn_seen_keys(p, c, cut, m0, lengths[which], contexts[which]), 0};
      }
      const int mine = t < tiles ? attn_units(cut, tile.seen) : 0;
      int64_t all;
      tile.start = units + block_scan((int64_t)(t < tiles ? mine + cut.overhead : 0), scan_units, all) - mine;
      units += all;
      if (t < tiles) p.tiles[before + t] = tile;
      int most = mine;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) most = max(most, __shfl_xor(most, o, 64));
      if ((threadIdx.x & 63) == 0) atomicMax(&longest, most);
    }
    before += tiles;
    __syncthreads();
  }
  const int64_t share = attn_share(cut, units);
  // (what this workgroup wrote is read back by other threads of it: the barriers order it)
  if (before >= kManyTiles * cut.shares && longest <= 2 * share) {
    for (int pass = 0; pass < 2; ++pass) {
      for (int t = threadIdx.x; t < before; t += kPlanThreads) {
        const AttnTile tile = p.tiles[t];
        const int n = attn_units(cut, tile.seen);
        const int at = atomicAdd(&places[kLengths - 1 - (int)((int64_t)n * (kLengths - 1) / longest)], 1);
        if (pass == 1) p.workers[at] = AttnWorker{tile.start, tile.start + n, t, 0};
      }
      __syncthreads();
      if (pass == 0) {
        if (threadIdx.x == 0) {
          int sum = 0;
          for (int l = 0; l < kLengths; ++l) {
            const int n = places[l];
            places[l] = sum;
            sum += n;
          }
        }
        __syncthreads();
      }
    }
    if (threadIdx.x == 0) {
      p.counts[0] = before;
      p.counts[1] = 0;
    }
    return;
  }
  const int shares = units ? attn_share_of(units - 1, share) + 1 : 0;
  for (int w = threadIdx.x; w < shares; w += kPlanThreads) p.joins[w].parts = 0;
  __syncthreads();
  for (int t = threadIdx.x; t < before; t += kPlanThreads) {
    const AttnTile tile = p.tiles[t];
    const int n = attn_units(cut, tile.seen);
    // shares that begin within the tile or its overhead, and the one before, which may end there
    const int first = attn_share_of(tile.start - cut.overhead + share - 1, share);
    const int last = attn_share_of(tile.start + n - 1, share);
    for (int w = max(first - 1, 0); w <= last; ++w) {
      const AttnWorker worker{w * share, min((w + 1) * share, units), t, attn_slack(share)};
      if (w >= first) p.workers[w] = worker;
      AttnItem it{tile.sequence, tile.begin, tile.length, tile.context, tile.m0, 0, 0, 0};
      if (attn_item(cut, worker, w, tile.seen, tile.start, it) && it.key0 == 0 && it.part >= 0)
        p.joins[w] = attn_join(cut, it, tile.seen, tile.start, share, w);
    }
  }
  if (threadIdx.x == 0) p.counts[0] = p.counts[1] = shares;
}

// ------------------------------------------------------------- keys and values
// Workgroup 0 makes the plan; `share` workgroups take the rows of each sequence.
template <typename Row, typename T>
__global__ __launch_bounds__(kPlanThreads) void attn_prepare_kernel(AttnPlan p, AttnCall c, AttnCut cut, int share) {
  if (blockIdx.x == 0) {
    plan(p, c, cut);
    return;
  }
  const int i = (blockIdx.x - 1) / share, part = (blockIdx.x - 1) % share;
  if (!offsets_hold(c)) {
    if (threadIdx.x == 0 && part == 0) p.run[i] = 0;
    return;
  }
  const Sequence s = sequence_of(c, i);
  const bool bad = s.length > 0 && sequence_refused(p, c, i, s);
  if (threadIdx.x == 0 && part == 0) p.run[i] = !bad;
  if (bad || s.length <= 0) return;
  if (c.parents && part == 0) {
    __shared__ int parents[kAttnTreeNodes];
    __shared__ uint32_t words[kAttnTreeNodes][kAttnTreeWords];
    const int j = threadIdx.x;
    static_assert(kAttnTreeNodes <= kPlanThreads, "a thread for each node");
    if (j < s.length) parents[j] = c.parents[s.begin + j];
    __syncthreads();
    if (j < s.length) {
#pragma unroll
      for (int w = 0; w < kAttnTreeWords; ++w) words[j][w] = 0;
      for (int n = j; n >= 0; n = parents[n]) words[j][n >> 5] |= 1u << (n & 31);
#pragma unroll
      for (int w = 0; w < kAttnTreeWords; ++w) p.tree[(size_t)(s.begin + j) * kAttnTreeWords + w] = words[j][w];
    }
  }
  const int pieces = p.kv_heads * p.head_dim / 8, per_head = p.head_dim / 8;
  for (int r = part; r < s.length; r += share) {
    const int pos = s.context + r;
    const size_t at = attn_cell(p, c.layer, c.table[i * c.table_stride + (pos >> p.page_shift)], pos);
    const Row* k = static_cast<const Row*>(c.k) + (s.begin + r) * c.k_stride;
    const Row* v = static_cast<const Row*>(c.v) + (s.begin + r) * c.v_stride;
    for (int e = threadIdx.x; e < 2 * pieces; e += kPlanThreads) {
      const bool value = e >= pieces;
      const int piece = value ? e - pieces : e;
      const size_t to = at + ((size_t)(piece / per_head) << p.page_shift) * p.head_dim + piece % per_head * 8;
      attn_put8(static_cast<T*>(value ? p.values : p.keys) + to,
                *reinterpret_cast<const attn_eight<Row>*>((value ? v : k) + 8 * piece));
    }
  }
}

// ----------------------------------------------------------------------- joins
// Row m of a join: parts' sums taken to one reference.  A wavefront per row; kJoinParts parts' sums are on their way at once.
constexpr int kJoinParts = 8;
template <typename Row>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnPlan p, AttnCall c, AttnCut cut, int padded, int blocks) {
  const int index = blockIdx.x / (p.kv_heads * blocks), rest = blockIdx.x % (p.kv_heads * blocks);
  if (index >= p.counts[1]) return;
  const AttnJoin j = p.joins[index];
  const int kv_head = rest / blocks, lane = threadIdx.x & 63;
  const int r = rest % blocks * 4 + (threadIdx.x >> 6);
  if (j.parts < 2 || r >= cut.rows || j.m0 + r >= j.length * (int)p.group.divisor || (!cut.few && !p.run[j.sequence])) return;
  auto row = [&](int k) {
    return ((size_t)(k == 0 ? j.part0 : j.part1 + 2 * (k - 1)) * p.kv_heads + kv_head) * cut.rows + r;
  };
  float reference = -__builtin_inff();
  for (int k = lane; k < j.parts; k += 64) reference = fmaxf(reference, p.part_ml[row(k)].x);
  reference = wave_max(reference);
  const int d = min(4 * lane, padded - 4);
  floatx4 v{};
  float total = 0.f;
  for (int k0 = 0; k0 < j.parts; k0 += 64) {
    float weight = 0.f;
    if (k0 + lane < j.parts) {
      const float2 ml = p.part_ml[row(k0 + lane)];
      // a part of which the row sees nothing has zeros
      weight = ml.x == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(ml.x - reference);
      total += weight * ml.y;
    }
    const int count = min(64, j.parts - k0);
    for (int k = 0; k < count; k += kJoinParts) {
      floatx4 y[kJoinParts];
#pragma unroll
      for (int i = 0; i < kJoinParts; ++i)
        y[i] = *reinterpret_cast<const floatx4*>(p.part_y + row(k0 + min(k + i, count - 1)) * padded + d);
#pragma unroll
      for (int i = 0; i < kJoinParts; ++i) {
        const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, weight), k + i));
        if (k + i < count) v += w * y[i];
      }
    }
  }
  total = wave_total(total);
  if (4 * lane >= p.head_dim) return;
  const int m = j.m0 + r;
  Row* y = static_cast<Row*>(c.y) + (j.begin + m / p.group) * c.y_stride +
           (kv_head * (int)p.group.divisor + m % p.group) * p.head_dim + d;
  typedef Row Row4 __attribute__((ext_vector_type(4)));
  *reinterpret_cast<Row4*>(y) = __builtin_convertvector(v * (1.f / total), Row4);
}

// The same where tiles have many rows, and few parts: four elements of two rows a thread.
constexpr int kJoinAtOnce = 2;
static __host__ __device__ __forceinline__ int join_rows(int padded) { return kJoinAtOnce * 256 / (padded / 4); }

template <typename Row>
__global__ __launch_bounds__(256) void attn_join_rows_kernel(AttnPlan p, AttnCall c, AttnCut cut, int padded, int blocks) {
  const int index = blockIdx.x / (p.kv_heads * blocks), rest = blockIdx.x % (p.kv_heads * blocks);
  if (index >= p.counts[1]) return;
  const AttnJoin j = p.joins[index];
  const int kv_head = rest / blocks, r0 = rest % blocks * join_rows(padded), rows = j.length * (int)p.group.divisor - j.m0;
  if (j.parts < 2 || r0 >= rows || !p.run[j.sequence]) return;
  const int pieces = padded / 4, d = threadIdx.x % pieces * 4, step = 256 / pieces;
  auto place = [&](int k) {
    return ((size_t)(k == 0 ? j.part0 : j.part1 + 2 * (k - 1)) * p.kv_heads + kv_head) * cut.rows;
  };
  const int r = r0 + threadIdx.x / pieces;
  float reference[kJoinAtOnce], total[kJoinAtOnce] = {};
  floatx4 v[kJoinAtOnce] = {};
#pragma unroll
  for (int i = 0; i < kJoinAtOnce; ++i) reference[i] = -__builtin_inff();
  for (int k = 0; k < j.parts; ++k)
#pragma unroll
    for (int i = 0; i < kJoinAtOnce; ++i)
      reference[i] = fmaxf(reference[i], p.part_ml[place(k) + r + i * step].x);
  for (int k = 0; k < j.parts; ++k)
#pragma unroll
    for (int i = 0; i < kJoinAtOnce; ++i) {
      const size_t row = place(k) + r + i * step;
      const float2 ml = p.part_ml[row];
      const floatx4 y = *reinterpret_cast<const floatx4*>(p.part_y + row * padded + d);
      // a part of which the row sees nothing has zeros
      const float weight = ml.x == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(ml.x - reference[i]);
      total[i] += weight * ml.y;
      v[i] += weight * y;
    }
#pragma unroll
  for (int i = 0; i < kJoinAtOnce; ++i) {
    const int row = r + i * step, m = j.m0 + row;
    if (row >= rows || d >= p.head_dim) continue;
    Row* y = static_cast<Row*>(c.y) + (j.begin + m / p.group) * c.y_stride +
             (kv_head * (int)p.group.divisor + m % p.group) * p.head_dim + d;
    typedef Row Row4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<Row4*>(y) = __builtin_convertvector(v[i] * (1.f / total[i]), Row4);
  }
}

// ------------------------------------------------------------------- accepting
// Workgroups per sequence and layer, each with a share of the elements.  Node n_j goes to place j: n_0 < n_1 < ... has
// n_j >= j, so that no place is written before it is read if nodes are taken in order, some at a time; a thread moves
// its own 16 bytes of every node.
constexpr int kAcceptAtOnce = 8;
template <typename T>
__global__ __launch_bounds__(kPlanThreads) void attn_accept_kernel(AttnPlan p, AttnAccept a) {
  const int i = blockIdx.x, count = a.counts[i], context = a.context[i];
  const int* path = a.paths + i * a.path_stride;
  const int* table = a.table + i * a.table_stride;
  int bad = 0;
  if (count < 0 || count > min((int64_t)kAttnTreeNodes, a.path_stride)) {
    bad = kAttnErrPath;
  } else if (count == 0) {
    return;
  } else {
    for (int j = threadIdx.x; j < count; j += kPlanThreads)
      if (path[j] < 0 || path[j] >= kAttnTreeNodes || (j > 0 && path[j] <= path[j - 1])) bad |= kAttnErrPath;
  }
  if (!__syncthreads_or(bad)) {
    if (context < 0 || (int64_t)context + path[count - 1] >= p.max_context) {
      bad = kAttnErrContext;
    } else {
      // the pages between the cached tokens' end and the last node
      const int first = context >> p.page_shift, last = (context + path[count - 1]) >> p.page_shift;
      for (int e = first + threadIdx.x; e <= last; e += kPlanThreads)
        if ((uint32_t)table[e] >= (uint32_t)p.pages) bad = kAttnErrPage;
    }
  }
  if (bad) atomicOr(p.error, bad);
  if (__syncthreads_or(bad)) return;
  __shared__ size_t from[kAttnTreeNodes], to[kAttnTreeNodes];
  static_assert(kAttnTreeNodes <= kPlanThreads, "a thread for each node");
  if ((int)threadIdx.x < count) {
    const int source = context + path[threadIdx.x], place = context + threadIdx.x;
    from[threadIdx.x] = attn_cell(p, blockIdx.y, table[source >> p.page_shift], source);
    to[threadIdx.x] = attn_cell(p, blockIdx.y, table[place >> p.page_shift], place);
  }
  __syncthreads();
  constexpr int E = 16 / sizeof(T);
  const int pieces = p.kv_heads * p.head_dim / E, per_head = p.head_dim / E;
  for (int e = blockIdx.z * kPlanThreads + threadIdx.x; e < 2 * pieces; e += gridDim.z * kPlanThreads) {
    T* const pool = static_cast<T*>(e >= pieces ? p.values : p.keys);
    const int piece = e >= pieces ? e - pieces : e;
    const size_t in = ((size_t)(piece / per_head) << p.page_shift) * p.head_dim + piece % per_head * E;
    for (int j = 0; j < count; j += kAcceptAtOnce) {
      u32x4 v[kAcceptAtOnce];
#pragma unroll
      for (int i = 0; i < kAcceptAtOnce; ++i)
        v[i] = *reinterpret_cast<const u32x4*>(pool + from[min(j + i, count - 1)] + in);
#pragma unroll
      for (int i = 0; i < kAcceptAtOnce; ++i)
        if (j + i < count) *reinterpret_cast<u32x4*>(pool + to[j + i] + in) = v[i];
    }
  }
}

// error[1] = what error[0] gathered, which starts anew: in one step, for calls on other streams may add to it.
__global__ void attn_take_error_kernel(int* error) {
  if (threadIdx.x == 0) error[1] = atomicExch(error, 0);
}

// ------------------------------------------------------------------------ host

constexpr int kCus = 256;
// Rows of a kv head in a sequence, on average, up to which waves share rows and not keys: those of two wavefronts, for
// with fewer than three of eight at work the other kernel loses more than reading the keys for each 32 rows costs (us, 16
// trees behind 2000 tokens, 8 kv heads of 128, fp32 rows over f16: 32 rows 53 against 69, 64 rows 68 and 72, 80 rows 86
// and 72; over fp32 157 and 193, 248 and 207, 353 and 211).  A call without a launch before has more to lose (one tree
// behind 4000 tokens: 160 rows 42 and 60; behind 30000, 160 rows 88 and 96, 224 rows 153 and 106), but not over
// fp32 (30000 tokens, 128 rows: 347 and 192).
constexpr int kFewRows = 64, kFewRowsAlone = 160;

static AttnCut cut_as(const AttnPlan& p, bool shared) {
  const int padded = attn_padded(p.head_dim), row_bytes = p.row_type == kAttnF32 ? 4 : 2;
  AttnCut cut{};
  cut.shared = shared;
  cut.rows = shared ? 32 * attn_shared_waves(p.cache_type, row_bytes, padded) : 32;
  // A unit is a tile of keys (two, where it has 32), or two for each wavefront (a step of one sequence 20 us, with twice
  // as many 22, a tree of 26 nodes 35 and 38).  What else a tile costs, about 8 us to load its rows, to fill the pipeline
  // and to store, is taken for some of them: (us for 2, 3, 4 and 5) prompts of 2311 tokens over f16 145, 129, 120, 126; 12 of 2000, heads of 256 and
  // fp32 rows, whose units take twice as long, 105, 98, 106, 107; 1501 tokens in fp32, four times, 124, 131, 131, 138.
  const int keys = attn_shared_keys(padded, row_bytes);
  cut.unit_log2 = !shared ? 8 : keys == 128 ? 7 : 6;
  cut.overhead = !shared || p.cache_type == kAttnF32 || keys == 128 ? 2 : keys == 32 ? 3 : 4;
  cut.shares = std::max(1, kCus / p.kv_heads);
  cut.each = 1.0 / cut.shares;
  return cut;
}
static AttnCut cut_of(const AttnPlan& p, const AttnCall& c) {
  const bool alone = c.tokens <= kAttnFewTokens && c.sequences <= kAttnFewSequences;
  const int64_t rows = ceil_div((int64_t)c.tokens * p.group.divisor, c.sequences);
  AttnCut cut = cut_as(p, rows > (alone && p.cache_type != kAttnF32 ? kFewRowsAlone : kFewRows));
  cut.few = !cut.shared && alone;
  return cut;
}

// Tiles of a call at most: one for each cut.rows rows and one more for each sequence.
static int64_t tiles_of(const AttnPlan& p, int64_t tokens, int64_t sequences, int rows) {
  return std::min(tokens * p.group.divisor / rows + sequences, tokens * p.group.divisor);
}
static int64_t workers_of(const AttnPlan& p, const AttnCall& c, const AttnCut& cut) {
  return cut.few ? cut.shares : std::max<int64_t>(cut.shares, tiles_of(p, c.tokens, c.sequences, cut.rows));
}

AttnSizes attn_sizes(const AttnPlan& p) {
  AttnSizes s{0, 0, 0, 0};
  for (int shared = 0; shared < 2; ++shared) {
    const AttnCut cut = cut_as(p, shared);
    s.tiles = std::max(s.tiles, tiles_of(p, p.max_tokens, p.max_sequences, cut.rows));
    s.shares = std::max<int64_t>(s.shares, cut.shares);
    s.part_rows = std::max(s.part_rows, (int64_t)2 * cut.shares * p.kv_heads * cut.rows);
  }
  s.workers = std::max(s.tiles, s.shares);
  return s;
}

static int64_t prepare_share(const AttnPlan& p, const AttnCall& c) {
  // a row is 1 or 2 rounds of a workgroup; some rows each, as many workgroups as the device holds several times over
  const int64_t rows = ceil_div(c.tokens, c.sequences);
  return std::max<int64_t>(1, std::min<int64_t>(ceil_div(rows, 2), 8 * kCus / c.sequences));
}
static int64_t join_blocks(const AttnCut& cut, const AttnPlan& p, const AttnCall& c) {
  if (cut.shared) return cut.rows / join_rows(attn_padded(p.head_dim));
  // 4 rows each; a step has only a group's
  return ceil_div(c.offsets ? cut.rows : std::min<int>(cut.rows, p.group.divisor), 4);
}
static int64_t join_grid(const AttnPlan& p, const AttnCall& c, const AttnCut& cut) {
  return (int64_t)cut.shares * p.kv_heads * join_blocks(cut, p, c);
}

bool attn_call_fits(const AttnPlan& p, const AttnCall& c) {
  const AttnCut cut = cut_of(p, c);
  const int64_t most = UINT32_MAX / 512;
  return workers_of(p, c, cut) * p.kv_heads <= most && 1 + c.sequences * prepare_share(p, c) <= most &&
         join_grid(p, c, cut) <= most;
}

template <typename Row>
static hipError_t join(const AttnPlan& p, const AttnCall& c, const AttnCut& cut, hipStream_t s) {
  const dim3 grid((uint32_t)join_grid(p, c, cut));
  const int padded = attn_padded(p.head_dim), blocks = (int)join_blocks(cut, p, c);
  if (cut.shared) hipLaunchKernelGGL(attn_join_rows_kernel<Row>, grid, dim3(256), 0, s, p, c, cut, padded, blocks);
  else hipLaunchKernelGGL(attn_join_kernel<Row>, grid, dim3(256), 0, s, p, c, cut, padded, blocks);
  return hipGetLastError();
}

template <typename Row, typename T>
static hipError_t prepare(const AttnPlan& p, const AttnCall& c, const AttnCut& cut, hipStream_t s) {
  const int share = (int)prepare_share(p, c);
  hipLaunchKernelGGL((attn_prepare_kernel<Row, T>), dim3((uint32_t)(1 + (int64_t)c.sequences * share)),
                     dim3(kPlanThreads), 0, s, p, c, cut, share);
  return hipGetLastError();
}

hipError_t attn_run_launch(const AttnPlan& p, const AttnCall& c, hipStream_t s) {
  const AttnCut cut = cut_of(p, c);
  hipError_t e = hipSuccess;
  if (cut.few) {
  } else if (p.row_type == kAttnF16) e = prepare<_Float16, _Float16>(p, c, cut, s);
  else if (p.row_type == kAttnBF16) e = prepare<__bf16, __bf16>(p, c, cut, s);
  else if (p.cache_type == kAttnF16) e = prepare<float, _Float16>(p, c, cut, s);
  else if (p.cache_type == kAttnBF16) e = prepare<float, __bf16>(p, c, cut, s);
  else e = prepare<float, float>(p, c, cut, s);
  if (e != hipSuccess) return e;
  const uint32_t grid = (uint32_t)(workers_of(p, c, cut) * p.kv_heads);
  switch (p.cache_type) {
    case kAttnF16: e = attn_attend_f16(p, c, cut, grid, s); break;
    case kAttnBF16: e = attn_attend_bf16(p, c, cut, grid, s); break;
    default: e = attn_attend_f32(p, c, cut, grid, s); break;
  }
  if (e != hipSuccess) return e;
  if (p.max_context <= 1 << cut.unit_log2) return hipSuccess;  // no tile has parts to join
  if (p.row_type == kAttnF16) return join<_Float16>(p, c, cut, s);
  if (p.row_type == kAttnBF16) return join<__bf16>(p, c, cut, s);
  return join<float>(p, c, cut, s);
}

hipError_t attn_accept_launch(const AttnPlan& p, const AttnAccept& a, hipStream_t s) {
  const int bytes = 2 * p.kv_heads * p.head_dim * (p.cache_type == kAttnF32 ? 4 : 2);
  const dim3 grid(a.sequences, p.layers, ceil_div(bytes, 16 * kPlanThreads));
  if (p.cache_type == kAttnF32) hipLaunchKernelGGL(attn_accept_kernel<float>, grid, dim3(kPlanThreads), 0, s, p, a);
  else hipLaunchKernelGGL(attn_accept_kernel<uint16_t>, grid, dim3(kPlanThreads), 0, s, p, a);
  return hipGetLastError();
}

hipError_t attn_take_error_launch(const AttnPlan& p, hipStream_t s) {
  hipLaunchKernelGGL(attn_take_error_kernel, dim3(1), dim3(64), 0, s, p.error);
  return hipGetLastError();
}

}  // namespace llhip
