// attention.hip -- attention over a paged cache: what comes before and after the
// products (attention_tile.h).
//
// A call is three launches.  attn_prepare_kernel checks the sequences, rounds the
// new rows' keys and values into their pages and notes each tree row's ancestors,
// while one workgroup cuts the call into items: the rows of a sequence and kv head
// in tiles (row m is token m / group, head m % group, so that the heads of a group
// share what is read of the cache), and the positions that a tile sees in parts
// where the tiles alone would not fill the device or one would outlast the rest.
// The attend kernel does the items; attn_join_kernel adds up parts.
#include "attention_cut.h"

#include <algorithm>
#include <climits>

#include "mfma.h"

namespace llhip {

constexpr int kPlanThreads = 256;
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float8_t __attribute__((ext_vector_type(8)));

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
__device__ int block_scan(int v, int* lds, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  if (lane == 63) lds[wave] = v;
  __syncthreads();
  total = 0;
  int before = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    if (w < wave) before += lds[w];
    total += lds[w];
  }
  __syncthreads();
  return v + before;
}

// Items and joins.  Long items come first, so that the short ones fill what they leave: a count of items by length, then
// their places.  (The order of items of like length, and of the partial results' places, is that of the counters: no
// result depends on it.)
constexpr int kLengths = 16;

__device__ void plan(const AttnPlan& p, const AttnCall& c, const AttnCut& cut) {
  __shared__ int scan[kPlanThreads / 64], ends[kPlanThreads], lengths[kPlanThreads], contexts[kPlanThreads],
      begins[kPlanThreads], places[kLengths], joins, parts;
  __shared__ unsigned long long keys;
  if (!offsets_hold(c)) {
    if (threadIdx.x == 0) {
      atomicOr(p.error, kAttnErrOffsets);
      p.counts[0] = p.counts[1] = 0;
    }
    return;
  }
  if (threadIdx.x == 0) keys = joins = parts = 0;
  if (threadIdx.x < kLengths) places[threadIdx.x] = 0;
  int chunk = 0;
  for (int pass = 0; pass < 3; ++pass) {
    for (int i0 = 0; i0 < c.sequences; i0 += kPlanThreads) {
      const int i = i0 + threadIdx.x;
      Sequence s{0, 0, 0};
      if (i < c.sequences) s = sequence_of(c, i);
      // a refused sequence's items do nothing; they only have to be few
      if (s.context < 0 || (int64_t)s.context + s.length > p.max_context) s.context = s.length = 0;
      int tiles;
      ends[threadIdx.x] = block_scan((s.length * (int)p.group.divisor + cut.rows - 1) / cut.rows, scan, tiles);
      lengths[threadIdx.x] = s.length;
      contexts[threadIdx.x] = s.context;
      begins[threadIdx.x] = s.begin;
      __syncthreads();
      for (int t = threadIdx.x; t < tiles; t += kPlanThreads) {
        int which = 0;
        for (int hi = kPlanThreads - 1; which < hi;) {  // the first sequence whose tiles end behind t
          const int mid = (which + hi) / 2;
          if (ends[mid] > t) hi = mid;
          else which = mid + 1;
        }
        const int m0 = (ends[which] - 1 - t) * cut.rows;
        const int seen = attn_seen_keys(p, c, cut, m0, lengths[which], contexts[which]);
        if (pass == 0) {
          atomicAdd(&keys, (unsigned long long)seen);
          continue;
        }
        const int n = attn_parts_of(seen, chunk);
        AttnItem it{i0 + which, begins[which], lengths[which], contexts[which], m0, 0, 0, 0};
        attn_part(it, seen, n, 0, 0);
        // all parts but the last have one length; the last takes its place among them
        const int length = kLengths - 1 - (int)((int64_t)min(it.key1, chunk) * (kLengths - 1) / chunk);
        const int at = atomicAdd(&places[length], n);
        if (pass == 1) continue;
        const int part = n > 1 ? atomicAdd(&parts, n) : 0;
        for (int k = 0; k < n; ++k) {
          attn_part(it, seen, n, k, part);
          p.items[at + k] = it;
        }
        if (n > 1) p.joins[atomicAdd(&joins, 1)] = AttnJoin{begins[which], lengths[which], m0, n, part, i0 + which};
      }
      __syncthreads();
    }
    if (pass == 0) chunk = attn_chunk(p, cut, (int64_t)keys);
    if (pass == 1) {
      if (threadIdx.x == 0) {
        int before = 0;
        for (int l = 0; l < kLengths; ++l) {
          const int n = places[l];
          places[l] = before;
          before += n;
        }
        p.counts[0] = before;
      }
      __syncthreads();
    }
  }
  if (threadIdx.x == 0) p.counts[1] = joins;
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
      attn_put8(static_cast<T*>(value ? p.values : p.keys) + to, (value ? v : k) + 8 * piece);
    }
  }
}

// ----------------------------------------------------------------------- joins
// Row m of a join: parts' sums taken to one reference.  A wavefront per row; eight parts' sums are on their way at once.
template <typename Row>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnPlan p, AttnCall c, AttnCut cut, int padded, int blocks) {
  const int index = blockIdx.x / (p.kv_heads * blocks), rest = blockIdx.x % (p.kv_heads * blocks);
  if (index >= p.counts[1]) return;
  const AttnJoin j = p.joins[index];
  const int kv_head = rest / blocks, lane = threadIdx.x & 63;
  const int r = rest % blocks * 4 + (threadIdx.x >> 6);
  if (j.parts < 2 || r >= cut.rows || j.m0 + r >= j.length * (int)p.group.divisor || (!cut.few && !p.run[j.sequence])) return;
  const size_t step = (size_t)p.kv_heads * cut.rows;
  const size_t row = ((size_t)j.part0 * p.kv_heads + kv_head) * cut.rows + r;
  float reference = -__builtin_inff();
  for (int k = lane; k < j.parts; k += 64) reference = fmaxf(reference, p.part_ml[row + k * step].x);
  reference = wave_max(reference);
  const int d = min(4 * lane, padded - 4);
  floatx4 v{};
  float total = 0.f;
  for (int k0 = 0; k0 < j.parts; k0 += 64) {
    float weight = 0.f;
    if (k0 + lane < j.parts) {
      const float2 ml = p.part_ml[row + (k0 + lane) * step];
      // a part of which the row sees nothing has zeros
      weight = ml.x == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(ml.x - reference);
      total += weight * ml.y;
    }
    const int count = min(64, j.parts - k0);
    for (int k = 0; k < count; k += 8) {
      floatx4 y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        y[i] = *reinterpret_cast<const floatx4*>(p.part_y + (row + (k0 + min(k + i, count - 1)) * step) * padded + d);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
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

// ------------------------------------------------------------------- accepting
// A workgroup per sequence and layer.  Node n_j goes to place j: n_0 < n_1 < ... has n_j >= j, so that in order no
// place is written before it is read; a thread moves its own 16 bytes of every node.
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
  constexpr int E = 16 / sizeof(T);
  const int pieces = p.kv_heads * p.head_dim / E, per_head = p.head_dim / E;
  for (int e = threadIdx.x; e < 2 * pieces; e += kPlanThreads) {
    T* const pool = static_cast<T*>(e >= pieces ? p.values : p.keys);
    const int piece = e >= pieces ? e - pieces : e;
    const size_t in = ((size_t)(piece / per_head) << p.page_shift) * p.head_dim + piece % per_head * E;
    for (int j = 0; j < count; ++j) {
      const int from = context + path[j], to = context + j;
      if (from == to) continue;
      const u32x4 v = *reinterpret_cast<const u32x4*>(
          pool + attn_cell(p, blockIdx.y, table[from >> p.page_shift], from) + in);
      *reinterpret_cast<u32x4*>(pool + attn_cell(p, blockIdx.y, table[to >> p.page_shift], to) + in) = v;
    }
  }
}

// error[1] = what error[0] gathered, which starts anew: in one step, for calls on other streams may add to it.
__global__ void attn_take_error_kernel(int* error) {
  if (threadIdx.x == 0) error[1] = atomicExch(error, 0);
}

// ------------------------------------------------------------------------ host

constexpr int kCus = 256;
#ifndef RT
#define SLS 8
#define MINS 256
#define SLP 9
#define MINP 256
#define RT 160
#endif

static int shared_waves(const AttnPlan& p) {
  const int padded = attn_padded(p.head_dim);
  return padded == 256 || (p.cache_type == kAttnBF16 && p.row_type == kAttnF32 && padded == 128) ? 4 : 8;
}

static AttnCut cut_as(const AttnPlan& p, bool shared) {
  AttnCut cut{};
  cut.shared = shared;
  cut.rows = shared ? 32 * shared_waves(p) : 32;
  cut.min_keys = shared ? MINS : MINP;
  cut.slots_log2 = shared ? SLS : SLP;
  return cut;
}
static AttnCut cut_of(const AttnPlan& p, const AttnCall& c) {
  // rows of a kv head in a sequence, on average; the lengths are on the device
  AttnCut cut = cut_as(p, ceil_div((int64_t)c.tokens * p.group.divisor, c.sequences) > RT);
  cut.few = !cut.shared && c.tokens <= kAttnFewTokens && c.sequences <= kAttnFewSequences;
  return cut;
}

// Items of a call at most: a tile for each cut.rows rows, one more for each sequence, and parts that are no shorter
// than the keys of all tiles over 2^slots_log2.
static int64_t tiles_of(const AttnPlan& p, int64_t tokens, int64_t sequences, int rows) {
  return std::min(tokens * p.group.divisor / rows + sequences, tokens * p.group.divisor);
}
static int64_t items_of(const AttnPlan& p, int64_t tokens, int64_t sequences, const AttnCut& cut) {
  return tiles_of(p, tokens, sequences, cut.rows) + (1 << cut.slots_log2) / p.kv_heads;
}

AttnSizes attn_sizes(const AttnPlan& p) {
  AttnSizes s{0, 0, 0};
  for (int shared = 0; shared < 2; ++shared) {
    const AttnCut cut = cut_as(p, shared);
    const int64_t tiles = tiles_of(p, p.max_tokens, p.max_sequences, cut.rows);
    const int64_t split = (1 << cut.slots_log2) / p.kv_heads;
    s.items = std::max(s.items, tiles + split);
    s.joins = std::max(s.joins, std::min(tiles, split));
    if (!shared)  // of a call of few rows one for each tile
      s.joins = std::max(s.joins, tiles_of(p, std::min(p.max_tokens, kAttnFewTokens),
                                           std::min(p.max_sequences, kAttnFewSequences), cut.rows));
    // n > 1 parts are at most twice the n - 1 that come beside the tile's own
    s.part_rows = std::max(s.part_rows, 2 * split * p.kv_heads * cut.rows);
  }
  return s;
}

static int64_t prepare_share(const AttnPlan& p, const AttnCall& c) {
  // a row is 1 or 2 rounds of a workgroup; some rows each, as many workgroups as the device holds several times over
  const int64_t rows = ceil_div(c.tokens, c.sequences);
  return std::max<int64_t>(1, std::min<int64_t>(ceil_div(rows, 2), 8 * kCus / c.sequences));
}
static int64_t join_blocks(const AttnCut& cut, const AttnPlan& p, const AttnCall& c) {
  // 4 rows each; a step has only a group's
  return ceil_div(c.offsets ? cut.rows : std::min<int>(cut.rows, p.group.divisor), 4);
}
static int64_t join_grid(const AttnPlan& p, const AttnCall& c, const AttnCut& cut) {
  const int64_t tiles = tiles_of(p, c.tokens, c.sequences, cut.rows);
  return (cut.few ? tiles : std::min<int64_t>(tiles, (1 << cut.slots_log2) / p.kv_heads)) * p.kv_heads * join_blocks(cut, p, c);
}

bool attn_call_fits(const AttnPlan& p, const AttnCall& c) {
  const AttnCut cut = cut_of(p, c);
  const int64_t most = UINT32_MAX / 512;
  return items_of(p, c.tokens, c.sequences, cut) * p.kv_heads <= most &&
         1 + c.sequences * prepare_share(p, c) <= most && join_grid(p, c, cut) <= most;
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
  const uint32_t grid = (uint32_t)(items_of(p, c.tokens, c.sequences, cut) * p.kv_heads);
  switch (p.cache_type) {
    case kAttnF16: e = attn_attend_f16(p, c, cut, grid, s); break;
    case kAttnBF16: e = attn_attend_bf16(p, c, cut, grid, s); break;
    default: e = attn_attend_f32(p, c, cut, grid, s); break;
  }
  if (e != hipSuccess) return e;
  // where no sequence can have two parts there is nothing to join
  if (p.max_context <= cut.min_keys) return hipSuccess;
  const uint32_t joins = (uint32_t)join_grid(p, c, cut);
  if (joins == 0) return hipSuccess;
  const int padded = attn_padded(p.head_dim), blocks = (int)join_blocks(cut, p, c);
  if (p.row_type == kAttnF16) hipLaunchKernelGGL(attn_join_kernel<_Float16>, dim3(joins), dim3(256), 0, s, p, c, cut, padded, blocks);
  else if (p.row_type == kAttnBF16) hipLaunchKernelGGL(attn_join_kernel<__bf16>, dim3(joins), dim3(256), 0, s, p, c, cut, padded, blocks);
  else hipLaunchKernelGGL(attn_join_kernel<float>, dim3(joins), dim3(256), 0, s, p, c, cut, padded, blocks);
  return hipGetLastError();
}

hipError_t attn_accept_launch(const AttnPlan& p, const AttnAccept& a, hipStream_t s) {
  const dim3 grid(a.sequences, p.layers);
  if (p.cache_type == kAttnF32) hipLaunchKernelGGL(attn_accept_kernel<float>, grid, dim3(kPlanThreads), 0, s, p, a);
  else hipLaunchKernelGGL(attn_accept_kernel<uint16_t>, grid, dim3(kPlanThreads), 0, s, p, a);
  return hipGetLastError();
}

hipError_t attn_take_error_launch(const AttnPlan& p, hipStream_t s) {
  hipLaunchKernelGGL(attn_take_error_kernel, dim3(1), dim3(64), 0, s, p.error);
  return hipGetLastError();
}

}  // namespace llhip
