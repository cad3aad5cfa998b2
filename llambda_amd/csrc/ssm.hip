// ssm.hip -- the Mamba-2 mixer's kernels (ssm.h).
//
// One token per sequence (ssm_step_kernel): a workgroup per sequence, head and
// 8192 state elements reads them, applies the recurrence and writes them;
// bound by the state's traffic.  ssm_finish_kernel then gates and norms the
// rows and shifts the convolution's state.
//
// Sequences of any lengths: the plan kernel checks the call and cuts the
// sequences into segments and chunks of Q = 32 tokens; ssm_prepare_kernel
// convolves B and C once for all heads and forms each chunk's decays; the scan
// kernel takes one segment of a few heads per workgroup, chunk by chunk, the
// state in registers.  With e_i the decay from the chunk's start to token i,
//   Y = (S o L) X + e (C s),  S = C B^T,  L_ij = dt_j e_i / e_j  (j <= i)
//   s' = e_Q s + sum_j B_j (x_j dt_j e_Q / e_j)^T
// are matrix products.  Every operand keeps the lane that made it: the state
// is held transposed, as the result tiles [16 n][16 p] that the next chunk's
// C s takes as its right operand without a move (a lane's four result rows are
// four of its K elements; which K element a lane holds is free as long as both
// operands agree), x likewise, and S is formed transposed so that its result
// is M's left operand.  Exponents are sums in 64 bits, kept as two floats,
// and subtracted before exp2 is taken, so a strong decay early in the chunk
// costs the later tokens no precision.
// Long sequences of few heads are cut into segments so that the grid fills the
// device: a first pass forms each segment's own state, a small kernel joins
// them in order, and the scan proper starts each segment from its state.
#include "mfma.h"
#include "ssm.h"

#include <algorithm>
#include <cfloat>
#include <climits>

namespace llhip {

typedef float f32x4a4 __attribute__((ext_vector_type(4), aligned(4)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr double kLog2eD = 1.44269504088896340736;

// exp(v) to about one unit: 2^(v log2 e) with the product's rounding error
// brought back in (v log2 e = t + r).
__device__ __forceinline__ float exp_f32(float v) {
  const float t = v * kLog2e;
  const float r = fmaf(v, kLog2e, -t) + v * 1.925963033500e-8f;  // log2 e - float(log2 e)
  const float e = __builtin_amdgcn_exp2f(t);
  // near the ends of the exponent range e is left as it is (inf, zero)
  return fabsf(t) < 126.f ? fmaf(e, r * 0.69314718056f, e) : e;
}
__device__ __forceinline__ float silu_f32(float v) {
  // large negative v: exp overflows and v / inf = -0, as the limit is
  return v / (1.f + exp_f32(-v));
}
// log(1 + e^v) = max(v, 0) + log1p(e^-|v|)
__device__ __forceinline__ float softplus_f32(float v) {
  return fmaxf(v, 0.f) + log1pf(exp_f32(-fabsf(v)));
}

// log2 of one token's decay, dt A log2 e.  Bounded below: 2^-4096 is zero in
// single precision times any single, and the sums and their differences stay
// finite.  (NaN passes through.)
__device__ __forceinline__ double log2_decay(float dt, float a) {
  const double v = (double)dt * (double)a * kLog2eD;
  return v < -4096.0 ? -4096.0 : v;
}

// ------------------------------------------------------------------ planning

// Slots of sequence i of a call: what it reads and what it writes.
__device__ __forceinline__ int slot_of(const int* list, int i) { return list ? list[i] : i; }

// Whether sequence i may run, by the block's threads together (uniform): its
// slots lie in the pool, and no other sequence reads or writes the slot that
// it writes.  `flag`: one int of LDS.
__device__ bool slots_allowed(const SsmLayerPlan& p, const SsmCall& c, int i, int* flag) {
  const int from = slot_of(c.from, i), to = slot_of(c.to, i);
  int bad = (from < -1 || from >= p.slots || to < -1 || to >= p.slots) ? kSsmErrSlot : 0;
  if (threadIdx.x == 0) *flag = bad;
  __syncthreads();
  if (!bad && to >= 0 && (c.from || c.to)) {
    bool hit = false;
    for (int j = threadIdx.x; j < c.sequences; j += blockDim.x)
      hit |= j != i && (slot_of(c.from, j) == to || slot_of(c.to, j) == to);
    if (hit) *flag = kSsmErrConflict;
  }
  __syncthreads();
  bad = *flag;
  __syncthreads();
  if (bad && threadIdx.x == 0) atomicOr(p.error, bad);
  return bad == 0;
}

constexpr int kPlanThreads = 256;

// One workgroup per sequence: its place in the tables.  The sums over the
// earlier sequences' chunks and segments are formed by each workgroup itself.
__global__ void __launch_bounds__(kPlanThreads) ssm_plan_kernel(SsmLayerPlan p, SsmCall c,
                                                                int segment_tokens) {
  __shared__ int flag, bad;
  __shared__ int part[3][kPlanThreads / 64];
  const int i = blockIdx.x, tid = threadIdx.x;
  if (tid == 0) bad = 0;
  __syncthreads();
  // offsets ascend within the tokens (every workgroup checks them all: the
  // tables' bounds rest on it)
  bool wrong = false;
  int chunks = 0, segments = 0, states = 0;
  for (int j = tid; j < c.sequences; j += kPlanThreads) {
    const int b = c.offsets[j], e = c.offsets[j + 1];
    const bool w = b < 0 || e < b || e > c.tokens;
    wrong |= w;
    if (!w && j < i) {
      const int len = e - b;
      chunks += (len + kSsmChunk - 1) / kSsmChunk;
      const int n = max(1, (len + segment_tokens - 1) / segment_tokens);
      segments += n;
      states += n > 1 ? n : 0;
    }
  }
  if (wrong) bad = 1;
  for (int o = 32; o > 0; o >>= 1) {
    chunks += __shfl_xor(chunks, o, 64);
    segments += __shfl_xor(segments, o, 64);
    states += __shfl_xor(states, o, 64);
  }
  if ((tid & 63) == 0) {
    part[0][tid >> 6] = chunks;
    part[1][tid >> 6] = segments;
    part[2][tid >> 6] = states;
  }
  __syncthreads();
  chunks = segments = states = 0;
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    chunks += part[0][w];
    segments += part[1][w];
    states += part[2][w];
  }
  if (bad) {
    if (tid == 0) {
      atomicOr(p.error, kSsmErrOffsets);
      SsmSequence s{};
      p.sequences[i] = s;
      p.counts[0] = p.counts[1] = 0;
    }
    return;
  }
  const bool run = slots_allowed(p, c, i, &flag);
  const int begin = c.offsets[i], length = c.offsets[i + 1] - begin;
  const int nc = (length + kSsmChunk - 1) / kSsmChunk;
  const int ns = max(1, (length + segment_tokens - 1) / segment_tokens);
  if (tid == 0) {
    p.sequences[i] = SsmSequence{begin,  length,   slot_of(c.from, i), slot_of(c.to, i),
                                 chunks, ns,       states,             run};
    if (i == c.sequences - 1) {
      p.counts[0] = segments + ns;
      p.counts[1] = chunks + nc;
    }
  }
  for (int j = tid; j < nc; j += kPlanThreads) p.chunks[chunks + j] = make_int2(i, j);
  for (int j = tid; j < ns; j += kPlanThreads) p.segments[segments + j] = make_int2(i, j);
}

// ------------------------------------------------------------------ convolution

// The raw row t of a sequence's x | B | C, t < 0 from the state it started
// with (zeros for a new sequence), four channels from `ch`.
__device__ __forceinline__ floatx4 raw4(const float* rows, int64_t stride, const float* taps,
                                        int channels, int conv, int t, int length, int ch) {
  if (t >= length) return floatx4{0.f, 0.f, 0.f, 0.f};
  if (t >= 0) return *reinterpret_cast<const f32x4a4*>(rows + (int64_t)t * stride + ch);
  if (!taps) return floatx4{0.f, 0.f, 0.f, 0.f};
  return *reinterpret_cast<const f32x4a4*>(taps + (int64_t)(conv - 1 + t) * channels + ch);
}
__device__ __forceinline__ float raw1(const float* rows, int64_t stride, const float* taps,
                                      int channels, int conv, int t, int length, int ch) {
  if (t >= length) return 0.f;
  if (t >= 0) return rows[(int64_t)t * stride + ch];
  return taps ? taps[(int64_t)(conv - 1 + t) * channels + ch] : 0.f;
}

__device__ __forceinline__ const float* conv_taps(const SsmLayerPlan& p, int slot) {
  const int channels = p.heads * p.head_dim + 2 * p.groups * p.state;
  return slot < 0 ? nullptr : p.conv_states + (int64_t)slot * (p.conv - 1) * channels;
}

// Block (chunk, y): y < blocks of 256 channels of B | C: their convolution,
// a thread taking four channels of eight tokens; then blocks of eight heads:
// dt and the decays, a lane per token.
constexpr int kPrepChannels = 256;
constexpr int kPrepHeads = 8;

template <int W>
__global__ void __launch_bounds__(256) ssm_prepare_kernel(SsmLayerPlan p, SsmCall c) {
  const int chunk = blockIdx.x;
  if (chunk >= p.counts[1]) return;
  const int2 at = p.chunks[chunk];
  const SsmSequence s = p.sequences[at.x];
  if (!s.run) return;
  const int inner = p.heads * p.head_dim, gn = p.groups * p.state, channels = inner + 2 * gn;
  const int64_t stride = inner + channels + p.heads;
  const float* rows = c.x + (int64_t)s.begin * stride + inner;
  const int tid = threadIdx.x, t0 = at.y * kSsmChunk;
  const int conv_blocks = (2 * gn + kPrepChannels - 1) / kPrepChannels;
  if ((int)blockIdx.y < conv_blocks) {
    const int bc = blockIdx.y * kPrepChannels + 4 * (tid & 63);  // within B | C
    if (bc >= 2 * gn) return;
    const int ch = inner + bc, q0 = 8 * (tid >> 6);
    const float* taps = conv_taps(p, s.from);
    floatx4 w[W], r[8 + W - 1];
#pragma unroll
    for (int k = 0; k < 8 + W - 1; ++k)
      r[k] = raw4(rows, stride, taps, channels, W, t0 + q0 - (W - 1) + k, s.length, ch);
#pragma unroll
    for (int k = 0; k < W; ++k)
      w[k] = *reinterpret_cast<const floatx4*>(p.conv_weight + (int64_t)k * channels + ch);
    const floatx4 b = *reinterpret_cast<const floatx4*>(p.conv_bias + ch);
    // [chunk][group][B, C][token][n]
    const int which = bc >= gn, inside = bc - which * gn;
    float* out = p.bc + ((((int64_t)chunk * p.groups + inside / p.state) * 2 + which) * kSsmChunk + q0) *
                            p.state + inside % p.state;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      floatx4 v = b;
#pragma unroll
      for (int k = 0; k < W; ++k) v += w[k] * r[q + k];
      floatx4 u;
#pragma unroll
      for (int e = 0; e < 4; ++e) u[e] = t0 + q0 + q < s.length ? silu_f32(v[e]) : 0.f;
      *reinterpret_cast<floatx4*>(out + (int64_t)q * p.state) = u;
    }
    return;
  }
  const int h = ((int)blockIdx.y - conv_blocks) * kPrepHeads + (tid >> 5), q = tid & 31;
  if (h >= p.heads) return;
  const bool in = t0 + q < s.length;
  const float dt = in ? softplus_f32(rows[(int64_t)(t0 + q) * stride + channels + h] + p.dt_bias[h]) : 0.f;
  double sum = in ? log2_decay(dt, p.a[h]) : 0.0;
  for (int o = 1; o < kSsmChunk; o <<= 1) {
    const double v = __shfl_up(sum, o, 32);
    if (q >= o) sum += v;
  }
  float* out = p.decay + ((int64_t)chunk * p.heads + h) * 3 * kSsmChunk + q;
  const float hi = (float)sum;
  out[0] = dt;
  out[kSsmChunk] = hi;
  out[2 * kSsmChunk] = (float)(sum - (double)hi);
}

// ------------------------------------------------------------------ the scan

// acc += A B over 32 K elements (16 with N8 = 4): a lane's element e of both
// operands is the same K element.
template <int N8>
__device__ __forceinline__ floatx4 mma(const float* a, const float* b, floatx4 acc) {
#pragma unroll
  for (int e = 0; e < N8; ++e) acc = mfma4f32(a[e], b[e], acc);
  return acc;
}

constexpr int kScanWaves = 4;
constexpr int kScanTiles = 8;  // column tiles of 16 channels per workgroup, two per wave

// Heads per workgroup: as many whole heads of one group as fit its tiles.
static int scan_heads(const SsmLayerPlan& p) {
  const int share = p.heads / p.groups;
  int n = std::max(1, kScanTiles * 16 / p.head_dim);
  while (share % n) --n;
  return n;
}

// One segment of `hw` heads.  STATES: only the segment's own state, from
// zeros, to the next segment's place; else outputs and, in a sequence's last
// segment, the state to its slot.
template <int NT, int W, bool STATES>
__global__ void __launch_bounds__(64 * kScanWaves) ssm_scan_kernel(SsmLayerPlan p, SsmCall c,
                                                                   int segment_tokens, int hw) {
  constexpr int N = 16 * NT, Q = kSsmChunk, LD = N + 4;
  extern __shared__ float lds[];
  float* sb = lds;                      // [Q][LD]
  float* sc = sb + Q * LD;              // [Q][LD]
  float* sm = sc + (STATES ? 0 : Q * LD);  // [hw][3 tiles][64 lanes][4]
  float* sd = sm + (STATES ? 0 : hw * 3 * 256);  // [hw][3][Q]
  const int sets = p.heads / hw;
  // groups vary fastest, so that the workgroups that read one group's B and C
  // sit on one XCD where there are eight groups
  const int set_in_group = sets / p.groups;
  const int seg = blockIdx.x / sets, rest = blockIdx.x - seg * sets;
  if (seg >= p.counts[0]) return;
  const int2 at = p.segments[seg];
  const SsmSequence s = p.sequences[at.x];
  if (!s.run) return;
  if (STATES && at.y == s.segments - 1) return;  // no segment follows
  const int group = rest % p.groups, h0 = (group * set_in_group + rest / p.groups) * hw;
  const int inner = p.heads * p.head_dim, channels = inner + 2 * p.groups * p.state;
  const int64_t stride = inner + channels + p.heads;
  const float* rows = c.x + (int64_t)s.begin * stride + inner;
  const float* taps = conv_taps(p, s.from);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, g = lane >> 4;
  const int t_begin = at.y * segment_tokens, t_end = min(s.length, t_begin + segment_tokens);

  // this wave's column tiles: channels [p0, p0 + 16) of a head
  const int per_head = p.head_dim / 16, tiles = hw * per_head;
  bool on[2];
  int head[2], ch[2];
  float skip[2], w[2][W], bias[2];
  floatx4 st[2][NT];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int tile = wave + kScanWaves * k;
    on[k] = tile < tiles;
    head[k] = on[k] ? tile / per_head : 0;
    ch[k] = (h0 + head[k]) * p.head_dim + (on[k] ? tile % per_head : 0) * 16 + col;
    skip[k] = p.d[h0 + head[k]];
    bias[k] = p.conv_bias[ch[k]];
#pragma unroll
    for (int j = 0; j < W; ++j) w[k][j] = p.conv_weight[(int64_t)j * channels + ch[k]];
    const float* src = nullptr;
    if (!STATES) {
      if (s.segments > 1) src = p.seg_states + (int64_t)(s.state0 + at.y) * inner * N;
      else if (s.from >= 0) src = p.ssm_states + (int64_t)s.from * inner * N;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
      st[k][n] = src && on[k] ? *reinterpret_cast<const floatx4*>(src + (int64_t)ch[k] * N + 16 * n + 4 * g)
                              : floatx4{0.f, 0.f, 0.f, 0.f};
  }
  float total_hi[2] = {0.f, 0.f}, total_lo[2] = {0.f, 0.f};

  for (int t0 = t_begin; t0 < t_end; t0 += Q) {
    const int64_t chunk = s.chunk0 + t0 / Q;
    __syncthreads();  // the last chunk's operands have been read
    {
      const floatx4* src = reinterpret_cast<const floatx4*>(p.bc + (chunk * p.groups + group) * 2 * Q * N);
      constexpr int kVec = Q * N / 4;
      for (int i = tid; i < (STATES ? 1 : 2) * kVec; i += 64 * kScanWaves) {
        const int which = i / kVec, r = (i - which * kVec) / (N / 4), q = i % (N / 4);
        *reinterpret_cast<floatx4*>((which ? sc : sb) + r * LD + 4 * q) = src[i];
      }
      const float* dsrc = p.decay + (chunk * p.heads + h0) * 3 * Q;
      for (int i = tid; i < hw * 3 * Q; i += 64 * kScanWaves) sd[i] = dsrc[i];
    }
    // x of the lane's tokens 4 g .. + 3 and 16 + 4 g .. + 3
    float x[2][8];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (!on[k]) continue;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float r[4 + W - 1];
        const int t = t0 + 16 * half + 4 * g;
#pragma unroll
        for (int j = 0; j < 4 + W - 1; ++j)
          r[j] = raw1(rows, stride, taps, channels, W, t - (W - 1) + j, t_end, ch[k]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = bias[k];
#pragma unroll
          for (int j = 0; j < W; ++j) v = fmaf(w[k][j], r[e + j], v);
          x[k][4 * half + e] = t + e < t_end ? silu_f32(v) : 0.f;
        }
      }
    }
    // A non-finite x_j would reach the tokens before it, as 0 x_j in the masked
    // part of the product: the products take zero in its place, and the
    // channel's outputs from token j on are NaN (its state too, by x itself).
    float xf[2][8];
    int first_bad[2] = {Q, Q};
    if constexpr (!STATES) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (!on[k]) continue;
        bool bad = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          xf[k][e] = x[k][e];
          bad |= !(fabsf(x[k][e]) <= FLT_MAX);
        }
        if (__ballot(bad)) {
          int f = Q;
#pragma unroll
          for (int e = 7; e >= 0; --e)
            if (!(fabsf(x[k][e]) <= FLT_MAX)) {
              f = 16 * (e >> 2) + 4 * g + (e & 3);
              xf[k][e] = 0.f;
            }
          f = min(f, __shfl_xor(f, 16, 64));
          first_bad[k] = min(f, __shfl_xor(f, 32, 64));
        }
      }
    }
    __syncthreads();
    if constexpr (!STATES) {
      // S^T tiles (j tile, i tile) = (0, 0), (0, 1), (1, 1), one per wave
      if (wave < 3) {
        const int jt = wave == 2, it = wave > 0;
        floatx4 acc{0.f, 0.f, 0.f, 0.f};
        const float* pa = sb + (16 * jt + col) * LD + 4 * g;
        const float* pb = sc + (16 * it + col) * LD + 4 * g;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const floatx4 a = *reinterpret_cast<const floatx4*>(pa + 16 * n);
          const floatx4 b = *reinterpret_cast<const floatx4*>(pb + 16 * n);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc = mfma4f32(a[e], b[e], acc);
        }
        const int i = 16 * it + col, j0 = 16 * jt + 4 * g;
        for (int h = 0; h < hw; ++h) {
          const float* dd = sd + h * 3 * Q;
          const float ihi = dd[Q + i], ilo = dd[2 * Q + i];
          floatx4 m;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = j0 + e;
            const float l = (ihi - dd[Q + j]) + (ilo - dd[2 * Q + j]);
            m[e] = j <= i ? acc[e] * (__builtin_amdgcn_exp2f(l) * dd[j]) : 0.f;
          }
          *reinterpret_cast<floatx4*>(sm + ((h * 3 + wave) * 64 + lane) * 4) = m;
        }
      }
      __syncthreads();
#pragma unroll
      for (int it = 0; it < 2; ++it) {
        floatx4 acc[2] = {floatx4{0.f, 0.f, 0.f, 0.f}, floatx4{0.f, 0.f, 0.f, 0.f}};
        const float* pa = sc + (16 * it + col) * LD + 4 * g;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const floatx4 a = *reinterpret_cast<const floatx4*>(pa + 16 * n);
#pragma unroll
          for (int k = 0; k < 2; ++k)
            if (on[k])
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[k] = mfma4f32(a[e], st[k][n][e], acc[k]);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (!on[k]) continue;
          const float* dd = sd + head[k] * 3 * Q;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = 16 * it + 4 * g + e;
            acc[k][e] = acc[k][e] * __builtin_amdgcn_exp2f(dd[Q + i] + dd[2 * Q + i]);
          }
          for (int jt = 0; jt <= it; ++jt) {
            const floatx4 a = *reinterpret_cast<const floatx4*>(sm + ((head[k] * 3 + it + jt) * 64 + lane) * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[k] = mfma4f32(a[e], xf[k][4 * jt + e], acc[k]);
          }
          float* out = c.y + (int64_t)(s.begin + t0 + 16 * it + 4 * g) * inner + ch[k];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (t0 + 16 * it + 4 * g + e < t_end)
              out[(int64_t)e * inner] = 16 * it + 4 * g + e < first_bad[k]
                                            ? fmaf(skip[k], xf[k][4 * it + e], acc[k][e])
                                            : __builtin_nanf("");
        }
      }
    }
    // the state: decayed, plus the tokens' products
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (!on[k]) continue;
      const float* dd = sd + head[k] * 3 * Q;
      const float qhi = dd[2 * Q - 1], qlo = dd[3 * Q - 1];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int j = 16 * (e >> 2) + 4 * g + (e & 3);
        x[k][e] *= dd[j] * __builtin_amdgcn_exp2f((qhi - dd[Q + j]) + (qlo - dd[2 * Q + j]));
      }
      const float e = __builtin_amdgcn_exp2f(qhi + qlo);
#pragma unroll
      for (int n = 0; n < NT; ++n) st[k][n] *= e;
      total_hi[k] += qhi;
      total_lo[k] += qlo;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float b[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) b[e] = sb[(16 * (e >> 2) + 4 * g + (e & 3)) * LD + 16 * n + col];
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (on[k]) st[k][n] = mma<8>(b, x[k], st[k][n]);
    }
  }

  float* dst = nullptr;
  if (STATES) dst = p.seg_states + (int64_t)(s.state0 + at.y + 1) * inner * N;
  else if (at.y == s.segments - 1 && s.to >= 0) dst = p.ssm_states + (int64_t)s.to * inner * N;
  if (!dst) return;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (!on[k]) continue;
#pragma unroll
    for (int n = 0; n < NT; ++n)
      *reinterpret_cast<floatx4*>(dst + (int64_t)ch[k] * N + 16 * n + 4 * g) = st[k][n];
    if (STATES && g == 0 && ch[k] % p.head_dim == 0)
      p.seg_decay[(int64_t)(s.state0 + at.y) * p.heads + h0 + head[k]] = total_hi[k] + total_lo[k];
  }
}

// The segments' states in order: what enters the first is the sequence's (the
// scan's last segment may be writing that slot while the first reads it, so
// it gets a copy), each later one its predecessor's, decayed, plus what that
// segment added.
__global__ void __launch_bounds__(256) ssm_join_kernel(SsmLayerPlan p) {
  const SsmSequence s = p.sequences[blockIdx.x];
  if (!s.run || s.segments <= 1) return;
  const int inner = p.heads * p.head_dim, per_head = p.head_dim * p.state;
  const int64_t size = (int64_t)inner * p.state, i = ((int64_t)blockIdx.y * 256 + threadIdx.x) * 4;
  if (i >= size) return;
  const int h = (int)(i / per_head);
  floatx4 v{0.f, 0.f, 0.f, 0.f};
  if (s.from >= 0) v = *reinterpret_cast<const floatx4*>(p.ssm_states + (int64_t)s.from * size + i);
  float* at = p.seg_states + (int64_t)s.state0 * size + i;
  *reinterpret_cast<floatx4*>(at) = v;
  constexpr int kAhead = 8;  // loads in flight
  for (int k0 = 1; k0 < s.segments; k0 += kAhead) {
    floatx4 add[kAhead];
    float e[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (k0 + k < s.segments) {
        add[k] = *reinterpret_cast<const floatx4*>(at + (int64_t)(k0 + k) * size);
        e[k] = p.seg_decay[(int64_t)(s.state0 + k0 + k - 1) * p.heads + h];
      }
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (k0 + k < s.segments) {
        v = v * __builtin_amdgcn_exp2f(e[k]) + add[k];
        *reinterpret_cast<floatx4*>(at + (int64_t)(k0 + k) * size) = v;
      }
  }
}

// ------------------------------------------------------------------ one token

// Block (sequence, head, part): kStepElements state elements of a head.  N / 4
// lanes share a channel's state row.
constexpr int kStepElements = 8192;

template <int N>
__global__ void __launch_bounds__(256) ssm_step_kernel(SsmLayerPlan p, SsmCall c) {
  constexpr int LANES = N / 4, ROWS = 256 / LANES;  // channels per round of the block
  constexpr int kRounds = kStepElements / (ROWS * N);
  __shared__ float sx[kSsmMaxHeadDim], sb[N], sc[N];
  __shared__ int flag;
  const int i = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  if (!slots_allowed(p, c, i, &flag)) return;
  const int from = slot_of(c.from, i), to = slot_of(c.to, i);
  const int P = p.head_dim, inner = p.heads * P, gn = p.groups * N, channels = inner + 2 * gn, W = p.conv;
  const int group = h / (p.heads / p.groups);
  const float* row = c.x + (int64_t)i * (inner + channels + p.heads);
  const float* taps = conv_taps(p, from);
  const int p0 = blockIdx.z * (kStepElements / N), np = min(P - p0, kStepElements / N);
  // the state first: its loads run while the convolution is formed
  const int q = tid % LANES, r0 = tid / LANES;
  const int64_t at = ((int64_t)h * P + p0) * N + 4 * q;
  floatx4 st[kRounds];
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const int r = r0 + ROWS * k;
    st[k] = from >= 0 && r < np
                ? *reinterpret_cast<const floatx4*>(p.ssm_states + (int64_t)from * inner * N + at + (int64_t)r * N)
                : floatx4{0.f, 0.f, 0.f, 0.f};
  }
  const float dt = softplus_f32(row[inner + channels + h] + p.dt_bias[h]);
  const float a = __builtin_amdgcn_exp2f((float)log2_decay(dt, p.a[h]));
  for (int k = tid; k < np + 2 * N; k += 256) {
    const int ch = k < np ? h * P + p0 + k
                          : inner + (k - np >= N ? gn : 0) + group * N + (k - np) % N;
    float v = p.conv_bias[ch];
    for (int j = 0; j < W - 1; ++j)
      v = fmaf(p.conv_weight[(int64_t)j * channels + ch], taps ? taps[(int64_t)j * channels + ch] : 0.f, v);
    v = silu_f32(fmaf(p.conv_weight[(int64_t)(W - 1) * channels + ch], row[inner + ch], v));
    if (k < np) sx[k] = v;
    else (k - np >= N ? sc : sb)[(k - np) % N] = v;
  }
  __syncthreads();
  const floatx4 b = *reinterpret_cast<const floatx4*>(sb + 4 * q);
  const floatx4 cc = *reinterpret_cast<const floatx4*>(sc + 4 * q);
  const float d = p.d[h];
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const int r = r0 + ROWS * k;
    const float x = r < np ? sx[r] : 0.f;
    st[k] = st[k] * a + b * (dt * x);
    float y = (st[k].x * cc.x + st[k].y * cc.y) + (st[k].z * cc.z + st[k].w * cc.w);
    y = segment_sum<LANES>(y);
    if (r >= np) continue;
    if (to >= 0)
      *reinterpret_cast<floatx4*>(p.ssm_states + (int64_t)to * inner * N + at + (int64_t)r * N) = st[k];
    if (q == 0) c.y[(int64_t)i * inner + h * P + p0 + r] = fmaf(d, x, y);
  }
}

// ------------------------------------------------------------------ gate, norm, convolution state

// Blocks [0, norm_blocks): rows y of (token, group), THREADS threads each:
// v = y silu(z), out = v / sqrt(mean v^2 + eps) * norm, in place.  The others:
// the convolution state of a sequence, 256 channels a block (a thread reads
// all of a channel's rows before it writes them: from and to may be one slot).
template <int THREADS>
__global__ void __launch_bounds__(256 > THREADS ? 256 : THREADS)
ssm_finish_kernel(SsmLayerPlan p, SsmCall c, int norm_blocks) {
  constexpr int BLOCK = 256 > THREADS ? 256 : THREADS;
  constexpr int kPer = 4;  // vectors of four channels per thread, THREADS * 16 channels at most
  __shared__ float red[BLOCK / 64];
  __shared__ int flag;
  const int tid = threadIdx.x, P = p.head_dim, inner = p.heads * P, gn = p.groups * p.state;
  const int channels = inner + 2 * gn;
  const int64_t stride = inner + channels + p.heads;
  if ((int)blockIdx.x >= norm_blocks) {
    const int per = (channels + BLOCK - 1) / BLOCK;
    const int i = ((int)blockIdx.x - norm_blocks) / per;
    const int ch = (((int)blockIdx.x - norm_blocks) - i * per) * BLOCK + tid;
    SsmSequence s;
    if (c.offsets) {
      s = p.sequences[i];
      if (!s.run) return;
    } else {
      if (!slots_allowed(p, c, i, &flag)) return;
      s = SsmSequence{i, 1, slot_of(c.from, i), slot_of(c.to, i), 0, 1, 0, 1};
    }
    if (s.to < 0 || ch >= channels) return;
    const int W = p.conv;
    const float* rows = c.x + (int64_t)s.begin * stride + inner;
    const float* taps = conv_taps(p, s.from);
    float v[kSsmMaxConv - 1];
#pragma unroll
    for (int k = 0; k < kSsmMaxConv - 1; ++k)
      if (k < W - 1) v[k] = raw1(rows, stride, taps, channels, W, s.length - (W - 1) + k, s.length, ch);
    float* out = p.conv_states + (int64_t)s.to * (W - 1) * channels + ch;
#pragma unroll
    for (int k = 0; k < kSsmMaxConv - 1; ++k)
      if (k < W - 1) out[(int64_t)k * channels] = v[k];
    return;
  }
  const int width = inner / p.groups;
  const int64_t item = (int64_t)blockIdx.x * (BLOCK / THREADS) + tid / THREADS;
  const int64_t t = item / p.groups;
  const int group = (int)(item - t * p.groups), l = tid % THREADS;
  // rows of refused sequences and behind the last sequence stay as they are
  bool live = t < c.tokens;
  if (c.offsets) {
    if (live) {
      int lo = 0, hi = c.sequences;  // the sequence that holds row t
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (c.offsets[mid + 1] <= t) lo = mid + 1;
        else hi = mid;
      }
      live = lo < c.sequences && c.offsets[lo] <= t && p.sequences[lo].run;
    }
  } else {
    // one token each: a row is a sequence
    live = live && slots_allowed(p, c, (int)min(t, (int64_t)c.sequences - 1), &flag);
  }
  float* y = c.y + (live ? t : 0) * inner + group * width;
  const float* z = c.x + (live ? t : 0) * stride + group * width;
  floatx4 v[kPer];
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int i = 4 * (l + THREADS * k);
    v[k] = floatx4{0.f, 0.f, 0.f, 0.f};
    if (live && i < width) {
      const floatx4 yv = *reinterpret_cast<const f32x4a4*>(y + i);
      const floatx4 zv = *reinterpret_cast<const f32x4a4*>(z + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[k][e] = yv[e] * silu_f32(zv[e]);
    }
    sum += (v[k].x * v[k].x + v[k].y * v[k].y) + (v[k].z * v[k].z + v[k].w * v[k].w);
  }
  sum = segment_sum<64>(sum);
  if constexpr (THREADS > 64) {
    if ((tid & 63) == 0) red[tid >> 6] = sum;
    __syncthreads();
    sum = 0.f;
    for (int k = 0; k < THREADS / 64; ++k) sum += red[k];
  }
  if (!live) return;
  const float scale = 1.f / sqrtf(sum / (float)width + p.epsilon);
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int i = 4 * (l + THREADS * k);
    if (i < width) {
      const floatx4 n = *reinterpret_cast<const floatx4*>(p.norm + group * width + i);
      *reinterpret_cast<f32x4a4*>(y + i) = v[k] * scale * n;
    }
  }
}

__global__ void ssm_reset_error_kernel(int* error) {
  if (threadIdx.x == 0) *error = 0;
}

// ------------------------------------------------------------------ host

int64_t ssm_max_chunks(int64_t tokens, int64_t sequences) { return tokens / kSsmChunk + sequences; }

// Workgroups that a scan should have before a sequence is cut no further.
constexpr int64_t kScanGroups = 1024;
constexpr int kMinSegment = 128;

int ssm_segment_tokens(const SsmLayerPlan& p, int64_t tokens) {
  const int64_t sets = p.heads / scan_heads(p);
  const int64_t n = (tokens * sets + kScanGroups - 1) / kScanGroups;
  return (int)std::max<int64_t>(kMinSegment, (n + kSsmChunk - 1) / kSsmChunk * kSsmChunk);
}
int64_t ssm_max_segments(const SsmLayerPlan& p, int64_t tokens, int64_t sequences) {
  // of any call of at most `tokens`: its segments hold kMinSegment tokens at
  // least, and no more than kScanGroups / sets are full ones
  return std::min<int64_t>(tokens / kMinSegment, kScanGroups / (p.heads / scan_heads(p))) + sequences;
}

int64_t ssm_max_states(const SsmLayerPlan& p, int64_t tokens) {
  // a sequence of n > 1 segments fills n - 1 >= n / 2 of them
  return 2 * (ssm_max_segments(p, tokens, 0) + 1);
}

template <typename Kernel, typename... Args>
static hipError_t launch(Kernel k, dim3 grid, dim3 block, size_t lds, hipStream_t s, Args... args) {
  if (lds > 65536) {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(k),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(k, grid, block, lds, s, args...);
  return hipGetLastError();
}

static hipError_t finish_launch(const SsmLayerPlan& p, const SsmCall& c, hipStream_t s) {
  const int inner = p.heads * p.head_dim, channels = inner + 2 * p.groups * p.state;
  const int width = inner / p.groups;
  const int64_t items = (int64_t)c.tokens * p.groups;
  auto blocks = [&](int block, int per_block) {
    const int64_t norm = (items + per_block - 1) / per_block;
    return std::pair<int, dim3>((int)norm, dim3((uint32_t)(norm + (int64_t)c.sequences * ((channels + block - 1) / block))));
  };
  if (width <= 1024 && c.offsets) {  // a row's refusal is the block's where a row is a sequence
    const auto b = blocks(256, 4);
    return launch(ssm_finish_kernel<64>, b.second, dim3(256), 0, s, p, c, b.first);
  }
  if (width <= 4096) {
    const auto b = blocks(256, 1);
    return launch(ssm_finish_kernel<256>, b.second, dim3(256), 0, s, p, c, b.first);
  }
  const auto b = blocks(1024, 1);
  return launch(ssm_finish_kernel<1024>, b.second, dim3(1024), 0, s, p, c, b.first);
}

hipError_t ssm_step_launch(const SsmLayerPlan& p, const SsmCall& c, hipStream_t s) {
  const dim3 grid(c.sequences, p.heads, (p.head_dim * p.state + kStepElements - 1) / kStepElements);
  hipError_t e;
  switch (p.state) {
    case 16: e = launch(ssm_step_kernel<16>, grid, dim3(256), 0, s, p, c); break;
    case 32: e = launch(ssm_step_kernel<32>, grid, dim3(256), 0, s, p, c); break;
    case 64: e = launch(ssm_step_kernel<64>, grid, dim3(256), 0, s, p, c); break;
    case 128: e = launch(ssm_step_kernel<128>, grid, dim3(256), 0, s, p, c); break;
    case 256: e = launch(ssm_step_kernel<256>, grid, dim3(256), 0, s, p, c); break;
    default: return hipErrorInvalidValue;
  }
  if (e != hipSuccess) return e;
  return finish_launch(p, c, s);
}

template <int NT, int W>
static hipError_t scan_launch(const SsmLayerPlan& p, const SsmCall& c, int segment_tokens,
                              int64_t max_segments, hipStream_t s) {
  constexpr int N = 16 * NT, Q = kSsmChunk;
  const int hw = scan_heads(p);
  const dim3 grid((uint32_t)(max_segments * (p.heads / hw)));
  const size_t tile = (size_t)Q * (N + 4) * sizeof(float), decays = (size_t)hw * 3 * Q * sizeof(float);
  if (c.tokens > segment_tokens) {
    hipError_t e = launch(ssm_scan_kernel<NT, W, true>, grid, dim3(64 * kScanWaves), tile + decays, s, p, c,
                          segment_tokens, hw);
    if (e != hipSuccess) return e;
    const int64_t size = (int64_t)p.heads * p.head_dim * N;
    e = launch(ssm_join_kernel, dim3(c.sequences, (uint32_t)((size / 4 + 255) / 256)), dim3(256), 0, s, p);
    if (e != hipSuccess) return e;
  }
  return launch(ssm_scan_kernel<NT, W, false>, grid, dim3(64 * kScanWaves),
                2 * tile + decays + (size_t)hw * 3 * 256 * sizeof(float), s, p, c, segment_tokens, hw);
}

template <int W>
static hipError_t run_launch(const SsmLayerPlan& p, const SsmCall& c, hipStream_t s) {
  const int segment_tokens = ssm_segment_tokens(p, c.tokens);
  const int64_t chunks = ssm_max_chunks(c.tokens, c.sequences);
  const int64_t segments = c.tokens / segment_tokens + c.sequences;
  hipError_t e = launch(ssm_plan_kernel, dim3(c.sequences), dim3(kPlanThreads), 0, s, p, c, segment_tokens);
  if (e != hipSuccess) return e;
  const int blocks = (2 * p.groups * p.state + kPrepChannels - 1) / kPrepChannels +
                     (p.heads + kPrepHeads - 1) / kPrepHeads;
  e = launch(ssm_prepare_kernel<W>, dim3((uint32_t)chunks, blocks), dim3(256), 0, s, p, c);
  if (e != hipSuccess) return e;
  switch (p.state) {
    case 16: e = scan_launch<1, W>(p, c, segment_tokens, segments, s); break;
    case 32: e = scan_launch<2, W>(p, c, segment_tokens, segments, s); break;
    case 64: e = scan_launch<4, W>(p, c, segment_tokens, segments, s); break;
    case 128: e = scan_launch<8, W>(p, c, segment_tokens, segments, s); break;
    case 256: e = scan_launch<16, W>(p, c, segment_tokens, segments, s); break;
    default: return hipErrorInvalidValue;
  }
  if (e != hipSuccess) return e;
  return finish_launch(p, c, s);
}

hipError_t ssm_run_launch(const SsmLayerPlan& p, const SsmCall& c, hipStream_t s) {
  switch (p.conv) {
    case 2: return run_launch<2>(p, c, s);
    case 3: return run_launch<3>(p, c, s);
    case 4: return run_launch<4>(p, c, s);
    default: return hipErrorInvalidValue;
  }
}

hipError_t ssm_reset_error_launch(const SsmLayerPlan& p, hipStream_t s) {
  return launch(ssm_reset_error_kernel, dim3(1), dim3(64), 0, s, p.error);
}

}  // namespace llhip
