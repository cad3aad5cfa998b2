// ssm.hip -- the Mamba-2 mixer's kernels (ssm.h).
//
// One token per sequence (ssm_step_kernel): a workgroup per sequence, head and
// 8192 or 2048 state elements reads them, applies the recurrence and writes
// them; bound by the state's traffic (48 sequences of 2 MiB: 44 us, 4.6 TB/s).
// ssm_finish_kernel then gates and norms the rows and shifts the convolution's
// state (8192 rows of 4096: 68 us, 5.9 TB/s).
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
// The products are of single precision on the matrix cores' 16-bit operands:
// C s and the state's, which need only scales that run along a row or column
// of the product, as two f16 parts and three products; (S o L) X, whose S o L
// has no such scale at hand, as three bf16 parts and six.  (All in bf16 parts
// 8192 tokens of 64 heads took 170 us for the scan and 77 for its first pass;
// so 142 and 67.  fp32 matrix instructions have an eighth of the rate.)
// Bound by latency: a chunk of 256 channels takes a workgroup 8.5 us, of which
// the matrix cores work 1.6, the vector units about 2 and the LDS about 1.2;
// its LDS (124 KB) and registers (238 of 256) leave no room for a second
// workgroup.  Half as many channels leave it, but two of those took longer:
// when the scan was at 154 us, 187 in the 128 registers of two workgroups (with
// 80 bytes of scratch) and 171 without that limit.
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
  // (the reciprocal is good to one unit); large negative v: exp overflows, the
  // reciprocal is 0 and the result -0, as the limit is
  return v * __builtin_amdgcn_rcpf(1.f + exp_f32(-v));
}
// The same without that correction, for the convolution's outputs: the product
// v log2 e rounds, so the result is off by about (|v| + 5) 2^-24 of it, which is
// below the rounding of the sum that v is unless v is large, and tiny then.
__device__ __forceinline__ float silu_conv(float v) {
  return v * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v * -kLog2e));
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
__device__ __forceinline__ bool slots_in_pool(const SsmLayerPlan& p, int from, int to) {
  return !(from < -1 || from >= p.slots || to < -1 || to >= p.slots);
}
__device__ bool slots_allowed(const SsmLayerPlan& p, const SsmCall& c, int i, int* flag) {
  const int from = slot_of(c.from, i), to = slot_of(c.to, i);
  int bad = slots_in_pool(p, from, to) ? 0 : kSsmErrSlot;
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

// x = hi + mid + lo in bf16, 24 significant bits and single precision's whole
// range, so products need no scales: |x - hi - mid - lo| <= 2^-25 |x|.  Eight
// values, packed as a matrix operand's lane holds them.
struct Split8 {
  u32x4 hi, mid, lo;
};
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(floatx2{a, b}, bf16x2));
}
__device__ __forceinline__ void split_pair(float a, float b, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
  hi = bf16_pair(a, b);
  a -= __builtin_bit_cast(float, hi << 16);
  b -= __builtin_bit_cast(float, hi & 0xFFFF0000u);
  mid = bf16_pair(a, b);
  a -= __builtin_bit_cast(float, mid << 16);
  b -= __builtin_bit_cast(float, mid & 0xFFFF0000u);
  lo = bf16_pair(a, b);
}
__device__ __forceinline__ Split8 split8(const float* v) {
  Split8 r;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t h, m, l;
    split_pair(v[2 * e], v[2 * e + 1], h, m, l);
    r.hi[e] = h;
    r.mid[e] = m;
    r.lo[e] = l;
  }
  return r;
}

// v s = hi + lo in f16 for values whose largest is brought to [2^14, 2^15) by
// the power of two s: 22 significant bits, or 2^-40 of the largest, whichever is
// more.  Three products (of 2^-22 of the whole the fourth) where the three bf16
// parts take six: the operands that are scaled in common by a row or column of
// a product, whose result takes the scale back, are held so.
struct Split2 {
  u32x4 hi, lo;
};
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ Split2 split_f16(const float* v) {
  Split2 r;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const f16x2 h = __builtin_convertvector(floatx2{v[2 * e], v[2 * e + 1]}, f16x2);
    const f16x2 l = __builtin_convertvector(floatx2{v[2 * e] - (float)h.x, v[2 * e + 1] - (float)h.y}, f16x2);
    r.hi[e] = __builtin_bit_cast(uint32_t, h);
    r.lo[e] = __builtin_bit_cast(uint32_t, l);
  }
  return r;
}
// The scale as a float's bits, at most 2^100, for values of at most |m| (its sign
// bit clear), and a power of two's reciprocal.
__device__ __forceinline__ int scale_bits(float m) {
  return (227 << 23) - max((__builtin_bit_cast(int, m) & 0x7F800000) - (41 << 23), 0);
}
__device__ __forceinline__ float power(int bits) { return __builtin_bit_cast(float, bits); }
constexpr int k2p14 = 14 << 23;  // to add to or take from such bits
__device__ __forceinline__ int reciprocal_bits(int bits) { return (254 << 23) - bits; }

// What a chunk's scan reads of its group, in operand order: fragments of 64
// lanes x 16 bytes, lane (r, g) = (lane & 15, lane >> 4).
//   C   [i tile][n block of 32][hi, lo]: token 16 it + r; element e is
//       n = 32 t + 16 (e / 4) + 4 g + e % 4, the elements of the state's result
//       tiles that the same lane holds (zeros past n)
//   B^T [n tile][hi, lo]: row n = 16 nt + r; element e is token
//       16 (e / 4) + 4 g + e % 4
//   (both f16, scaled per token: 2^14 over the scales lies in p.scales)
//   S^T [(j, i) tiles (0, 0), (0, 1), (1, 1)], fp32: rows j = 16 jt + 4 g ..
//       + 3, column i = 16 it + r
constexpr int kFragment = 1024;
constexpr int n_blocks(int nt) { return (nt + 1) / 2; }
constexpr int c_fragments(int nt) { return 4 * n_blocks(nt); }
constexpr int b_fragments(int nt) { return 2 * nt; }
constexpr int image_fragments(int nt) { return c_fragments(nt) + b_fragments(nt) + 3; }

size_t ssm_image_bytes(int state) { return (size_t)image_fragments(state / 16) * kFragment; }

// Block (chunk, y): y < groups: that group's B and C after the convolution (a
// thread takes four channels of eight tokens), as the images above; then
// blocks of eight heads: dt and the decays, a lane per token.
constexpr int kPrepHeads = 8;

template <int NT, int W>
__global__ void __launch_bounds__(256) ssm_prepare_kernel(SsmLayerPlan p, SsmCall c) {
  constexpr int N = 16 * NT, Q = kSsmChunk, LD = N + 4, NB = n_blocks(NT);
  __shared__ float sbc[2][Q * LD], scale[2][Q];
  const int chunk = blockIdx.x;
  if (chunk >= p.counts[1]) return;
  const int2 at = p.chunks[chunk];
  const SsmSequence s = p.sequences[at.x];
  if (!s.run) return;
  const int inner = p.heads * p.head_dim, gn = p.groups * N, channels = inner + 2 * gn;
  const int64_t stride = inner + channels + p.heads;
  const float* rows = c.x + (int64_t)s.begin * stride + inner;
  const int tid = threadIdx.x, t0 = at.y * Q;
  if ((int)blockIdx.y < p.groups) {
    const int group = blockIdx.y;
    const float* taps = conv_taps(p, s.from);
    for (int item = tid; item < 2 * N; item += 256) {
      const int quad = item % (N / 2), q0 = 8 * (item / (N / 2));
      const int which = quad >= N / 4, n = 4 * (quad - which * (N / 4));
      const int ch = inner + which * gn + group * N + n;
      floatx4 w[W], r[8 + W - 1];
#pragma unroll
      for (int k = 0; k < 8 + W - 1; ++k)
        r[k] = raw4(rows, stride, taps, channels, W, t0 + q0 - (W - 1) + k, s.length, ch);
#pragma unroll
      for (int k = 0; k < W; ++k)
        w[k] = *reinterpret_cast<const floatx4*>(p.conv_weight + (int64_t)k * channels + ch);
      const floatx4 b = *reinterpret_cast<const floatx4*>(p.conv_bias + ch);
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        floatx4 v = b;
#pragma unroll
        for (int k = 0; k < W; ++k) v += w[k] * r[q + k];
        floatx4 u;
#pragma unroll
        for (int e = 0; e < 4; ++e) u[e] = t0 + q0 + q < s.length ? silu_conv(v[e]) : 0.f;
        *reinterpret_cast<floatx4*>(&sbc[which][(q0 + q) * LD + n]) = u;
      }
    }
    __syncthreads();
    {
      // a token's scale: four threads take its B and C (what is not finite has none to give)
      const int which = tid >> 7, q = (tid >> 2) & 31, part = tid & 3;
      float m = 0.f;
      for (int n = 4 * part; n < N; n += 16) {
        const floatx4 v = *reinterpret_cast<const floatx4*>(&sbc[which][q * LD + n]);
#pragma unroll
        for (int e = 0; e < 4; ++e) m = fmaxf(m, fabsf(v[e]) <= FLT_MAX ? fabsf(v[e]) : 0.f);
      }
      m = fmaxf(m, dpp<kDppXor1>(m));
      m = fmaxf(m, dpp<kDppXor2>(m));
      if (part == 0) {
        const int bits = scale_bits(m);
        scale[which][q] = power(bits);
        p.scales[((int64_t)chunk * p.groups + group) * 2 * Q + which * Q + q] = power(reciprocal_bits(bits) + k2p14);
      }
    }
    __syncthreads();
    const int lane = tid & 63, wave = tid >> 6, col = lane & 15, g = lane >> 4;
    uint8_t* image = p.images + ((int64_t)chunk * p.groups + group) * image_fragments(NT) * kFragment;
    if (wave < 3) {
      const int jt = wave == 2, it = wave > 0;
      floatx4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const floatx4 a = *reinterpret_cast<const floatx4*>(&sbc[0][(16 * jt + col) * LD + 16 * n + 4 * g]);
        const floatx4 b = *reinterpret_cast<const floatx4*>(&sbc[1][(16 * it + col) * LD + 16 * n + 4 * g]);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc = mfma4f32(a[e], b[e], acc);
      }
      *reinterpret_cast<floatx4*>(image + (c_fragments(NT) + b_fragments(NT) + wave) * kFragment + 16 * lane) = acc;
    }
    for (int f = wave; f < 2 * NB + NT; f += 4) {
      float v[8];
      int first;
      if (f < 2 * NB) {
        const int it = f / NB, t = f - it * NB;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          floatx4 q{0.f, 0.f, 0.f, 0.f};
          if (2 * t + half < NT)
            q = *reinterpret_cast<const floatx4*>(&sbc[1][(16 * it + col) * LD + 32 * t + 16 * half + 4 * g]);
          const float by = scale[1][16 * it + col];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[4 * half + e] = q[e] * by;
        }
        first = 2 * f;
      } else {
        const int nt = f - 2 * NB;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int q = 16 * (e >> 2) + 4 * g + (e & 3);
          v[e] = sbc[0][q * LD + 16 * nt + col] * scale[0][q];
        }
        first = c_fragments(NT) + 2 * nt;
      }
      const Split2 r = split_f16(v);
      u32x4* out = reinterpret_cast<u32x4*>(image + first * kFragment) + lane;
      out[0] = r.hi;
      out[kFragment / 16] = r.lo;
    }
    return;
  }
  const int h = ((int)blockIdx.y - p.groups) * kPrepHeads + (tid >> 5), q = tid & 31;
  if (h >= p.heads) return;
  const bool in = t0 + q < s.length;
  const float dt = in ? softplus_f32(rows[(int64_t)(t0 + q) * stride + channels + h] + p.dt_bias[h]) : 0.f;
  double sum = in ? log2_decay(dt, p.a[h]) : 0.0;
  for (int o = 1; o < Q; o <<= 1) {
    const double v = __shfl_up(sum, o, 32);
    if (q >= o) sum += v;
  }
  float* out = p.decay + ((int64_t)chunk * p.heads + h) * 3 * Q + q;
  const float hi = (float)sum;
  out[0] = dt;
  out[Q] = hi;
  out[2 * Q] = (float)(sum - (double)hi);
}

// ------------------------------------------------------------------ the scan

// acc += A B over 32 K elements to single precision: the six products of
// parts above 2^-24 of the whole.  A lane's element e of both operands is the
// same K element.
__device__ __forceinline__ floatx4 mma_one(const u32x4& a, const u32x4& b, const floatx4& c) {
  return mfma32(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c);
}

__device__ __forceinline__ floatx4 mma_f16(const u32x4& a, const u32x4& b, const floatx4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// The maximum over the four lanes that hold one column (row swaps as in
// row_pair_sum).
__device__ __forceinline__ float column_max(float v) {
  float a = v, b = v;
  asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
  a = b = fmaxf(a, b);
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
  return fmaxf(a, b);
}

// Wait for every load, in a form that the compiler counts too (it would wait
// again for the registers, behind the loads that follow).
__device__ __forceinline__ void wait_all_loads() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  asm volatile("" ::: "memory");
}

constexpr int kScanWaves = 8;

// Column tiles of 16 channels per wavefront at most (the state of one takes
// N / 4 registers) and heads per workgroup at most (their masked products take
// 12 KB of LDS each).
constexpr int scan_max_tiles(int nt) { return nt > 8 ? 1 : 2; }
constexpr int scan_max_heads(int nt) { return nt > 8 ? 2 : 4; }

// Heads per workgroup: as many whole heads of one group as fit its tiles.
static int scan_heads(const SsmLayerPlan& p, int tiles) {
  const int share = p.heads / p.groups;
  int n = std::min(scan_max_heads(p.state / 16), std::max(1, kScanWaves * tiles * 16 / p.head_dim));
  while (share % n) --n;
  return n;
}

// LDS of a scan workgroup, in bytes: B, raw rows, decays and scales (two of each in the first
// pass), C, S, decays, masked products (two), decay tables (two).
template <int NT, int W, bool STATES>
struct ScanLds {
  static constexpr int buffers = STATES ? 2 : 1;  // of B, the rows and the decays
  static constexpr int b = b_fragments(NT) * kFragment;
  static constexpr int c = STATES ? 0 : c_fragments(NT) * kFragment;
  static constexpr int s = STATES ? 0 : 3 * kFragment;
  static constexpr int decays = 3 * kSsmChunk * 4;             // per head
  static constexpr int products = STATES ? 0 : 6 * kFragment;  // per head: [i tile][hi, mid, lo]
  static constexpr int tables = (2 * kSsmChunk + 4) * 4;       // per head: [e, w], the chunk's whole decay
  static constexpr int scales = 2 * kSsmChunk * 4;             // B's, C's
  // raw rows of the workgroup's channels.  The pitch puts the rows 4 apart
  // that a wavefront reads together 16 banks apart.
  static constexpr int rows = kSsmChunk + W - 1;
  __host__ __device__ static constexpr int pitch(int width) { return 4 * (width + 4); }
  static constexpr int at_c = buffers * b, at_s = at_c + c, at_decays = at_s + s;
  __host__ __device__ static constexpr int at_scales(int hw) { return at_decays + buffers * hw * decays; }
  __host__ __device__ static constexpr int at_products(int hw) { return at_scales(hw) + buffers * scales; }
  __host__ __device__ static constexpr int at_tables(int hw) { return at_products(hw) + 2 * hw * products; }
  __host__ __device__ static constexpr int at_rows(int hw) { return at_tables(hw) + 2 * hw * tables; }
  __host__ __device__ static constexpr int bytes(int hw, int width) {
    return at_rows(hw) + buffers * rows * pitch(width);
  }
};

// A 4 x 4 transpose over each four neighbouring lanes: lane q's v[e] becomes
// lane e's v[q].
__device__ __forceinline__ void transpose_quads(floatx4& v, bool odd, bool high) {
  // (every lane takes part in each exchange, so they stand outside the selects)
  const float x1 = dpp<kDppXor1>(v.x), y1 = dpp<kDppXor1>(v.y), z1 = dpp<kDppXor1>(v.z), w1 = dpp<kDppXor1>(v.w);
  const float a = odd ? y1 : v.x, b = odd ? v.y : x1, c = odd ? w1 : v.z, d = odd ? v.w : z1;
  const float a2 = dpp<kDppXor2>(a), b2 = dpp<kDppXor2>(b), c2 = dpp<kDppXor2>(c), d2 = dpp<kDppXor2>(d);
  v.x = high ? c2 : a;
  v.z = high ? c : a2;
  v.y = high ? d2 : b;
  v.w = high ? d : b2;
}

// One segment of `hw` heads.  STATES: only the segment's own state, from
// zeros, to the next segment's place; else outputs and, in a sequence's last
// segment, the state to its slot.
//
// A wavefront owns column tiles (16 channels of a head): their part of the
// state, x, and outputs.  Per chunk each forms its tiles' outputs, then their
// state; beside the state's products, which leave the vector unit idle, the
// wavefronts convolve x of the next chunk and share the work of its masked
// products M = S o L (six half tiles a head) and decay tables.  Images and raw
// rows come into LDS by loads that need no registers, each requested a phase
// or more ahead: a load of one dword per lane costs the memory pipeline as
// much as one of sixteen bytes, and reading x that way took it 5000 cycles of
// a chunk's 17000.
template <int NT, int W, int TPW, bool STATES>
__global__ void __launch_bounds__(64 * kScanWaves) ssm_scan_kernel(SsmLayerPlan p, SsmCall c,
                                                                   int segment_tokens, int hw) {
  using Lds = ScanLds<NT, W, STATES>;
  constexpr int N = 16 * NT, Q = kSsmChunk, NB = n_blocks(NT);
  constexpr int kC = c_fragments(NT), kB = b_fragments(NT), kImage = image_fragments(NT) * kFragment;
  extern __shared__ __align__(16) uint8_t lds[];
  const int width = hw * p.head_dim, pitch = Lds::pitch(width);
  const int sets = p.heads / hw;
  // groups vary fastest, so that the workgroups that read one group's images
  // sit on one XCD where there are eight groups
  const int set_in_group = sets / p.groups;
  const int seg = blockIdx.x / sets, rest = blockIdx.x - seg * sets;
  if (seg >= p.counts[0]) return;
  const int2 at = p.segments[seg];
  const SsmSequence s = p.sequences[at.x];
  if (!s.run) return;
  if (STATES && at.y == s.segments - 1) return;  // no segment follows
  const int group = rest % p.groups, h0 = (group * set_in_group + rest / p.groups) * hw;
  const int inner = p.heads * p.head_dim, channels = inner + 2 * p.groups * N;
  const int64_t stride = inner + channels + p.heads;
  const float* rows = c.x + (int64_t)s.begin * stride + inner + h0 * p.head_dim;
  const float* taps = conv_taps(p, s.from);
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int t_begin = at.y * segment_tokens, t_end = min(s.length, t_begin + segment_tokens);

  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_address(lds));
  // `n` fragments of a chunk's image from `first` on, to LDS at `to`
  auto request_image = [&](int t, int first, int n, int to) {
    const uint8_t* img = uniform_ptr(p.images + ((int64_t)(s.chunk0 + t / Q) * p.groups + group) * kImage +
                                     first * kFragment);
    const uint32_t off = wave * kFragment + 16 * lane;
#pragma unroll
    for (int f = 0; f < n; f += kScanWaves)
      if (f + wave < n) load_lds16(img, off + f * kFragment, lds0 + to + (f + wave) * kFragment);
  };
  auto request_decays = [&](int t, int buf) {
    const uint8_t* dec = uniform_ptr(reinterpret_cast<const uint8_t*>(
        p.decay + ((int64_t)(s.chunk0 + t / Q) * p.heads + h0) * 3 * Q));
    // the last two wavefronts, which have the fewest fragments
    const int first = (kScanWaves - 1 - wave) * kFragment;
    if (first + 16 * lane < hw * Lds::decays)
      load_lds16(dec, first + 16 * lane, lds0 + Lds::at_decays + buf * hw * Lds::decays + first);
    // and the group's scales
    if (wave == kScanWaves - 3 && 16 * lane < Lds::scales)
      load_lds16(uniform_ptr(reinterpret_cast<const uint8_t*>(
                     p.scales + ((int64_t)(s.chunk0 + t / Q) * p.groups + group) * 2 * Q)),
                 16 * lane, lds0 + Lds::at_scales(hw) + buf * Lds::scales);
  };
  // the raw rows that a chunk's convolution reads: before the sequence those
  // it started with (zeros for a new one), past its end the last row again
  // (their outputs are not stored, and the state takes zeros for them)
  auto request_rows = [&](int t0, int buf) {
    const uint32_t to = lds0 + Lds::at_rows(hw) + buf * Lds::rows * pitch;
    if (4 * lane >= width) return;
    if (t0 >= W - 1 && t0 + Q <= t_end) {
      const float* src = rows + (int64_t)(t0 - (W - 1) + wave) * stride;
#pragma unroll
      for (int r = 0; r < Lds::rows; r += kScanWaves, src += kScanWaves * stride)
        if (r + wave < Lds::rows)
          load_lds16(uniform_ptr(reinterpret_cast<const uint8_t*>(src)), 16 * lane, to + (r + wave) * pitch);
    } else {
      for (int r = wave; r < Lds::rows; r += kScanWaves) {
        const int t = t0 - (W - 1) + r;
        const float* src = t >= 0 ? rows + (int64_t)min(t, t_end - 1) * stride
                                  : taps ? taps + (int64_t)(W - 1 + t) * channels + h0 * p.head_dim : nullptr;
        if (src)
          load_lds16(uniform_ptr(reinterpret_cast<const uint8_t*>(src)), 16 * lane, to + r * pitch);
        else
          *reinterpret_cast<floatx4*>(lds + Lds::at_rows(hw) + (buf * Lds::rows + r) * pitch + 16 * lane) =
              floatx4{0.f, 0.f, 0.f, 0.f};
      }
    }
  };
  if (t_begin < t_end) {
    // all that the first chunk needs, and what its state phase reads of the second
    request_rows(t_begin, 0);
    request_decays(t_begin, 0);
    if (STATES) {
      request_image(t_begin, kC, kB, 0);
    } else {
      request_image(t_begin, kC + kB, 3, Lds::at_s);
      request_image(t_begin, 0, kC, Lds::at_c);
    }
  }

  // this wave's column tiles: channels [p0, p0 + 16) of a head
  const int per_head = p.head_dim / 16, tiles = hw * per_head;
  bool on[TPW];
  int head[TPW], ch[TPW];  // ch: within the workgroup's channels
  float skip[TPW], w[TPW][W], bias[TPW];
  floatx4 st[TPW][2 * NB];
#pragma unroll
  for (int k = 0; k < TPW; ++k) {
    const int tile = wave + kScanWaves * k;
    on[k] = tile < tiles;
    head[k] = on[k] ? tile / per_head : 0;
    ch[k] = (on[k] ? tile * 16 : 0) + col;
    const int at_ch = h0 * p.head_dim + ch[k];
    skip[k] = p.d[h0 + head[k]];
    bias[k] = p.conv_bias[at_ch];
#pragma unroll
    for (int j = 0; j < W; ++j) w[k][j] = p.conv_weight[(int64_t)j * channels + at_ch];
    const float* src = nullptr;
    if (!STATES) {
      if (s.segments > 1) src = p.seg_states + (int64_t)(s.state0 + at.y) * inner * N;
      else if (s.from >= 0) src = p.ssm_states + (int64_t)s.from * inner * N;
    }
#pragma unroll
    for (int n = 0; n < 2 * NB; ++n)
      st[k][n] = src && on[k] && n < NT ? *reinterpret_cast<const floatx4*>(src + (int64_t)at_ch * N + 16 * n + 4 * g)
                                        : floatx4{0.f, 0.f, 0.f, 0.f};
  }
  double total[TPW] = {};
  // The state is held times a power of two per column, which changes with the
  // inputs (below); `most` bounds it there.
  int held[TPW];
  float most[TPW];
  auto state_max = [&](int k) {
    float m = 0.f;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) m = fmaxf(m, fabsf(st[k][n][e]));
    return column_max(m);
  };
#pragma unroll
  for (int k = 0; k < TPW; ++k) {
    held[k] = 227 << 23;  // (of zeros)
    most[k] = 0.f;
    if (!STATES) {
      held[k] = max(scale_bits(state_max(k)), (1 << 23) + k2p14);
#pragma unroll
      for (int n = 0; n < NT; ++n) st[k][n] *= power(held[k]);
    }
  }

  // x of the lane's tokens 4 g .. + 3 and 16 + 4 g .. + 3 after the convolution
  float x[TPW][8];
  // (half a tile's at a time: its reads, and what is made of them)
  float raw[4 + W - 1];
  auto convolve_read = [&](int buf, int k, int half) {
    const uint8_t* from = lds + Lds::at_rows(hw) + buf * Lds::rows * pitch + (4 * g + 16 * half) * pitch + 4 * ch[k];
#pragma unroll
    for (int j = 0; j < 4 + W - 1; ++j) raw[j] = *reinterpret_cast<const float*>(from + j * pitch);
  };
  auto convolve = [&](int k, int half) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float v = bias[k];
#pragma unroll
      for (int j = 0; j < W; ++j) v = fmaf(w[k][j], raw[e + j], v);
      v = silu_conv(v);
      asm("" : "+v"(v));  // one by one: as a vector the taps would be held eight times each
      x[k][4 * half + e] = v;
    }
  };
  auto decays_at = [&](int buf) { return reinterpret_cast<const float*>(lds + Lds::at_decays + buf * hw * Lds::decays); };
  auto tables_at = [&](int buf) { return reinterpret_cast<float*>(lds + Lds::at_tables(hw) + buf * hw * Lds::tables); };
  // decays from the chunk's start (e) and to its end, with dt (w), and C's and
  // B's scales taken back; the same
  // values from as many threads as there are
  auto make_tables = [&](int from, int to) {
    const int h = (tid / Q) % hw, q = tid % Q;
    const float* d = decays_at(from) + h * 3 * Q;
    const float* scale = reinterpret_cast<const float*>(lds + Lds::at_scales(hw) + from * Lds::scales);
    float* t = tables_at(to) + h * (Lds::tables / 4) + q;
    const float e = __builtin_amdgcn_exp2f(d[Q + q] + d[2 * Q + q]);
    t[0] = e * scale[Q + q];
    t[Q] = d[q] * __builtin_amdgcn_exp2f((d[2 * Q - 1] - d[Q + q]) + (d[3 * Q - 1] - d[2 * Q + q])) * scale[q];
    if (q == Q - 1) t[Q + 1] = e;
  };
  // M = S o L of the workgroup's heads, as left operands: job (head, tile,
  // half), a lane's two neighbouring j of column i.  (Past the last job that
  // one again.)
  constexpr int kJobs = STATES ? 0 : (6 * scan_max_heads(NT) + kScanWaves - 1) / kScanWaves;
  auto make_products = [&](int n, int to) {
    const float* dec = decays_at(0);
    if (n * kScanWaves < 6 * hw) {
      const int job = min(n * kScanWaves + wave, 6 * hw - 1);
      const int h = job / 6, tile = job % 6 / 2, half = job % 2, jt = tile == 2, it = tile > 0;
      const floatx2 sv = *reinterpret_cast<const floatx2*>(lds + Lds::at_s + tile * kFragment + 16 * lane + 8 * half);
      const int i = 16 * it + col, j0 = 16 * jt + 4 * g + 2 * half;
      const float* d = dec + h * 3 * Q;
      const float ihi = d[Q + i], ilo = d[2 * Q + i];
      const floatx2 dt = *reinterpret_cast<const floatx2*>(d + j0);
      const floatx2 jhi = *reinterpret_cast<const floatx2*>(d + Q + j0);
      const floatx2 jlo = *reinterpret_cast<const floatx2*>(d + 2 * Q + j0);
      float m[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        // (masked exponents may be large: the product is not used)
        const float v = sv[e] * (__builtin_amdgcn_exp2f((ihi - jhi[e]) + (ilo - jlo[e])) * dt[e]);
        m[e] = j0 + e <= i ? v : 0.f;
      }
      uint32_t hi, mid, lo;
      split_pair(m[0], m[1], hi, mid, lo);
      uint32_t* out = reinterpret_cast<uint32_t*>(lds + Lds::at_products(hw) + (to * hw + h) * Lds::products +
                                                  it * 3 * kFragment + 16 * lane + 8 * jt + 4 * half);
      out[0] = hi;
      out[kFragment / 4] = mid;
      out[2 * kFragment / 4] = lo;
    }
  };

  // the first pass: log2 of the decay over the chunks so far (in 64 bits: a segment may have hundreds,
  // and sums of single precision would round at each)
  auto add_total = [&](int from) {
#pragma unroll
    for (int k = 0; k < TPW; ++k) {
      const float* d = decays_at(from) + head[k] * 3 * Q;
      total[k] += (double)d[2 * Q - 1] + (double)d[3 * Q - 1];
    }
  };

  if constexpr (!STATES) {
    // M's upper right quarter is zero throughout
    for (int i = tid; i < 2 * hw * 3 * 64; i += 64 * kScanWaves)
      *reinterpret_cast<u32x2*>(lds + Lds::at_products(hw) + i / 192 * Lds::products + i % 192 * 16 + 8) = u32x2{0u, 0u};
  }
  if (t_begin < t_end) {
    wait_all_loads();
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2 * TPW; ++k) {
      convolve_read(0, k >> 1, k & 1);
      convolve(k >> 1, k & 1);
    }
    make_tables(0, 0);
#pragma unroll
    for (int n = 0; n < kJobs; ++n) make_products(n, 0);
    if (STATES) add_total(0);
    if (STATES && t_begin + Q < t_end) {
      request_rows(t_begin + Q, 1);
      request_decays(t_begin + Q, 1);
    }
  }
  int buf = 0;  // of the chunk's tables and masked products; in the first pass of B, rows and decays too
  for (int t0 = t_begin; t0 < t_end; t0 += Q, buf ^= 1) {
    const int next = t0 + Q;
    wait_all_loads();
    // the chunk's images, products and tables are there (in the first pass
    // also the next one's rows and decays); what the last chunk read is free
    __syncthreads();
    const float* tables = tables_at(buf);
    if constexpr (STATES) {
      if (next < t_end) request_image(next, kC, kB, (buf ^ 1) * Lds::b);
      if (next + Q < t_end) {
        request_rows(next + Q, buf);
        request_decays(next + Q, buf);
      }
    } else {
      floatx4 acc[2][TPW];
#pragma unroll
      for (int it = 0; it < 2; ++it)
#pragma unroll
        for (int k = 0; k < TPW; ++k) acc[it][k] = floatx4{0.f, 0.f, 0.f, 0.f};
      int by[TPW];  // the state's scale as an operand, beyond the held one
#pragma unroll
      for (int k = 0; k < TPW; ++k) {
        most[k] = state_max(k);
        by[k] = scale_bits(most[k]);
      }
      // the next block's fragments are read ahead, and no further ahead: read
      // where the compiler likes they crowd the state out of the registers
      auto c_at = [&](int t, int it, int part) {
        return *reinterpret_cast<const u32x4*>(lds + Lds::at_c + ((it * NB + t) * 2 + part) * kFragment + 16 * lane);
      };
      u32x4 a[2][2], ahead[2][2];
#pragma unroll
      for (int part = 0; part < 4; ++part) ahead[part / 2][part % 2] = c_at(0, part / 2, part % 2);
#pragma unroll
      for (int t = 0; t < NB; ++t) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int part = 0; part < 4; ++part) {
          a[part / 2][part % 2] = ahead[part / 2][part % 2];
          if (t + 1 < NB) ahead[part / 2][part % 2] = c_at(t + 1, part / 2, part % 2);
        }
        Split2 sp[TPW];
#pragma unroll
        for (int k = 0; k < TPW; ++k) {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = st[k][2 * t + (e >> 2)][e & 3] * power(by[k]);
          sp[k] = split_f16(v);
        }
        // neighbouring products belong to different accumulators
#define LLHIP_SSM_PRODUCT(MMA, A, B)                                       \
  _Pragma("unroll") for (int it = 0; it < 2; ++it)                         \
      _Pragma("unroll") for (int k = 0; k < TPW; ++k)                      \
          acc[it][k] = MMA(A, B, acc[it][k]);
        LLHIP_SSM_PRODUCT(mma_f16, a[it][0], sp[k].lo)
        LLHIP_SSM_PRODUCT(mma_f16, a[it][1], sp[k].hi)
        LLHIP_SSM_PRODUCT(mma_f16, a[it][0], sp[k].hi)
        // loads for the state phase: in parts, for a wavefront waits where
        // the memory pipeline is busy with the others'
        if (t == 0) request_image(t0, kC, kB, 0);
        if (t == std::min(1, NB - 1) && next < t_end) request_rows(next, 0);
        if (t == std::min(2, NB - 1) && next < t_end) {
          request_decays(next, 0);
          request_image(next, kC + kB, 3, Lds::at_s);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      // A non-finite x_j would reach the tokens before it, as 0 x_j in the
      // masked part of the product: the products take zero in its place, and
      // the channel's outputs from token j on are NaN (its state too, by x
      // itself).
      float xf[TPW][8], largest = 0.f;
      int first_bad[TPW];
#pragma unroll
      for (int k = 0; k < TPW; ++k) {
        first_bad[k] = Q;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          xf[k][e] = x[k][e];
          largest = __builtin_elementwise_maximum(largest, fabsf(x[k][e]));  // NaN if one is
        }
      }
      const bool all_finite = !__ballot(!(largest <= FLT_MAX));
      if (!all_finite) {
#pragma unroll
        for (int k = 0; k < TPW; ++k) {
#pragma unroll
          for (int e = 7; e >= 0; --e)
            if (!(fabsf(x[k][e]) <= FLT_MAX)) {
              first_bad[k] = 16 * (e >> 2) + 4 * g + (e & 3);
              xf[k][e] = 0.f;
            }
          first_bad[k] = min(first_bad[k], __shfl_xor(first_bad[k], 16, 64));
          first_bad[k] = min(first_bad[k], __shfl_xor(first_bad[k], 32, 64));
        }
      }
      Split8 xs[TPW];
      u32x4 m[2][TPW][3];
#pragma unroll
      for (int k = 0; k < TPW; ++k) {
        xs[k] = split8(xf[k]);
        // (one by one, so that none of them leaves single precision's range)
        const float back = power(reciprocal_bits(by[k]) - k2p14), own = power(reciprocal_bits(held[k]));
        const uint8_t* from = lds + Lds::at_products(hw) + (buf * hw + head[k]) * Lds::products + 16 * lane;
#pragma unroll
        for (int it = 0; it < 2; ++it) {
          acc[it][k] = acc[it][k] * back * own *
                       *reinterpret_cast<const floatx4*>(tables + head[k] * (Lds::tables / 4) + 16 * it + 4 * g);
#pragma unroll
          for (int part = 0; part < 3; ++part)
            m[it][k][part] = *reinterpret_cast<const u32x4*>(from + (it * 3 + part) * kFragment);
        }
      }
      LLHIP_SSM_PRODUCT(mma_one, m[it][k][2], xs[k].hi)
      LLHIP_SSM_PRODUCT(mma_one, m[it][k][0], xs[k].lo)
      LLHIP_SSM_PRODUCT(mma_one, m[it][k][1], xs[k].mid)
      LLHIP_SSM_PRODUCT(mma_one, m[it][k][1], xs[k].hi)
      LLHIP_SSM_PRODUCT(mma_one, m[it][k][0], xs[k].mid)
      LLHIP_SSM_PRODUCT(mma_one, m[it][k][0], xs[k].hi)
#undef LLHIP_SSM_PRODUCT
      // the lane's four tokens of a channel become four channels of a token
      const bool odd = lane & 1, high = lane & 2;
#pragma unroll
      for (int it = 0; it < 2; ++it)
#pragma unroll
        for (int k = 0; k < TPW; ++k) {
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[it][k][e] = fmaf(skip[k], xf[k][4 * it + e], acc[it][k][e]);
          if (!all_finite)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (16 * it + 4 * g + e >= first_bad[k]) acc[it][k][e] = __builtin_nanf("");
          transpose_quads(acc[it][k], odd, high);
        }
      wait_all_loads();  // B, the rows and S, requested a phase ago (and not the stores that follow)
#pragma unroll
      for (int it = 0; it < 2; ++it) {
        const int t = t0 + 16 * it + 4 * g + (lane & 3);
        float* out = c.y + (int64_t)(s.begin + t) * inner + h0 * p.head_dim + 4 * (col >> 2) - col;
#pragma unroll
        for (int k = 0; k < TPW; ++k)
          if (on[k] && t < t_end) *reinterpret_cast<f32x4a4*>(out + ch[k]) = acc[it][k];
      }
      __syncthreads();  // B and what the next chunk needs have come; C is free
    }
    // Past the sequence's end x is of repeated rows, whose sum of taps may be
    // infinite where no token's is: times a step of zero it would be NaN.
    if (!STATES && next > t_end) {  // (segments that another follows end with a chunk)
#pragma unroll
      for (int k = 0; k < TPW; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[k][e] = t0 + 16 * (e >> 2) + 4 * g + (e & 3) < t_end ? x[k][e] : 0.f;
    }
    // The state: decayed, plus the tokens' products.  These inputs' scale
    // becomes the one that the state is held times, unless that brought it
    // near the end of single precision (inputs of next to nothing: they keep
    // the digits that matter beside it).
    Split2 xs[TPW];
#pragma unroll
    for (int k = 0; k < TPW; ++k) {
      const float* tab = tables + head[k] * (Lds::tables / 4);
      const floatx4 w0 = *reinterpret_cast<const floatx4*>(tab + Q + 4 * g);
      const floatx4 w1 = *reinterpret_cast<const floatx4*>(tab + Q + 16 + 4 * g);
      float v[8], m = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = x[k][e] * (e < 4 ? w0[e & 3] : w1[e & 3]);
        m = fmaxf(m, fabsf(v[e]));
      }
      const int room = (100 << 23) - max((__builtin_bit_cast(int, most[k]) & 0x7F800000) - (127 << 23), 0);
      const int now = max(held[k] + min(scale_bits(column_max(m)) + k2p14 - held[k], room), (1 << 23) + k2p14);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= power(now - k2p14);
      xs[k] = split_f16(v);
      const float e = tab[2 * Q] * (power(now) * power(reciprocal_bits(held[k])));
      held[k] = now;
      // (32 products of two operands below 2^15)
      if (STATES) most[k] = fmaf(most[k], e, 0x1p35f);
#pragma unroll
      for (int n = 0; n < NT; ++n) st[k][n] *= e;
    }
    auto b_at = [&](int n, int part) {
      return *reinterpret_cast<const u32x4*>(lds + (STATES ? buf * Lds::b : 0) + (2 * n + part) * kFragment + 16 * lane);
    };
    // Between the products of the n tiles, what the next chunk needs (past the
    // last one it is not used): the wavefronts of a SIMD take turns with the
    // matrix cores and the vector unit.
    constexpr int kPieces = 2 * TPW + kJobs + 1;
    auto piece_read = [&](int i) {
      if (i < 2 * TPW) convolve_read(STATES ? buf ^ 1 : 0, i >> 1, i & 1);
    };
    auto piece = [&](int i) {
      if (i < 2 * TPW) convolve(i >> 1, i & 1);
      else if (i < 2 * TPW + kJobs) make_products(i - 2 * TPW, buf ^ 1);
      else make_tables(STATES ? buf ^ 1 : 0, buf ^ 1);
    };
    u32x4 b[2], ahead[2];
#pragma unroll
    for (int part = 0; part < 2; ++part) ahead[part] = b_at(0, part);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        b[part] = ahead[part];
        if (n + 1 < NT) ahead[part] = b_at(n + 1, part);
      }
      const int first = n * kPieces / NT, last = (n + 1) * kPieces / NT;
      if (first < last) piece_read(first);
#define LLHIP_SSM_UPDATE(PART, FIELD)                                      \
  _Pragma("unroll") for (int k = 0; k < TPW; ++k)                          \
      st[k][n] = mma_f16(b[PART], xs[k].FIELD, st[k][n]);
      LLHIP_SSM_UPDATE(0, lo)
      LLHIP_SSM_UPDATE(1, hi)
      LLHIP_SSM_UPDATE(0, hi)
#undef LLHIP_SSM_UPDATE
#pragma unroll
      for (int i = first; i < last; ++i) {
        if (i > first) piece_read(i);
        piece(i);
      }
      if (!STATES && n == 0 && next < t_end) request_image(next, 0, kC, Lds::at_c);
    }
    if (STATES && next < t_end) add_total(buf ^ 1);
  }

  float* dst = nullptr;
  if (STATES) dst = p.seg_states + (int64_t)(s.state0 + at.y + 1) * inner * N;
  else if (at.y == s.segments - 1 && s.to >= 0) dst = p.ssm_states + (int64_t)s.to * inner * N;
  if (!dst) return;
#pragma unroll
  for (int k = 0; k < TPW; ++k) {
    if (!on[k]) continue;
    const int at_ch = h0 * p.head_dim + ch[k];
#pragma unroll
    for (int n = 0; n < NT; ++n)
      *reinterpret_cast<floatx4*>(dst + (int64_t)at_ch * N + 16 * n + 4 * g) = st[k][n] * power(reciprocal_bits(held[k]));
    if (STATES && g == 0 && ch[k] % p.head_dim == 0)
      p.seg_decay[(int64_t)(s.state0 + at.y) * p.heads + h0 + head[k]] = (float)total[k];
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

// Block (sequence, head, part): ELEMENTS state elements of a head.  N / 4 lanes share a channel's
// state row.  The states are read and written past the caches' ordinary policy (48 states of 2 MiB in
// rotation: 44 us, 55 with plain accesses): a layer's are not met again before all others'.
template <int N, int ELEMENTS>
__global__ void __launch_bounds__(256) ssm_step_kernel(SsmLayerPlan p, SsmCall c) {
  constexpr int LANES = N / 4, ROWS = 256 / LANES;  // channels per round of the block
  constexpr int kRounds = ELEMENTS / (ROWS * N);
  __shared__ float sx[kSsmMaxHeadDim], sb[N], sc[N];
  __shared__ int flag;
  const int i = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  const int to = slot_of(c.to, i);
  int from = slot_of(c.from, i);
  if (!slots_in_pool(p, from, to)) from = -1;  // (refused below)
  const int P = p.head_dim, inner = p.heads * P, gn = p.groups * N, channels = inner + 2 * gn, W = p.conv;
  const int group = h / (p.heads / p.groups);
  const float* row = c.x + (int64_t)i * (inner + channels + p.heads);
  const float* taps = conv_taps(p, from);
  const int p0 = blockIdx.z * (ELEMENTS / N), np = min(P - p0, ELEMENTS / N);
  // the state first: its loads run while the slots are checked and the convolution is formed
  const int q = tid % LANES, r0 = tid / LANES;
  const int64_t at = ((int64_t)h * P + p0) * N + 4 * q;
  floatx4 st[kRounds];
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const int r = r0 + ROWS * k;
    st[k] = from >= 0 && r < np
                ? __builtin_nontemporal_load(reinterpret_cast<const floatx4*>(
                      p.ssm_states + (int64_t)from * inner * N + at + (int64_t)r * N))
                : floatx4{0.f, 0.f, 0.f, 0.f};
  }
  if (!slots_allowed(p, c, i, &flag)) return;
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
      __builtin_nontemporal_store(st[k], reinterpret_cast<floatx4*>(p.ssm_states + (int64_t)to * inner * N + at +
                                                                    (int64_t)r * N));
    if (q == 0) c.y[(int64_t)i * inner + h * P + p0 + r] = fmaf(d, x, y);
  }
}

// ------------------------------------------------------------------ gate, norm, convolution state

template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)(uint32_t)dpp_i<CTRL>((int)(u >> 32)) << 32 | (uint32_t)dpp_i<CTRL>((int)u));
}
__device__ __forceinline__ double readlane_f64(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(u >> 32), lane) << 32 |
                                        (uint32_t)__builtin_amdgcn_readlane((int)u, lane));
}
__device__ __forceinline__ double wave_sum_f64(double v) {
  v += dpp_f64<kDppXor1>(v);
  v += dpp_f64<kDppXor2>(v);
  v += dpp_f64<kDppHalfMirror>(v);
  v += dpp_f64<kDppMirror>(v);
  return (readlane_f64(v, 0) + readlane_f64(v, 16)) + (readlane_f64(v, 32) + readlane_f64(v, 48));
}

// Blocks [0, norm_blocks): rows y of (token, group), THREADS threads each:
// v = y silu(z), out = v / sqrt(mean v^2 + eps) * norm, in place.  The others:
// the convolution state of a sequence, 256 channels a block (a thread reads
// all of a channel's rows before it writes them: from and to may be one slot).
template <int THREADS>
__global__ void __launch_bounds__(256 > THREADS ? 256 : THREADS)
ssm_finish_kernel(SsmLayerPlan p, SsmCall c, int norm_blocks) {
  constexpr int BLOCK = 256 > THREADS ? 256 : THREADS;
  constexpr int kPer = 4;  // vectors of four channels per thread, THREADS * 16 channels at most
  __shared__ double red[BLOCK / 64];
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
  double sum = 0.0;  // (squares leave single precision's range before what is normed does)
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
#pragma unroll
    for (int e = 0; e < 4; ++e) sum = fma((double)v[k][e], (double)v[k][e], sum);
  }
  sum = wave_sum_f64(sum);
  if constexpr (THREADS > 64) {
    if ((tid & 63) == 0) red[tid >> 6] = sum;
    __syncthreads();
    sum = 0.0;
    for (int k = 0; k < THREADS / 64; ++k) sum += red[k];
  }
  if (!live) return;
  const float scale = (float)(1.0 / sqrt(sum / (double)width + (double)p.epsilon));
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int i = 4 * (l + THREADS * k);
    if (i < width) {
      const floatx4 n = *reinterpret_cast<const floatx4*>(p.norm + group * width + i);
      *reinterpret_cast<f32x4a4*>(y + i) = v[k] * scale * n;
    }
  }
}

// error[1] = what error[0] gathered, which starts anew: in one step, for calls on other streams may add to it.
__global__ void ssm_take_error_kernel(int* error) {
  if (threadIdx.x == 0) error[1] = atomicExch(error, 0);
}

// ------------------------------------------------------------------ host

int64_t ssm_max_chunks(int64_t tokens, int64_t sequences) { return tokens / kSsmChunk + sequences; }

// How a call is cut: column tiles per wavefront and tokens per segment.  A
// scan workgroup has a CU to itself (its LDS), so a pass takes as many rounds
// as it has workgroups to the device's 256 CUs.  The times are measured ones of
// N = 128 (us) and stand for all: a chunk of N = 256 takes one tile 6.6 instead of
// 4.75, those of smaller states were not timed alone.  Two tiles a wavefront share
// a group's operands between twice the channels; one tile halves a chunk's latency
// where there are CUs to spare.  Segments add the first pass, the join and the
// launches of both.
struct ScanCut {
  int tiles, segment_tokens;
};
constexpr int kScanCus = 256;
constexpr int kMinSegment = 64;
static double scan_begin_us(int tiles) { return tiles == 2 ? 6.0 : 5.0; }
static double scan_chunk_us(int tiles) { return tiles == 2 ? 8.8 : 4.75; }
constexpr double kFirstPassShare = 0.45, kJoinUs = 12.0;

// Segments that the whole segments of a call may number.
static int64_t scan_segment_limit(const SsmLayerPlan& p, int tiles) {
  return 2 * kScanCus / (p.heads / scan_heads(p, tiles)) + 1;
}

static ScanCut scan_cut(const SsmLayerPlan& p, int64_t tokens, int64_t sequences) {
  ScanCut best{1, 0};
  double least = 1e30;
  for (int tiles = 1; tiles <= scan_max_tiles(p.state / 16); ++tiles) {
    const int64_t sets = p.heads / scan_heads(p, tiles);
    const int64_t most = std::max<int64_t>(1, std::min(tokens / kMinSegment, scan_segment_limit(p, tiles)));
    for (int64_t m = 1; m <= most; m += std::max<int64_t>(1, m / 8)) {
      const int64_t part = (tokens + m - 1) / m;
      const int64_t seg = std::max<int64_t>(kMinSegment, (part + kSsmChunk - 1) / kSsmChunk * kSsmChunk);
      // the sequences' lengths are on the device: each ends half a segment on
      // average, and the longest is taken for twice the average
      const int64_t cut = sequences == 1 ? (tokens + seg - 1) / seg
                                         : std::max(sequences, tokens / seg + sequences / 2);
      const int64_t longest = std::min(seg, sequences == 1 ? tokens : 2 * tokens / sequences + kSsmChunk);
      const double rounds = (double)((cut * sets + kScanCus - 1) / kScanCus);
      const double chunks = (double)((longest + kSsmChunk - 1) / kSsmChunk);
      double us = rounds * (scan_begin_us(tiles) + chunks * scan_chunk_us(tiles));
      if (tokens > seg) us += kJoinUs + rounds * (scan_begin_us(tiles) + kFirstPassShare * chunks * scan_chunk_us(tiles));
      if (us < least) {
        least = us;
        best = ScanCut{tiles, (int)seg};
      }
    }
  }
  return best;
}

int64_t ssm_max_segments(const SsmLayerPlan& p, int64_t tokens, int64_t sequences) {
  int64_t limit = 0;
  for (int tiles = 1; tiles <= scan_max_tiles(p.state / 16); ++tiles)
    limit = std::max(limit, scan_segment_limit(p, tiles));
  return std::min(tokens / kMinSegment, limit) + sequences;
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

// The last launch: threads to a row, and to a block; blocks that norm rows, and all.
struct FinishGrid {
  int threads, block;
  int64_t norm, all;
};
static FinishGrid finish_grid(const SsmLayerPlan& p, const SsmCall& c) {
  const int inner = p.heads * p.head_dim, channels = inner + 2 * p.groups * p.state;
  const int width = inner / p.groups;
  FinishGrid g{256, 256, (int64_t)c.tokens * p.groups, 0};
  if (width <= 1024 && c.offsets) {  // a row's refusal is the block's where a row is a sequence
    g.threads = 64;
    g.norm = (g.norm + 3) / 4;
  } else if (width > 4096) {
    g.threads = g.block = 1024;
  }
  g.all = g.norm + (int64_t)c.sequences * ((channels + g.block - 1) / g.block);
  return g;
}

static hipError_t finish_launch(const SsmLayerPlan& p, const SsmCall& c, hipStream_t s) {
  const FinishGrid g = finish_grid(p, c);
  const dim3 grid((uint32_t)g.all), block(g.block);
  switch (g.threads) {
    case 64: return launch(ssm_finish_kernel<64>, grid, block, 0, s, p, c, (int)g.norm);
    case 256: return launch(ssm_finish_kernel<256>, grid, block, 0, s, p, c, (int)g.norm);
    default: return launch(ssm_finish_kernel<1024>, grid, block, 0, s, p, c, (int)g.norm);
  }
}

template <int ELEMENTS>
static hipError_t step_launch(const SsmLayerPlan& p, const SsmCall& c, hipStream_t s) {
  const dim3 grid(c.sequences, p.heads, (p.head_dim * p.state + ELEMENTS - 1) / ELEMENTS);
  switch (p.state) {
    case 16: return launch(ssm_step_kernel<16, ELEMENTS>, grid, dim3(256), 0, s, p, c);
    case 32: return launch(ssm_step_kernel<32, ELEMENTS>, grid, dim3(256), 0, s, p, c);
    case 64: return launch(ssm_step_kernel<64, ELEMENTS>, grid, dim3(256), 0, s, p, c);
    case 128: return launch(ssm_step_kernel<128, ELEMENTS>, grid, dim3(256), 0, s, p, c);
    case 256: return launch(ssm_step_kernel<256, ELEMENTS>, grid, dim3(256), 0, s, p, c);
    default: return hipErrorInvalidValue;
  }
}

hipError_t ssm_step_launch(const SsmLayerPlan& p, const SsmCall& c, hipStream_t s) {
  // Parts of 2048 elements put a short call on more CUs, each of whose workgroups forms B and C again:
  // 64 heads of 64 x 128, one sequence 6.0 us (8.3 in parts of 8192), 8 sequences 12.1 (13.0), 10 16.1
  // (13.7), 48 57 (44).
  const int64_t parts = (int64_t)c.sequences * p.heads * ((p.head_dim * p.state + 8191) / 8192);
  const hipError_t e = parts <= 512 ? step_launch<2048>(p, c, s) : step_launch<8192>(p, c, s);
  if (e != hipSuccess) return e;
  return finish_launch(p, c, s);
}

static int64_t scan_blocks(const SsmLayerPlan& p, const SsmCall& c, ScanCut cut) {
  return (int64_t)(c.tokens / cut.segment_tokens + c.sequences) * (p.heads / scan_heads(p, cut.tiles));
}

// A launch has fewer than 2^32 threads.  (The most blocks of any cut come from the shortest segments and one tile
// a wavefront: a call that fits so needs no cut made for it here.)
bool ssm_call_fits(const SsmLayerPlan& p, const SsmCall& c) {
  const FinishGrid g = finish_grid(p, c);
  if (g.all * g.block > UINT32_MAX) return false;
  if (!c.offsets || scan_blocks(p, c, ScanCut{1, kMinSegment}) * 64 * kScanWaves <= UINT32_MAX) return true;
  return scan_blocks(p, c, scan_cut(p, c.tokens, c.sequences)) * 64 * kScanWaves <= UINT32_MAX;
}

template <int NT, int W, int TPW>
static hipError_t scan_launch(const SsmLayerPlan& p, const SsmCall& c, int segment_tokens, hipStream_t s) {
  const int hw = scan_heads(p, TPW), width = hw * p.head_dim;
  const dim3 grid((uint32_t)scan_blocks(p, c, ScanCut{TPW, segment_tokens})), block(64 * kScanWaves);
  if (c.tokens > segment_tokens) {
    hipError_t e = launch(ssm_scan_kernel<NT, W, TPW, true>, grid, block, ScanLds<NT, W, true>::bytes(hw, width), s,
                          p, c, segment_tokens, hw);
    if (e != hipSuccess) return e;
    const int64_t size = (int64_t)p.heads * p.head_dim * 16 * NT;
    e = launch(ssm_join_kernel, dim3(c.sequences, (uint32_t)((size / 4 + 255) / 256)), dim3(256), 0, s, p);
    if (e != hipSuccess) return e;
  }
  return launch(ssm_scan_kernel<NT, W, TPW, false>, grid, block, ScanLds<NT, W, false>::bytes(hw, width), s, p, c,
                segment_tokens, hw);
}

template <int NT, int W>
static hipError_t run_launch(const SsmLayerPlan& p, const SsmCall& c, hipStream_t s) {
  const ScanCut cut = scan_cut(p, c.tokens, c.sequences);
  hipError_t e = launch(ssm_plan_kernel, dim3(c.sequences), dim3(kPlanThreads), 0, s, p, c, cut.segment_tokens);
  if (e != hipSuccess) return e;
  e = launch(ssm_prepare_kernel<NT, W>,
             dim3((uint32_t)ssm_max_chunks(c.tokens, c.sequences), p.groups + (p.heads + kPrepHeads - 1) / kPrepHeads),
             dim3(256), 0, s, p, c);
  if (e != hipSuccess) return e;
  if constexpr (scan_max_tiles(NT) == 2)
    if (cut.tiles == 2) e = scan_launch<NT, W, 2>(p, c, cut.segment_tokens, s);
  if (cut.tiles == 1) e = scan_launch<NT, W, 1>(p, c, cut.segment_tokens, s);
  if (e != hipSuccess) return e;
  return finish_launch(p, c, s);
}

template <int W>
static hipError_t run_state(const SsmLayerPlan& p, const SsmCall& c, hipStream_t s) {
  switch (p.state) {
    case 16: return run_launch<1, W>(p, c, s);
    case 32: return run_launch<2, W>(p, c, s);
    case 64: return run_launch<4, W>(p, c, s);
    case 128: return run_launch<8, W>(p, c, s);
    case 256: return run_launch<16, W>(p, c, s);
    default: return hipErrorInvalidValue;
  }
}

hipError_t ssm_run_launch(const SsmLayerPlan& p, const SsmCall& c, hipStream_t s) {
  switch (p.conv) {
    case 2: return run_state<2>(p, c, s);
    case 3: return run_state<3>(p, c, s);
    case 4: return run_state<4>(p, c, s);
    default: return hipErrorInvalidValue;
  }
}

hipError_t ssm_take_error_launch(const SsmLayerPlan& p, hipStream_t s) {
  return launch(ssm_take_error_kernel, dim3(1), dim3(64), 0, s, p.error);
}

}  // namespace llhip
