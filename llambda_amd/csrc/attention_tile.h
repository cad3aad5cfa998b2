// attention_tile.h -- the attention kernels over one range of positions (attention.h).
//
// A wavefront takes 32 rows and forms both products transposed, S^T = K Q^T and
// Y^T = V^T P^T, on 32 x 32 tiles: a lane then holds one row of the softmax, half
// of its keys, so maximum, sum and every factor of a row are that lane's own (one
// exchange with lane ^ 32), and the results of S^T are the operand P^T of the
// second product without a move: which key an operand's K element stands for is
// free as long as both operands agree, and the lane's keys 8 i + 4 (lane / 32) +
// 0..3 are what two transposing LDS reads bring of V.
//
// Softmax runs over the keys once, with the running maximum and sum in fp32.
//
// Operands.  A cache in 16 bits is an operand as it is.  fp32 rows, and the fp32
// probabilities of such rows, are split into parts of the cache's type whose
// products are added: two of f16 (22 bits; q times a power of two for each row, p
// times 2^9, so that the parts stay normal), three of bf16 (24 bits).  Rows in 16
// bits are one part, and so are their probabilities: rounding those to 8 or 11 bits
// costs what rounding the output costs.  An fp32 cache uses the fp32 products.
//
// Keys and values pass through LDS, loaded there directly, a tile ahead, 16-byte
// pieces permuted so that neither read meets a bank twice.
//
// Two kernels.  Where a sequence has many rows, eight wavefronts with 32 rows each
// share every tile (attn_shared_kernel): a tile's bytes serve 256 rows, and the two
// wavefronts of a SIMD are a phase apart, one's products beside the other's softmax
// (8192 tokens 1014 us, all in step 1105).  Those 8192 tokens, 32 heads of 128, fp32
// rows over f16, are 550 GFLOP in two parts, in 940 to 1015 us 1080 to 1170 TFLOP/s of
// products, next to 1070 of a large library product of f16 (random operands hold the
// card to about 1500 from registers alone): the matrix pipes are busy in 66% of the
// cycles that wavefronts live, the VALU in 45%.  6000 tokens of bf16, one part, take
// 357 to 395 us or 750 to 830 TFLOP/s, 43% and 45%: each fragment of 1 KB feeds one
// product of 32 cycles there, so that the four SIMDs ask the LDS for all of its 128
// bytes a cycle.  1501 tokens in fp32, 70% and 15%, read fragments where they are
// needed.  Where a sequence has few rows, wavefronts share 32 of them and take a tile of
// keys each (attn_split_kernel), so that the keys' way through the device is all that
// counts: a step of 48 sequences, 614 MB, in 125 us, 4.9 TB/s (a large copy 5.1).
#pragma once

#include "attention_cut.h"
#include "mfma.h"

namespace llhip {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) const uint8_t* lds_bytes;
__device__ __forceinline__ lds_bytes lds_at(uint32_t address) { return reinterpret_cast<lds_bytes>(address); }

__device__ __forceinline__ float half_pair_max(float v) {
  float a = v, b = v;
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
  return fmaxf(a, b);
}

// ---------------------------------------------------------------- operands
template <int TYPE>
struct Cell;
template <>
struct Cell<kAttnF32> {
  typedef float T;
  static constexpr float kLift = 0.f;
};
template <>
struct Cell<kAttnF16> {
  typedef _Float16 T;
  typedef halfx8 Frag;
  // p times 2^9, 2^15 at most: down to 2^-23 of the reference its first part is a normal number
  static constexpr float kLift = 9.f;
  static __device__ __forceinline__ floatx16 mfma(Frag a, Frag b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(floatx2{a, b}, halfx2));
  }
  static __device__ __forceinline__ floatx2 unpack(uint32_t v) {
    return __builtin_convertvector(__builtin_bit_cast(halfx2, v), floatx2);
  }
};
template <>
struct Cell<kAttnBF16> {
  typedef __bf16 T;
  typedef bf16x8 Frag;
  static constexpr float kLift = 0.f;
  static __device__ __forceinline__ floatx16 mfma(Frag a, Frag b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(floatx2{a, b}, bf16x2));
  }
  static __device__ __forceinline__ floatx2 unpack(uint32_t v) {
    return floatx2{__builtin_bit_cast(float, v << 16), __builtin_bit_cast(float, v & 0xFFFF0000u)};
  }
};

// Parts of the cache's type that a number of the rows' type takes.
template <int TYPE, typename Row>
constexpr int attn_parts() {
  return sizeof(Row) == 2 ? 1 : TYPE == kAttnF16 ? 2 : 3;
}

// (a, b) as N packed pairs whose sums they are.
template <int TYPE, int N>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t (&out)[N]) {
  float minus = -1.f;  // hidden, so that an f16's conversion becomes part of the (exact) difference
  asm("" : "+s"(minus));
#pragma unroll
  for (int n = 0; n < N; ++n) {
    out[n] = Cell<TYPE>::pack(a, b);
    if (n + 1 < N) {
      const floatx2 u = Cell<TYPE>::unpack(out[n]);
      a = fmaf(u.x, minus, a);
      b = fmaf(u.y, minus, b);
    }
  }
}

// COUNT fragments read from LDS, each AHEAD of its use, in this order: left to itself the compiler reads one ahead, and
// every product waits for the LDS.
template <int COUNT, int AHEAD, typename Frag, typename Read, typename Use>
__device__ __forceinline__ void read_ahead(Read&& read, Use&& use) {
  Frag f[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) f[i] = read(i);
#pragma unroll
  for (int i = 0; i < COUNT; ++i) {
    __builtin_amdgcn_sched_barrier(0);
    use(i, f[i % AHEAD]);
    __builtin_amdgcn_sched_barrier(0);
    if (i + AHEAD < COUNT) f[i % AHEAD] = read(i + AHEAD);
  }
  __builtin_amdgcn_sched_barrier(0);
}

template <typename Row>
__device__ __forceinline__ void store4(Row* p, floatx4 v) {
  if constexpr (sizeof(Row) == 4) {
    *reinterpret_cast<floatx4*>(p) = v;
  } else {
    typedef Row Row4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<Row4*>(p) = __builtin_convertvector(v, Row4);
  }
}

// ------------------------------------------------------------------- layout
// A tile of keys (or values) in LDS: rows of kRow bytes, their 16-byte pieces permuted.
template <int SIZE, int DP>
struct TileLayout {
  static constexpr int kRow = DP * SIZE;
  static constexpr int kPieces = kRow / 16;
  static constexpr int kRowsPerLoad = 64 / kPieces;  // 64 lanes load 16 bytes each
  // Where a piece of keys goes: 16-byte reads of 16 rows (rows n and n + 8 among them) fill the banks once.
  static __device__ __forceinline__ int key_swizzle(int row) { return kPieces == 8 ? (row >> 1) & 7 : row & 15; }
  // Of values in 16 bits: transposing reads of 64 bytes of 4 neighbouring rows do.  fp32 reads need none.
  static __device__ __forceinline__ int value_swizzle(int row) {
    return SIZE == 4 ? 0 : kPieces == 8 ? 4 * ((row >> 1) & 1) : 4 * (row & 3);
  }
};

// The pages of one kv head of one sequence, for loads of tiles into LDS.
template <int SIZE, int DP, int KT>
struct TileLoader {
  typedef TileLayout<SIZE, DP> L;
  static constexpr int kLoads = KT / L::kRowsPerLoad;  // of keys, and of values, by one wavefront
  const uint8_t* keys;    // of the head in page 0
  const uint8_t* values;
  uint64_t page_bytes;    // of all heads
  int page_shift, head_dim;
  int last;  // the sequence's last position; tiles past it hold rows near it again
  __device__ __forceinline__ TileLoader(const AttnPlan& p, int layer, int kv_head, const AttnItem& it)
      : page_bytes(((uint64_t)p.kv_heads * p.head_dim * SIZE) << p.page_shift),
        page_shift(p.page_shift),
        head_dim(p.head_dim),
        last(it.context + it.length - 1) {
    const uint64_t at = (uint64_t)layer * p.pages * page_bytes + (((uint64_t)kv_head * p.head_dim * SIZE) << page_shift);
    keys = static_cast<const uint8_t*>(p.keys) + at;
    values = static_cast<const uint8_t*>(p.values) + at;
  }

  // Lane l's page: the one of position base + kApart l.
  static constexpr int kApart = KT > 64 ? KT / 64 : 1;
  static_assert(kApart == 1 || L::kRowsPerLoad % kApart == 0, "a load begins at a position whose page a lane has");
  __device__ __forceinline__ int entry(int base, int lane) const {
    return min(base + lane * kApart, last) >> page_shift;
  }
  // Of the loads of the keys, or values, of tile `base` to LDS every STEP-th from `from` on; pages: entry()'s, by lane.
  // What depends on the lane alone is the same for every tile.
  template <bool VALUES, int STEP>
  __device__ __forceinline__ void load(int base, int pages, uint32_t to, int from, int lane) const {
    constexpr int R = L::kRowsPerLoad;
    static_assert(kLoads % STEP == 0, "as many loads for every wavefront");
    const int row = lane / L::kPieces, piece = lane % L::kPieces;
    const uint32_t bytes = head_dim * SIZE;
    const uint32_t in_page = (1u << page_shift) - 1;
#pragma unroll
    for (int j = 0; j < kLoads / STEP; ++j) {
      const int i = from + j * STEP, r0 = i * R;
      uint32_t source = 16 * (piece ^ (VALUES ? L::value_swizzle(r0 + row) : L::key_swizzle(r0 + row)));
      // a row shorter than the tile's: its first piece again (the row's q has zeros there, its y is not stored; rows whose
      // zeros meet an infinite key come to whole_row)
      if (source >= bytes) source = 0;
      const uint32_t pos = min(base + r0, last & ~(R - 1));
      const uint32_t page = __builtin_amdgcn_readlane(pages, r0 / kApart);
      load_lds16((VALUES ? values : keys) + (uint64_t)page * page_bytes + (pos & in_page) * bytes, row * bytes + source,
                 to + 1024u * i);
    }
  }
};

// ---------------------------------------------------------- a wavefront's rows
// Bits of the keys base .. base + 31 that a lane's row sees.
struct Sight {
  int limit;             // causal: positions below it; a tree's: the cached ones
  const uint32_t* tree;  // null: causal
  __device__ __forceinline__ uint32_t bits(int base) const {
    const int n = limit - base;
    if (!tree) return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1;
    if (n >= 32) return ~0u;
    if (n > 0) return ((1u << n) - 1) | (tree[0] << n);
    const int w = -n >> 5, s = -n & 31;
    if (w >= kAttnTreeWords) return 0;
    const uint32_t lo = tree[w], hi = w + 1 < kAttnTreeWords ? tree[w + 1] : 0;
    return (uint32_t)((((uint64_t)hi << 32) | lo) >> s);
  }
};

// How far a row's maximum may grow, in powers of two, before its sums are scaled.
constexpr float kSlack = 6.f;
// Exponents from here on are off by one half and more, as products with the row's factor are rounded, and more than f16 has
// room for beside the slack; from 2^31 on by more than fp32 has.
constexpr float kMostExponent = 0x1p22f;

// Sums of 32 rows over the keys so far: y holds rows 32 b + 8 (i / 4) + 4 (lane / 32) + i % 4 of Y^T, column lane % 32.
template <int DP>
struct RowSums {
  floatx16 y[DP / 32];
  float reference;  // the exponent that p is taken against; -inf: no key yet
  float sum;        // of this lane's keys
  uint32_t bad[DP / 32];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int b = 0; b < DP / 32; ++b) y[b] = floatx16{}, bad[b] = 0;
    reference = -__builtin_inff();
    sum = 0.f;
  }
  // Notes the elements that are no numbers in keys that the row sees.
  template <int KB>
  __device__ __forceinline__ void spoil(const uint32_t* bits, const uint32_t (&sight)[KB]) {
#pragma unroll
    for (int b = 0; b < KB; ++b)
      for (int k = 0; k < 32; ++k)
        if (sight[b] >> k & 1)
#pragma unroll
          for (int d = 0; d < DP / 32; ++d) bad[d] |= bits[(32 * b + k) * (DP / 32) + d];
  }
  // y's rows 32 b + 8 i + 4 half + 0..3.
  __device__ __forceinline__ floatx4 piece(int b, int i, int half) const {
    floatx4 v;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = bad[b] >> (8 * i + 4 * half + k) & 1 ? __builtin_nanf("") : y[b][4 * i + k];
    return v;
  }
  // The scores s of KB blocks of 32 keys become probabilities, 2^lift for the reference's.
  template <int KB>
  __device__ __forceinline__ void softmax(floatx16 (&s)[KB], float factor, float lift) {
    float top = s[0][0];
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
    top = half_pair_max(top) * factor;
    // the sums are scaled again only where a maximum has grown by more than the probabilities' range leaves room for
    if (__ballot(top > reference + kSlack)) {
      const float next = fmaxf(reference, top);
      // a row that has seen nothing has nothing to scale (and no reference)
      const float scale = next == reference ? 1.f : __builtin_amdgcn_exp2f(reference - next);
      sum *= scale;
      // such a row is formed anew in the end (whole_row)
      if (next != reference && fabsf(next) >= kMostExponent) sum = __builtin_nanf("");
      reference = next;
#pragma unroll
      for (int b = 0; b < DP / 32; ++b) y[b] *= scale;
    }
    const float shift = lift - (reference == -__builtin_inff() ? 0.f : reference);
    float part[4] = {};
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[b][i] = __builtin_amdgcn_exp2f(fmaf(s[b][i], factor, shift));
        part[i & 3] += s[b][i];
      }
    sum += (part[0] + part[1]) + (part[2] + part[3]);
  }
};

template <int KB>
__device__ __forceinline__ void mask_scores(floatx16 (&s)[KB], const uint32_t (&sight)[KB], int half) {
#pragma unroll
  for (int b = 0; b < KB; ++b) {
    const uint32_t v = sight[b] >> (4 * half);
#pragma unroll
    for (int i = 0; i < 16; ++i) s[b][i] = v >> (8 * (i / 4) + i % 4) & 1 ? s[b][i] : -__builtin_inff();
  }
}

// Values that are infinite or NaN, where a row may see only part of a tile: a masked probability of 0 would make NaN
// of them.  They become zeros in LDS, noted by key and element, and rows that see one get NaN there afterwards.
template <int SIZE, int DP, int KT>
struct Spoiled {
  static constexpr int kWords = DP / 32;
  static constexpr int kBytes = (KT * kWords + 1) * 4;
  uint32_t* bits;  // LDS: [KT][kWords], then whether there are any
  __device__ __forceinline__ void clear(int thread, int threads) const {
    for (int i = thread; i <= KT * kWords; i += threads) bits[i] = 0;
  }
  // The tile at `tile`, by `threads` threads; the words are clear.
  __device__ __forceinline__ void scan(uint8_t* tile, int thread, int threads) const {
    typedef TileLayout<SIZE, DP> L;
    // an exponent of ones carries into the sign's place
    constexpr uint32_t kSigns = SIZE == 4 ? 0x80000000u : 0x80008000u;
#pragma unroll 4
    for (int i = thread; i < KT * L::kPieces; i += threads) {
      u32x4 v = *reinterpret_cast<const u32x4*>(tile + 16 * i);
      uint32_t carry = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) carry |= (v[k] & ~kSigns) + one;
      if (carry & kSigns) {
        const int key = i / L::kPieces;
        const int d = ((i % L::kPieces) ^ L::value_swizzle(key)) * (16 / SIZE);
        uint32_t bad = 0;
        if constexpr (SIZE == 4) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if ((v[k] & ~kSigns) + one & kSigns) bad |= 1u << k, v[k] = 0;
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if ((v[k / 2] & ~kSigns) + one & (k & 1 ? 0x80000000u : 0x8000u))
              bad |= 1u << k, v[k / 2] &= k & 1 ? 0xFFFFu : 0xFFFF0000u;
        }
        *reinterpret_cast<u32x4*>(tile + 16 * i) = v;
        atomicOr(bits + key * kWords + d / 32, bad << (d % 32));
        bits[KT * kWords] = 1;
      }
    }
  }
  __device__ __forceinline__ bool any() const { return __builtin_amdgcn_readfirstlane(bits[KT * kWords]) != 0; }
  uint32_t one;  // the lowest bit of an element's exponent, for each in 32 bits
};

template <int TYPE, typename Row, int DP>
struct RowTile {
  typedef Cell<TYPE> C;
  typedef typename C::Frag Frag;
  typedef TileLayout<2, DP> L;
  static constexpr int N = attn_parts<TYPE, Row>(), kSteps = DP / 16, kBlocks = DP / 32;
  static constexpr int kAhead = N == 1 ? 4 : 3;  // what registers are left for
  Frag q[N][kSteps];
  RowSums<DP> sums;
  float factor;  // of the products, into exponents of two
  uint32_t key_at, value_at;
  int half;

  // A row as it is on its way.  Lane l holds elements 16 s + 8 (l / 32) + 0..7 of row l % 32.
  typedef Row Row8 __attribute__((ext_vector_type(8)));
  struct Raw {
    Row8 v[kSteps];
  };
  // row: null for rows behind the last.
  __device__ __forceinline__ static void fetch(Raw& raw, const Row* row, int head_dim, int lane) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      raw.v[s] = Row8{};
      if (row && 16 * s < head_dim) raw.v[s] = *reinterpret_cast<const Row8*>(row + 16 * s + 8 * (lane >> 5));
    }
  }
  __device__ __forceinline__ void start(const Raw& raw, float scale_log2, int lane) {
    half = lane >> 5;
    sums.clear();
    const int r = lane & 31, j = lane & 15;
    key_at = r * L::kRow + 16 * (half ^ L::key_swizzle(r));
    value_at = (4 * half + (j >> 2)) * L::kRow + 16 * L::value_swizzle(j >> 2) + ((lane >> 4) & 1) * 32 + (j & 3) * 8;
    if constexpr (N == 1) {
      factor = scale_log2;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) q[0][s] = __builtin_bit_cast(Frag, raw.v[s]);
      return;
    }
    float v[kSteps][8], top = 0.f;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[s][i] = (float)raw.v[s][i];
        top = fmaxf(top, fabsf(v[s][i]));
      }
    float lift = 1.f;
    if (N == 2) {
      // the row's largest between 2^13 and 2^14 (rows next to zero, infinities and NaN as they are)
      top = half_pair_max(top);
      const int e = (int)(__builtin_bit_cast(uint32_t, top) >> 23);
      if (e > 20 && e < 255) {
        lift = __builtin_bit_cast(float, (uint32_t)(127 + 13 + 127 - e) << 23);
        factor = scale_log2 * __builtin_bit_cast(float, (uint32_t)(e - 13) << 23);
      } else {
        factor = scale_log2;
      }
    } else {
      // rows of less than 2^-64 times 2^64: the third part of a number below 2^-110 would be next to nothing
      top = half_pair_max(top);
      const bool small = top < 0x1p-64f;
      lift = small ? 0x1p64f : 1.f;
      factor = small ? scale_log2 * 0x1p-64f : scale_log2;
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      u32x4 packed[N];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t p[N];
        split_pair<TYPE, N>(v[s][2 * i] * lift, v[s][2 * i + 1] * lift, p);
#pragma unroll
        for (int n = 0; n < N; ++n) packed[n][i] = p[n];
      }
#pragma unroll
      for (int n = 0; n < N; ++n) q[n][s] = __builtin_bit_cast(Frag, packed[n]);
    }
  }

  // A tile of KB blocks of 32 keys between its steps: scores, then packed probabilities.
  template <int KB>
  struct Work {
    floatx16 s[KB];
    u32x4 p[KB][2][N];
  };
  template <int KB>
  __device__ __forceinline__ void scores(Work<KB>& w, uint32_t lds_k) const {
#pragma unroll
    for (int b = 0; b < KB; ++b) w.s[b] = floatx16{};
    // the blocks in turn: a product does not follow one of the same sum
    read_ahead<KB * kSteps, kAhead, Frag>(
        [&](int i) {
          return *reinterpret_cast<const __attribute__((address_space(3))) Frag*>(
              lds_at(lds_k + (key_at ^ (32u * (i / KB)))) + 32 * (i % KB) * L::kRow);
        },
        [&](int i, const Frag& k) {
#pragma unroll
          for (int n = 0; n < N; ++n) w.s[i % KB] = C::mfma(k, q[n][i / KB], w.s[i % KB]);
        });
  }
  // sight: what each lane's row sees of the tile, if masked.
  template <int KB>
  __device__ __forceinline__ void softmax(Work<KB>& w, bool masked, const uint32_t (&sight)[KB]) {
    if (masked) mask_scores(w.s, sight, half);
    sums.softmax(w.s, factor, C::kLift);
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t part[N];
          split_pair<TYPE, N>(w.s[b][8 * t + 2 * i], w.s[b][8 * t + 2 * i + 1], part);
#pragma unroll
          for (int n = 0; n < N; ++n) w.p[b][t][n][i] = part[n];
        }
  }
  template <int KB>
  __device__ __forceinline__ void add(const Work<KB>& w, uint32_t lds_v) {
    read_ahead<KB * 2 * kBlocks, kAhead, Frag>(
        [&](int i) { return __builtin_bit_cast(Frag, value(lds_v, i / kBlocks * 16, i % kBlocks)); },
        [&](int i, const Frag& v) {
          const int d = i % kBlocks, step = i / kBlocks;
#pragma unroll
          for (int n = 0; n < N; ++n)
            sums.y[d] = C::mfma(v, __builtin_bit_cast(Frag, w.p[step / 2][step % 2][n]), sums.y[d]);
        });
  }

  // Keys key .. key + 15, elements 32 d .. 32 d + 31: lane l holds element l % 32 of keys 4 (l / 32) + 0..3 and
  // 8 more on.
  __device__ __forceinline__ u32x4 value(uint32_t lds_v, int key, int d) const {
    const lds_bytes at = lds_at(lds_v + (value_at ^ (64u * d)));
    typedef short shortx4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) shortx4* ptr;
    const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(at + key * L::kRow)));
    const u32x2 c = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(at + (key + 8) * L::kRow)));
    return u32x4{a.x, a.y, c.x, c.y};
  }
};

// fp32 rows over an fp32 cache: the 32x32x2 products, lane l's K element is the one of its half.
template <typename Row, int DP>
struct RowTile<kAttnF32, Row, DP> {
  typedef TileLayout<4, DP> L;
  static constexpr int kSteps = DP / 8, kBlocks = DP / 32;
  floatx4 q[kSteps];  // elements 8 s + 4 (lane / 32) + 0..3
  RowSums<DP> sums;
  float factor;
  uint32_t key_at, value_at;
  int half;

  static __device__ __forceinline__ floatx16 mfma(float a, float b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
  }
  struct Raw {
    floatx4 v[kSteps];
  };
  __device__ __forceinline__ static void fetch(Raw& raw, const Row* row, int head_dim, int lane) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      raw.v[s] = floatx4{};
      if (row && 8 * s < head_dim) raw.v[s] = *reinterpret_cast<const floatx4*>(row + 8 * s + 4 * (lane >> 5));
    }
  }
  __device__ __forceinline__ void start(const Raw& raw, float scale_log2, int lane) {
    half = lane >> 5;
    sums.clear();
    const int r = lane & 31;
    key_at = r * L::kRow + 16 * (half ^ L::key_swizzle(r));
    value_at = 4 * half * L::kRow + 4 * r;
    factor = scale_log2;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) q[s] = raw.v[s];
  }
  template <int KB>
  struct Work {
    floatx16 s[KB];
  };
  template <int KB>
  __device__ __forceinline__ void scores(Work<KB>& w, uint32_t lds_k) const {
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      w.s[b] = floatx16{};
#pragma unroll
      for (int t = 0; t < kSteps; ++t) {
        const floatx4 k = *reinterpret_cast<const __attribute__((address_space(3))) floatx4*>(
            lds_at(lds_k + (key_at ^ (32u * t))) + 32 * b * L::kRow);
#pragma unroll
        for (int i = 0; i < 4; ++i) w.s[b] = mfma(k[i], q[t][i], w.s[b]);
      }
    }
  }
  template <int KB>
  __device__ __forceinline__ void softmax(Work<KB>& w, bool masked, const uint32_t (&sight)[KB]) {
    if (masked) mask_scores(w.s, sight, half);
    sums.softmax(w.s, factor, Cell<kAttnF32>::kLift);
  }
  template <int KB>
  __device__ __forceinline__ void add(const Work<KB>& w, uint32_t lds_v) {
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int d = 0; d < kBlocks; ++d)
          sums.y[d] = mfma(value(lds_v, 32 * b + 8 * (i / 4) + i % 4, d), w.s[b][i], sums.y[d]);
  }
  __device__ __forceinline__ float value(uint32_t lds_v, int key, int d) const {
    return *reinterpret_cast<const __attribute__((address_space(3))) float*>(lds_at(lds_v + value_at) +
                                                                             key * L::kRow + 128 * d);
  }
};

// -------------------------------------------------------------------- kernels
constexpr float kAttnLog2e = 1.44269504088896340736f;
constexpr int kAttnPageList = 1024;  // entries of a table's row in LDS

template <int TYPE>
constexpr int attn_cell_bytes() {
  return TYPE == kAttnF32 ? 4 : 2;
}

template <int TYPE>
constexpr uint32_t attn_exponent() {
  return TYPE == kAttnF16 ? 0x04000400u : TYPE == kAttnBF16 ? 0x00800080u : 0x00800000u;
}
// LDS accesses of this wavefront so far are done before those that follow.
__device__ __forceinline__ void wave_lds_order() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// Hides where a pointer comes from.
template <typename T>
__device__ __forceinline__ const T* opaque_pointer(const T* p) {
  asm("" : "+s"(p));
  return p;
}

// The kernel's first arguments, read again: where they are rarely needed, no register holds them meanwhile.
struct AttnArgs {
  AttnPlan p;
  AttnCall c;
};
static_assert(sizeof(AttnPlan) % alignof(AttnCall) == 0, "arguments follow each other as a struct's members do");
__device__ __forceinline__ const AttnArgs& args_again() {
  typedef const __attribute__((address_space(4))) AttnArgs* Args;
  Args a = (Args)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(a));
  return *(const AttnArgs*)a;
}

// A struct of the workspace, in scalar registers.
template <typename T>
__device__ __forceinline__ T uniform_load(const T* at) {
  union {
    T t;
    int v[sizeof(T) / 4];
  } u;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 4); ++i)
    u.v[i] = __builtin_amdgcn_readfirstlane(reinterpret_cast<const int*>(at)[i]);
  return u.t;
}

// What an item's rows are, for one of its wavefronts (32 rows from m on).
template <typename Row>
struct ItemRows {
  int rows;    // of the sequence's kv head
  int m;       // this lane's
  int token;   // its token, the last one's for rows behind it
  bool real;
  __device__ __forceinline__ ItemRows(const AttnPlan& p, const AttnItem& it, int m0, int lane) {
    rows = it.length * (int)p.group.divisor;
    m = m0 + (lane & 31);
    real = m < rows;
    token = min(m, rows - 1) / p.group;
  }
  __device__ __forceinline__ int head(const AttnPlan& p, int kv_head) const {
    return kv_head * (int)p.group.divisor + min(m, rows - 1) % p.group;
  }
  __device__ __forceinline__ const Row* q(const AttnPlan& p, const AttnCall& c, const AttnItem& it, int kv_head) const {
    return real ? static_cast<const Row*>(c.q) + (it.begin + token) * c.q_stride + head(p, kv_head) * p.head_dim
                : nullptr;
  }
  __device__ __forceinline__ Row* y(const AttnPlan& p, const AttnCall& c, const AttnItem& it, int kv_head) const {
    return static_cast<Row*>(c.y) + (it.begin + token) * c.y_stride + head(p, kv_head) * p.head_dim;
  }
  __device__ __forceinline__ Sight sight(const AttnPlan& p, const AttnCall& c, const AttnItem& it) const {
    if (c.parents) return Sight{it.context, p.tree + (size_t)(it.begin + token) * kAttnTreeWords};
    return Sight{it.context + token + 1, nullptr};
  }
};

// Row m of a tile of ROWS by its definition, by one wavefront: a row whose sum is no number is formed anew here, in fp32, with
// products of whole elements and differences of scores before all else, twice over its keys: for the largest score and for
// the sums, or as far as a score that is +inf or no number.  Such rows are those of
//   parts of q, which are of either sign or zero, so that their products with a key's infinity make no number of a score that
//   is -inf and has no weight; an element next to the end of fp32 has a first part that is infinite;
//   heads narrower than their tile, whose zeros behind q meet a key's infinity (zeros behind the keys instead, written by
//   each wavefront behind its loads, took steps at width 80 from 53 to 60 us and at 192 from 135 to 163);
//   exponents from kMostExponent on;
//   and those that are no numbers by the definition.
// (5000 tokens, 32 heads of 128 in fp32 over f16, one infinite key: 25 ms in place of 0.43; a mend within the loop would cost
// every call.)
// tree: the ancestors of the item's tokens in LDS, null where they are in the workspace.
template <int TYPE, typename Row, int DP, int ROWS>
__device__ __forceinline__ void whole_row(const AttnPlan& p, const AttnCall& c, const AttnItem& it, int kv_head, int m,
                                          const uint32_t* tree) {
  typedef typename Cell<TYPE>::T T;
  typedef T T4 __attribute__((ext_vector_type(4)));
  typedef float float8 __attribute__((ext_vector_type(8)));
  const int lane = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0));
  const ItemRows<Row> rows(p, it, m, 0);
  Sight sight = rows.sight(p, c, it);
  if (tree && c.parents) sight.tree = tree + (rows.token - it.m0 / p.group) * kAttnTreeWords;
  const Row* const q = rows.q(p, c, it, kv_head);
  const int* const table = c.table + it.sequence * c.table_stride;
  const float factor = p.scale * kAttnLog2e;
  auto cells = [&](void* pool, int page, int pos) {
    return static_cast<const T*>(pool) + attn_cell(p, c.layer, page, pos) + ((size_t)kv_head << p.page_shift) * p.head_dim;
  };
  auto sees = [&](int base) { return base + lane < it.key1 && (sight.bits(base + (lane & 32)) >> (lane & 31) & 1); };
  int page = 0;
  auto score = [&](int base) {  // of key base + lane, in exponents of two
    if (!sees(base)) return -__builtin_inff();
    page = table[(base + lane) >> p.page_shift];
    const T* const key = cells(p.keys, page, base + lane);
    float v = 0.f;
#pragma unroll 1
    for (int d = 0; d < p.head_dim; d += 8) {
      const float8 a = __builtin_convertvector(*reinterpret_cast<const attn_eight<Row>*>(q + d), float8);
      const float8 b = __builtin_convertvector(*reinterpret_cast<const attn_eight<T>*>(key + d), float8);
#pragma unroll
      for (int i = 0; i < 8; ++i) v = fmaf(a[i], b[i], v);
    }
    return v * factor;
  };
  float reference = -__builtin_inff(), sum = 0.f;
  floatx4 y{};
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    const float least = reference == -__builtin_inff() ? 0.f : reference;
    for (int base = it.key0; base < it.key1; base += 64) {
      const float v = score(base);
      if (pass == 0) {
        reference = fmaxf(reference, v);
        if (!__ballot(!(v < __builtin_inff()))) continue;
        sum = __builtin_nanf("");
        break;
      }
      const float weight = __builtin_amdgcn_exp2f(v - least + Cell<TYPE>::kLift);
      sum += weight;
      floatx4 some{};  // of 64 keys, then of all: no long chains
      for (uint64_t left = __ballot(sees(base)); left; left &= left - 1) {
        const int k = __builtin_ctzll(left);
        const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, weight), k));
        const T* const value = cells(p.values, __builtin_amdgcn_readlane(page, k), base + k);
        if (4 * lane < p.head_dim) some += w * __builtin_convertvector(*reinterpret_cast<const T4*>(value + 4 * lane), floatx4);
      }
      y += some;
    }
    reference = wave_max(reference);
    if (__ballot(sum != sum)) {  // no softmax
      reference = -__builtin_inff();
      break;
    }
  }
  sum = wave_total(sum);
  if (it.part < 0) {
    if (4 * lane < p.head_dim) store4(rows.y(p, c, it, kv_head) + 4 * lane, y * (1.f / sum));
  } else {
    const size_t row = ((size_t)it.part * p.kv_heads + kv_head) * ROWS + m - it.m0;
    if (lane == 0) p.part_ml[row] = make_float2(reference, sum);
    if (4 * lane < DP) *reinterpret_cast<floatx4*>(p.part_y + row * DP + 4 * lane) = y;
  }
}

// Waves share tiles of KT keys, two of which are in LDS; each has 32 rows of its own.
template <int TYPE, typename Row, int DP, int WAVES, int KT>
__device__ __forceinline__ void shared_item(const AttnPlan& p, const AttnCall& c, const AttnItem& it, int kv_head,
                                            uint8_t* lds) {
  constexpr int SIZE = attn_cell_bytes<TYPE>(), KB = KT / 32;
  typedef TileLoader<SIZE, DP, KT> Loader;
  constexpr uint32_t kTile = KT * DP * SIZE;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m0 = it.m0 + 32 * wave;
  const bool any = m0 < it.length * (int)p.group.divisor;
  auto see_tile = [&](int key, uint32_t (&see)[KB]) {
    const Sight sight = ItemRows<Row>(p, it, m0, (int)opaque((uint32_t)lane)).sight(p, c, it);
#pragma unroll
    for (int b = 0; b < KB; ++b) see[b] = sight.bits(key + 32 * b);
  };
  // below all_sure every row of the item sees everything
  const int all_sure = c.parents ? it.context : it.context + it.m0 / p.group + 1;
  const Spoiled<SIZE, DP, KT> spoiled{reinterpret_cast<uint32_t*>(lds + 4 * kTile), attn_exponent<TYPE>()};
  spoiled.clear(threadIdx.x, 64 * WAVES);
  typedef RowTile<TYPE, Row, DP> Tile;
  Tile tile;

  const Loader loader(p, c.layer, kv_head, it);
  const int* table = c.table + it.sequence * c.table_stride;
  const uint32_t base = lds_address(lds);
  const int tiles = (it.key1 - it.key0 + KT - 1) / KT;
  auto key_of = [&](int t) { return it.key0 + t * KT; };
  auto keys_at = [&](int t) { return base + (t & 1) * kTile; };
  auto values_at = [&](int t) { return base + (2 + (t & 1)) * kTile; };
  auto pages_of = [&](int t) { return table[loader.entry(key_of(t), lane)]; };
  auto barrier = [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
  // the pages of tiles t and t + 1 when loads(t) is next
  int pages = pages_of(0), next_pages = pages_of(1);
  auto loads = [&](int t) {
    if (t + 1 < tiles) loader.template load<false, WAVES>(key_of(t + 1), next_pages, keys_at(t + 1), wave, lane);
    if (t < tiles) loader.template load<true, WAVES>(key_of(t), pages, values_at(t), wave, lane);
    pages = next_pages;
    next_pages = pages_of(t + 2);
  };
  // after the loads of tile t's values have ended, before they are read
  auto look = [&](int t) {
    if (t >= tiles || key_of(t) + KT <= all_sure) return;
    spoiled.scan(lds + (values_at(t) - base), threadIdx.x, 64 * WAVES);
    barrier();
    if (spoiled.any()) {
      uint32_t see[KB];
      see_tile(key_of(t), see);
      tile.sums.template spoil<KB>(spoiled.bits, see);
      barrier();
      spoiled.clear(threadIdx.x, 64 * WAVES);
    }
  };
  typename Tile::template Work<KB> work;
  if (tiles > 0) loader.template load<false, WAVES>(it.key0, pages, keys_at(0), wave, lane);
  typename Tile::Raw raw;
  Tile::fetch(raw, ItemRows<Row>(p, it, m0, lane).q(p, c, it, kv_head), p.head_dim, lane);
  tile.start(raw, p.scale * kAttnLog2e, lane);
  wait_loads<0>();
  barrier();
  // Two phases a tile: products (of the probabilities before and of this tile's scores), then the softmax.  Waves 4 to
  // 7, which share the SIMDs of waves 0 to 3, are a phase behind, so that one's products run beside the other's softmax.
  const bool behind = WAVES > 4 && wave >= 4;
  if (behind) {
    loads(0);
    barrier();
  }
  for (int t = 0; t <= tiles; ++t) {
    if (!behind) loads(t);
    if (any) {
      if (t > 0) tile.add(work, values_at(t - 1));
      if (t < tiles) tile.scores(work, keys_at(t));
    }
    if (behind) wait_loads<0>();
    barrier();
    if (behind) {
      look(t);
      loads(t + 1);
    }
    if (any && t < tiles) {
      const bool partly = key_of(t) + KT > all_sure;  // for some row of the workgroup
      uint32_t see[KB] = {};
      if (partly) see_tile(key_of(t), see);
      tile.softmax(work, partly, see);
    }
    if (!behind) wait_loads<0>();
    barrier();
    if (!behind) look(t);
  }
  if (WAVES > 4 && !behind) barrier();
  const float sum = half_pair_sum(tile.sums.sum);
  // made again, so that the loop's registers need not hold it
  const ItemRows<Row> rows(p, it, m0, (int)opaque((uint32_t)lane));
  const bool again = rows.real && sum != sum;
  if (!rows.real || again) {
  } else if (it.part < 0) {
    const float scale = 1.f / sum;
    Row* y = rows.y(p, c, it, kv_head);
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = 32 * b + 8 * i + 4 * tile.half;
        if (d < p.head_dim) store4(y + d, tile.sums.piece(b, i, tile.half) * scale);
      }
  } else {
    const size_t row = ((size_t)it.part * p.kv_heads + kv_head) * (32 * WAVES) + 32 * wave + (lane & 31);
    if (tile.half == 0) p.part_ml[row] = make_float2(tile.sums.reference, sum);
    float* y = p.part_y + row * DP;
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<floatx4*>(y + 32 * b + 8 * i + 4 * tile.half) = tile.sums.piece(b, i, tile.half);
  }
  for (uint32_t left = (uint32_t)__ballot(again); left; left &= left - 1) {
    const AttnArgs& args = args_again();
    whole_row<TYPE, Row, DP, 32 * WAVES>(args.p, args.c, it, kv_head, m0 + __builtin_ctz(left), nullptr);
  }
}

template <int TYPE, typename Row, int DP, int WAVES, int KT>
__global__ __launch_bounds__(64 * WAVES, WAVES / 4) void attn_shared_kernel(AttnPlan p, AttnCall c, AttnCut cut) {
  extern __shared__ __align__(16) uint8_t lds[];
  const int index = blockIdx.x / p.kv_heads, kv_head = blockIdx.x % p.kv_heads;
  if (index >= p.counts[0]) return;
  for (int t = uniform_load(p.workers + index).tile;; ++t) {
    // read again for every item, so that no register holds it meanwhile
    const AttnWorker worker = uniform_load(opaque_pointer(p.workers) + index);
    const AttnTile tile = uniform_load(p.tiles + t);
    const bool last = tile.start + attn_units(cut, tile.seen) >= worker.to;
    AttnItem it{tile.sequence, tile.begin, tile.length, tile.context, tile.m0, 0, 0, 0};
    if (attn_item(cut, worker, index, tile.seen, tile.start, it) && p.run[it.sequence])
      shared_item<TYPE, Row, DP, WAVES, KT>(p, c, it, kv_head, lds);
    if (last) break;
  }
}

// A call of few rows, of at most kAttnFewSequences sequences, needs no launch before the attend kernel: each of its
// workgroups makes the plan for itself, checks its sequence, and puts those of the new rows' keys and values that it
// is about to read into their pages.  (Others that read them put the same bytes there.)
struct FewLds {
  int64_t ends[kAttnFewSequences];  // units of a sequence's tiles and those before
  int64_t waves[4];
  int lengths[kAttnFewSequences], contexts[kAttnFewSequences];
  int first;                        // the sequence of the share's first unit
  int parents[kAttnTreeNodes];
  uint32_t tree[32][kAttnTreeWords];
};

// Share `index` of the call, by a workgroup of 64 WAVES threads; whether it has one.
template <int WAVES>
__device__ __forceinline__ bool few_share(const AttnPlan& p, const AttnCall& c, const AttnCut& cut, FewLds& m, int index,
                                          int kv_head, int64_t& from, int64_t& to, int64_t& share) {
  constexpr int B = 64 * WAVES;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const bool speaks = index == 0 && kv_head == 0;
  bool ascend = true;
  int64_t units = 0;
  for (int i0 = 0; i0 < c.sequences; i0 += B) {
    const int i = i0 + t;
    int64_t mine = 0;
    if (i < c.sequences) {
      int begin = i, length = 1, context = c.context[i];
      if (c.offsets) {
        begin = c.offsets[i];
        const int end = c.offsets[i + 1];
        ascend = ascend && begin >= 0 && end >= begin && end <= c.tokens;
        length = ascend ? end - begin : 0;
      }
      if (context < 0 || (int64_t)context + length > p.max_context) {
        if (speaks && length > 0) atomicOr(p.error, kAttnErrContext);
        context = length = 0;
      }
      m.lengths[i] = length;
      m.contexts[i] = context;
      for (int m0 = 0; m0 < length * (int)p.group.divisor; m0 += cut.rows)
        mine += attn_units(cut, attn_seen_keys(p, c, cut, m0, length, context)) + cut.overhead;
    }
    int64_t sum = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t u = __shfl_up(sum, o, 64);
      if (lane >= o) sum += u;
    }
    if (i0) __syncthreads();
    if (lane == 63) m.waves[wave] = sum;
    __syncthreads();
    int64_t all = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      if (w < wave) sum += m.waves[w];
      all += m.waves[w];
    }
    if (i < c.sequences) m.ends[i] = units + sum;
    units += all;
  }
  const bool holds = __syncthreads_and(ascend);
  if (speaks && t == 0) {
    if (!holds) atomicOr(p.error, kAttnErrOffsets);
    p.counts[1] = holds ? cut.shares : 0;
  }
  if (!holds) return false;
  share = attn_share(cut, units);
  from = index * share;
  to = min(from + share, units);
  if (t == 0 && kv_head == 0) p.joins[index].parts = 0;
  if (from >= units) return false;
  for (int i = t; i < c.sequences; i += B)
    if (m.ends[i] > from && (i == 0 || m.ends[i - 1] <= from)) m.first = i;
  __syncthreads();
  return true;
}

// Checks an item's sequence; then the new keys and values of its positions, the ancestors of its rows' tokens, and the
// list of its first pages.
template <int TYPE, typename Row, int WAVES>
__device__ __forceinline__ bool few_checked(const AttnPlan& p, const AttnCall& c, const AttnItem& it, int kv_head,
                                            FewLds& m, int* list) {
  typedef typename Cell<TYPE>::T T;
  constexpr int B = 64 * WAVES;
  const int t = threadIdx.x, first_page = it.key0 >> p.page_shift;
  const int pieces = p.head_dim / 8, first = max(it.key0, it.context), all = max(it.key1 - first, 0) * 2 * pieces;
  // some pieces of the rows at once, the first on their way beside the checks (a prompt of 33 tokens 19.6 us, one by one
  // behind the checks 20.5)
  constexpr int kAtOnce = 4;
  attn_eight<Row> v[kAtOnce];
  auto fetch = [&](int e0) {
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int e = min(e0 + i * B, all - 1), pos = first + e / (2 * pieces), piece = e % pieces;
      const bool value = e / pieces & 1;
      const int64_t row = it.begin + pos - it.context;
      v[i] = *reinterpret_cast<const attn_eight<Row>*>(static_cast<const Row*>(value ? c.v : c.k) +
                                                       row * (value ? c.v_stride : c.k_stride) +
                                                       kv_head * p.head_dim + piece * 8);
    }
  };
  if (t < all) fetch(t);
  int bad = 0;
  for (int e = t; e <= (it.context + it.length - 1) >> p.page_shift; e += B) {
    const int page = c.table[it.sequence * c.table_stride + e];
    if ((uint32_t)page >= (uint32_t)p.pages) bad = kAttnErrPage;
    if ((uint32_t)(e - first_page) < (uint32_t)kAttnPageList) list[e - first_page] = page;
  }
  if (c.parents) {
    if (it.length > kAttnTreeNodes) {
      bad |= kAttnErrTree;
    } else {
      for (int j = t; j < it.length; j += B) {
        m.parents[j] = c.parents[it.begin + j];
        if (m.parents[j] < -1 || m.parents[j] >= j) bad |= kAttnErrTree;
      }
    }
  }
  if (bad) atomicOr(p.error, bad);
  if (__syncthreads_or(bad)) return false;
  if (all == 0 && !c.parents) return true;
  for (int e0 = t; e0 < all;) {
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int e = e0 + i * B;
      if (e >= all) break;
      const int pos = first + e / (2 * pieces), piece = e % pieces;
      const bool value = e / pieces & 1;
      const int entry = (pos >> p.page_shift) - first_page;
      const int page = entry < kAttnPageList ? list[entry] : c.table[it.sequence * c.table_stride + first_page + entry];
      attn_put8(static_cast<T*>(value ? p.values : p.keys) + attn_cell(p, c.layer, page, pos) +
                    ((size_t)kv_head << p.page_shift) * p.head_dim + piece * 8,
                v[i]);
    }
    e0 += kAtOnce * B;
    if (e0 < all) fetch(e0);
  }
  if (c.parents && t < 32) {
    const int token = it.m0 / p.group + t;
    if (token < it.length) {
      uint32_t* words = m.tree[t];
#pragma unroll
      for (int w = 0; w < kAttnTreeWords; ++w) words[w] = 0;
      for (int n = token; n >= 0; n = m.parents[n]) words[n >> 5] |= 1u << (n & 31);
    }
  }
  wait_loads<0>();  // and stores: what the tiles' loads read is there
  __syncthreads();
  return true;
}

// Waves share 32 rows and take tiles of 32 keys in turn, each from LDS of its own; their sums are joined at the end.
template <int TYPE, typename Row, int DP, int WAVES>
struct SplitLds {
  static constexpr int kTile = 32 * DP * attn_cell_bytes<TYPE>();
  static constexpr int kWave = 4 * kTile;           // two tiles of keys and two of values
  static constexpr int kRow = DP + 4;               // floats of a row of sums, in the same memory
  static_assert(32 * kRow * 4 <= kWave, "a wavefront's sums fit its tiles");
  static constexpr int kSpoiled = Spoiled<attn_cell_bytes<TYPE>(), DP, 32>::kBytes / 4;
  static constexpr int kSums = (WAVES * 64 + kAttnPageList + WAVES * kSpoiled + 1) / 2 * 8;  // the few's are 8-byte aligned
  static constexpr int kBytes = WAVES * kWave + kSums + (int)sizeof(FewLds);
};

// Whether the item was done: not if its sequence is refused.
template <int TYPE, typename Row, int DP, int WAVES>
__device__ __forceinline__ bool split_item(const AttnPlan& p, const AttnCall& c, const AttnCut& cut, const AttnItem& it,
                                           int kv_head, uint8_t* lds) {
  constexpr int SIZE = attn_cell_bytes<TYPE>(), KT = 32;
  typedef TileLoader<SIZE, DP, KT> Loader;
  typedef SplitLds<TYPE, Row, DP, WAVES> M;
  typedef RowTile<TYPE, Row, DP> Tile;
  constexpr int kLoads = 2 * Loader::kLoads;
  float* const ml = reinterpret_cast<float*>(lds + WAVES * M::kWave);  // [WAVES][2][32]
  int* const list = reinterpret_cast<int*>(ml + WAVES * 64);
  FewLds& few = *reinterpret_cast<FewLds*>(lds + WAVES * M::kWave + M::kSums);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const ItemRows<Row> rows(p, it, it.m0, lane);
  typename Tile::Raw raw;
  constexpr bool kEarly = DP < 256;  // wide rows would take the registers of the checks
  if (kEarly) Tile::fetch(raw, rows.q(p, c, it, kv_head), p.head_dim, lane);
  if (cut.few && !few_checked<TYPE, Row, WAVES>(p, c, it, kv_head, few, list)) return false;
  Sight sight = rows.sight(p, c, it);
  if (cut.few && c.parents) sight.tree = few.tree[rows.token - it.m0 / p.group];
  const int sure = c.parents ? it.context : it.context + it.m0 / p.group + 1;
  Tile tile;  // started behind the first loads, which its rows need not wait for
  const Loader loader(p, c.layer, kv_head, it);
  const int* table = c.table + it.sequence * c.table_stride;
  const uint32_t lds_base = lds_address(lds), base = lds_base + wave * M::kWave;
  const Spoiled<SIZE, DP, KT> spoiled{reinterpret_cast<uint32_t*>(list + kAttnPageList) + wave * M::kSpoiled,
                                      attn_exponent<TYPE>()};
  // as many keys at a time as the list has pages for
  const int stretch = kAttnPageList << p.page_shift;
  for (int key0 = it.key0; key0 < it.key1;) {
    const int first = key0 >> p.page_shift;
    const int key1 = (int)min((int64_t)it.key1, ((int64_t)first << p.page_shift) + stretch);
    const int entries = loader.entry(key1 - 1, 0) - first + 1;
    if (!cut.few || key0 != it.key0) {
      if (key0 != it.key0) __syncthreads();
      for (int i = threadIdx.x; i < entries; i += 64 * WAVES) list[i] = table[first + i];
      __syncthreads();
    }
    auto load = [&](int key, int buffer) {
      const int pages = list[min(loader.entry(key, lane) - first, entries - 1)];
      loader.template load<false, 1>(key, pages, base + buffer * 2 * M::kTile, 0, lane);
      loader.template load<true, 1>(key, pages, base + buffer * 2 * M::kTile + M::kTile, 0, lane);
    };
    int key = key0 + KT * wave;
    if (key < key1) load(key, 0);
    if (key0 == it.key0) {
      if (!kEarly) Tile::fetch(raw, rows.q(p, c, it, kv_head), p.head_dim, lane);
      tile.start(raw, p.scale * kAttnLog2e, lane);
    }
    for (int t = 0; key < key1; ++t, key += KT * WAVES) {
      if (key + KT * WAVES < key1) {
        load(key + KT * WAVES, ~t & 1);
        wait_loads<kLoads <= 63 ? kLoads : 0>();
      } else {
        wait_loads<0>();
      }
      const uint32_t now = base + (t & 1) * 2 * M::kTile;
      uint32_t see[1] = {};
      const bool partly = key + KT > sure;
      if (partly) {
        see[0] = sight.bits(key);
        spoiled.clear(lane, 64);
        wave_lds_order();
        spoiled.scan(lds + (now - lds_base) + M::kTile, lane, 64);
        wave_lds_order();
      }
      typename Tile::template Work<1> work;
      tile.scores(work, now);
      tile.softmax(work, partly, see);
      tile.add(work, now + M::kTile);
      if (partly && spoiled.any()) tile.sums.template spoil<1>(spoiled.bits, see);
      wave_lds_order();  // the next load into this tile's place follows its reads
    }
    key0 = key1;
  }
  const float sum = half_pair_sum(tile.sums.sum);
  if (lane < 32) {
    ml[wave * 64 + lane] = tile.sums.reference;
    ml[wave * 64 + 32 + lane] = sum;
  }
  float* const own = reinterpret_cast<float*>(lds + wave * M::kWave) + (lane & 31) * M::kRow;
#pragma unroll
  for (int b = 0; b < DP / 32; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<floatx4*>(own + 32 * b + 8 * i + 4 * tile.half) = tile.sums.piece(b, i, tile.half);
  __syncthreads();
  const int count = min(32, rows.rows - it.m0);
  uint32_t again = 0;
#pragma unroll 2
  for (int i = threadIdx.x; i < count * (DP / 4); i += 64 * WAVES) {
    const int r = i / (DP / 4), d = 4 * (i % (DP / 4));
    if (d >= p.head_dim) continue;
    float reference = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) reference = fmaxf(reference, ml[w * 64 + r]);
    floatx4 v{};
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      // a wavefront that saw nothing for this row has zeros
      const float mine = ml[w * 64 + r];
      const float weight = mine == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(mine - reference);
      total += weight * ml[w * 64 + 32 + r];
      v += weight * *reinterpret_cast<const floatx4*>(lds + w * M::kWave + (r * M::kRow + d) * 4);
    }
    if (total != total) {  // formed anew below (a row's threads are one wavefront's)
      again |= 1u << r;
      continue;
    }
    if (it.part < 0) {
      const int m = it.m0 + r;
      Row* y = static_cast<Row*>(c.y) + (it.begin + m / p.group) * c.y_stride +
               (kv_head * (int)p.group.divisor + m % p.group) * p.head_dim;
      store4(y + d, v * (1.f / total));
    } else {
      const size_t row = ((size_t)it.part * p.kv_heads + kv_head) * 32 + r;
      if (d == 0) p.part_ml[row] = make_float2(reference, total);
      *reinterpret_cast<floatx4*>(p.part_y + row * DP + d) = v;
    }
  }
  if (__builtin_expect(__ballot(again != 0) != 0, 0))
    for (int r = 0; r < count; ++r) {
      if (!__ballot(again >> r & 1)) continue;
      const AttnArgs& args = args_again();
      whole_row<TYPE, Row, DP, 32>(args.p, args.c, it, kv_head, it.m0 + r, cut.few ? few.tree[0] : nullptr);
    }
  return true;
}

template <int TYPE, typename Row, int DP, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 1) void attn_split_kernel(AttnPlan p, AttnCall c, AttnCut cut) {
  typedef SplitLds<TYPE, Row, DP, WAVES> M;
  extern __shared__ __align__(16) uint8_t lds[];
  const int index = blockIdx.x / p.kv_heads, kv_head = blockIdx.x % p.kv_heads;
  if (!cut.few) {
    if (index >= p.counts[0]) return;
    const AttnWorker worker = uniform_load(p.workers + index);
    int64_t end = worker.from;
    for (int t = worker.tile; end < worker.to; ++t) {
      const AttnTile tile = uniform_load(p.tiles + t);
      end = tile.start + attn_units(cut, tile.seen);
      AttnItem it{tile.sequence, tile.begin, tile.length, tile.context, tile.m0, 0, 0, 0};
      if (!attn_item(cut, worker, index, tile.seen, tile.start, it) || !p.run[it.sequence]) continue;
      split_item<TYPE, Row, DP, WAVES>(p, c, cut, it, kv_head, lds);
      __syncthreads();  // the sums have been read
    }
    return;
  }
  FewLds& few = *reinterpret_cast<FewLds*>(lds + WAVES * M::kWave + M::kSums);
  int64_t from, to, share;
  if (!few_share<WAVES>(p, c, cut, few, index, kv_head, from, to, share)) return;
  auto uniform = [](int64_t v) {
    return (int64_t)((uint64_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 |
                     (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
  };
  AttnItem it;
  it.sequence = __builtin_amdgcn_readfirstlane(few.first);
  int64_t start = it.sequence ? uniform(few.ends[it.sequence - 1]) : 0;  // of a tile's overhead
  const AttnWorker worker{uniform(from), uniform(to), 0, attn_slack(uniform(share))};
  it.m0 = 0;
  while (start < worker.to) {
    it.length = __builtin_amdgcn_readfirstlane(few.lengths[it.sequence]);
    it.context = __builtin_amdgcn_readfirstlane(few.contexts[it.sequence]);
    if (it.m0 >= it.length * (int)p.group.divisor) {
      ++it.sequence;
      it.m0 = 0;
      continue;
    }
    const int seen = attn_seen_keys(p, c, cut, it.m0, it.length, it.context), units = attn_units(cut, seen);
    start += cut.overhead;
    if (attn_item(cut, worker, index, seen, start, it)) {
      it.begin = c.offsets ? __builtin_amdgcn_readfirstlane(c.offsets[it.sequence]) : it.sequence;
      const bool done = split_item<TYPE, Row, DP, WAVES>(p, c, cut, it, kv_head, lds);
      if (done && it.key0 == 0 && it.part >= 0 && threadIdx.x == 0 && kv_head == 0)
        p.joins[index] = attn_join(cut, it, seen, start, share, index);
      __syncthreads();  // the sums have been read
    }
    start += units;
    it.m0 += cut.rows;
  }
}

// ------------------------------------------------------------------ launches
template <typename Kernel>
hipError_t attn_launch(Kernel k, uint32_t grid, int threads, int lds, hipStream_t s, const AttnPlan& p,
                       const AttnCall& c, const AttnCut& cut) {
  if (lds > 65536) {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(k, dim3(grid), dim3(threads), lds, s, p, c, cut);
  return hipGetLastError();
}

// Waves that split keys: what LDS holds of their tiles.
template <int TYPE, int DP>
constexpr int attn_split_waves() {
  return DP * attn_cell_bytes<TYPE>() <= 256 ? 4 : DP * attn_cell_bytes<TYPE>() == 512 ? 2 : 1;
}

template <int TYPE, typename Row, int DP>
hipError_t attn_attend(const AttnPlan& p, const AttnCall& c, const AttnCut& cut, uint32_t grid, hipStream_t s) {
  if (cut.shared) {
    constexpr int W = attn_shared_waves(TYPE, sizeof(Row), DP), KT = attn_shared_keys(DP, sizeof(Row));
    return attn_launch(attn_shared_kernel<TYPE, Row, DP, W, KT>, grid, 64 * W,
                       4 * KT * DP * attn_cell_bytes<TYPE>() + Spoiled<attn_cell_bytes<TYPE>(), DP, KT>::kBytes, s, p, c, cut);
  }
  constexpr int W = attn_split_waves<TYPE, DP>();
  return attn_launch(attn_split_kernel<TYPE, Row, DP, W>, grid, 64 * W, SplitLds<TYPE, Row, DP, W>::kBytes, s, p, c, cut);
}

template <int TYPE, typename Row>
hipError_t attn_attend_width(const AttnPlan& p, const AttnCall& c, const AttnCut& cut, uint32_t grid, hipStream_t s) {
  switch (attn_padded(p.head_dim)) {
    case 64: return attn_attend<TYPE, Row, 64>(p, c, cut, grid, s);
    case 128: return attn_attend<TYPE, Row, 128>(p, c, cut, grid, s);
    default: return attn_attend<TYPE, Row, 256>(p, c, cut, grid, s);
  }
}

}  // namespace llhip
