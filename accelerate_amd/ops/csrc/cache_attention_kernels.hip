// Attention of a few new tokens of each sequence over a cache of keys and
// values in 16 or 8 bits.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale q_i . k_j - max_j)
//
// over the slots j before the new tokens and those new ones that the mask (a
// tree of drafted tokens) or the causal chain lets i see. One pass over the
// cache, with the running maximum and sum of the softmax in 32 bits.
//
// Bound by memory: all q heads of a group and all new tokens ("rows") share
// one reading of the group's keys and values. So the product is laid out for
// the reading:
//  * a wave takes 32 keys at a time and holds them in registers, straight
//    from memory: no LDS, and no wave waits for another until the end.
//  * S^T = K Q^T: a lane's operand is 16 bytes of one key, as it lies in
//    memory. The lane then holds, of one row, the scores of the keys
//    {4 g + r, 16 + 4 g + r} (g = lane / 16, r = 0..3).
//  * O^T = V^T P^T: those are taken as the lane's 8 summation indices, so
//    that the probabilities go from the first product to the second in
//    place. Each lane loads the same 8 keys' values, D / 16 neighbours of
//    each (16 lanes read one row of V), and the j-th of these makes the
//    operand of the j-th product, whose 16 output rows are the dimensions
//    j, j + D / 16, ...: the transposition of V is a choice of elements.
//  * 8-bit codes are exact in bf16 and fp16, e4m3 codes times their scale (a
//    power of two) in bf16. Other scales multiply, in 32 bits, the scores (the
//    keys') and the probabilities (the values'). Probabilities times scales
//    need more than fp16's range, so those values are operands in bf16 then.
// The cache's length is split over workgroups where there are too few heads
// and sequences to fill the chip; a second kernel joins the parts.
//
// Measured: 32 sequences of 8000 to 16000 int8 tokens, 64 query heads on 8:
// 151 us, 5.4 TB/s; one of 130001 bf16 tokens: 93 us, 5.7 TB/s (a stream that
// only reads: 5.9 to 6.2). One of 300: 7.7 us, the latency of a launch and three readings in turn.
// Of 108 rows (27 drafted tokens, 4 heads a group) over 8 sequences of 2000 to
// 4000 e4m3 tokens: 36 us, where the bytes would take 11: two waves a SIMD take
// about 1600 cycles a tile (1130 of vector and 770 of matrix instructions, which
// overlap in part), and the start, the end and the join 12 us.

#include <type_traits>

#include "serving.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int uint4v __attribute__((ext_vector_type(4)));

typedef float f32x2 __attribute__((ext_vector_type(2)));

template <typename T> struct Operand;
template <> struct Operand<__bf16> {
  typedef __bf16 V __attribute__((ext_vector_type(8)));
  typedef __bf16 Pair __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Operand<_Float16> {
  typedef _Float16 V __attribute__((ext_vector_type(8)));
  typedef _Float16 Pair __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

constexpr int kWaves = 4;
constexpr int kTile = 32;              // keys a wave takes at a time
constexpr int kStep = kWaves * kTile;  // keys a workgroup takes at a time
constexpr int kShort = 512;        // slots of a cache whose keys are not split
constexpr int kMaxSplits = 512, kFewSplits = 8;
constexpr float kNegInf = -__builtin_inff();
constexpr float kNothing = -0x1p127f;  // the maximum of no scores: finite, so that its difference to them is a number

// Two values as a word of an operand. (Values that are converted one by one
// are put together by two instructions more.)
template <typename T>
__device__ __forceinline__ unsigned pack2(float x, float y) {
  return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{x, y}, typename Operand<T>::Pair));
}

template <typename T>
__device__ __forceinline__ f32x2 unpack2(unsigned word) {
  return __builtin_convertvector(__builtin_bit_cast(typename Operand<T>::Pair, word), f32x2);
}

// The codes of the two low or high bytes of a word, exact; e4m3 times a power
// of two.
template <typename T, CacheKind kKind, bool kHigh>
__device__ __forceinline__ unsigned decode2(unsigned word, float scale = 1.f) {
  if constexpr (kKind == CacheKind::kInt8)
    return pack2<T>((float)(int8_t)(word >> (kHigh ? 16 : 0)), (float)(int8_t)(word >> (kHigh ? 24 : 8)));
  else if constexpr (__is_same(T, __bf16))
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, kHigh));
  else
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, scale, kHigh));
}

// The codes of byte j of two words.
template <typename T, CacheKind kKind>
__device__ __forceinline__ unsigned decode_bytes(unsigned a, unsigned b, int j) {
  if constexpr (kKind == CacheKind::kInt8) return pack2<T>((float)(int8_t)(a >> (8 * j)), (float)(int8_t)(b >> (8 * j)));
  else return decode2<T, kKind, false>(__builtin_amdgcn_perm(b, a, 0x0400u + 0x0101u * j));
}

// The largest of a value over the lanes c + 16 g of a row; and the sum.
template <typename F>
__device__ __forceinline__ float over_groups(float x, F f) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ float max_over_groups(float x) {
  return over_groups(x, [](float a, float b) { return fmaxf(a, b); });
}

__device__ __forceinline__ float sum_over_groups(float x) {
  return over_groups(x, [](float a, float b) { return a + b; });
}

// bytes of a lane's neighbours in one row, as words (a 2-byte one in the low half)
template <int kBytes>
struct Raw {
  static constexpr int kWords = (kBytes + 3) / 4;
  unsigned w[kWords];
  __device__ __forceinline__ void load(const uint8_t* p) {
    if constexpr (kBytes == 2) {
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    } else if constexpr (kBytes >= 16) {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4v x = *reinterpret_cast<const uint4v*>(p + 4 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[i + j] = x[j];
      }
    } else {
      typedef unsigned V __attribute__((ext_vector_type(kWords)));
      if constexpr (kWords == 1) {
        w[0] = *reinterpret_cast<const unsigned*>(p);
      } else {
        const V x = *reinterpret_cast<const V*>(p);
#pragma unroll
        for (int j = 0; j < kWords; ++j) w[j] = x[j];
      }
    }
  }
};

__device__ __forceinline__ int clamped_length(const AttendArgs& a, int b) {
  return min(max(a.lengths[b], 0), a.max_len);
}

// how many keys each split of the grid has: the sequence's own length is shared
// out in steps of a workgroup's keys, not the cache's. Splits whose keys would
// start behind all of them have none.
struct Share {
  int steps, all;
  __device__ __forceinline__ bool has(int split) const { return (int64_t)split * steps < all; }
};

__device__ __forceinline__ Share share_of(int end, const AttendArgs& a) {
  const int all = max(1, (end + kStep - 1) / kStep);
  return {(int)a.by_splits.quotient(all + a.splits - 1), all};
}

// A row of a group: its token, and its head of all.
struct RowOf {
  int t, head;
};

__device__ __forceinline__ RowOf row_of(const AttendArgs& a, int h, int row) {
  const int t = a.by_rep.quotient(row);
  return {t, h * a.rep + row - t * a.rep};
}

// A row whose probabilities sum to zero saw nothing and is zero, or all that
// it saw has a score of minus infinity, where the quotient is NaN.
__device__ __forceinline__ float empty_row(const AttendArgs& a, int b, int t, int n0) {
  bool any = n0 > 0;
  const int w_end = min(a.W, a.max_len - n0);
  if (!a.mask) any |= w_end > 0;
  else
    for (int j = 0; j < w_end && !any; ++j) any = a.mask[b * a.mb + t * a.mt + j] != 0;
  return any ? __builtin_nanf("") : 0.f;
}

// What a workgroup works on: a split of one sequence's and head's keys, and a
// block of rows. Workgroups go round the 8 XCDs in turn; those that read the
// same keys for other rows are 8 apart, so that they share an L2.
struct Work {
  int split, bh, b, h, rb, n0, end, from, stop;
  bool any;
};

template <bool kOne>
__device__ __forceinline__ Work work_of(const AttendArgs& a) {
  Work w;
  const int splits = kOne ? 1 : a.splits, parts = splits * a.Hkv * a.B;
  int part = blockIdx.x;
  w.rb = 0;
  if (a.row_blocks > 1) {
    const int xcd = blockIdx.x & 7, at = blockIdx.x >> 3;
    const int of = a.by_row_blocks.quotient(at);
    w.rb = at - of * a.row_blocks;
    part = of * 8 + xcd;
  }
  w.any = part < parts;
  const int bh = kOne ? part : a.by_splits.quotient(part);
  w.split = part - bh * splits;
  w.bh = w.any ? bh : 0;
  w.b = a.by_heads.quotient(w.bh);
  w.h = w.bh - w.b * a.Hkv;
  w.n0 = clamped_length(a, w.b);
  w.end = (int)min((int64_t)w.n0 + a.W, (int64_t)a.max_len);
  if constexpr (kOne) {
    w.from = 0;
    w.stop = w.end;
  } else {
    const Share share = share_of(w.end, a);
    w.any = w.any && share.has(w.split);
    const int64_t from = (int64_t)w.split * share.steps * kStep;
    w.from = (int)from;
    w.stop = (int)min((int64_t)w.end, from + share.steps * kStep);
  }
  return w;
}

template <typename T, CacheKind kKind, int kD>
struct Shape {
  static constexpr bool kSame = kKind == CacheKind::kSame;
  // e4m3 codes times their scale, a power of two, are exact in bf16's range.
  // Other scales multiply scores and probabilities, in 32 bits.
  static constexpr bool kFolded = kKind == CacheKind::kFp8 && __is_same(T, __bf16);
  static constexpr bool kScaled = !kSame && !kFolded;
  typedef std::conditional_t<kScaled, __bf16, T> VT;  // of the second product's operands
  static constexpr int kBytes = kSame ? 2 : 1;
  static constexpr int kRowBytes = kD * kBytes;
  static constexpr int kQK = kD / 32;  // products a tile of 16 keys
  static constexpr int kND = kD / 16;  // a lane's neighbours of a row of V, and products
  // 8-bit keys are loaded 16 values at a time, the two halves of which belong
  // to two products; the queries follow that order
  static constexpr bool kPaired = !kSame && kD >= 64;
  static constexpr unsigned kExp = __is_same(T, __bf16) ? 0x7F80u : 0x7C00u;  // of an infinity or NaN
};

// 32 keys and their values, as a wave loads them, and as operands.
template <typename T, CacheKind kKind, int kD>
struct Tile : Shape<T, kKind, kD> {
  using S = Shape<T, kKind, kD>;
  using OV = typename Operand<T>::V;
  using VT = typename S::VT;
  using VOV = typename Operand<VT>::V;
  static constexpr int kLoad = S::kSame || S::kPaired ? 16 : 8;
  static constexpr int kLoads = S::kPaired ? S::kQK / 2 : S::kQK;
  Raw<kLoad> k[2][kLoads];
  Raw<S::kND * S::kBytes> v[8];
  float kown[2];          // kFolded: the scales of the keys c of the two halves
  f32x4 kscale[2], vscale[2];  // of the keys 4 g + r of the two halves

  __device__ __forceinline__ void load_keys(const uint8_t* keys, const float* scales, int key0, int c, int g) {
    const uint8_t* p = keys + (int64_t)key0 * S::kRowBytes + c * S::kRowBytes + g * kLoad;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) k[t][i].load(p + t * 16 * S::kRowBytes + i * 64);
      if constexpr (S::kFolded) kown[t] = scales[key0 + t * 16 + c];
      if constexpr (S::kScaled) kscale[t] = *reinterpret_cast<const f32x4*>(scales + key0 + t * 16 + g * 4);
    }
  }

  __device__ __forceinline__ void load_values(const uint8_t* values, const float* scales, int key0, int c, int g) {
    const uint8_t* p = values + (int64_t)key0 * S::kRowBytes + g * 4 * S::kRowBytes + c * S::kND * S::kBytes;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e].load(p + ((e >> 2) * 16 + (e & 3)) * S::kRowBytes);
    if constexpr (!S::kSame) {
#pragma unroll
      for (int t = 0; t < 2; ++t) vscale[t] = *reinterpret_cast<const f32x4*>(scales + key0 + t * 16 + g * 4);
    }
  }

  __device__ __forceinline__ OV key(int t, int ds) const {
    if constexpr (S::kSame) {
      return __builtin_bit_cast(OV, k[t][ds]);
    } else {
      const auto& raw = k[t][S::kPaired ? ds / 2 : ds];
      const int w0 = S::kPaired ? (ds & 1) * 2 : 0;
      const float scale = S::kFolded ? kown[t] : 1.f;
      return __builtin_bit_cast(
          OV, uint4v{decode2<T, kKind, false>(raw.w[w0], scale), decode2<T, kKind, true>(raw.w[w0], scale),
                     decode2<T, kKind, false>(raw.w[w0 + 1], scale), decode2<T, kKind, true>(raw.w[w0 + 1], scale)});
    }
  }

  // Operands j and j + 1: the j-th and next values of the lane's eight keys.
  __device__ __forceinline__ void value2(int j, VOV& x, VOV& y) const {
    uint4v lo, hi;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      if constexpr (S::kScaled) {
        lo[e / 2] = decode_bytes<VT, kKind>(v[e].w[j / 4], v[e + 1].w[j / 4], j & 3);
        hi[e / 2] = decode_bytes<VT, kKind>(v[e].w[j / 4], v[e + 1].w[j / 4], (j & 3) + 1);
      } else {
        unsigned a, b;
        if constexpr (S::kSame) {
          a = v[e].w[j / 2];
          b = v[e + 1].w[j / 2];
        } else if (j & 2) {
          a = decode2<T, kKind, true>(v[e].w[j / 4], vscale[e >> 2][e & 3]);
          b = decode2<T, kKind, true>(v[e + 1].w[j / 4], vscale[e >> 2][(e & 3) + 1]);
        } else {
          a = decode2<T, kKind, false>(v[e].w[j / 4], vscale[e >> 2][e & 3]);
          b = decode2<T, kKind, false>(v[e + 1].w[j / 4], vscale[e >> 2][(e & 3) + 1]);
        }
        lo[e / 2] = __builtin_amdgcn_perm(b, a, 0x05040100u);
        hi[e / 2] = __builtin_amdgcn_perm(b, a, 0x07060302u);
      }
    }
    x = __builtin_bit_cast(VOV, lo);
    y = __builtin_bit_cast(VOV, hi);
  }

  // A probability of zero does not hide an infinite or NaN value. In a tile
  // with slots that some rows do not see, slots behind the new tokens (which
  // hold anything) are cleared; of the others, values that are not finite are
  // left out and found again at the end, for the rows that see them. Says
  // whether there are any.
  __device__ __forceinline__ bool clear(int key0, int end, int g) {
    bool odd = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool in = key0 + (e >> 2) * 16 + g * 4 + (e & 3) < end;
      if constexpr (S::kSame) {
#pragma unroll
        for (int w = 0; w < Raw<S::kND * S::kBytes>::kWords; ++w) {
          unsigned& x = v[e].w[w];
          const unsigned low = (x & S::kExp) == S::kExp ? 0xFFFFu : 0u;
          const unsigned high = ((x >> 16) & S::kExp) == S::kExp ? 0xFFFF0000u : 0u;
          odd |= in & ((low | high) != 0);
          x = in ? x & ~(low | high) : 0u;
        }
      } else {  // codes are finite, their scale may not be
        const float x = vscale[e >> 2][e & 3];
        const bool finite = x < __builtin_inff();
        odd |= in & !finite;
        vscale[e >> 2][e & 3] = in & finite ? x : 0.f;
      }
    }
    return odd;
  }
};

// A wave's rows: queries, running maximum and sum of the softmax, and sums of
// values. Row c of tile mt belongs to the four lanes c + 16 g.
template <typename T, CacheKind kKind, int kD, int kMT>
struct Rows : Shape<T, kKind, kD> {
  using S = Shape<T, kKind, kD>;
  using OV = typename Operand<T>::V;
  using VT = typename S::VT;
  using VOV = typename Operand<VT>::V;
  // Probabilities of at most 1 use fp16's range from below alone: they are
  // operands in units of 2^-15, and what is lost then is below 2^-40.
  static constexpr float kLift = __is_same(VT, _Float16) ? 0x1p15f : 1.f;
  OV q[kMT][S::kQK];
  f32x4 o[kMT][S::kND];
  float m[kMT], l[kMT];
  float scale;  // of the scores where the keys' are none, not negative

  __device__ __forceinline__ void start(const AttendArgs& a, const Work& w, int row0, int c, int g) {
    // Rows behind the last repeat it; no row reaches another's result, and
    // they are not written.
    const int rows = a.T * a.rep;
    // The largest score is the largest product, so that only one a row has to
    // be scaled before the exponentials. A negative scale turns the queries.
    scale = fmaxf(fabsf(a.scale_log2), 0x1p-126f);  // not zero: times minus infinity that is NaN
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt) {
      const int row = min(row0 + mt * 16 + c, rows - 1);
      const RowOf r = row_of(a, w.h, row);
      const T* src = reinterpret_cast<const T*>(a.q) + w.b * a.qb + r.head * a.qh + r.t * a.qt;
#pragma unroll
      for (int ds = 0; ds < S::kQK; ++ds) {
        const int d = S::kPaired ? (ds / 2) * 64 + g * 16 + (ds & 1) * 8 : ds * 32 + g * 8;
        q[mt][ds] = __builtin_bit_cast(OV, *reinterpret_cast<const uint4v*>(src + d));
      }
      m[mt] = kNothing;
      l[mt] = 0.f;
#pragma unroll
      for (int j = 0; j < S::kND; ++j) o[mt][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }

  __device__ __forceinline__ void turn(const AttendArgs& a) {
    if constexpr (!S::kScaled) {
      const unsigned sign = a.scale_log2 < 0.f ? 0x80008000u : 0u;
#pragma unroll
      for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
        for (int ds = 0; ds < S::kQK; ++ds) q[mt][ds] = __builtin_bit_cast(OV, __builtin_bit_cast(uint4v, q[mt][ds]) ^ sign);
    }
  }

  // Scores of the 32 keys from key0 on to probabilities, as operands; o and l
  // follow the maximum.
  __device__ __forceinline__ void soften(const AttendArgs& a, const Work& w, const f32x4 (&s)[kMT][2],
                                         const f32x4* kscale, const f32x4* vscale, int key0, int row0, int c, int g,
                                         VOV (&pv)[kMT][2]) {
    const bool masked = key0 + kTile > w.n0;  // the tile has slots that some rows do not see
    bool grew = false;
    float p[kMT][8], keep[kMT];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float ksc = S::kScaled ? kscale[e >> 2][e & 3] * a.scale_log2 : 1.f;
#pragma unroll
      for (int mt = 0; mt < kMT; ++mt) p[mt][e] = S::kScaled ? s[mt][e >> 2][e & 3] * ksc : s[mt][e >> 2][e & 3];
    }
    if (masked) {
      // Selects, no branches: an array element written under a lane's own
      // condition was lost by the compiler.
#pragma unroll
      for (int mt = 0; mt < kMT; ++mt) {
        const int t_row = a.by_rep.quotient(row0 + mt * 16 + c);
        // all of a lane's mask values are read at once, from inside the mask
        const bool chain = a.mask == nullptr;
        const uint8_t* bits = a.mask + w.b * a.mb + min(t_row, a.T - 1) * a.mt;
        uint8_t bit[8] = {};
        if (!chain && a.W > 0) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            bit[e] = bits[min(max(key0 + (e >> 2) * 16 + g * 4 + (e & 3) - w.n0, 0), a.W - 1)];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int key = key0 + (e >> 2) * 16 + g * 4 + (e & 3);
          const bool sees = (key < w.n0) | ((key < w.end) & (chain ? key - w.n0 <= t_row : bit[e] != 0));
          p[mt][e] = sees ? p[mt][e] : kNegInf;
        }
      }
    }
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt) {
      float top = fmaxf(p[mt][0], p[mt][1]);
#pragma unroll
      for (int e = 2; e < 8; ++e) top = fmaxf(top, p[mt][e]);
      top = max_over_groups(top);
      if constexpr (!S::kScaled) top *= scale;
      // Not below the product as it is, half a step of which was rounded off:
      // a probability above 1 would leave fp16's range (from scores of 2^24 on).
      if constexpr (kLift != 1.f) top = __builtin_fmaf(fabsf(top), 0x1p-23f, top);
      const float m_new = fmaxf(m[mt], top);
      keep[mt] = __builtin_amdgcn_exp2f(m[mt] - m_new);
      grew |= m_new > m[mt];
      m[mt] = m_new;
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[mt][e] = __builtin_amdgcn_exp2f(S::kScaled ? p[mt][e] - m_new : __builtin_fmaf(p[mt][e], scale, -m_new));
        sum += p[mt][e];
      }
      l[mt] = l[mt] * keep[mt] + sum;
    }

    if (__any(grew)) {
#pragma unroll
      for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
        for (int j = 0; j < S::kND; ++j) o[mt][j] *= keep[mt];
    }

    // Probabilities as operands: rounded to the type, and the rounding of what
    // that left out. One alone adds half a step of the type a key to the
    // result's own (an error of 0.0023 of random bf16 values, 0.0017 with two).
    // The second product costs nothing where the reading of the keys bounds,
    // and 3 to 6 % at 108 rows. Two of bf16 hold 16 bits of a probability, two
    // of fp16 22, where the result has 8 or 11.
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt) {
      uint4v x, rest;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        float p0 = p[mt][e], p1 = p[mt][e + 1];
        if constexpr (S::kScaled) {
          p0 *= vscale[e >> 2][e & 3];
          p1 *= vscale[e >> 2][(e & 3) + 1];
        } else if constexpr (kLift != 1.f) {
          p0 *= kLift;
          p1 *= kLift;
        }
        x[e / 2] = pack2<VT>(p0, p1);
        const f32x2 is = unpack2<VT>(x[e / 2]);
        rest[e / 2] = pack2<VT>(p0 - is[0], p1 - is[1]);
      }
      pv[mt][0] = __builtin_bit_cast(VOV, x);
      pv[mt][1] = __builtin_bit_cast(VOV, rest);
    }
  }

  // The sums of a row over its four lanes; o in units of 1.
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt) {
      l[mt] = sum_over_groups(l[mt]);
      if constexpr (kLift != 1.f) {
#pragma unroll
        for (int j = 0; j < S::kND; ++j) o[mt][j] *= 1.f / kLift;
      }
    }
  }
};

// Where the workgroup's slots that row t sees have infinite or NaN values (8
// bits: scales), their sum is the row's, whatever the others are: N dimensions
// from d on. The masked tiles left them out, and elsewhere a product with one
// of a probability's two operands may have made NaN of an infinity.
template <typename T, int N>
__device__ void take_odd(const AttendArgs& a, const Work& w, int t, const uint8_t* values, const float* scales, int d,
                         float* y) {
  struct alignas(N * 2 < 16 ? N * 2 : 16) Values { T v[N]; };
  float odd[N] = {};
  for (int j = w.from; j < w.stop; ++j) {
    if (j >= w.n0 && !(a.mask ? a.mask[w.b * a.mb + t * a.mt + (j - w.n0)] != 0 : j - w.n0 <= t)) continue;
    if (scales) {
      if (!__builtin_isfinite(scales[j])) odd[0] = __builtin_nanf("");
    } else {
      const Values v = *reinterpret_cast<const Values*>(reinterpret_cast<const T*>(values) + (int64_t)j * a.D + d);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (!__builtin_isfinite((float)v.v[i])) odd[i] += (float)v.v[i];
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float x = scales ? odd[0] : odd[i];
    if (x != 0.f) y[i] = x;  // NaN too
  }
}

// N dimensions of a row from d on, as the result or as a split's part of it.
template <typename T, int N, bool kOne>
__device__ __forceinline__ void write_row(const AttendArgs& a, const Work& w, int row, int d, const float* y, float top,
                                          float sum) {
  if (kOne || a.splits == 1) {
    const RowOf r = row_of(a, w.h, row);
    const float inverse = 1.f / sum;
    const float none = sum == 0.f ? empty_row(a, w.b, r.t, w.n0) : 0.f;
    struct alignas(N * 2 < 16 ? N * 2 : 16) { T v[N]; } out;
#pragma unroll
    for (int j = 0; j < N; ++j) out.v[j] = (T)(sum == 0.f ? none : y[j] * inverse);
    *reinterpret_cast<decltype(out)*>(reinterpret_cast<T*>(a.out) + w.b * a.ob + r.head * a.oh + r.t * a.ot + d) = out;
  } else {
    const int64_t at = ((int64_t)w.bh * a.T * a.rep + row) * a.splits + w.split;
    struct alignas(N * 4 < 16 ? N * 4 : 16) { float v[N]; } out;
#pragma unroll
    for (int j = 0; j < N; ++j) out.v[j] = y[j];
    *reinterpret_cast<decltype(out)*>(a.part_o + at * a.D + d) = out;
    if (d == 0) {
      a.part_ml[at * 2] = top;
      a.part_ml[at * 2 + 1] = sum;
    }
  }
}

// The four waves of a workgroup take tiles of keys in turn, all for the same
// 16 kMT rows, and join in the end. Where a short cache's keys are all one
// workgroup's (kOne) the first tiles are loaded before the length is known, which
// took 0.4 us off 300 keys. (Eight waves there: 300 keys of 8 heads 7.9 us for
// 7.7, 510 10.2 for 9.0, of 64 sequences 26.5 for 23.3.)
template <typename T, CacheKind kKind, int kD, int kMT, bool kOne>
__global__ void __launch_bounds__(256, (kD == 256 ? 1 : 2)) attend_kernel(AttendArgs a) {
  using S = Shape<T, kKind, kD>;
  using OV = typename Operand<T>::V;
  using VT = typename S::VT;
  using VOV = typename Operand<VT>::V;
  constexpr int kND = S::kND;
  constexpr int kV = kND < 4 ? kND : 4;
  typedef float Some __attribute__((ext_vector_type(kV)));
  __shared__ Some red[kWaves][kMT][4][kND / kV][64];
  __shared__ float red_m[kWaves][kMT][16], red_l[kWaves][kMT][16];
  __shared__ int red_odd[kWaves];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const Work w = work_of<kOne>(a);
  if (!w.any) return;
  const int row0 = w.rb * kMT * 16;
  const uint8_t* keys = reinterpret_cast<const uint8_t*>(a.k) + (int64_t)w.bh * a.slots * S::kRowBytes;
  const uint8_t* values = reinterpret_cast<const uint8_t*>(a.v) + (int64_t)w.bh * a.slots * S::kRowBytes;
  const float* ks = S::kSame ? nullptr : a.k_scale + (int64_t)w.bh * a.slots;
  const float* vs = S::kSame ? nullptr : a.v_scale + (int64_t)w.bh * a.slots;
  bool odd = false;  // whether masked tiles have values that are not finite

  // A tile's keys are loaded while the tile before is exponentiated and
  // multiplied with its values, its values while its own scores are made: the
  // registers of one are free when the other's next loads start. No load is
  // conditional: a wave without keys, or without more, reads its last tile or
  // the sequence's first once more, from a cache. Registers that a branch may
  // leave unwritten were given away by the compiler while they were in use.
  // The order of the first loads (queries, keys, values) is held fixed: the
  // loop's waits are for the worst of its entries, and with the keys or the
  // queries last each tile's values were waited for before its scores (32
  // sequences of 8000 to 16000 int8 tokens: 154.9 us for 151.3).
  Tile<T, kKind, kD> tile;
  const int first = w.from + wave * kTile;
  const int safe = kOne ? min(first, a.slots - kTile) : first < w.stop ? first : 0;
  Rows<T, kKind, kD, kMT> rows;
  rows.start(a, w, row0, c, g);
  __builtin_amdgcn_sched_barrier(0);
  tile.load_keys(keys, ks, safe, c, g);
  __builtin_amdgcn_sched_barrier(0);
  tile.load_values(values, vs, safe, c, g);
  __builtin_amdgcn_sched_barrier(0);
  rows.turn(a);
  for (int key0 = first; key0 < w.stop; key0 += kStep) {
    const int next = key0 + kStep < w.stop ? key0 + kStep : key0;
    f32x4 s[kMT][2];
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt) s[mt][0] = s[mt][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ds = 0; ds < S::kQK; ++ds) {
      const OV k0 = tile.key(0, ds), k1 = tile.key(1, ds);
#pragma unroll
      for (int mt = 0; mt < kMT; ++mt) {
        s[mt][0] = Operand<T>::mfma(k0, rows.q[mt][ds], s[mt][0]);
        s[mt][1] = Operand<T>::mfma(k1, rows.q[mt][ds], s[mt][1]);
      }
    }
    const f32x4 kscale[2] = {tile.kscale[0], tile.kscale[1]};
    tile.load_keys(keys, ks, next, c, g);
    if (key0 + kTile > w.n0) odd |= tile.clear(key0, w.end, g);
    VOV pv[kMT][2];
    rows.soften(a, w, s, kscale, tile.vscale, key0, row0, c, g, pv);
#pragma unroll
    for (int j = 0; j < kND; j += 2) {
      VOV v0, v1;
      tile.value2(j, v0, v1);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt) {
          rows.o[mt][j] = Operand<VT>::mfma(v0, pv[mt][i], rows.o[mt][j]);
          rows.o[mt][j + 1] = Operand<VT>::mfma(v1, pv[mt][i], rows.o[mt][j + 1]);
        }
    }
    tile.load_values(values, vs, next, c, g);
  }

  // The four waves' parts of a row, joined: wave i sums the elements r = i,
  // neighbours of row c from (4 g + i) D / 16 on.
  rows.finish();
  const bool wave_odd = __any(odd);
  if (lane == 0) red_odd[wave] = wave_odd;
  if (g == 0) {
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt) {
      red_m[wave][mt][c] = rows.m[mt];
      red_l[wave][mt][c] = rows.l[mt];
    }
  }
#pragma unroll
  for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < kND; j += kV) {
        Some x;
#pragma unroll
        for (int i = 0; i < kV; ++i) x[i] = rows.o[mt][j + i][r];
        red[wave][mt][r][j / kV][lane] = x;
      }
  __syncthreads();
  const bool any_odd = (red_odd[0] | red_odd[1] | red_odd[2] | red_odd[3]) != 0;
#pragma unroll
  for (int mt = 0; mt < kMT; ++mt) {
    float top = kNothing, sum = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) top = fmaxf(top, red_m[i][mt][c]);
    float y[kND] = {};
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      const float weight = __builtin_amdgcn_exp2f(red_m[i][mt][c] - top);
      sum += red_l[i][mt][c] * weight;
#pragma unroll
      for (int j = 0; j < kND; j += kV) {
        const Some x = red[i][mt][wave][j / kV][lane];
#pragma unroll
        for (int e = 0; e < kV; ++e) y[j + e] += x[e] * weight;
      }
    }
    const int row = row0 + mt * 16 + c;
    if (row < a.T * a.rep) {
      const int d = (g * 4 + wave) * kND;
      bool nan = false;
#pragma unroll
      for (int j = 0; j < kND; ++j) nan |= y[j] != y[j];
      if (any_odd || (nan && sum == sum)) take_odd<T, kND>(a, w, a.by_rep.quotient(row), values, vs, d, y);
      write_row<T, kND, kOne>(a, w, row, d, y, top, sum);
    }
  }
}

// A split's part of a sum. One that is infinite or NaN is the sum's, however
// little the split weighs: its weight may be zero in 32 bits.
__device__ __forceinline__ float weighted(float x, float weight) { return __builtin_isfinite(x) ? x * weight : x; }

// The splits of a row, joined, where they are few: D / 4 lanes a row, each of
// four dimensions. (With a workgroup a row, below, calls of 2 to 8 splits take
// 1 us more, 6 where the rows are many: 8 x 8 x 108 rows.)
template <typename T, int kD>
__global__ void __launch_bounds__(256) attend_join_few_kernel(AttendArgs a) {
  constexpr int kLanes = kD / 4;
  const int rows = a.T * a.rep;
  const int lane = threadIdx.x % kLanes;
  const int64_t at_row = (int64_t)blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  if (at_row >= (int64_t)a.B * a.Hkv * rows) return;
  const int bh = a.by_rows.quotient((unsigned)at_row), row = (int)at_row - bh * rows;
  const int b = a.by_heads.quotient(bh), h = bh - b * a.Hkv;
  const int n0 = clamped_length(a, b);
  const Share share = share_of((int)min((int64_t)n0 + a.W, (int64_t)a.max_len), a);
  const float* ml = a.part_ml + at_row * a.splits * 2;
  const float* part = a.part_o + at_row * a.splits * kD + lane * 4;
  float m[kFewSplits], l[kFewSplits];
  f32x4 o[kFewSplits];
  float top = kNothing;
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) {  // in place of a split without keys the first, with no weight
    const int at = s < a.splits && share.has(s) ? s : 0;
    m[s] = ml[at * 2];
    l[s] = ml[at * 2 + 1];
    o[s] = *reinterpret_cast<const f32x4*>(part + at * kD);
    top = fmaxf(top, m[s]);
  }
  float sum = 0.f;
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) {
    const float weight = __builtin_amdgcn_exp2f(m[s] - top);
    const bool is = s < a.splits && share.has(s);
    sum += is ? l[s] * weight : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] += is ? weighted(o[s][i], weight) : 0.f;
  }
  const RowOf r = row_of(a, h, row);
  const float none = sum == 0.f ? empty_row(a, b, r.t, n0) : 0.f, inverse = 1.f / sum;
  struct alignas(8) { T v[4]; } out;
#pragma unroll
  for (int i = 0; i < 4; ++i) out.v[i] = (T)(sum == 0.f ? none : y[i] * inverse);
  *reinterpret_cast<decltype(out)*>(reinterpret_cast<T*>(a.out) + b * a.ob + r.head * a.oh + r.t * a.ot + lane * 4) = out;
}

// Where they are many: a workgroup a row. Its threads take four
// dimensions each and share the splits out, so that few rows of many splits
// (one long sequence) still have many reads under way.
template <typename T, int kD>
__global__ void __launch_bounds__(256) attend_join_kernel(AttendArgs a) {
  constexpr int kLanes = kD / 4, kGroups = 256 / kLanes;
  __shared__ f32x4 red[kGroups][kLanes];
  __shared__ float weight[kMaxSplits], red_m[4], red_l[4];
  const int rows = a.T * a.rep, tid = threadIdx.x;
  const int bh = a.by_rows.quotient(blockIdx.x), row = blockIdx.x - bh * rows;
  const int b = a.by_heads.quotient(bh), h = bh - b * a.Hkv;
  const int n0 = clamped_length(a, b);
  const Share share = share_of((int)min((int64_t)n0 + a.W, (int64_t)a.max_len), a);
  const int64_t at = (int64_t)blockIdx.x * a.splits;

  float m[kMaxSplits / 256], l[kMaxSplits / 256], top = kNothing;
#pragma unroll
  for (int i = 0; i < kMaxSplits / 256; ++i) {
    const int s = tid + i * 256;
    m[i] = kNothing;
    l[i] = 0.f;
    if (s < a.splits && share.has(s)) {
      m[i] = a.part_ml[(at + s) * 2];
      l[i] = a.part_ml[(at + s) * 2 + 1];
    }
    top = fmaxf(top, m[i]);
  }
#pragma unroll
  for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
  if ((tid & 63) == 0) red_m[tid >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(red_m[0], red_m[1]), fmaxf(red_m[2], red_m[3]));
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kMaxSplits / 256; ++i) {
    const float w = __builtin_amdgcn_exp2f(m[i] - top);
    weight[tid + i * 256] = w;
    sum += l[i] * w;
  }
#pragma unroll
  for (int x = 32; x; x >>= 1) sum += __shfl_xor(sum, x);
  if ((tid & 63) == 0) red_l[tid >> 6] = sum;
  __syncthreads();
  sum = red_l[0] + red_l[1] + red_l[2] + red_l[3];

  const int lane = tid % kLanes, group = tid / kLanes;
  const float* part = a.part_o + at * kD + lane * 4;
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = group; s < a.splits && share.has(s); s += kGroups) {
    const f32x4 x = *reinterpret_cast<const f32x4*>(part + (int64_t)s * kD);
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] += weighted(x[i], weight[s]);
  }
  red[group][lane] = y;
  __syncthreads();
  if (tid >= kD) return;
  float out = 0.f;
#pragma unroll
  for (int i = 0; i < kGroups; ++i) out += red[i][tid / 4][tid % 4];
  const RowOf r = row_of(a, h, row);
  out = sum == 0.f ? empty_row(a, b, r.t, n0) : out / sum;
  reinterpret_cast<T*>(a.out)[b * a.ob + r.head * a.oh + r.t * a.ot + tid] = (T)out;
}

template <typename T, CacheKind kKind, int kD, bool kOne>
void attend_rows(const AttendArgs& a, hipStream_t stream) {
  const int64_t parts = (int64_t)a.splits * a.Hkv * a.B;
  const int64_t blocks = a.row_blocks == 1 ? parts : (parts + 7) / 8 * 8 * a.row_blocks;
  const dim3 grid((unsigned)blocks), block(256);
  if (a.T * a.rep <= 16) hipLaunchKernelGGL((attend_kernel<T, kKind, kD, 1, kOne>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((attend_kernel<T, kKind, kD, 2, kOne>), grid, block, 0, stream, a);
}

template <typename T, CacheKind kKind, int kD>
hipError_t attend_by_rows(const AttendArgs& a, hipStream_t stream) {
  if (a.max_len <= kShort) attend_rows<T, kKind, kD, true>(a, stream);
  else attend_rows<T, kKind, kD, false>(a, stream);
  const int64_t rows = (int64_t)a.B * a.Hkv * a.T * a.rep, per = 256 / (kD / 4);
  if (a.splits > kFewSplits)
    hipLaunchKernelGGL((attend_join_kernel<T, kD>), dim3((unsigned)rows), dim3(256), 0, stream, a);
  else if (a.splits > 1)
    hipLaunchKernelGGL((attend_join_few_kernel<T, kD>), dim3((unsigned)((rows + per - 1) / per)), dim3(256), 0, stream, a);
  return hipGetLastError();
}

template <typename T, CacheKind kKind>
hipError_t attend_by_dim(const AttendArgs& a, hipStream_t stream) {
  switch (a.D) {
    case 32: return attend_by_rows<T, kKind, 32>(a, stream);
    case 64: return attend_by_rows<T, kKind, 64>(a, stream);
    case 128: return attend_by_rows<T, kKind, 128>(a, stream);
    default: return attend_by_rows<T, kKind, 256>(a, stream);
  }
}

template <typename T>
hipError_t attend_by_kind(const AttendArgs& a, CacheKind kind, hipStream_t stream) {
  switch (kind) {
    case CacheKind::kInt8: return attend_by_dim<T, CacheKind::kInt8>(a, stream);
    case CacheKind::kFp8: return attend_by_dim<T, CacheKind::kFp8>(a, stream);
    default: return attend_by_dim<T, CacheKind::kSame>(a, stream);
  }
}

}  // namespace

// Row blocks: 32 rows leave two waves a SIMD room. 64 (one wave) took 68 us
// where these take 41 (8 sequences, 8 heads, 108 rows, 4000 e4m3 keys); a
// workgroup that shares its decoded keys among 128 rows, in LDS, took 43.
//
// Splits of the keys: the host does not know the lengths, so the cache's size
// stands for them; a shorter sequence is shared out over the same number, as
// far as its steps go.
//  * Up to 4 steps there is one, and no second launch (300 keys of 8 heads: 7.7
//    us bf16 and 6.0 e4m3 with one, 7.9 and 7.3 with three; 500: 9.0 and 6.9, 8.0
//    and 7.2 with four; a second launch takes the host 3 us more).
//  * Else one workgroup a CU: 16000 keys of 8 heads take 17.3 (bf16) and 11.8
//    us (int8) with 32 splits, 19.1 and 14.1 with 64; 130000 95.0 and 46.8, 96.4
//    and 48.3.
//  * Two for several sequences whose parts stay long: those of unlike length
//    even out (32 of 8000 to 16000 int8 keys: 160.8 us with one, 150.3 with two;
//    16 of 15000 to 30000, 2 heads of 64: 31.7 and 27.5. Equal lengths take up to
//    5 % longer: 32 of 16000 174 and 182).
void plan_attend(AttendArgs& a) {
  const int rows = a.T * a.rep, per = rows <= 16 ? 16 : 32;
  a.row_blocks = (rows + per - 1) / per;
  a.splits = 1;
  if (a.max_len > kShort) {
    const int64_t groups = (int64_t)a.B * a.Hkv * a.row_blocks;
    int64_t splits = (256 + groups - 1) / groups;
    if (a.B > 1 && a.max_len / splits >= 2048) splits = (512 + groups - 1) / groups;
    a.splits = (int)std::min<int64_t>(splits, (a.max_len + kStep - 1) / kStep);
  }
  a.by_splits = Divisor(a.splits);
  a.by_row_blocks = Divisor(a.row_blocks);
  a.by_rep = Divisor(a.rep);
  a.by_heads = Divisor(a.Hkv);
  a.by_rows = Divisor(rows);
}

hipError_t launch_attend(const AttendArgs& a, ServingType type, CacheKind kind, hipStream_t stream) {
  return type == ServingType::kBf16 ? attend_by_kind<__bf16>(a, kind, stream) : attend_by_kind<_Float16>(a, kind, stream);
}
