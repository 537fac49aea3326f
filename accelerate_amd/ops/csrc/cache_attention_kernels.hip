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
//  * 8-bit codes are exact in bf16 and fp16. The keys' scales multiply the
//    scores, the values' scales the probabilities, both in 32 bits.
// The cache's length is split over workgroups where there are too few heads
// and sequences to fill the chip; a second kernel joins the parts.

#include "serving.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int uint4v __attribute__((ext_vector_type(4)));

template <typename T> struct Operand;
template <> struct Operand<__bf16> {
  typedef __bf16 V __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Operand<_Float16> {
  typedef _Float16 V __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

constexpr int kWaves = 4;
constexpr int kTile = 32;                // keys a wave takes at a time
constexpr int kStep = kWaves * kTile;    // keys a workgroup takes at a time
constexpr int kMaxSplits = 512;
constexpr float kNegInf = -__builtin_inff();

// the value of the code in byte i of a word, exact
template <CacheKind kKind>
__device__ __forceinline__ float decode(unsigned word, int i) {
  if constexpr (kKind == CacheKind::kInt8) return (float)(int8_t)(word >> (8 * i));
  switch (i) {  // the byte is an immediate of the instruction
    case 0: return __builtin_amdgcn_cvt_f32_fp8(word, 0);
    case 1: return __builtin_amdgcn_cvt_f32_fp8(word, 1);
    case 2: return __builtin_amdgcn_cvt_f32_fp8(word, 2);
    default: return __builtin_amdgcn_cvt_f32_fp8(word, 3);
  }
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
  template <typename T>
  __device__ __forceinline__ T as16(int i) const {  // the i-th 16-bit element
    return __builtin_bit_cast(T, (uint16_t)(w[i / 2] >> (16 * (i & 1))));
  }
};

__device__ __forceinline__ int clamped_length(const AttendArgs& a, int b) {
  return min(max(a.lengths[b], 0), a.max_len);
}

// how many splits of the grid have keys, and how many steps of kStep each has:
// the sequence's own length is shared out, not the cache's
struct Share {
  int steps, active;
};

__device__ __forceinline__ Share share_of(int end, int splits) {
  const int all = max(1, (end + kStep - 1) / kStep);
  Share s;
  s.steps = (all + splits - 1) / splits;
  s.active = (all + s.steps - 1) / s.steps;
  return s;
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

// The infinite and NaN values that the masked tiles left out, of the slots
// [from, to) that row t sees, added to its sums of N dimensions from d on.
template <typename T, int N>
__device__ void add_odd_row(const AttendArgs& a, int b, int t, int n0, int from, int to,
                                         const uint8_t* values, int d, float* y) {
  for (int j = max(from, n0 / kTile * kTile); j < to; ++j) {
    if (j >= n0 && !(a.mask ? a.mask[b * a.mb + t * a.mt + (j - n0)] != 0 : j - n0 <= t)) continue;
    const T* v = reinterpret_cast<const T*>(values) + (int64_t)j * a.D + d;
    for (int i = 0; i < N; ++i)
      if (!__builtin_isfinite((float)v[i])) y[i] += (float)v[i];
  }
}

template <typename T, CacheKind kKind, int kD, int kMT>
__global__ void __launch_bounds__(256, (kMT * kD > 256 || kD == 256 ? 1 : 2)) attend_kernel(AttendArgs a) {
  using Op = Operand<T>;
  using OV = typename Op::V;
  constexpr bool kSame = kKind == CacheKind::kSame;
  constexpr int kBytes = kSame ? 2 : 1;
  constexpr int kQK = kD / 32;  // products a tile of 16 keys
  constexpr int kND = kD / 16;  // a lane's neighbours of a row of V, and products
  // 8-bit keys are loaded 16 values at a time, the two halves of which belong
  // to two products; the queries follow that order
  constexpr bool kPaired = !kSame && kD >= 64;
  constexpr int kRowBytes = kD * kBytes;
  __shared__ float red[kWaves][4][kND][64];
  __shared__ float red_m[kWaves][kMT][16], red_l[kWaves][kMT][16];
  __shared__ int red_odd;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  // Workgroups go round the 8 XCDs in turn. Those that read the same keys for
  // other rows are 8 apart, so that they share an L2.
  const int parts = a.splits * a.Hkv * a.B;
  int part, rb;
  if (a.row_blocks == 1) {
    part = blockIdx.x;
    rb = 0;
  } else {
    const int xcd = blockIdx.x & 7, at = blockIdx.x >> 3;
    rb = at % a.row_blocks;
    part = (at / a.row_blocks) * 8 + xcd;
    if (part >= parts) return;
  }
  const int split = part % a.splits;
  const int bh = part / a.splits;
  const int b = bh / a.Hkv, h = bh - b * a.Hkv;
  const int n0 = clamped_length(a, b);
  const int end = min(n0 + a.W, a.max_len);
  const Share share = share_of(end, a.splits);
  if (split >= share.active) return;
  const int rows = a.T * a.rep;
  const int row0 = rb * kMT * 16;

  // the queries, as operands: 8 values of row c. Rows behind the last repeat
  // it; no row reaches another's result, and they are not written.
  OV q[kMT][kQK];
#pragma unroll
  for (int mt = 0; mt < kMT; ++mt) {
    const int row = min(row0 + mt * 16 + c, rows - 1);
    const int t = row / a.rep, head = h * a.rep + row % a.rep;
    const T* src = reinterpret_cast<const T*>(a.q) + b * a.qb + head * a.qh + t * a.qt;
#pragma unroll
    for (int ds = 0; ds < kQK; ++ds) {
      const int d = kPaired ? (ds / 2) * 64 + g * 16 + (ds & 1) * 8 : ds * 32 + g * 8;
      q[mt][ds] = *reinterpret_cast<const OV*>(src + d);
    }
  }

  f32x4 o[kMT][kND];
  float m[kMT], l[kMT];
#pragma unroll
  for (int mt = 0; mt < kMT; ++mt) {
    m[mt] = kNegInf;
    l[mt] = 0.f;
#pragma unroll
    for (int j = 0; j < kND; ++j) o[mt][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  constexpr unsigned kExp = __is_same(T, __bf16) ? 0x7F80u : 0x7C00u;  // of an infinity or NaN
  bool odd = false;  // whether masked tiles have such values
  int unit = -126;  // fp16, 8 bits: o is held in units of 2^unit (below)

  const uint8_t* kbase = reinterpret_cast<const uint8_t*>(a.k) + (int64_t)bh * a.slots * kRowBytes;
  const uint8_t* vbase = reinterpret_cast<const uint8_t*>(a.v) + (int64_t)bh * a.slots * kRowBytes;
  const float* ks = kSame ? nullptr : a.k_scale + (int64_t)bh * a.slots;
  const float* vs = kSame ? nullptr : a.v_scale + (int64_t)bh * a.slots;
  const int first = split * share.steps * kStep + wave * kTile;
  const int stop = min(end, (split + 1) * share.steps * kStep);

  // A tile's keys are loaded while the tile before is exponentiated and
  // multiplied with its values, its values while its own scores are made: the
  // registers of one are free when the other's next loads start.
  constexpr int kLoad = kSame || kPaired ? 16 : 8;
  constexpr int kLoads = kPaired ? kQK / 2 : kQK;
  Raw<kLoad> kraw[2][kLoads];
  Raw<kND * kBytes> vraw[8];
  f32x4 kscale[2], vscale[2];
  const auto load_keys = [&](int key0) {
    const uint8_t* kp = kbase + (int64_t)key0 * kRowBytes + c * kRowBytes + g * kLoad;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < kLoads; ++i) kraw[t][i].load(kp + t * 16 * kRowBytes + i * 64);
    if constexpr (!kSame) {
#pragma unroll
      for (int t = 0; t < 2; ++t) kscale[t] = *reinterpret_cast<const f32x4*>(ks + key0 + t * 16 + g * 4);
    }
  };
  const auto load_values = [&](int key0) {
    const uint8_t* vp = vbase + (int64_t)key0 * kRowBytes + g * 4 * kRowBytes + c * kND * kBytes;
#pragma unroll
    for (int e = 0; e < 8; ++e) vraw[e].load(vp + ((e >> 2) * 16 + (e & 3)) * kRowBytes);
    if constexpr (!kSame) {
#pragma unroll
      for (int t = 0; t < 2; ++t) vscale[t] = *reinterpret_cast<const f32x4*>(vs + key0 + t * 16 + g * 4);
    }
  };
  // No load is conditional: a wave without keys, or without more, reads its
  // last tile or the sequence's first once more, from a cache. Registers that
  // a branch may leave unwritten were given away by the compiler while they
  // were in use.
  const int safe = first < stop ? first : 0;
  load_keys(safe);
  load_values(safe);
  for (int key0 = first; key0 < stop; key0 += kStep) {
    const int next = key0 + kStep < stop ? key0 + kStep : key0;

    // scores
    f32x4 s[kMT][2];
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt) s[mt][0] = s[mt][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ds = 0; ds < kQK; ++ds) {
      OV k[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if constexpr (kSame) {
          k[t] = __builtin_bit_cast(OV, kraw[t][ds]);
        } else {
          const auto& raw = kraw[t][kPaired ? ds / 2 : ds];
          const int w0 = kPaired ? (ds & 1) * 2 : 0;
#pragma unroll
          for (int i = 0; i < 8; ++i) k[t][i] = (T)decode<kKind>(raw.w[w0 + i / 4], i & 3);
        }
      }
#pragma unroll
      for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
        for (int t = 0; t < 2; ++t) s[mt][t] = Op::mfma(k[t], q[mt][ds], s[mt][t]);
    }
    float ksc[8], vsc[8];
    if constexpr (!kSame) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        ksc[e] = kscale[e >> 2][e & 3] * a.scale_log2;
        vsc[e] = vscale[e >> 2][e & 3];
      }
    }
    load_keys(next);

    const bool masked = key0 + kTile > n0;  // the tile has slots that some rows do not see
    float p[kMT][8];
    bool grew = false;
    float keep[kMT];
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt) {
      const int t_row = (row0 + mt * 16 + c) / a.rep;
#pragma unroll
      for (int e = 0; e < 8; ++e) p[mt][e] = s[mt][e >> 2][e & 3] * (kSame ? a.scale_log2 : ksc[e]);
      if (masked) {
        // all of a lane's mask values are read at once, from inside the mask
        const bool chain = a.mask == nullptr;
        const uint8_t* bits = a.mask + b * a.mb + min(t_row, a.T - 1) * a.mt;
        uint8_t bit[8] = {};
        if (!chain && a.W > 0) {
#pragma unroll
          for (int e = 0; e < 8; ++e) bit[e] = bits[min(max(key0 + (e >> 2) * 16 + g * 4 + (e & 3) - n0, 0), a.W - 1)];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int key = key0 + (e >> 2) * 16 + g * 4 + (e & 3);
          // selects, no branches: an array element written under a lane's own
          // condition was lost by the compiler
          const bool sees = (key < n0) | ((key < end) & (chain ? key - n0 <= t_row : bit[e] != 0));
          p[mt][e] = sees ? p[mt][e] : kNegInf;
        }
      }
      float top = p[mt][0];
#pragma unroll
      for (int e = 1; e < 8; ++e) top = fmaxf(top, p[mt][e]);
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float m_new = fmaxf(m[mt], top);
      const float base = m_new == kNegInf ? 0.f : m_new;  // nothing seen so far
      keep[mt] = __builtin_amdgcn_exp2f(m[mt] - base);
      grew |= m_new > m[mt];
      m[mt] = m_new;
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[mt][e] = __builtin_amdgcn_exp2f(p[mt][e] - base);
        sum += p[mt][e];
      }
      l[mt] = l[mt] * keep[mt] + sum;
    }

    if constexpr (!kSame) {
      if (masked) {  // slots behind the new tokens hold anything
#pragma unroll
        for (int e = 0; e < 8; ++e)
          vsc[e] = key0 + (e >> 2) * 16 + g * 4 + (e & 3) < end ? vsc[e] : 0.f;
      }
    }
    float unit_scale = 1.f;
    if constexpr (!kSame && __is_same(T, _Float16)) {
      // Probabilities times the values' scales would be lost below fp16's
      // range. They are held relative to the power of two of the largest
      // scale so far, which is the same for all rows.
      float most = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) most = fmaxf(most, vsc[e]);
#pragma unroll
      for (int x = 16; x < 64; x <<= 1) most = fmaxf(most, __shfl_xor(most, x));
      const int wanted = min(max(unit, (int)(__float_as_uint(most) >> 23) - 126), 120);
      if (wanted > unit) {
        grew = true;
        const float less = __builtin_ldexpf(1.f, max(unit - wanted, -126));
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt) keep[mt] *= less;
        unit = wanted;
      }
      unit_scale = __builtin_ldexpf(1.f, -unit);
    }
    if (__any(grew)) {
#pragma unroll
      for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
        for (int j = 0; j < kND; ++j) o[mt][j] *= keep[mt];
    }

    // Probabilities are rounded to the type of the product's operands: half a
    // step of it for each, without a common sign.
    OV pv[kMT];
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float x = p[mt][e];
        if constexpr (!kSame) {
          x *= vsc[e] * unit_scale;
          // the scale of a token that the row does not see may be anything
          x = masked & (p[mt][e] == 0.f) ? 0.f : x;
        }
        pv[mt][e] = (T)x;
      }

    if constexpr (kSame) {
      if (masked) {
        // A probability of zero does not hide an infinite or NaN value. Slots
        // behind the new tokens are cleared; of the others, those values that
        // are not finite are left out here and added at the end, to the rows
        // that see them alone.
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool in = key0 + (e >> 2) * 16 + g * 4 + (e & 3) < end;
#pragma unroll
          for (int w = 0; w < Raw<kND * kBytes>::kWords; ++w) {
            unsigned& x = vraw[e].w[w];
            const unsigned low = (x & kExp) == kExp ? 0xFFFFu : 0u;
            const unsigned high = ((x >> 16) & kExp) == kExp ? 0xFFFF0000u : 0u;
            odd |= in & ((low | high) != 0);
            x = in ? x & ~(low | high) : 0u;
          }
        }
      }
    }

#pragma unroll
    for (int j = 0; j < kND; ++j) {
      OV v;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (kSame) v[e] = vraw[e].template as16<T>(j);
        else v[e] = (T)decode<kKind>(vraw[e].w[j / 4], j & 3);
      }
#pragma unroll
      for (int mt = 0; mt < kMT; ++mt) o[mt][j] = Op::mfma(v, pv[mt], o[mt][j]);
    }
    load_values(next);
  }

  // the four waves' parts of a row, joined
  if (threadIdx.x == 0) red_odd = 0;
  __syncthreads();
  if (kSame && odd) red_odd = 1;
#pragma unroll
  for (int mt = 0; mt < kMT; ++mt) {
    l[mt] += __shfl_xor(l[mt], 16);
    l[mt] += __shfl_xor(l[mt], 32);
    if (g == 0) {
      red_m[wave][mt][c] = m[mt];
      red_l[wave][mt][c] = l[mt];
    }
  }
  __syncthreads();
#pragma unroll
  for (int mt = 0; mt < kMT; ++mt) {
    float top = kNegInf, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, red_m[w][mt][c]);
    const float base = top == kNegInf ? 0.f : top;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += red_l[w][mt][c] * __builtin_amdgcn_exp2f(red_m[w][mt][c] - base);
    float mine = __builtin_amdgcn_exp2f(m[mt] - base);
    if constexpr (!kSame && __is_same(T, _Float16)) mine *= __builtin_ldexpf(1.f, unit);
#pragma unroll
    for (int j = 0; j < kND; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) red[wave][r][j][lane] = o[mt][j][r] * mine;
    __syncthreads();
    // wave w sums the elements r = w: neighbours of row c from (4 g + w) D / 16 on
    const int row = row0 + mt * 16 + c;
    float y[kND];
#pragma unroll
    for (int j = 0; j < kND; ++j) {
      y[j] = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) y[j] += red[w][wave][j][lane];
    }
    __syncthreads();
    if (row < rows) {
      const int d = (g * 4 + wave) * kND;
      if (kSame && red_odd) add_odd_row<T, kND>(a, b, row / a.rep, n0, first - wave * kTile, stop, vbase, d, y);
      if (a.splits == 1) {
        const int t = row / a.rep, head = h * a.rep + row % a.rep;
        const float inverse = 1.f / sum;
        T* dst = reinterpret_cast<T*>(a.out) + b * a.ob + head * a.oh + t * a.ot + d;
        const float none = sum == 0.f ? empty_row(a, b, t, n0) : 0.f;
        struct alignas(kND * 2 < 16 ? kND * 2 : 16) { T v[kND]; } out;
#pragma unroll
        for (int j = 0; j < kND; ++j) out.v[j] = (T)(sum == 0.f ? none : y[j] * inverse);
        *reinterpret_cast<decltype(out)*>(dst) = out;
      } else {
        const int64_t at = ((int64_t)bh * rows + row) * a.splits + split;
        struct alignas(kND * 4 < 16 ? kND * 4 : 16) { float v[kND]; } out;
#pragma unroll
        for (int j = 0; j < kND; ++j) out.v[j] = y[j];
        *reinterpret_cast<decltype(out)*>(a.part_o + at * kD + d) = out;
        if (d == 0) {
          a.part_ml[at * 2] = top;
          a.part_ml[at * 2 + 1] = sum;
        }
      }
    }
  }
}

// The splits of a row, joined: a workgroup a row. Its threads take four
// dimensions each and share the splits out, so that few rows of many splits
// (one long sequence) still have many reads under way.
template <typename T, int kD>
__global__ void __launch_bounds__(256) attend_join_kernel(AttendArgs a) {
  constexpr int kLanes = kD / 4, kGroups = 256 / kLanes;
  __shared__ f32x4 red[kGroups][kLanes];
  __shared__ float weight[kMaxSplits], red_m[4], red_l[4];
  const int rows = a.T * a.rep, tid = threadIdx.x;
  const int bh = blockIdx.x / rows, row = blockIdx.x - bh * rows;
  const int b = bh / a.Hkv, h = bh - b * a.Hkv;
  const int n0 = clamped_length(a, b);
  const int active = share_of(min(n0 + a.W, a.max_len), a.splits).active;
  const int64_t at = (int64_t)blockIdx.x * a.splits;

  float m[kMaxSplits / 256], l[kMaxSplits / 256], top = kNegInf;
#pragma unroll
  for (int i = 0; i < kMaxSplits / 256; ++i) {
    const int s = tid + i * 256;
    m[i] = kNegInf;
    l[i] = 0.f;
    if (s < active) {
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
  const float base = top == kNegInf ? 0.f : top;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kMaxSplits / 256; ++i) {
    const float w = __builtin_amdgcn_exp2f(m[i] - base);
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
  for (int s = group; s < active; s += kGroups) y += *reinterpret_cast<const f32x4*>(part + (int64_t)s * kD) * weight[s];
  red[group][lane] = y;
  __syncthreads();
  if (tid >= kD) return;
  float out = 0.f;
#pragma unroll
  for (int i = 0; i < kGroups; ++i) out += red[i][tid / 4][tid % 4];
  const int t = row / a.rep, head = h * a.rep + row % a.rep;
  out = sum == 0.f ? empty_row(a, b, t, n0) : out / sum;
  reinterpret_cast<T*>(a.out)[b * a.ob + head * a.oh + t * a.ot + tid] = (T)out;
}

template <typename T, CacheKind kKind, int kD>
hipError_t attend_by_rows(const AttendArgs& a, hipStream_t stream) {
  const int64_t parts = (int64_t)a.splits * a.Hkv * a.B;
  const int64_t blocks = a.row_blocks == 1 ? parts : (parts + 7) / 8 * 8 * a.row_blocks;
  const dim3 grid((unsigned)blocks), block(256);
  switch (attend_row_tiles(a.T * a.rep, kD)) {
    case 1: hipLaunchKernelGGL((attend_kernel<T, kKind, kD, 1>), grid, block, 0, stream, a); break;
    case 2: hipLaunchKernelGGL((attend_kernel<T, kKind, kD, 2>), grid, block, 0, stream, a); break;
    default:
      if constexpr (kD <= 128) hipLaunchKernelGGL((attend_kernel<T, kKind, kD, 4>), grid, block, 0, stream, a);
      break;
  }
  if (a.splits > 1)
    hipLaunchKernelGGL((attend_join_kernel<T, kD>), dim3((unsigned)(a.B * a.Hkv * a.T * a.rep)), block, 0, stream, a);
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

// Tiles of 16 rows a workgroup holds. More rows share one reading of the keys;
// at D = 256 four tiles of accumulators would not fit the registers.
int attend_row_tiles(int rows, int D) {
  if (rows <= 16) return 1;
  return rows <= 32 || D == 256 ? 2 : 4;
}

// Parts that a sequence's keys are split into: enough workgroups for two on
// each of the 256 CUs, and none with less than one step of keys. The host does
// not know the lengths, so the cache's size stands for them; a shorter
// sequence is shared out over the same number, as far as its steps go.
int attend_splits(const AttendArgs& a) {
  const int64_t groups = (int64_t)a.B * a.Hkv * a.row_blocks;
  const int64_t wanted = (kMaxSplits + groups - 1) / groups;
  const int64_t most = (a.max_len + kStep - 1) / kStep;
  return (int)std::max<int64_t>(1, std::min(wanted, most));
}

hipError_t launch_attend(const AttendArgs& a, ServingType type, CacheKind kind, hipStream_t stream) {
  return type == ServingType::kBf16 ? attend_by_kind<__bf16>(a, kind, stream) : attend_by_kind<_Float16>(a, kind, stream);
}
