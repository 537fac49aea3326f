// A cache of keys and values in 8 bits: quantised as it is written, read back
// in 16 or 32 bits, and the accepted path of a tree of drafted tokens moved
// together.
//
// A row is the D values of one token and one head. Its scale s is one float:
//   int8: s = amax / 127, code = x / s to the nearest integer, ties to even;
//   fp8 (e4m3): s = the least power of two with amax / s <= 448, code = x / s
//         rounded by the hardware's convert, ties to even. s is at most 2^119,
//         where codes saturate: the rounded 256 * 2^120 would be no number.
// A value of a row that is infinite or NaN has no code: the row's scale is
// NaN then, and it reads back as NaN. A row whose int8 scale would be
// subnormal (amax below 127 * 2^-126) is held as zeros.
//
// All of these are bound by memory, and nearly by the instructions around it:
// a lane holds 16 values (32 bytes of input, 16 of codes), D / 16 lanes a row,
// and the grid's y and z are the sequence and the tensor, so that one division
// finds a row. Rows of a call go over heads first where the input has the
// heads of a token side by side, so that whole pages of it are read at a time.
// 4 sequences of 7001 tokens, 8 heads of 128 in e4m3: 31.9 us to append (5.4
// TB/s), 29.5 to read back in bf16 (5.8); a large copy reaches 5.1. One token
// of 64 sequences: 4.2 and 2.8, a launch and a reading.

#include "serving.h"

namespace {

typedef unsigned int uint4v __attribute__((ext_vector_type(4)));

constexpr int kPer = 16;  // values a lane

template <typename T>
struct alignas(16) Values { T v[kPer]; };

constexpr unsigned kInfBits = 0x7F800000u;

__device__ __forceinline__ unsigned codes4_int8(const float* x, float scale, float inverse) {
  unsigned word = 0;
  const float half = 0.5f * scale;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // x * (1 / s) can fall on the wrong side of a border between two codes.
    // The remainder x - q s has at most 24 bits (x has 11, or it is s times
    // an integer within a step), so fma gives it exactly and the comparison
    // with half a step decides as the quotient in full would.
    float q = rintf(x[i] * inverse);
    const float rest = __builtin_fmaf(-q, scale, x[i]);
    const bool odd = ((int)q & 1) != 0;
    if (rest > half || (rest == half && odd)) q += 1.f;
    else if (rest < -half || (rest == -half && odd)) q -= 1.f;
    word |= ((unsigned)(int)q & 0xFFu) << (8 * i);
  }
  return word;
}

__device__ __forceinline__ unsigned codes4_fp8(const float* x, float inverse) {
  // by a power of two, exact; above 448 (where the convert gives NaN) only at the largest scale
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = __builtin_amdgcn_fmed3f(x[i] * inverse, -448.f, 448.f);
  unsigned word = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0u, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], word, true);
}

template <CacheKind kKind>
__device__ __forceinline__ void values4(unsigned word, float scale, float* y) {
  if constexpr (kKind == CacheKind::kInt8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = (float)(int8_t)(word >> (8 * i)) * scale;
  } else {
    y[0] = __builtin_amdgcn_cvt_f32_fp8(word, 0) * scale;
    y[1] = __builtin_amdgcn_cvt_f32_fp8(word, 1) * scale;
    y[2] = __builtin_amdgcn_cvt_f32_fp8(word, 2) * scale;
    y[3] = __builtin_amdgcn_cvt_f32_fp8(word, 3) * scale;
  }
}

// The head and token of a thread's row of its sequence.
struct Row {
  int h, t;
};

__device__ __forceinline__ Row row_of(unsigned row, const CacheArgs& a) {
  const unsigned inner = a.heads_first ? a.H : a.T;
  const unsigned q = row / inner, r = row - q * inner;
  return a.heads_first ? Row{(int)r, (int)q} : Row{(int)q, (int)r};
}

template <typename T, CacheKind kKind, int kD>
__global__ void __launch_bounds__(256) cache_append_kernel(CacheArgs a) {
  constexpr int kLanes = kD / kPer;
  const int lane = threadIdx.x % kLanes, b = blockIdx.y, which = blockIdx.z;
  const unsigned row = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  if (row >= (unsigned)a.H * a.T) return;  // whole groups of kLanes lanes leave together
  const Row r = row_of(row, a);
  if (a.counts && r.t >= a.counts[b]) return;
  const int64_t slot = (a.start ? (int64_t)a.start[b] : 0) + a.offset + r.t;
  if (slot < 0 || slot >= a.max_len) return;
  const T* x = reinterpret_cast<const T*>(a.x[which]) + b * a.sb[which] + r.h * a.sh[which] + r.t * a.st[which] +
               lane * kPer;
  const Values<T> in = *reinterpret_cast<const Values<T>*>(x);
  const CacheTensor& out = which ? a.v : a.k;
  const int64_t at = ((int64_t)b * a.H + r.h) * a.slots + slot;
  if constexpr (kKind == CacheKind::kSame) {
    *reinterpret_cast<Values<T>*>(reinterpret_cast<T*>(out.data) + at * kD + lane * kPer) = in;
  } else {
    float f[kPer];
    unsigned most = 0;  // of the absolute values' bits: infinities and NaN are above all others
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      f[i] = (float)in.v[i];
      most = max(most, __float_as_uint(f[i]) & 0x7FFFFFFFu);
    }
#pragma unroll
    for (int m = 1; m < kLanes; m <<= 1) most = max(most, (unsigned)__shfl_xor((int)most, m));
    float scale, inverse;
    if constexpr (kKind == CacheKind::kInt8) {
      scale = __uint_as_float(most) / 127.f;
      if (scale < 1.17549435e-38f) scale = 0.f;
      inverse = 1.f / scale;
    } else {
      // amax = 1.f * 2^(E - 127), 448 = 1.75 * 2^8
      const int e = min(max((int)(most >> 23) - 135 + ((most & 0x7FFFFFu) > 0x600000u ? 1 : 0), -126), 119);
      scale = most ? __uint_as_float((unsigned)(e + 127) << 23) : 0.f;
      inverse = __uint_as_float((unsigned)(127 - e) << 23);
    }
    uint4v codes = {0u, 0u, 0u, 0u};
    if (most >= kInfBits) {
      scale = __builtin_nanf("");
    } else if (scale > 0.f) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (kKind == CacheKind::kInt8) codes[i] = codes4_int8(f + 4 * i, scale, inverse);
        else codes[i] = codes4_fp8(f + 4 * i, inverse);
      }
    }
    *reinterpret_cast<uint4v*>(reinterpret_cast<uint8_t*>(out.data) + at * kD + lane * kPer) = codes;
    if (lane == 0) out.scale[at] = scale;
  }
}

template <typename T, CacheKind kKind, typename Out, int kD>
__global__ void __launch_bounds__(256) cache_read_kernel(CacheArgs a) {
  constexpr int kLanes = kD / kPer;
  const int lane = threadIdx.x % kLanes, b = blockIdx.y, which = blockIdx.z;
  const unsigned row = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  if (row >= (unsigned)a.H * a.T) return;
  const Row r = row_of(row, a);  // tokens first, as the output has them
  const int64_t slot = (a.start ? (int64_t)a.start[b] : 0) + a.offset + r.t;
  const CacheTensor& in = which ? a.v : a.k;
  const int64_t at = ((int64_t)b * a.H + r.h) * a.slots + slot;
  float f[kPer] = {};  // slots that the cache does not have read as zeros
  if (slot >= 0 && slot < a.max_len) {
    if constexpr (kKind == CacheKind::kSame) {
      const Values<T> held = *reinterpret_cast<const Values<T>*>(reinterpret_cast<const T*>(in.data) + at * kD + lane * kPer);
#pragma unroll
      for (int i = 0; i < kPer; ++i) f[i] = (float)held.v[i];
    } else {
      const uint4v codes =
          *reinterpret_cast<const uint4v*>(reinterpret_cast<const uint8_t*>(in.data) + at * kD + lane * kPer);
      const float scale = in.scale[at];
#pragma unroll
      for (int i = 0; i < 4; ++i) values4<kKind>(codes[i], scale, f + 4 * i);
    }
  }
  Out* y = reinterpret_cast<Out*>(a.y[which]) + ((int64_t)b * a.H * a.T + row) * kD + lane * kPer;
  Values<Out> o;
#pragma unroll
  for (int i = 0; i < kPer; ++i) o.v[i] = (Out)f[i];
  *reinterpret_cast<Values<Out>*>(y) = o;
}

// The kept tokens of a sequence, in order: slot start + path[i] to start + i.
// A path ascends, so path[i] >= i and no slot is written before it is read;
// a thread moves the same 16 bytes of every row, so it needs no others' order.
__global__ void __launch_bounds__(64) cache_keep_kernel(CacheArgs a, const int64_t* path, int row_bytes) {
  const int which = blockIdx.x & 1;
  const int bh = blockIdx.x >> 1;
  const int b = bh / a.H;
  const CacheTensor& c = which ? a.v : a.k;
  const int64_t start = (int64_t)a.start[b] + a.offset;
  const int at = threadIdx.x * 16;
  const bool moves = at < row_bytes, scales = c.scale && threadIdx.x == 63;
  if (start < 0 || !(moves || scales)) return;
  uint8_t* rows = reinterpret_cast<uint8_t*>(c.data) + ((int64_t)bh * a.slots + start) * row_bytes + at;
  float* scale = c.scale + (int64_t)bh * a.slots + start;
  int64_t last = -1;
  for (int i = 0; i < a.T; ++i) {
    const int64_t from = path[(int64_t)b * a.T + i];
    if (from <= last || from >= a.T || start + from >= a.max_len) return;  // the path's end, or no path
    last = from;
    if (from == i) continue;
    if (moves) *reinterpret_cast<uint4v*>(rows + (int64_t)i * row_bytes) = *reinterpret_cast<uint4v*>(rows + from * row_bytes);
    if (scales) scale[i] = scale[from];
  }
}

template <typename T, CacheKind kKind, int kD>
hipError_t append_launch(const CacheArgs& a, hipStream_t stream) {
  const unsigned rows = (unsigned)a.H * a.T, per = 256 / (kD / kPer);
  hipLaunchKernelGGL((cache_append_kernel<T, kKind, kD>), dim3((rows + per - 1) / per, a.B, 2), dim3(256), 0, stream, a);
  return hipGetLastError();
}

template <typename T, CacheKind kKind>
hipError_t append_by_dim(const CacheArgs& a, hipStream_t stream) {
  switch (a.D) {
    case 32: return append_launch<T, kKind, 32>(a, stream);
    case 64: return append_launch<T, kKind, 64>(a, stream);
    case 128: return append_launch<T, kKind, 128>(a, stream);
    default: return append_launch<T, kKind, 256>(a, stream);
  }
}

template <typename T, CacheKind kKind, typename Out, int kD>
hipError_t read_launch(const CacheArgs& a, hipStream_t stream) {
  const unsigned rows = (unsigned)a.H * a.T, per = 256 / (kD / kPer);
  hipLaunchKernelGGL((cache_read_kernel<T, kKind, Out, kD>), dim3((rows + per - 1) / per, a.B, 2), dim3(256), 0, stream, a);
  return hipGetLastError();
}

template <typename T, CacheKind kKind, typename Out>
hipError_t read_by_dim(const CacheArgs& a, hipStream_t stream) {
  switch (a.D) {
    case 32: return read_launch<T, kKind, Out, 32>(a, stream);
    case 64: return read_launch<T, kKind, Out, 64>(a, stream);
    case 128: return read_launch<T, kKind, Out, 128>(a, stream);
    default: return read_launch<T, kKind, Out, 256>(a, stream);
  }
}

template <typename T, CacheKind kKind>
hipError_t read_by_out(const CacheArgs& a, ServingType out, hipStream_t stream) {
  switch (out) {
    case ServingType::kBf16: return read_by_dim<T, kKind, __bf16>(a, stream);
    case ServingType::kFp16: return read_by_dim<T, kKind, _Float16>(a, stream);
    default: return read_by_dim<T, kKind, float>(a, stream);
  }
}

}  // namespace

hipError_t launch_cache_append(const CacheArgs& a, ServingType type, CacheKind kind, hipStream_t stream) {
  const bool bf = type == ServingType::kBf16;
  switch (kind) {
    case CacheKind::kInt8:
      return bf ? append_by_dim<__bf16, CacheKind::kInt8>(a, stream) : append_by_dim<_Float16, CacheKind::kInt8>(a, stream);
    case CacheKind::kFp8:
      return bf ? append_by_dim<__bf16, CacheKind::kFp8>(a, stream) : append_by_dim<_Float16, CacheKind::kFp8>(a, stream);
    default:  // 16 bits are moved as they are
      return append_by_dim<__bf16, CacheKind::kSame>(a, stream);
  }
}

hipError_t launch_cache_read(const CacheArgs& a, ServingType type, CacheKind kind, ServingType out, hipStream_t stream) {
  switch (kind) {  // 8-bit codes do not depend on the 16-bit type
    case CacheKind::kInt8: return read_by_out<__bf16, CacheKind::kInt8>(a, out, stream);
    case CacheKind::kFp8: return read_by_out<__bf16, CacheKind::kFp8>(a, out, stream);
    default:
      return type == ServingType::kBf16 ? read_by_out<__bf16, CacheKind::kSame>(a, out, stream)
                                        : read_by_out<_Float16, CacheKind::kSame>(a, out, stream);
  }
}

hipError_t launch_cache_keep(const CacheArgs& a, const int64_t* path, int row_bytes, hipStream_t stream) {
  hipLaunchKernelGGL(cache_keep_kernel, dim3(2u * a.B * a.H), dim3(64), 0, stream, a, path, row_bytes);
  return hipGetLastError();
}
