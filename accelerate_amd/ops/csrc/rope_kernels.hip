// Fused rotary position embedding (half-split layout) for CDNA4.
//
// One kernel replaces torch's slice + 4 muls + 2 adds + cat chain (~7
// kernels, 6× the memory traffic). bf16 activations, fp32 cos/sin tables
// (host-precomputed — CDNA4 guide: on-device trig turns memory-bound ops
// VALU-bound). Backward is rotation by −θ (pass negate_sin).

#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>

#include "serving.h"

namespace {

typedef ushort ushort8r __attribute__((ext_vector_type(8)));

__device__ __forceinline__ float rbf2f(ushort u) {
  union { unsigned int i; float f; } cv;
  cv.i = ((unsigned int)u) << 16;
  return cv.f;
}

__device__ __forceinline__ ushort rf2bf(float f) {
  union { float f; unsigned int i; } cv;
  cv.f = f;
  if ((cv.i & 0x7F800000u) == 0x7F800000u) return (ushort)(cv.i >> 16) | (ushort)((cv.i & 0xFFFFu) ? 0x40 : 0);
  cv.i += 0x7FFFu + ((cv.i >> 16) & 1u);
  return (ushort)(cv.i >> 16);
}

}  // namespace

// x,y: [BH, S, D] contiguous bf16; cos/sin: [>=S, D/2] fp32 (pre-offset).
// Each thread rotates 8 pairs: loads 16 B from each half.
__global__ void rope_bf16_kernel(const ushort* __restrict__ x, ushort* __restrict__ y,
                                 const float* __restrict__ cos_t, const float* __restrict__ sin_t,
                                 int64_t n_bh, int S, int D, float sin_sign) {
  const int half = D >> 1;
  const int chunks_per_row = half >> 3;  // 8-pair chunks per (bh, s)
  const int64_t total = n_bh * S * chunks_per_row;
  for (int64_t idx = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; idx < total;
       idx += (int64_t)gridDim.x * blockDim.x) {
    const int c8 = (int)(idx % chunks_per_row);
    const int64_t row = idx / chunks_per_row;  // bh*S + s
    const int s = (int)(row % S);
    const int d0 = c8 * 8;
    const ushort* x1p = x + row * D + d0;
    const ushort* x2p = x1p + half;
    ushort8r x1 = *reinterpret_cast<const ushort8r*>(x1p);
    ushort8r x2 = *reinterpret_cast<const ushort8r*>(x2p);
    float4 c0 = *reinterpret_cast<const float4*>(cos_t + (int64_t)s * half + d0);
    float4 c1 = *reinterpret_cast<const float4*>(cos_t + (int64_t)s * half + d0 + 4);
    float4 s0 = *reinterpret_cast<const float4*>(sin_t + (int64_t)s * half + d0);
    float4 s1 = *reinterpret_cast<const float4*>(sin_t + (int64_t)s * half + d0 + 4);
    ushort8r y1, y2;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float a = rbf2f(x1[k]);
      float b = rbf2f(x2[k]);
      float ck = (k < 4) ? (&c0.x)[k] : (&c1.x)[k - 4];
      float sk = ((k < 4) ? (&s0.x)[k] : (&s1.x)[k - 4]) * sin_sign;
      y1[k] = rf2bf(a * ck - b * sk);
      y2[k] = rf2bf(b * ck + a * sk);
    }
    *reinterpret_cast<ushort8r*>(y + row * D + d0) = y1;
    *reinterpret_cast<ushort8r*>(y + row * D + d0 + half) = y2;
  }
}

// ---------------------------------------------------------------------------
// Rotary positions of q and k in one launch: positions per token, the first R
// of D elements, half or interleaved pairs, any (b, h, s) strides.
//
//   (a, b) -> (a cos - b sin, b cos + a sin)     for the pair i of position p,
//   cos = cos_t[p][i], sin = sin_t[p][i]; the inverse (and so the gradient)
//   negates sin.
//
// Bound by memory: 3 flops a value against 2 reads and writes of it. A thread
// holds the table's values of V pairs of one token and goes over heads with
// them, so the fp32 table is read once a token and not once a head (it would
// be twice the bytes of bf16 heads); neighbouring threads take the rest of the
// head, then the next head, so that a wave reads and writes whole lines. A
// training pass over 16384 tokens of 40 heads reads and writes at 5.1 TB/s, as
// a large copy does.
// ---------------------------------------------------------------------------

namespace {

template <typename T>
__device__ __forceinline__ float to_f32(T x) { return (float)x; }

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec { T v[N]; };

// V pairs a thread. V * sizeof(T) bytes is the width of every access: the
// host takes the largest V that sizes, strides and addresses allow.
template <typename T, int V, bool kInterleaved>
__global__ void __launch_bounds__(256) rotary_kernel(RotaryArgs a) {
  using VT = Vec<T, V>;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t unit = idx / a.chunks;
  const int chunk = (int)(idx - unit * a.chunks);
  const int64_t token = unit / a.head_step;
  if (token >= a.tokens) return;
  const int first_head = (int)(unit - token * a.head_step);
  const int64_t b = token / a.S, s = token - b * a.S;
  const int half = a.R >> 1;
  const bool rotated = chunk < a.rotary_chunks;

  float c[V], sn[V];
  if (rotated) {
    int64_t pos = s;
    if (a.positions) {
      const int64_t at = b * a.pos_b + s * a.pos_s;
      pos = a.pos_is_64 ? reinterpret_cast<const int64_t*>(a.positions)[at]
                        : (int64_t)reinterpret_cast<const int*>(a.positions)[at];
    }
    if (pos >= 0 && pos < a.table_rows) {
      // float4 where V allows it: the table's rows are half floats apart and
      // V divides half
      using FV = Vec<float, (V < 4 ? V : 4)>;
      const float* cp = a.cos_t + pos * half + chunk * V;
      const float* sp = a.sin_t + pos * half + chunk * V;
#pragma unroll
      for (int i = 0; i < V; i += (V < 4 ? V : 4)) {
        const FV cv = *reinterpret_cast<const FV*>(cp + i), sv = *reinterpret_cast<const FV*>(sp + i);
#pragma unroll
        for (int j = 0; j < (V < 4 ? V : 4); ++j) {
          c[i + j] = cv.v[j];
          sn[i + j] = sv.v[j] * a.sin_sign;
        }
      }
    } else {  // no such position: the values say so
#pragma unroll
      for (int i = 0; i < V; ++i) c[i] = sn[i] = __builtin_nanf("");
    }
  }
  // the two vectors of a chunk: V firsts and V seconds of its pairs, or 2 V neighbours
  const int off0 = rotated ? (kInterleaved ? chunk * 2 * V : chunk * V) : a.R + (chunk - a.rotary_chunks) * 2 * V;
  const int off1 = rotated && !kInterleaved ? off0 + half : off0 + V;
  const bool has0 = off0 < a.D, has1 = off1 < a.D;  // the rest of an odd head may end inside its chunk

#pragma unroll 4
  for (int h = first_head; h < a.Hq + a.Hk; h += a.head_step) {
    const bool is_k = h >= a.Hq;
    const RotaryTensor& t = is_k ? a.k : a.q;
    const int64_t head = is_k ? h - a.Hq : h;
    const T* x = reinterpret_cast<const T*>(t.x) + b * t.xb + head * t.xh + s * t.xs;
    T* y = reinterpret_cast<T*>(t.y) + b * t.yb + head * t.yh + s * t.ys;
    VT u, w;
    if (has0) u = *reinterpret_cast<const VT*>(x + off0);
    if (has1) w = *reinterpret_cast<const VT*>(x + off1);
    if (rotated) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if constexpr (kInterleaved) {
          T& p = 2 * i < V ? u.v[2 * i < V ? 2 * i : 0] : w.v[2 * i < V ? 0 : 2 * i - V];
          T& q = 2 * i + 1 < V ? u.v[2 * i + 1 < V ? 2 * i + 1 : 0] : w.v[2 * i + 1 < V ? 0 : 2 * i + 1 - V];
          const float fa = to_f32(p), fb = to_f32(q);
          p = (T)(fa * c[i] - fb * sn[i]);
          q = (T)(fb * c[i] + fa * sn[i]);
        } else {
          const float fa = to_f32(u.v[i]), fb = to_f32(w.v[i]);
          u.v[i] = (T)(fa * c[i] - fb * sn[i]);
          w.v[i] = (T)(fb * c[i] + fa * sn[i]);
        }
      }
    }
    if (has0) *reinterpret_cast<VT*>(y + off0) = u;
    if (has1) *reinterpret_cast<VT*>(y + off1) = w;
  }
}

template <typename T, int V>
hipError_t rotary_launch(const RotaryArgs& a, bool interleaved, hipStream_t stream) {
  const int64_t threads = a.tokens * a.head_step * a.chunks;
  const dim3 grid((unsigned)((threads + 255) / 256));
  if (interleaved) hipLaunchKernelGGL((rotary_kernel<T, V, true>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((rotary_kernel<T, V, false>), grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

template <typename T>
hipError_t rotary_by_width(const RotaryArgs& a, int V, bool interleaved, hipStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    if (V == 8) return rotary_launch<T, 8>(a, interleaved, stream);
  }
  if (V == 4) return rotary_launch<T, 4>(a, interleaved, stream);
  return rotary_launch<T, 1>(a, interleaved, stream);
}

}  // namespace

hipError_t launch_rotary(RotaryArgs a, ServingType type, int V, bool interleaved, hipStream_t stream) {
  a.rotary_chunks = a.R / (2 * V);
  a.chunks = a.rotary_chunks + (a.D - a.R + 2 * V - 1) / (2 * V);
  const int heads = a.Hq + a.Hk;
  // Few tokens: a thread for each head, the chip is not full anyway (400 tokens
  // of 40 heads of 128 take 4.0 us, 5.6 with four heads; 819: 5.2 and 6.4; 1600:
  // 8.7 and 8.7). Many: four heads a thread, with the table's values in its
  // registers (3200: 13.0 us, 13.8 with one; 8192 of 72 heads 58 us, 65 with
  // one, 72 with nine).
  const bool few = a.tokens * heads * a.chunks <= 256 * 1024;
  a.head_step = few ? heads : (heads + 3) / 4;
  switch (type) {
    case ServingType::kBf16: return rotary_by_width<__bf16>(a, V, interleaved, stream);
    case ServingType::kFp16: return rotary_by_width<_Float16>(a, V, interleaved, stream);
    default: return rotary_by_width<float>(a, V, interleaved, stream);
  }
}
