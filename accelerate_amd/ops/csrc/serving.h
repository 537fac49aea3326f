// Shared between the serving kernels (rotary positions, key/value cache,
// cache attention, draft verification) and their bindings.
#pragma once
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

enum class ServingType : int { kBf16 = 0, kFp16 = 1, kFp32 = 2 };
enum class CacheKind : int { kSame = 0, kInt8 = 1, kFp8 = 2 };

// Slots of a cache are allocated in multiples of this, so that a tile of keys
// that starts inside a sequence ends inside its storage.
constexpr int kSlotTile = 32;

struct RotaryTensor {
  const void* x;
  void* y;
  int64_t xb, xh, xs, yb, yh, ys;  // element strides; the last dimension is contiguous
};

struct RotaryArgs {
  RotaryTensor q, k;
  const float *cos_t, *sin_t;  // [table_rows, R / 2]
  const void* positions;       // [B, S] int64 or int32, or null: 0..S-1
  int64_t pos_b, pos_s, table_rows, tokens, S;
  int pos_is_64, Hq, Hk, D, R;
  int chunks, rotary_chunks, head_step;  // set by the launcher
  float sin_sign;
};

struct CacheTensor {
  void* data;    // [B, H, slots, D]: 16-bit values, int8 or e4m3 codes
  float* scale;  // [B, H, slots], or null for 16-bit values
};

// rows of D values between a [B, H, T, D] view and a window of the cache
struct CacheArgs {
  CacheTensor k, v;
  const void* x[2];        // append: the inputs of k and v
  void* y[2];              // read: the outputs, [B, H, T, D] contiguous
  int64_t sb[2], sh[2], st[2];
  const int* start;        // [B] first slot of each sequence, or null
  int64_t offset;          // added to it
  const int* counts;       // [B] tokens that are written, or null: all T
  int B, H, T, D, slots, max_len;
  int heads_first;         // rows in the order of their heads, then tokens
};

// Division of numbers below 2^31 by one that the host knows: with l the bits of
// d - 1, the quotient is (n + n m / 2^32) / 2^l, m = 2^32 (2^l - d) / d + 1.
struct Divisor {
  unsigned multiplier = 1, shift = 0;
  Divisor() = default;
  explicit Divisor(unsigned d) {
    while ((1ull << shift) < d) ++shift;
    multiplier = (unsigned)((((1ull << shift) - d) << 32) / d + 1);
  }
  __host__ __device__ unsigned quotient(unsigned n) const {
    return (n + (unsigned)(((uint64_t)n * multiplier) >> 32)) >> shift;
  }
};

struct AttendArgs {
  const void *q, *k, *v;
  const float *k_scale, *v_scale;
  void* out;
  const int* lengths;          // [B]
  const uint8_t* mask;         // [B, T, W] truth values, or null: the causal chain
  float *part_o, *part_ml;     // [B * Hkv, rows, splits, D] and [.., 2]
  int64_t qb, qh, qt, ob, oh, ot, mb, mt;
  int B, Hkv, rep, T, W, D, slots, max_len;
  int splits, row_blocks;      // set by plan_attend, as are
  Divisor by_splits, by_row_blocks, by_rep, by_heads, by_rows;
  float scale_log2;            // the softmax scale times log2(e)
};

struct VerifyArgs {
  const void* target;      // [B, T, V] probabilities
  const void* draft;       // [B, T - 1, V] or null
  const int64_t* tokens;   // [B, T]
  const int64_t* parents;  // [B, T] or null: a chain
  const void* uniforms;    // [B, T]
  int64_t* out_tokens;     // [B, T]
  int64_t* counts;         // [B]
  int64_t* path;           // [B, T]
  double* partial;         // [B, chunks]
  int* meta;               // [B, 3 + T]: last node, residual, how many tokens are left out, those
  int64_t tb, tt, db, dt, kb, pb, ub;  // element strides
  int B, T, chunks, uniform_is_64;
  int64_t V;
};

hipError_t launch_rotary(RotaryArgs a, ServingType type, int V, bool interleaved, hipStream_t stream);
hipError_t launch_cache_append(const CacheArgs& a, ServingType type, CacheKind kind, hipStream_t stream);
hipError_t launch_cache_read(const CacheArgs& a, ServingType type, CacheKind kind, ServingType out, hipStream_t stream);
hipError_t launch_cache_keep(const CacheArgs& a, const int64_t* path, int row_bytes, hipStream_t stream);
void plan_attend(AttendArgs& a);
hipError_t launch_attend(const AttendArgs& a, ServingType type, CacheKind kind, hipStream_t stream);
hipError_t launch_verify(const VerifyArgs& a, ServingType type, hipStream_t stream);
