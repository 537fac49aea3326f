// Verification of drafted tokens against the target's probabilities, from
// given random numbers.
//
// Node 0 is the last token that stands; a drafted node i > 0 follows its
// parent, and target row i is the target's distribution after node i. From
// the root on, with w the weights of the current node's row:
//   sampled drafts (a chain, with the distribution q that each was drawn
//     from): take token x of the child iff u_i q(x) < p(x); at the first
//     refusal the answer comes from max(p - q, 0).
//   certain drafts (a chain or a tree): the children in order; take child i
//     iff u_i r < p(x), where r = 1 - the mass of the siblings refused before
//     it; where none is taken the answer comes from p without those.
// The answer is the first token whose cumulative weight exceeds u_0 times the
// sum of all. So the tokens that come out are distributed as the target's.
//
// All comparisons and sums are in 64 bits: they decide whole numbers, and the
// sum over a vocabulary of 10^5 in 32 bits would move the borders between
// tokens by about their own width.
//
// Bound by latency and then by reading one row (with q two) a sequence: 8 chains
// of 5 drafts over 128256 tokens take 5.4 us for each of the two kernels and
// 10.8 a captured call, 2 trees of 22 nodes over 50257 4.9 each and 9.8. The
// walk needs one value (two) a node, read by a thread each, and is done by
// every workgroup for itself, so that a grid over chunks of the vocabulary
// can sum its row at once, without a launch between; a second kernel finds
// the chunk and the token in it.

#include "serving.h"

namespace {

constexpr int kThreads = 256;
constexpr int kRun = 8;           // vocabulary entries a thread sums,
constexpr int kChunk = kRun * kThreads;  // and a workgroup
constexpr int kMaxNodes = 1024;  // of a tree, root included

template <typename T>
__device__ __forceinline__ double wide(T x) { return (double)(float)x; }

__device__ __forceinline__ double uniform_at(const VerifyArgs& a, int b, int i) {
  return a.uniform_is_64 ? reinterpret_cast<const double*>(a.uniforms)[b * a.ub + i]
                         : (double)reinterpret_cast<const float*>(a.uniforms)[b * a.ub + i];
}

// What the answer is drawn from: 0 the row as it is, 1 less the draft's, 2 without tokens
enum Residual { kRow = 0, kLess = 1, kWithout = 2 };

// meta of a sequence: last node, residual, tokens left out, those tokens
constexpr int kMetaHead = 3;

// A thread's weights x = from, from + kThreads, ...: all reads before their use.
template <typename T>
__device__ __forceinline__ void weights_at(const T* p, const T* q, int residual, int64_t from, int64_t to, double* w) {
  T pv[kRun], qv[kRun];
#pragma unroll
  for (int i = 0; i < kRun; ++i) {
    const int64_t x = from + i * kThreads;
    pv[i] = x < to ? p[x] : (T)0.f;
    qv[i] = (T)0.f;
  }
  if (residual == kLess) {
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const int64_t x = from + i * kThreads;
      if (x < to) qv[i] = q[x];
    }
  }
#pragma unroll
  for (int i = 0; i < kRun; ++i) {
    const double y = wide(pv[i]) - wide(qv[i]);
    w[i] = y > 0. ? y : 0.;  // NaN too
  }
}

template <typename T>
__device__ __forceinline__ double weight_at(const T* p, const T* q, int residual, int64_t x) {
  double w = wide(p[x]);
  if (residual == kLess) w -= wide(q[x]);
  return w > 0. ? w : 0.;  // NaN too
}

// The first (last) thread of the workgroup for which a condition holds, or
// kThreads (-1). By votes: an atomic of all threads is done a lane at a time.
__device__ __forceinline__ int first_thread(bool is, int* votes) {
  const unsigned long long lanes = __ballot(is);
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) votes[wave] = lanes ? wave * 64 + __builtin_ctzll(lanes) : kThreads;
  __syncthreads();
  return min(min(votes[0], votes[1]), min(votes[2], votes[3]));
}

__device__ __forceinline__ int last_thread(bool is, int* votes) {
  const unsigned long long lanes = __ballot(is);
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) votes[wave] = lanes ? wave * 64 + 63 - __builtin_clzll(lanes) : -1;
  __syncthreads();
  return max(max(votes[0], votes[1]), max(votes[2], votes[3]));
}

// A lane's value; the lane is the same for the whole wave.
__device__ __forceinline__ double of_lane(double x, int lane) {
  const unsigned long long bits = __double_as_longlong(x);
  const unsigned low = __builtin_amdgcn_readlane((int)bits, lane), high = __builtin_amdgcn_readlane((int)(bits >> 32), lane);
  return __longlong_as_double((long long)((unsigned long long)high << 32 | low));
}

template <typename T>
__global__ void __launch_bounds__(kThreads) verify_walk_kernel(VerifyArgs a) {
  __shared__ double p_of[kMaxNodes], test_of[kMaxNodes];  // taken iff test (times what is left) < p
  __shared__ int token_of[kMaxNodes], parent_of[kMaxNodes], without[kMaxNodes];
  __shared__ int path[kMaxNodes];
  __shared__ int s_last, s_residual, s_without, s_count;
  __shared__ int votes[2][kThreads / 64];
  __shared__ unsigned left_out[kChunk / 32];  // a bit of each token of the chunk
  __shared__ double sums[kThreads / 64];
  const int b = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x;
  const T* target = reinterpret_cast<const T*>(a.target) + b * a.tb;
  const T* draft = a.draft ? reinterpret_cast<const T*>(a.draft) + b * a.db : nullptr;

  for (int i = tid; i < a.T; i += kThreads) {
    const int64_t token = a.tokens[b * a.kb + i];
    const int64_t parent = i == 0 ? -1 : (a.parents ? a.parents[b * a.pb + i] : (int64_t)i - 1);
    // a node without a token of the vocabulary, or that follows none before it, is none
    const bool is = i > 0 && token >= 0 && token < a.V && parent >= 0 && parent < i;
    token_of[i] = is ? (int)token : -1;
    parent_of[i] = is ? (int)parent : -1;
    p_of[i] = is ? wide(target[parent * a.tt + token]) : 0.;
    const double u = uniform_at(a, b, i);
    test_of[i] = is && draft ? u * wide(draft[parent * a.dt + token]) : u;
  }
  if (tid < kChunk / 32) left_out[tid] = 0;
  __syncthreads();

  if (!a.parents) {  // a chain ends at the first node that is none or not taken
    int first = a.T;
    for (int from = 1; from < a.T && first == a.T; from += kThreads) {
      const int i = from + tid;
      const int thread = first_thread(i < a.T && !(token_of[i] >= 0 && test_of[i] < p_of[i]), votes[from / kThreads & 1]);
      if (thread < kThreads) first = from + thread;
    }
    if (tid == 0) {
      const int last = first - 1;
      const bool refused = first < a.T && token_of[first] >= 0;
      s_last = last;
      s_count = last;
      s_residual = !refused ? kRow : draft ? kLess : kWithout;
      s_without = refused && !draft ? 1 : 0;
      if (s_without) without[0] = token_of[first];
    }
    for (int i = tid; i < first; i += kThreads) path[i] = i;
  } else if (tid < 64) {
    // Children come after their parents, so one pass in order is the walk: 64
    // nodes at a time, each in a lane, and the open children of the current
    // node as a vote: trees of 22 nodes take 10.1 us, of 200 11.3. (One thread
    // that reads node after node from LDS takes 11.6 and 22.6.)
    int cur = 0, n = 0, count = 0;
    double left = 1.;
    path[0] = 0;
    for (int base = 0; base < a.T; base += 64) {
      const int i = base + tid;
      const bool in = i < a.T;
      const int parent = in ? parent_of[i] : -1, token = in ? token_of[i] : -1;
      const double p = in ? p_of[i] : 0., test = in ? test_of[i] : 0.;
      bool again = false;  // a token refused before has nothing left
#pragma unroll 8
      for (int j = 0; j < n; ++j) again |= without[j] == token;
      unsigned long long open = __ballot(parent == cur && !again);
      while (open) {
        const int at = __builtin_ctzll(open);
        const double pi = of_lane(p, at);
        if (of_lane(test, at) * left < pi) {
          cur = base + at;
          n = 0;
          left = 1.;
          path[++count] = cur;
          open = __ballot(parent == cur);
        } else {
          const int x = __builtin_amdgcn_readlane(token, at);
          left -= pi > 0. ? pi : 0.;  // NaN too
          without[n++] = x;
          open &= ~__ballot(token == x);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // lanes read what all of them wrote
    }
    if (tid == 0) {
      s_last = cur;
      s_count = count;
      s_residual = n ? kWithout : kRow;
      s_without = n;
    }
  }
  __syncthreads();

  const int last = s_last, residual = s_residual, n_without = s_without;
  if (chunk == 0) {
    int* meta = a.meta + (int64_t)b * (kMetaHead + a.T);
    if (tid == 0) {
      meta[0] = last;
      meta[1] = residual;
      meta[2] = n_without;
      a.counts[b] = s_count;
    }
    for (int i = tid; i < n_without; i += kThreads) meta[kMetaHead + i] = without[i];
    for (int i = tid; i < a.T; i += kThreads) {
      a.path[(int64_t)b * a.T + i] = i <= s_count ? path[i] : -1;
      if (i != s_count) a.out_tokens[(int64_t)b * a.T + i] = i < s_count ? token_of[path[i + 1]] : -1;
    }
  }

  const T* p = target + last * a.tt;
  const T* q = residual == kLess ? draft + last * a.dt : nullptr;
  const int64_t from = (int64_t)chunk * kChunk, to = min(from + kChunk, a.V);
  double w[kRun], sum = 0.;
  weights_at(p, q, residual, from + tid, to, w);
  if (n_without) {
    for (int j = tid; j < n_without; j += kThreads) {
      const int64_t x = without[j] - from;
      if (x >= 0 && x < kChunk) atomicOr(&left_out[x / 32], 1u << (x % 32));
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const int x = tid + i * kThreads;
      w[i] = left_out[x / 32] >> (x % 32) & 1 ? 0. : w[i];
    }
  }
#pragma unroll
  for (int i = 0; i < kRun; ++i) sum += w[i];
#pragma unroll
  for (int m = 32; m; m >>= 1) sum += __shfl_xor(sum, m);
  if ((tid & 63) == 0) sums[tid >> 6] = sum;
  __syncthreads();
  if (tid == 0) a.partial[(int64_t)b * a.chunks + chunk] = sums[0] + sums[1] + sums[2] + sums[3];
}

// The sums of a value over the threads up to each one, into ends[1..kThreads];
// ends[0] = 0. Sums that are joined in another order may fall by a rounding
// where a value is tiny, so a border is looked for as the first that passes it.
__device__ __forceinline__ void scan(double x, double* ends, double* shared) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const double y = __shfl_up(x, m);
    if (lane >= m) x += y;
  }
  if (lane == 63) shared[wave] = x;
  __syncthreads();
  for (int w = 0; w < wave; ++w) x += shared[w];
  ends[tid + 1] = x;
  if (tid == 0) ends[0] = 0.;
  __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kThreads) verify_answer_kernel(VerifyArgs a) {
  __shared__ double weights[kChunk + kThreads];  // a gap after each thread's run: no two start in one bank
  __shared__ double ends[kThreads + 1], shared[kThreads / 64];
  __shared__ double s_base;
  __shared__ int s_chunk, votes[6][kThreads / 64];
  const int b = blockIdx.x, tid = threadIdx.x;
  const int* meta = a.meta + (int64_t)b * (kMetaHead + a.T);
  const int last = meta[0], residual = meta[1], n_without = meta[2];
  const int gone = tid < n_without ? meta[kMetaHead + tid] : 0;  // read while the sums are
  const T* p = reinterpret_cast<const T*>(a.target) + b * a.tb + last * a.tt;
  const T* q = residual == kLess ? reinterpret_cast<const T*>(a.draft) + b * a.db + last * a.dt : nullptr;
  int64_t* out = a.out_tokens + (int64_t)b * a.T + a.counts[b];
  const double u = fmax(uniform_at(a, b, 0), 0.);
  const double* partial = a.partial + (int64_t)b * a.chunks;

  // the chunk: each thread has a run of them
  const int per = (a.chunks + kThreads - 1) / kThreads;
  const int c0 = min(tid * per, a.chunks), c1 = min(c0 + per, a.chunks);
  double sum = 0.;
  int positive = -1;
  for (int i = c0; i < c1; ++i) {
    sum += partial[i];
    if (partial[i] > 0.) positive = i;
  }
  scan(sum, ends, shared);
  double threshold = u * ends[kThreads];
  const int passing = first_thread(ends[tid + 1] > threshold && positive >= 0, votes[0]);
  const int last_positive = last_thread(positive >= 0, votes[1]);

  if (last_positive < 0) {
    // No weight at all. A residual that has none (a draft that covered all of
    // the target) gives way to the row itself; that, to token 0. Rare: the
    // whole workgroup goes over the row, twice.
    double row = 0.;
    if (residual != kRow)
      for (int64_t x = tid; x < a.V; x += kThreads) row += weight_at(p, q, kRow, x);
    __syncthreads();
    scan(row, ends, shared);
    threshold = u * ends[kThreads];
    int64_t token = 0;
    bool crossed = false;
    double base = 0.;
    for (int64_t from = 0; residual != kRow && from < a.V && !crossed; from += kThreads) {
      const int64_t x = from + tid;
      const double w = x < a.V ? weight_at(p, q, kRow, x) : 0.;
      __syncthreads();
      scan(w, ends, shared);
      const int thread = first_thread(w > 0. && base + ends[tid + 1] > threshold, votes[2]);
      const int some = last_thread(w > 0., votes[3]);
      crossed = thread < kThreads;
      if (crossed) token = from + thread;
      else if (some >= 0) token = from + some;
      base += ends[kThreads];
    }
    if (tid == 0) *out = token;
    return;
  }

  // Where rounding leaves no crossing, it is the last chunk, and in it the
  // last token, that has any weight.
  const bool crossed = passing < kThreads;
  if (tid == (crossed ? passing : last_positive)) {
    double base = ends[tid];
    int found = positive;
    for (int i = c0; crossed && i < positive; ++i) {
      if (base + partial[i] > threshold) {
        found = i;
        break;
      }
      base += partial[i];
    }
    s_chunk = found;
    s_base = base;
  }
  __syncthreads();
  const int64_t from = (int64_t)s_chunk * kChunk;
  const double base = s_base;
  const int n = (int)(min(from + kChunk, a.V) - from);
  double w[kRun];
  weights_at(p, q, residual, from + tid, from + n, w);
#pragma unroll
  for (int i = 0; i < kRun; ++i) weights[tid + i * kThreads + (tid + i * kThreads) / kRun] = w[i];
  __syncthreads();
  for (int j = tid; j < n_without; j += kThreads) {
    const int64_t x = (j < kThreads ? gone : meta[kMetaHead + j]) - from;
    if (x >= 0 && x < n) weights[x + x / kRun] = 0.;
  }
  __syncthreads();
  // the token in it: each thread has a run of eight
  sum = 0.;
  positive = -1;
#pragma unroll
  for (int i = 0; i < kRun; ++i) {
    w[i] = weights[tid * (kRun + 1) + i];
    sum += w[i];
    if (w[i] > 0.) positive = tid * kRun + i;
  }
  scan(sum, ends, shared);
  const int holder = first_thread(crossed && positive >= 0 && base + ends[tid + 1] > threshold, votes[4]);
  const int final = last_thread(positive >= 0, votes[5]);
  if (holder == kThreads) {  // rounding left no crossing in it
    if (tid == max(final, 0)) *out = from + max(positive, 0);
  } else if (tid == holder) {
    double at = base + ends[tid];
    int found = positive;
#pragma unroll
    for (int i = kRun - 1; i >= 0; --i) {  // the first is found last
      double upto = at;
#pragma unroll
      for (int j = 0; j <= i; ++j) upto += w[j];
      if (w[i] > 0. && upto > threshold) found = tid * kRun + i;
    }
    *out = from + found;
  }
}

template <typename T>
hipError_t verify_by_type(const VerifyArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((verify_walk_kernel<T>), dim3(a.chunks, a.B), dim3(kThreads), 0, stream, a);
  hipLaunchKernelGGL((verify_answer_kernel<T>), dim3(a.B), dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace

int verify_chunks(int64_t V) { return (int)((V + kChunk - 1) / kChunk); }
int verify_max_nodes() { return kMaxNodes; }
int verify_meta_ints(int T) { return kMetaHead + T; }

hipError_t launch_verify(const VerifyArgs& a, ServingType type, hipStream_t stream) {
  switch (type) {
    case ServingType::kBf16: return verify_by_type<__bf16>(a, stream);
    case ServingType::kFp16: return verify_by_type<_Float16>(a, stream);
    default: return verify_by_type<float>(a, stream);
  }
}
