// Bindings of the serving kernels: rotary positions, the key/value cache,
// attention over it, and the verification of drafted tokens. Everything that
// the kernels assume of shapes, strides, types and devices is checked here.

#include <torch/extension.h>
#include <ATen/DeviceGuard.h>
#include <ATen/ExpandUtils.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/HIPContext.h>
#include <c10/hip/HIPStream.h>

#include <limits>
#include <tuple>

#include "serving.h"

int verify_chunks(int64_t V);
int verify_max_nodes();
int verify_meta_ints(int T);

namespace {

using OptTensor = c10::optional<at::Tensor>;

bool aligned16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

ServingType type_of(const at::Tensor& t, const char* who, bool fp32) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return ServingType::kBf16;
    case at::kHalf: return ServingType::kFp16;
    case at::kFloat:
      if (fp32) return ServingType::kFp32;
    default: break;
  }
  TORCH_CHECK(false, who, ": ", fp32 ? "bfloat16, float16 or float32" : "bfloat16 or float16", " expected, got ",
              t.scalar_type());
}

void check_device(const at::Tensor& t, const at::Tensor& as, const char* who, const char* name) {
  TORCH_CHECK(t.device() == as.device(), who, ": ", name, " is on ", t.device(), ", expected ", as.device());
}

hipStream_t current_stream() { return at::hip::getCurrentHIPStream().stream(); }

void check_launch(hipError_t e, const char* who) {
  TORCH_CHECK(e == hipSuccess, who, " launch failed: ", hipGetErrorString(e));
}

// Memory on the device of a tensor, past the dispatcher: small calls are bound
// by what the host does for them.
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& as) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, as.device(), c10::nullopt));
}

// One like t, its last dimension contiguous where t's is.
at::Tensor fresh_like(const at::Tensor& t) {
  if (t.is_non_overlapping_and_dense())
    return at::Tensor(at::detail::empty_strided_cuda(t.sizes(), t.strides(), t.scalar_type(), t.device()));
  const auto strides = at::infer_dense_strides(t.sizes(), t.strides());
  return at::Tensor(at::detail::empty_strided_cuda(t.sizes(), strides, t.scalar_type(), t.device()));
}

// A forward-mode derivative of a tensor, which the kernels would drop.
void check_not_dual(const at::Tensor& t, const char* who) {
  TORCH_CHECK(!t._fw_grad(0).defined(), who, " has no forward-mode derivative on the GPU");
}

constexpr int64_t kMaxInt = std::numeric_limits<int>::max();

}  // namespace

namespace {

std::tuple<at::Tensor, OptTensor> rotate(at::Tensor q, OptTensor k, at::Tensor cos_t, at::Tensor sin_t,
                                         OptTensor positions, bool interleaved, bool inverse) {
  const char* who = "rotary_embedding";
  TORCH_CHECK(q.is_cuda() && q.dim() == 4, who, ": q must be a [B, H, S, D] tensor on the GPU");
  const ServingType type = type_of(q, who, true);
  for (const at::Tensor* t : {&q, k.has_value() ? &*k : &q, &cos_t, &sin_t}) check_not_dual(*t, who);
  const int64_t B = q.size(0), S = q.size(2), D = q.size(3);
  if (k.has_value()) {
    check_device(*k, q, who, "k");
    TORCH_CHECK(k->dim() == 4 && k->scalar_type() == q.scalar_type() && k->size(0) == B && k->size(2) == S && k->size(3) == D,
                who, ": k must be [B, Hk, S, D] of q's type");
  }
  check_device(cos_t, q, who, "cos");
  check_device(sin_t, q, who, "sin");
  TORCH_CHECK(cos_t.dim() == 2 && cos_t.sizes() == sin_t.sizes() && cos_t.scalar_type() == at::kFloat &&
                  sin_t.scalar_type() == at::kFloat,
              who, ": cos and sin must be float32 tables [positions, rotary_dim / 2]");
  const int64_t R = 2 * cos_t.size(1);
  TORCH_CHECK(R <= D && D <= kMaxInt, who, ": the tables rotate ", R, " elements, head_dim is ", D);
  cos_t = cos_t.contiguous();
  sin_t = sin_t.contiguous();
  if (!positions.has_value())
    TORCH_CHECK(S <= cos_t.size(0), who, ": ", S, " positions, the tables have ", cos_t.size(0));

  const c10::OptionalDeviceGuard guard(at::device_of(q));
  RotaryArgs a{};
  if (positions.has_value()) {
    check_device(*positions, q, who, "positions");
    TORCH_CHECK(positions->scalar_type() == at::kLong || positions->scalar_type() == at::kInt, who,
                ": positions must be int64 or int32");
    TORCH_CHECK(positions->dim() <= 2 && positions->dim() >= 1 && positions->size(-1) == S &&
                    (positions->dim() == 1 || positions->size(0) == B || positions->size(0) == 1),
                who, ": positions must be [S] or [B, S]");
    a.positions = positions->data_ptr();
    a.pos_is_64 = positions->scalar_type() == at::kLong;
    a.pos_s = positions->stride(-1);
    a.pos_b = positions->dim() == 2 && positions->size(0) == B ? positions->stride(0) : 0;
  }
  if (q.stride(3) != 1) q = q.contiguous();
  auto yq = fresh_like(q);
  if (yq.stride(3) != 1) yq = fresh(q.sizes(), q.scalar_type(), q);
  OptTensor yk;
  if (k.has_value()) {
    if (k->stride(3) != 1) k = k->contiguous();
    yk = fresh_like(*k);
    if (yk->stride(3) != 1) yk = fresh(k->sizes(), k->scalar_type(), q);
  }
  a.table_rows = cos_t.size(0);
  a.cos_t = cos_t.data_ptr<float>();
  a.sin_t = sin_t.data_ptr<float>();
  a.tokens = B * S;
  a.S = S;
  a.D = (int)D;
  a.R = (int)R;
  a.sin_sign = inverse ? -1.f : 1.f;

  // the widest access that every address and stride allows
  const int esize = (int)q.element_size();
  int V = 16 / esize;
  const auto fits = [&](int v) {
    bool ok = (R / 2) % v == 0 && D % v == 0 && aligned16(cos_t) && aligned16(sin_t);
    for (const at::Tensor* t : {&q, &yq, k.has_value() ? &*k : &q, yk.has_value() ? &*yk : &yq}) {
      ok = ok && reinterpret_cast<uintptr_t>(t->data_ptr()) % (v * esize) == 0;
      for (int i = 0; i < 3; ++i) ok = ok && (t->size(i) == 1 || t->stride(i) % v == 0);
    }
    return ok;
  };
  if (!fits(V)) V = V > 4 && fits(4) ? 4 : 1;

  const auto fill = [](RotaryTensor& r, const at::Tensor& x, const at::Tensor& y) {
    r = {x.data_ptr(), y.data_ptr(), x.stride(0), x.stride(1), x.stride(2), y.stride(0), y.stride(1), y.stride(2)};
  };
  fill(a.q, q, yq);
  if (k.has_value()) fill(a.k, *k, *yk);
  TORCH_CHECK(q.size(1) + (k.has_value() ? k->size(1) : 0) <= 1 << 20, who, ": too many heads");
  a.Hq = (int)q.size(1);
  a.Hk = k.has_value() ? (int)k->size(1) : 0;
  if (a.tokens == 0 || a.Hq + a.Hk == 0 || D == 0) return {yq, yk};
  // a thread takes at least one element and one head
  TORCH_CHECK((double)a.tokens * (a.Hq + a.Hk) * (double)D < 256. * kMaxInt, who, ": too many tokens");
  check_launch(launch_rotary(a, type, V, interleaved, current_stream()), who);
  return {yq, yk};
}

// The gradient is the rotation back; being linear, that of the gradient is the
// rotation itself. In C++, as a Python backward costs more than the kernels of
// most calls.
class RotaryFunction : public torch::autograd::Function<RotaryFunction> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, at::Tensor q, OptTensor k,
                                                at::Tensor cos_t, at::Tensor sin_t, OptTensor positions,
                                                bool interleaved, bool inverse) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({cos_t, sin_t, positions.value_or(at::Tensor())});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["inverse"] = inverse;
    auto [yq, yk] = rotate(q, k, cos_t, sin_t, positions, interleaved, inverse);
    if (yk.has_value()) return {yq, *yk};
    return {yq};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const OptTensor positions = saved[2].defined() ? OptTensor(saved[2]) : OptTensor();
    const bool interleaved = ctx->saved_data["interleaved"].toBool(), back = !ctx->saved_data["inverse"].toBool();
    torch::autograd::variable_list defined, result(7);
    for (const auto& g : grads)
      if (g.defined()) defined.push_back(g);
    if (defined.empty()) return result;
    const OptTensor second = defined.size() > 1 ? OptTensor(defined[1]) : OptTensor();
    if (at::GradMode::is_enabled()) {
      defined = apply(defined[0], second, saved[0], saved[1], positions, interleaved, back);
    } else {
      auto [yq, yk] = rotate(defined[0], second, saved[0], saved[1], positions, interleaved, back);
      defined[0] = yq;
      if (yk.has_value()) defined[1] = *yk;
    }
    size_t next = 0;
    for (size_t i = 0; i < grads.size(); ++i)
      if (grads[i].defined()) result[i] = defined[next++];
    return result;
  }
};

}  // namespace

std::tuple<at::Tensor, OptTensor> rotary(at::Tensor q, OptTensor k, at::Tensor cos_t, at::Tensor sin_t,
                                         OptTensor positions, bool interleaved) {
  if (at::GradMode::is_enabled() && (q.requires_grad() || (k.has_value() && k->requires_grad()))) {
    auto y = RotaryFunction::apply(q, k, cos_t, sin_t, positions, interleaved, false);
    return {y[0], y.size() > 1 ? OptTensor(y[1]) : OptTensor()};
  }
  return rotate(q, k, cos_t, sin_t, positions, interleaved, false);
}

namespace {

// The cache's storage, as KVCache allocates it.
struct Cache {
  CacheKind kind;
  int B, H, slots, D;
};

Cache check_cache(const at::Tensor& k, const at::Tensor& v, const OptTensor& k_scale, const OptTensor& v_scale,
                  int64_t max_len, const char* who) {
  TORCH_CHECK(k.is_cuda() && k.dim() == 4 && k.is_contiguous() && v.is_contiguous() && k.sizes() == v.sizes() &&
                  k.scalar_type() == v.scalar_type(),
              who, ": the cache's keys and values must be contiguous [B, H, slots, D] tensors on the GPU");
  check_device(v, k, who, "the cache's values");
  Cache c;
  switch (k.scalar_type()) {
    case at::kChar: c.kind = CacheKind::kInt8; break;
    case at::kFloat8_e4m3fn: c.kind = CacheKind::kFp8; break;
    case at::kBFloat16:
    case at::kHalf: c.kind = CacheKind::kSame; break;
    default: TORCH_CHECK(false, who, ": a cache of ", k.scalar_type(), " is not supported");
  }
  for (int i = 0; i < 4; ++i) TORCH_CHECK(k.size(i) <= kMaxInt, who, ": the cache is too large");
  c.B = (int)k.size(0);
  c.H = (int)k.size(1);
  c.slots = (int)k.size(2);
  c.D = (int)k.size(3);
  TORCH_CHECK(c.D == 32 || c.D == 64 || c.D == 128 || c.D == 256, who, ": head_dim must be 32, 64, 128 or 256, got ", c.D);
  TORCH_CHECK(c.slots % kSlotTile == 0 && max_len >= 0 && max_len <= c.slots && max_len < kMaxInt - 1024, who,
              ": bad slots for max_len ", max_len);
  TORCH_CHECK(c.B <= 65535, who, ": at most 65535 sequences");
  TORCH_CHECK(aligned16(k) && aligned16(v), who, ": the cache must be aligned to 16 bytes");
  if (c.kind != CacheKind::kSame) {
    for (const OptTensor* s : {&k_scale, &v_scale}) {
      TORCH_CHECK(s->has_value() && (*s)->is_contiguous() && (*s)->scalar_type() == at::kFloat && (*s)->dim() == 3 &&
                      (*s)->size(0) == c.B && (*s)->size(1) == c.H && (*s)->size(2) == c.slots && aligned16(**s),
                  who, ": an 8-bit cache has float32 scales [B, H, slots]");
      check_device(**s, k, who, "the cache's scales");
    }
  }
  return c;
}

const int* check_lengths(const OptTensor& t, const Cache& c, const at::Tensor& as, const char* who, const char* name) {
  if (!t.has_value()) return nullptr;
  check_device(*t, as, who, name);
  TORCH_CHECK(t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == c.B && t->is_contiguous(), who, ": ", name,
              " must be a contiguous int32 tensor [B]");
  return t->data_ptr<int>();
}

void fill_cache(CacheArgs& a, const Cache& c, const at::Tensor& k, const at::Tensor& v, const OptTensor& k_scale,
                const OptTensor& v_scale, int64_t max_len) {
  a.k = {k.data_ptr(), c.kind == CacheKind::kSame ? nullptr : k_scale->data_ptr<float>()};
  a.v = {v.data_ptr(), c.kind == CacheKind::kSame ? nullptr : v_scale->data_ptr<float>()};
  a.B = c.B;
  a.H = c.H;
  a.D = c.D;
  a.slots = c.slots;
  a.max_len = (int)max_len;
}

// 16 bytes at a time: the last dimension contiguous, the others in steps of 8
at::Tensor rows16(const at::Tensor& t) {
  bool ok = t.stride(3) == 1 && aligned16(t);
  for (int i = 0; i < 3; ++i) ok = ok && (t.size(i) == 1 || t.stride(i) % 8 == 0);
  if (ok) return t;
  return at::empty(t.sizes(), t.options()).copy_(t);
}

}  // namespace

void kv_cache_append(at::Tensor cache_k, at::Tensor cache_v, OptTensor k_scale, OptTensor v_scale, int64_t max_len,
                     at::Tensor k, at::Tensor v, OptTensor start, int64_t offset, OptTensor counts) {
  const char* who = "KVCache.append";
  const Cache c = check_cache(cache_k, cache_v, k_scale, v_scale, max_len, who);
  check_device(k, cache_k, who, "k");
  check_device(v, cache_k, who, "v");
  check_not_dual(k, who);
  check_not_dual(v, who);
  const ServingType type = type_of(k, who, false);
  TORCH_CHECK(k.dim() == 4 && k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type() && k.size(0) == c.B &&
                  k.size(1) == c.H && k.size(3) == c.D,
              who, ": k and v must be [", c.B, ", ", c.H, ", T, ", c.D, "] of one type");
  TORCH_CHECK(c.kind != CacheKind::kSame || k.scalar_type() == cache_k.scalar_type(), who, ": the cache holds ",
              cache_k.scalar_type(), ", got ", k.scalar_type());
  TORCH_CHECK(2 * c.B * (int64_t)c.H * k.size(2) < kMaxInt, who, ": too many tokens in one call");
  TORCH_CHECK(offset >= 0 && offset <= kMaxInt, who, ": bad offset ", offset);
  const c10::OptionalDeviceGuard guard(at::device_of(cache_k));
  CacheArgs a{};
  fill_cache(a, c, cache_k, cache_v, k_scale, v_scale, max_len);
  a.start = check_lengths(start, c, cache_k, who, "lengths");
  a.counts = check_lengths(counts, c, cache_k, who, "counts");
  a.offset = offset;
  a.T = (int)k.size(2);
  if (c.B == 0 || c.H == 0 || a.T == 0) return;
  // the cache's own rows would be written while others of them are read
  const auto own = [&](const at::Tensor& t) { return t.is_alias_of(cache_k) || t.is_alias_of(cache_v); };
  const at::Tensor in[2] = {rows16(own(k) ? k.clone() : k), rows16(own(v) ? v.clone() : v)};
  for (int i = 0; i < 2; ++i) {
    a.x[i] = in[i].data_ptr();
    a.sb[i] = in[i].stride(0);
    a.sh[i] = in[i].stride(1);
    a.st[i] = in[i].stride(2);
  }
  a.heads_first = a.sh[0] < a.st[0];
  check_launch(launch_cache_append(a, type, c.kind, current_stream()), who);
}

std::tuple<at::Tensor, at::Tensor> kv_cache_read(at::Tensor cache_k, at::Tensor cache_v, OptTensor k_scale,
                                                 OptTensor v_scale, int64_t max_len, OptTensor start, int64_t offset,
                                                 int64_t length, at::ScalarType dtype) {
  const char* who = "KVCache.read";
  const Cache c = check_cache(cache_k, cache_v, k_scale, v_scale, max_len, who);
  TORCH_CHECK(length >= 0 && offset >= 0 && offset <= kMaxInt && 2 * std::max<int64_t>(c.B, 1) * std::max<int64_t>(c.H, 1) <= kMaxInt &&
                  length < kMaxInt / (2 * std::max<int64_t>(c.B, 1) * std::max<int64_t>(c.H, 1)),
              who, ": bad length ", length, " or offset ", offset);
  const c10::OptionalDeviceGuard guard(at::device_of(cache_k));
  auto yk = fresh({c.B, c.H, length, c.D}, dtype, cache_k);
  auto yv = fresh({c.B, c.H, length, c.D}, dtype, cache_k);
  const ServingType out = type_of(yk, who, true);
  CacheArgs a{};
  fill_cache(a, c, cache_k, cache_v, k_scale, v_scale, max_len);
  a.start = check_lengths(start, c, cache_k, who, "start");
  a.offset = offset;
  a.T = (int)length;
  a.y[0] = yk.data_ptr();
  a.y[1] = yv.data_ptr();
  if (yk.numel() == 0) return {yk, yv};
  const ServingType type = cache_k.scalar_type() == at::kHalf ? ServingType::kFp16 : ServingType::kBf16;
  check_launch(launch_cache_read(a, type, c.kind, out, current_stream()), who);
  return {yk, yv};
}

void kv_cache_keep(at::Tensor cache_k, at::Tensor cache_v, OptTensor k_scale, OptTensor v_scale, int64_t max_len,
                   at::Tensor start, at::Tensor path) {
  const char* who = "KVCache.keep";
  const Cache c = check_cache(cache_k, cache_v, k_scale, v_scale, max_len, who);
  check_device(path, cache_k, who, "path");
  TORCH_CHECK(path.scalar_type() == at::kLong && path.dim() == 2 && path.size(0) == c.B && path.size(1) <= kMaxInt, who,
              ": path must be an int64 tensor [B, T]");
  const c10::OptionalDeviceGuard guard(at::device_of(cache_k));
  path = path.contiguous();
  CacheArgs a{};
  fill_cache(a, c, cache_k, cache_v, k_scale, v_scale, max_len);
  a.start = check_lengths(start, c, cache_k, who, "lengths");
  a.T = (int)path.size(1);
  TORCH_CHECK(2 * (int64_t)c.B * c.H < kMaxInt, who, ": the cache is too large");
  if (c.B == 0 || c.H == 0 || a.T == 0) return;
  check_launch(launch_cache_keep(a, path.data_ptr<int64_t>(), (int)(c.D * cache_k.element_size()), current_stream()), who);
}

at::Tensor kv_cache_attend(at::Tensor q, at::Tensor cache_k, at::Tensor cache_v, OptTensor k_scale, OptTensor v_scale,
                           int64_t max_len, at::Tensor lengths, OptTensor mask, double scale) {
  const char* who = "cache_attention";
  const Cache c = check_cache(cache_k, cache_v, k_scale, v_scale, max_len, who);
  check_device(q, cache_k, who, "q");
  check_not_dual(q, who);
  const ServingType type = type_of(q, who, false);
  TORCH_CHECK(q.dim() == 4 && q.size(0) == c.B && q.size(3) == c.D, who, ": q must be [", c.B, ", Hq, T, ", c.D, "]");
  TORCH_CHECK(c.H > 0 ? q.size(1) % c.H == 0 : q.size(1) == 0, who, ": ", q.size(1),
              " query heads are no multiple of the cache's ", c.H);
  TORCH_CHECK(c.kind != CacheKind::kSame || q.scalar_type() == cache_k.scalar_type(), who, ": the cache holds ",
              cache_k.scalar_type(), ", q is ", q.scalar_type());
  const c10::OptionalDeviceGuard guard(at::device_of(cache_k));
  AttendArgs a{};
  const int64_t Hq = q.size(1), T = q.size(2);
  a.B = c.B;
  a.Hkv = c.H;
  a.rep = c.H ? (int)(Hq / c.H) : 0;
  a.T = (int)T;
  a.W = (int)T;
  a.D = c.D;
  a.slots = c.slots;
  a.max_len = (int)max_len;
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  a.lengths = check_lengths(lengths, c, cache_k, who, "lengths");
  if (mask.has_value()) {
    check_device(*mask, q, who, "mask");
    TORCH_CHECK(mask->scalar_type() == at::kBool && (mask->dim() == 2 || mask->dim() == 3) && mask->size(-2) == T &&
                    (mask->dim() == 2 || mask->size(0) == c.B || mask->size(0) == 1),
                who, ": mask must be a bool tensor [T, W] or [B, T, W]");
    TORCH_CHECK(mask->size(-1) <= max_len, who, ": the mask covers ", mask->size(-1), " slots, the cache has ", max_len);
    if (mask->stride(-1) != 1) mask = mask->contiguous();
    a.mask = reinterpret_cast<const uint8_t*>(mask->data_ptr<bool>());
    a.W = (int)mask->size(-1);
    a.mt = mask->stride(-2);
    a.mb = mask->dim() == 3 && mask->size(0) == c.B ? mask->stride(0) : 0;
  }
  // where the model reshapes [B, T, Hq * D] next, this is a view
  at::Tensor out(at::detail::empty_strided_cuda({c.B, Hq, T, c.D}, {T * Hq * c.D, c.D, Hq * c.D, 1}, q.scalar_type(),
                                                q.device()));
  if (out.numel() == 0) return out;
  if (max_len == 0 && mask.has_value()) return out.zero_();  // nothing to see
  TORCH_CHECK(T <= max_len || mask.has_value(), who, ": ", T, " new tokens, the cache has ", max_len, " slots");
  TORCH_CHECK(c.B * Hq * T < kMaxInt && T * a.rep < kMaxInt, who, ": too many rows");
  q = rows16(q);
  a.q = q.data_ptr();
  a.qb = q.stride(0);
  a.qh = q.stride(1);
  a.qt = q.stride(2);
  a.k = cache_k.data_ptr();
  a.v = cache_v.data_ptr();
  if (c.kind != CacheKind::kSame) {
    a.k_scale = k_scale->data_ptr<float>();
    a.v_scale = v_scale->data_ptr<float>();
  }
  a.out = out.data_ptr();
  a.ob = out.stride(0);
  a.oh = out.stride(1);
  a.ot = out.stride(2);
  const int rows = (int)(T * a.rep);
  plan_attend(a);
  TORCH_CHECK((int64_t)a.splits * c.H * c.B * a.row_blocks < kMaxInt - 8 * (int64_t)a.row_blocks, who, ": too many workgroups");
  at::Tensor part;
  if (a.splits > 1) {
    const int64_t parts = (int64_t)c.B * c.H * rows * a.splits;
    part = fresh({parts * (c.D + 2)}, at::kFloat, q);
    a.part_o = part.data_ptr<float>();
    a.part_ml = a.part_o + parts * c.D;
  }
  check_launch(launch_attend(a, type, c.kind, current_stream()), who);
  return out;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> verify_draft(at::Tensor target, at::Tensor tokens, at::Tensor uniforms,
                                                            OptTensor draft, OptTensor parents) {
  const char* who = "verify_draft";
  TORCH_CHECK(target.is_cuda() && target.dim() == 3, who, ": target_probs must be a [B, T, V] tensor on the GPU");
  const ServingType type = type_of(target, who, true);
  const int64_t B = target.size(0), T = target.size(1), V = target.size(2);
  TORCH_CHECK(T >= 1 && T <= verify_max_nodes(), who, ": 1 to ", verify_max_nodes(), " nodes, got ", T);
  TORCH_CHECK(V >= 1 && V < kMaxInt / 2 && B <= 65535, who, ": bad sizes [", B, ", ", T, ", ", V, "]");
  TORCH_CHECK(!(draft.has_value() && parents.has_value()), who,
              ": draft_probs are for chains; the tokens of a tree are taken as certain drafts");
  check_device(tokens, target, who, "tokens");
  check_device(uniforms, target, who, "uniforms");
  TORCH_CHECK(tokens.scalar_type() == at::kLong && tokens.dim() == 2 && tokens.size(0) == B && tokens.size(1) == T, who,
              ": tokens must be int64 [B, T]");
  TORCH_CHECK((uniforms.scalar_type() == at::kFloat || uniforms.scalar_type() == at::kDouble) && uniforms.dim() == 2 &&
                  uniforms.size(0) == B && uniforms.size(1) == T,
              who, ": uniforms must be float32 or float64 [B, T]");
  const c10::OptionalDeviceGuard guard(at::device_of(target));
  VerifyArgs a{};
  if (draft.has_value()) {
    check_device(*draft, target, who, "draft_probs");
    TORCH_CHECK(draft->scalar_type() == target.scalar_type() && draft->dim() == 3 && draft->size(0) == B &&
                    draft->size(1) == T - 1 && draft->size(2) == V,
                who, ": draft_probs must be [B, T - 1, V] of target_probs' type");
    if (draft->stride(2) != 1) draft = draft->contiguous();
    a.draft = draft->data_ptr();
    a.db = draft->stride(0);
    a.dt = draft->stride(1);
  }
  if (parents.has_value()) {
    check_device(*parents, target, who, "parents");
    TORCH_CHECK(parents->scalar_type() == at::kLong && parents->size(-1) == T &&
                    (parents->dim() == 1 || (parents->dim() == 2 && (parents->size(0) == B || parents->size(0) == 1))),
                who, ": parents must be int64 [T] or [B, T]");
    if (parents->stride(-1) != 1) parents = parents->contiguous();
    a.parents = parents->data_ptr<int64_t>();
    a.pb = parents->dim() == 2 && parents->size(0) == B ? parents->stride(0) : 0;
  }
  if (target.stride(2) != 1) target = target.contiguous();
  tokens = tokens.contiguous();
  uniforms = uniforms.contiguous();
  auto out_tokens = fresh({B, T}, at::kLong, tokens);
  auto counts = fresh({B}, at::kLong, tokens);
  auto path = fresh({B, T}, at::kLong, tokens);
  if (B == 0) return {out_tokens, counts, path};
  a.chunks = verify_chunks(V);
  const int64_t meta_ints = verify_meta_ints((int)T);
  const int64_t sums = B * a.chunks;
  auto work = fresh({sums + (B * meta_ints + 1) / 2}, at::kDouble, target);  // the chunks' sums, then meta
  a.target = target.data_ptr();
  a.tb = target.stride(0);
  a.tt = target.stride(1);
  a.tokens = tokens.data_ptr<int64_t>();
  a.kb = tokens.stride(0);
  a.uniforms = uniforms.data_ptr();
  a.ub = uniforms.stride(0);
  a.uniform_is_64 = uniforms.scalar_type() == at::kDouble;
  a.out_tokens = out_tokens.data_ptr<int64_t>();
  a.counts = counts.data_ptr<int64_t>();
  a.path = path.data_ptr<int64_t>();
  a.partial = work.data_ptr<double>();
  a.meta = reinterpret_cast<int*>(a.partial + sums);
  a.B = (int)B;
  a.T = (int)T;
  a.V = V;
  check_launch(launch_verify(a, type, current_stream()), who);
  return {out_tokens, counts, path};
}

void bind_serving(pybind11::module_& m) {
  m.def("rotary", &rotary, "rotary positions of q and k (positions per token, part of the head, both layouts)");
  m.def("kv_cache_append", &kv_cache_append, "write keys and values behind a cache, quantised to 8 bits");
  m.def("kv_cache_read", &kv_cache_read, "read a window of a cache back in 16 or 32 bits",
        pybind11::arg("k"), pybind11::arg("v"), pybind11::arg("k_scale"), pybind11::arg("v_scale"),
        pybind11::arg("max_len"), pybind11::arg("start"), pybind11::arg("offset"), pybind11::arg("length"),
        pybind11::arg("dtype"));
  m.def("kv_cache_keep", &kv_cache_keep, "move the accepted path of a draft tree together");
  m.def("kv_cache_attend", &kv_cache_attend, "attention of a few tokens over a cache (tree mask, 16 or 8 bits)");
  m.def("verify_draft", &verify_draft, "verification of drafted tokens -> (tokens, counts, path)");
}
