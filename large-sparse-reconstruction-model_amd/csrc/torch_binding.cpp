// Eager PyTorch entry points of the operators whose smallest calls take less
// time on the GPU than their binding does in Python: sliding-window attention,
// its single-token form and the residual norm.  Argument checks, output and
// workspace allocation, autograd nodes and the calls of the C ABI
// (lsrm_hip.h) in one extension module, lsrm_hip._native; traced calls go
// through the operators that lsrm_hip/torch_ops.py registers, to the same
// kernels.  A call of five rows of the residual norm takes 6 us of the
// host this way (3.5 of them the launch), 20 through the registered operator.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <optional>
#include <tuple>

#include "lsrm_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

constexpr int64_t MAX_STRIDE = int64_t{1} << 22;  // elements between tokens

bool given(const OptTensor& t) { return t.has_value() && t->defined(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor tensor_or_none(const OptTensor& t) { return given(t) ? *t : Tensor(); }

void check(int rc, const char* what) {
  TORCH_CHECK(rc == LSRM_OK, what, " failed: ", lsrm_status_string(rc), " (status ", rc, ")");
}

void on_device(const Tensor& t, const Tensor& first) {
  TORCH_CHECK(t.is_cuda(), "lsrm_hip kernels need ROCm device tensors; got a tensor on ",
              t.device(), " (there is no CPU fallback)");
  TORCH_CHECK(t.device() == first.device(), "all tensors must live on the same device");
  TORCH_CHECK(!t._fw_grad(0).defined(), "no forward-mode derivative");
}

int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return LSRM_F32;
    case at::kHalf: return LSRM_F16;
    case at::kBFloat16: return LSRM_BF16;
    default: return -1;
  }
}

hipStream_t stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

Tensor int32(const Tensor& t) { return t.to(at::kInt).contiguous(); }

Tensor workspace(size_t bytes, const Tensor& like) {
  return at::empty({(int64_t)(bytes ? bytes : 1)}, like.options().dtype(at::kByte));
}

// ------------------------------------------------------- sliding windows --

// The tensor and the elements between its tokens for [N, H, D]; a contiguous
// copy where a token's heads are not contiguous or its rows cannot be read in
// 16-byte pieces.
std::pair<Tensor, int64_t> token_rows(const Tensor& t) {
  const int64_t n = t.size(0), h = t.size(1), d = t.size(2), dense = h * d;
  int64_t stride = -1;
  if (t.is_contiguous())
    stride = dense;
  else if (t.stride(2) == 1 && (h == 1 || t.stride(1) == d))
    stride = n > 1 ? t.stride(0) : dense;
  if (stride < dense || stride % 8 || stride > MAX_STRIDE || (uintptr_t)t.data_ptr() % 16)
    return {t.clone(at::MemoryFormat::Contiguous), dense};
  return {t, stride};
}

Tensor aligned(const Tensor& t) {
  const Tensor c = t.contiguous();
  return (uintptr_t)c.data_ptr() % 16 ? c.clone() : c;
}

void check_qkv(const Tensor& q, const Tensor& k, const Tensor& v) {
  for (const Tensor* t : {&q, &k, &v}) on_device(*t, q);
  TORCH_CHECK_VALUE(q.dim() == 3 && k.dim() == 3 && v.sizes() == k.sizes() &&
                        q.size(2) == k.size(2),
                    "q [Nq, Hq, D], k and v [Nk, Hkv, D] expected");
  TORCH_CHECK_TYPE((q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16) &&
                       k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                   "q, k and v must share dtype float16 or bfloat16");
  TORCH_CHECK_VALUE(k.size(1) != 0 && q.size(1) % k.size(1) == 0,
                    "num_q_heads must be a multiple of num_kv_heads");
}

struct Bias {
  Tensor table, buckets;
  int64_t n_buckets = 0, range = -1;
};

Bias bias_args(const Tensor& q, const OptTensor& table, const OptTensor& buckets) {
  Bias b;
  TORCH_CHECK_VALUE(given(table) == given(buckets), "bias_table and bias_buckets go together");
  if (!given(table)) return b;
  on_device(*table, q);
  on_device(*buckets, q);
  TORCH_CHECK_VALUE(table->dim() == 2 && table->size(1) == q.size(1) && table->size(0) > 0,
                    "bias_table must be [num_buckets, num_q_heads = ", q.size(1), "]");
  TORCH_CHECK_TYPE(table->scalar_type() == q.scalar_type(),
                   "bias_table must share the dtype of q");
  TORCH_CHECK_VALUE(buckets->dim() == 1 && buckets->numel() % 2 == 1,
                    "bias_buckets must be [2 * max_distance + 1]");
  b.table = table->contiguous();
  b.buckets = int32(*buckets);
  b.n_buckets = table->size(0);
  b.range = buckets->numel() / 2;
  return b;
}

struct Rule {
  int64_t left, right, sinks;
  double scale;
};

// -> (out, lse, out_low); lse and out_low are undefined where they are not wanted.
std::tuple<Tensor, Tensor, Tensor> window_fwd(const Tensor& q_, const Tensor& k_,
                                              const Tensor& v_, const Tensor& cu_q,
                                              const Tensor& cu_k, const Rule& r,
                                              const Bias& bias, bool with_lse, bool low) {
  const auto [q, qs] = token_rows(q_);
  const auto [k, ks] = token_rows(k_);
  const auto [v, vs] = token_rows(v_);
  const int64_t nq = q.size(0), hq = q.size(1), d = q.size(2);
  Tensor out = at::empty({nq, hq, d}, q.options());
  Tensor lse, out_low;
  if (with_lse) lse = at::empty({hq, nq}, q.options().dtype(at::kFloat));
  if (low) out_low = at::empty({nq, hq, d}, q.options().dtype(at::kChar));
  check(lsrm_window_attn_fwd(ptr(q), ptr(k), ptr(v), dtype_code(q), qs, ks, vs, nq, k.size(0),
                             hq, k.size(1), d, cu_q.data_ptr<int32_t>(),
                             cu_k.data_ptr<int32_t>(), cu_q.numel() - 1, r.left, r.right, r.sinks,
                             ptr(bias.table), bias.n_buckets, (const int32_t*)ptr(bias.buckets),
                             bias.range, (float)r.scale, ptr(out), ptr(out_low),
                             (float*)ptr(lse), stream_of(q)),
        "lsrm_window_attn_fwd");
  return {out, lse, out_low};
}

struct WindowNode : public torch::autograd::Function<WindowNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k,
                               const Tensor& v, const OptTensor& table, const Tensor& cu_q,
                               const Tensor& cu_k, const OptTensor& buckets, int64_t left,
                               int64_t right, int64_t sinks, double scale) {
    const Bias bias = bias_args(q, table, buckets);
    auto [out, lse, low] =
        window_fwd(q, k, v, cu_q, cu_k, Rule{left, right, sinks, scale}, bias, true, true);
    ctx->save_for_backward({q, k, v, tensor_or_none(table), out, lse, cu_q, cu_k,
                            tensor_or_none(buckets), low});
    ctx->saved_data["left"] = left;
    ctx->saved_data["right"] = right;
    ctx->saved_data["sinks"] = sinks;
    ctx->saved_data["scale"] = scale;
    ctx->mark_non_differentiable({lse});
    ctx->set_materialize_grads(false);
    return {out, lse};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list result(11);
    if (!grads[0].defined()) return result;
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "sliding_window_attention is differentiable once (no create_graph)");
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &cu_q = saved[6], &cu_k = saved[7];
    const c10::DeviceGuard guard(saved[0].device());
    const auto [q, qs] = token_rows(saved[0]);
    const auto [k, ks] = token_rows(saved[1]);
    const auto [v, vs] = token_rows(saved[2]);
    Bias bias;
    if (saved[3].defined()) bias = bias_args(q, saved[3], saved[8]);
    const Tensor dout = aligned(grads[0].to(q.scalar_type())), o = aligned(saved[4]);
    const int64_t nq = q.size(0), hq = q.size(1), d = q.size(2), nk = k.size(0), hkv = k.size(1);
    const int64_t left = ctx->saved_data["left"].toInt(), right = ctx->saved_data["right"].toInt(),
                  sinks = ctx->saved_data["sinks"].toInt(), batch = cu_q.numel() - 1;
    result[0] = at::empty({nq, hq, d}, q.options());
    result[1] = at::empty({nk, hkv, d}, q.options());
    result[2] = at::empty({nk, hkv, d}, q.options());
    if (bias.table.defined()) result[3] = at::empty_like(bias.table);
    const size_t bytes = lsrm_window_attn_bwd_workspace_size(nq, nk, hq, hkv, d, batch, left,
                                                             sinks, bias.range);
    const Tensor ws = workspace(bytes, q);
    check(lsrm_window_attn_bwd(
              ptr(dout), ptr(q), ptr(k), ptr(v), ptr(o), ptr(saved[9]),
              saved[5].data_ptr<float>(), dtype_code(q), qs, ks, vs, nq, nk, hq, hkv, d,
              cu_q.data_ptr<int32_t>(), cu_k.data_ptr<int32_t>(), batch, left, right, sinks,
              ptr(bias.table), bias.n_buckets, (const int32_t*)ptr(bias.buckets), bias.range,
              (float)ctx->saved_data["scale"].toDouble(), ptr(result[0]), ptr(result[1]),
              ptr(result[2]), ptr(result[3]), ptr(ws), (size_t)ws.numel(), stream_of(q)),
          "lsrm_window_attn_bwd");
    return result;
  }
};

// The flag word of a check in flight: pinned memory that the device writes, not
// given back before it has.  The host reads it in a short loop (an event's
// record and wait take 4 us longer) and falls back to waiting for the stream.
struct PendingCheck {
  static constexpr int32_t UNSET = -1;
  Tensor flags;
  hipStream_t stream = nullptr;
  bool open = false;
  volatile int32_t* word() { return flags.data_ptr<int32_t>(); }
  int32_t wait() {
    for (int i = 0; i < 200000 && *word() == UNSET; ++i) __builtin_ia32_pause();
    if (*word() == UNSET) {
      const hipError_t rc = hipStreamSynchronize(stream);
      open = false;
      TORCH_CHECK(rc == hipSuccess, "hipStreamSynchronize failed: ", hipGetErrorString(rc));
    }
    open = false;
    return *word();
  }
  ~PendingCheck() {
    if (open && *word() == UNSET) (void)hipStreamSynchronize(stream);
  }
};

// -> (out, lse or None, lsrm_meta_error bits).  validate: the offsets and the bucket
// map are checked on the device; the attention is launched behind the check,
// whose answer the host waits for (in pinned memory).
std::tuple<Tensor, Tensor, int64_t> window_attention(
    const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu_seqlens_q,
    const Tensor& cu_seqlens_k, int64_t left, int64_t right, int64_t sinks,
    const OptTensor& table, const OptTensor& buckets, double scale, bool with_lse,
    bool validate) {
  check_qkv(q, k, v);
  on_device(cu_seqlens_q, q);
  on_device(cu_seqlens_k, q);
  TORCH_CHECK_VALUE(cu_seqlens_q.dim() == 1 && cu_seqlens_q.sizes() == cu_seqlens_k.sizes() &&
                        cu_seqlens_q.numel() > 0,
                    "cu_seqlens_q and cu_seqlens_k must both have batch_size + 1 entries");
  const c10::DeviceGuard guard(q.device());
  const Tensor cu_q = int32(cu_seqlens_q), cu_k = int32(cu_seqlens_k);
  const Bias bias = bias_args(q, table, buckets);
  const hipStream_t st = stream_of(q);
  if (validate) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    validate = hipStreamIsCapturing(st, &status) == hipSuccess &&
               status == hipStreamCaptureStatusNone;
  }
  PendingCheck pending;
  if (validate) {
    pending.flags = at::empty({1}, at::TensorOptions().dtype(at::kInt).pinned_memory(true));
    *pending.word() = PendingCheck::UNSET;
    pending.stream = st;
    check(lsrm_window_validate(cu_q.data_ptr<int32_t>(), cu_k.data_ptr<int32_t>(),
                               cu_q.numel() - 1, q.size(0), k.size(0),
                               (const int32_t*)ptr(bias.buckets), bias.range < 0 ? 0 : bias.range,
                               bias.n_buckets, pending.flags.data_ptr<int32_t>(), st),
          "lsrm_window_validate");
    pending.open = true;
  }
  Tensor out, lse;
  if (at::GradMode::is_enabled() &&
      (q.requires_grad() || k.requires_grad() || v.requires_grad() ||
       (given(table) && table->requires_grad()))) {
    const OptTensor map = given(table) ? OptTensor(bias.buckets) : OptTensor();
    const variable_list r = WindowNode::apply(q, k, v, given(table) ? table : OptTensor(), cu_q,
                                              cu_k, map, left, right, sinks, scale);
    out = r[0];
    lse = r[1];
  } else {
    std::tie(out, lse, std::ignore) =
        window_fwd(q, k, v, cu_q, cu_k, Rule{left, right, sinks, scale}, bias, with_lse, false);
  }
  const int64_t bits = validate ? pending.wait() : 0;
  return {out, lse, bits};
}

struct CacheStrides {
  int64_t batch = 0, token = 0, head = 0;
};

CacheStrides cache_strides(const char* name, const Tensor& t) {
  CacheStrides s;
  if (t.numel() == 0) return s;
  // the stride of a dimension of one element is never used
  const auto at = [&](int i) { return t.size(i) > 1 ? t.stride(i) : 0; };
  s = CacheStrides{at(0), at(1), at(2)};
  TORCH_CHECK_VALUE((t.size(3) == 1 || t.stride(3) == 1) && s.batch % 8 == 0 &&
                        s.token % 8 == 0 && s.head % 8 == 0 && s.token <= MAX_STRIDE &&
                        (uintptr_t)t.data_ptr() % 16 == 0,
                    name, ": channels must be contiguous, the other strides multiples of 8 ",
                    "elements and the start 16-byte aligned (a cache is not copied)");
  return s;
}

std::tuple<Tensor, Tensor> window_decode(const Tensor& q_, const Tensor& k, const Tensor& v,
                                         const Tensor& seqlens, int64_t left, int64_t sinks,
                                         const OptTensor& table, const OptTensor& buckets,
                                         double scale, bool with_lse) {
  for (const Tensor* t : {&q_, &k, &v, &seqlens}) on_device(*t, q_);
  TORCH_CHECK_VALUE(q_.dim() == 3 && k.dim() == 4 && v.sizes() == k.sizes() &&
                        q_.size(0) == k.size(0) && q_.size(2) == k.size(3),
                    "q [B, Hq, D], k_cache and v_cache [B, capacity, Hkv, D] expected");
  TORCH_CHECK_TYPE((q_.scalar_type() == at::kHalf || q_.scalar_type() == at::kBFloat16) &&
                       k.scalar_type() == q_.scalar_type() &&
                       v.scalar_type() == q_.scalar_type(),
                   "q and the caches must share dtype float16 or bfloat16");
  const int64_t batch = q_.size(0), hq = q_.size(1), d = q_.size(2), capacity = k.size(1),
                hkv = k.size(2);
  TORCH_CHECK_VALUE(hkv != 0 && hq % hkv == 0, "num_q_heads must be a multiple of num_kv_heads");
  TORCH_CHECK_VALUE(seqlens.dim() == 1 && seqlens.size(0) == batch &&
                        (seqlens.scalar_type() == at::kInt || seqlens.scalar_type() == at::kLong),
                    "seqlens must be int32 [B]");
  const c10::DeviceGuard guard(q_.device());
  const Bias bias = bias_args(q_, table, buckets);
  const auto [q, qs] = token_rows(q_);
  const Tensor lens = int32(seqlens);
  const CacheStrides ks = cache_strides("k_cache", k), vs = cache_strides("v_cache", v);
  Tensor out = at::empty({batch, hq, d}, q.options());
  Tensor lse;
  if (with_lse) lse = at::empty({hq, batch}, q.options().dtype(at::kFloat));
  const size_t bytes =
      lsrm_window_decode_workspace_size(batch, capacity, hq, hkv, d, left, sinks);
  Tensor ws;
  if (bytes) ws = workspace(bytes, q);
  check(lsrm_window_decode(ptr(q), ptr(k), ptr(v), dtype_code(q), qs, ks.batch, ks.token, ks.head,
                           vs.batch, vs.token, vs.head, lens.data_ptr<int32_t>(), batch, capacity,
                           hq, hkv, d, left, sinks, ptr(bias.table), bias.n_buckets,
                           (const int32_t*)ptr(bias.buckets), bias.range, (float)scale, ptr(out),
                           (float*)ptr(lse), ptr(ws), bytes, stream_of(q)),
        "lsrm_window_decode");
  return {out, lse};
}

// --------------------------------------------------------- residual norm --

void check_rows(const Tensor& x, const Tensor& residual, const Tensor& weight) {
  on_device(x, x);
  on_device(weight, x);
  if (residual.defined()) on_device(residual, x);
  TORCH_CHECK_TYPE(dtype_code(x) >= 0 && weight.scalar_type() == x.scalar_type() &&
                       (!residual.defined() || residual.scalar_type() == x.scalar_type()),
                   "x, residual and weight must share one of bf16 / fp16 / fp32");
  TORCH_CHECK_VALUE(x.dim() >= 1 && weight.dim() == 1 && x.size(-1) == weight.size(0) &&
                        (!residual.defined() || residual.sizes() == x.sizes()),
                    "x and residual [.., hidden] of one shape and weight [hidden] expected");
  TORCH_CHECK_VALUE(x.size(-1) > 0 && x.size(-1) <= 16384, "hidden must be in 1 .. 16384");
}

std::tuple<Tensor, Tensor, Tensor, Tensor> norm_fwd(const Tensor& x_, const Tensor& residual_,
                                                    const Tensor& weight_, double eps,
                                                    int64_t least, const Tensor& rng_) {
  const Tensor x = x_.contiguous(), weight = weight_.contiguous();
  const Tensor residual = residual_.defined() ? residual_.contiguous() : residual_;
  const Tensor rng = rng_.defined() ? rng_.contiguous() : rng_;
  const int64_t hidden = x.size(-1), n = x.numel() / hidden;
  Tensor y = at::empty(x.sizes(), x.options()), h = at::empty(x.sizes(), x.options());
  Tensor rstd = at::empty({n}, x.options().dtype(at::kFloat));
  Tensor used;
  if (least > 0) used = at::empty({2}, rng.options());
  check(lsrm_residual_norm_fwd(ptr(x), ptr(residual), ptr(weight), dtype_code(x), n, hidden,
                               (float)eps, (int)least, (const int64_t*)ptr(rng),
                               (int64_t*)ptr(used), ptr(y), ptr(h), rstd.data_ptr<float>(),
                               stream_of(x)),
        "lsrm_residual_norm_fwd");
  return {y, h, rstd, used};
}

struct NormNode : public torch::autograd::Function<NormNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x,
                               const OptTensor& residual_, const Tensor& weight,
                               const OptTensor& rng_, double eps, int64_t least) {
    const Tensor residual = tensor_or_none(residual_), rng = tensor_or_none(rng_);
    auto [y, h, rstd, used] = norm_fwd(x, residual, weight, eps, least, rng);
    ctx->save_for_backward({h, weight, rstd, used});
    ctx->saved_data["least"] = least;
    ctx->saved_data["residual"] = residual.defined();
    ctx->set_materialize_grads(false);
    return {y, h};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list result(6);
    if (!grads[0].defined() && !grads[1].defined()) return result;
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "residual_rms_norm is differentiable once (no create_graph)");
    const variable_list saved = ctx->get_saved_variables();
    const int64_t least = ctx->saved_data["least"].toInt();
    const Tensor h = saved[0].contiguous(), weight = saved[1].contiguous();
    const Tensor &rstd = saved[2], &used = saved[3];
    const c10::DeviceGuard guard(h.device());
    const auto dense = [&](const Tensor& t) {
      return t.defined() ? t.to(h.scalar_type()).contiguous() : t;
    };
    const Tensor dy = dense(grads[0]), dh = dense(grads[1]);
    const int64_t hidden = h.size(-1), n = h.numel() / hidden;
    Tensor d_residual = at::empty(h.sizes(), h.options());
    Tensor d_weight = at::empty(weight.sizes(), weight.options());
    Tensor dx;
    if (least > 0) dx = at::empty(h.sizes(), h.options());
    const Tensor ws = workspace(lsrm_residual_norm_bwd_workspace_size(n, hidden), h);
    check(lsrm_residual_norm_bwd(ptr(dy), ptr(dh), ptr(h), ptr(weight), rstd.data_ptr<float>(),
                                 dtype_code(h), n, hidden, (int)least,
                                 (const int64_t*)ptr(used), ptr(dx), ptr(d_residual),
                                 ptr(d_weight), ptr(ws), (size_t)ws.numel(), stream_of(h)),
          "lsrm_residual_norm_bwd");
    // without dropout x and the residual have one gradient
    result[0] = least > 0 ? dx : d_residual;
    if (ctx->saved_data["residual"].toBool()) result[1] = d_residual;
    result[2] = d_weight;
    return result;
  }
};

std::tuple<Tensor, Tensor> residual_norm(const Tensor& x, const OptTensor& residual_,
                                         const Tensor& weight, double eps, int64_t least,
                                         const OptTensor& rng_) {
  const Tensor residual = tensor_or_none(residual_);
  check_rows(x, residual, weight);
  Tensor rng;
  if (least > 0) {
    TORCH_CHECK_VALUE(given(rng_), "dropout needs rng_state");
    rng = *rng_;
    on_device(rng, x);
    TORCH_CHECK_VALUE(rng.scalar_type() == at::kLong && rng.dim() == 1 && rng.size(0) == 2,
                      "rng_state must be int64 [2] (seed, offset)");
  }
  const c10::DeviceGuard guard(x.device());
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || weight.requires_grad() ||
       (residual.defined() && residual.requires_grad()))) {
    const auto optional = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    const variable_list r =
        NormNode::apply(x, optional(residual), weight, optional(rng), eps, least);
    return {r[0], r[1]};
  }
  const auto [y, h, rstd, used] = norm_fwd(x, residual, weight, eps, least, rng);
  return {y, h};
}

std::tuple<Tensor, Tensor, Tensor> residual_norm_fp8(const Tensor& x_, const OptTensor& residual_,
                                                     const Tensor& weight_, double eps,
                                                     int64_t group) {
  const Tensor given_residual = tensor_or_none(residual_);
  check_rows(x_, given_residual, weight_);
  const c10::DeviceGuard guard(x_.device());
  const Tensor x = x_.contiguous(), weight = weight_.contiguous();
  const Tensor residual = given_residual.defined() ? given_residual.contiguous() : given_residual;
  const int64_t hidden = x.size(-1), n = x.numel() / hidden;
  TORCH_CHECK_VALUE((group == 0 || group == 32 || group == 64 || group == 128) &&
                        (group == 0 || hidden % group == 0),
                    "group_size must be 0 (the row), 32, 64 or 128 and divide hidden");
  Tensor h = at::empty(x.sizes(), x.options());
  Tensor y8 = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn));
  auto shape = x.sizes().vec();
  shape.back() = group ? hidden / group : 1;
  Tensor scales = at::empty(shape, x.options().dtype(at::kFloat));
  check(lsrm_residual_norm_fp8(ptr(x), ptr(residual), ptr(weight), dtype_code(x), n, hidden,
                               (float)eps, group, ptr(y8), scales.data_ptr<float>(), ptr(h),
                               stream_of(x)),
        "lsrm_residual_norm_fp8");
  return {y8, scales, h};
}

}  // namespace

PYBIND11_MODULE(_native, m) {
  m.doc() = "Eager entry points of lsrm_hip (csrc/torch_binding.cpp).";
  // without the interpreter's lock: a check may wait for the device
  using Unlocked = pybind11::call_guard<pybind11::gil_scoped_release>;
  m.def("window_attention", &window_attention, Unlocked());
  m.def("window_decode", &window_decode, Unlocked());
  m.def("residual_norm", &residual_norm, Unlocked());
  m.def("residual_norm_fp8", &residual_norm_fp8, Unlocked());
}
