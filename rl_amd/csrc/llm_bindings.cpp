// Bindings of the language-model operators: token log-probabilities, the
// token policy loss, the paged key-value append and the attention over it.
//
// The argument checks are plain functions of tensors on any device (the
// `*_check` entries), so that the CPU forms in rl_amd/ops/language.py refuse
// exactly what the kernels refuse.  Autograd nodes are C++: a small loss is
// bound by the host, and a Python node costs several times its kernel.

#include "llm_bindings.h"

#include <ATen/core/grad_mode.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <tuple>
#include <vector>

#include "paged_kv.h"
#include "token_loss.h"

#ifdef RL_AMD_WITH_HIP
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#endif

namespace rl_amd {
namespace {

using torch::Tensor;
using OptTensor = std::optional<Tensor>;

bool real16_32(const Tensor& t) {
  return t.scalar_type() == torch::kFloat32 || t.scalar_type() == torch::kBFloat16 ||
         t.scalar_type() == torch::kFloat16;
}

bool index_type(const Tensor& t) {
  return t.scalar_type() == torch::kInt64 || t.scalar_type() == torch::kInt32;
}

int code_of(const Tensor& t, const char* op) {
  switch (t.scalar_type()) {
    case torch::kFloat32: return RL_F32;
    case torch::kBFloat16: return RL_BF16;
    case torch::kFloat16: return RL_F16;
    case torch::kBool:
    case torch::kUInt8: return RL_U8;
    case torch::kInt32: return RL_I32;
    case torch::kInt64: return RL_I64;
    case torch::kInt8: return RL_I8;
    case torch::kInt16: return RL_I16;
    case torch::kFloat64: return RL_F64;
    default: break;
  }
  TORCH_CHECK_TYPE(false, op, ": unsupported dtype ", t.scalar_type());
}

void same_device(const Tensor& a, const Tensor& b, const char* op, const char* name) {
  TORCH_CHECK_VALUE(a.device() == b.device(), op, ": ", name, " is on ", b.device(),
                    ", expected ", a.device());
}

// The largest launch: 2^32 threads in all, 256 to a workgroup.
constexpr int64_t kMostBlocks = (int64_t(1) << 24) - 1;

// ------------------------------ log-probs -------------------------------- //
void token_log_probs_check(const Tensor& logits, const Tensor& tokens, double temperature) {
  const char* op = "token_log_probs";
  TORCH_CHECK_TYPE(real16_32(logits), op, ": logits must be float32, bfloat16 or float16, got ",
                   logits.scalar_type());
  TORCH_CHECK_TYPE(index_type(tokens), op, ": tokens must be int64 or int32, got ",
                   tokens.scalar_type());
  TORCH_CHECK_VALUE(logits.dim() >= 1 && tokens.sizes() == logits.sizes().slice(0, logits.dim() - 1),
                    op, ": tokens must have the shape of logits without its last dim, got ",
                    tokens.sizes(), " for logits ", logits.sizes());
  TORCH_CHECK_VALUE(logits.size(-1) >= 1 && logits.size(-1) <= INT32_MAX, op,
                    ": the vocabulary must hold 1 to 2**31 - 1 tokens, got ", logits.size(-1));
  // its reciprocal times log2(e) has to be a float32
  TORCH_CHECK_VALUE(temperature >= 1e-30 && temperature <= 1e30, op,
                    ": temperature must be positive and within 1e-30 to 1e30, got ", temperature);
  same_device(logits, tokens, op, "tokens");
}

// ----------------------------- policy loss ------------------------------- //
void token_policy_loss_check(const Tensor& log_probs, const Tensor& old_log_probs,
                             const Tensor& advantage, const OptTensor& mask, const OptTensor& ref,
                             double clip_low, double clip_high, double kl_coeff,
                             double entropy_coeff) {
  const char* op = "token_policy_loss";
  TORCH_CHECK_TYPE(real16_32(log_probs), op,
                   ": log_probs must be float32, bfloat16 or float16, got ",
                   log_probs.scalar_type());
  TORCH_CHECK_VALUE(log_probs.numel() > 0, op, ": log_probs is empty");
  auto like = [&](const Tensor& t, const char* name, bool real) {
    TORCH_CHECK_VALUE(t.sizes() == log_probs.sizes(), op, ": ", name, " must have log_probs' shape ",
                      log_probs.sizes(), ", got ", t.sizes());
    same_device(log_probs, t, op, name);
    TORCH_CHECK_TYPE(!real || real16_32(t), op, ": ", name,
                     " must be float32, bfloat16 or float16, got ", t.scalar_type());
    TORCH_CHECK_VALUE(!(at::GradMode::is_enabled() && t.requires_grad()), op, ": ", name,
                      " is data and must not require a gradient");
  };
  like(old_log_probs, "old_log_probs", true);
  if (mask) like(*mask, "mask", false);
  if (ref) like(*ref, "ref_log_probs", true);
  same_device(log_probs, advantage, op, "advantage");
  TORCH_CHECK_TYPE(real16_32(advantage), op,
                   ": advantage must be float32, bfloat16 or float16, got ",
                   advantage.scalar_type());
  TORCH_CHECK_VALUE(!(at::GradMode::is_enabled() && advantage.requires_grad()), op,
                    ": advantage is data and must not require a gradient");
  bool fits = advantage.dim() <= log_probs.dim();
  for (int64_t d = 1; fits && d <= advantage.dim(); ++d)
    fits = advantage.size(-d) == 1 || advantage.size(-d) == log_probs.size(-d);
  TORCH_CHECK_VALUE(fits, op, ": advantage ", advantage.sizes(),
                    " does not broadcast to log_probs ", log_probs.sizes());
  if (mask) code_of(*mask, op);
  TORCH_CHECK_VALUE(std::isfinite(clip_low) && clip_low >= 0 && std::isfinite(clip_high) &&
                        clip_high >= 0,
                    op, ": clip_low and clip_high must be finite and not negative, got ", clip_low,
                    " and ", clip_high);
  TORCH_CHECK_VALUE(std::isfinite(kl_coeff) && std::isfinite(entropy_coeff), op,
                    ": kl_coeff and entropy_coeff must be finite, got ", kl_coeff, " and ",
                    entropy_coeff);
}

// ------------------------------ paged cache ------------------------------ //
void cache_check(const char* op, const Tensor& k_cache, const Tensor& v_cache,
                 const Tensor& page_table, int64_t batch, int64_t kv_heads, int64_t dim) {
  TORCH_CHECK_TYPE(real16_32(k_cache) && v_cache.scalar_type() == k_cache.scalar_type(), op,
                   ": k_cache and v_cache must share one dtype of float32, bfloat16 and float16, got ",
                   k_cache.scalar_type(), " and ", v_cache.scalar_type());
  TORCH_CHECK_VALUE(k_cache.dim() == 4 && v_cache.sizes() == k_cache.sizes(), op,
                    ": k_cache and v_cache must be [pages, kv_heads, page_size, dim] alike, got ",
                    k_cache.sizes(), " and ", v_cache.sizes());
  same_device(k_cache, v_cache, op, "v_cache");
  same_device(k_cache, page_table, op, "page_table");
  const int64_t page = k_cache.size(2);
  TORCH_CHECK_VALUE(page >= 1 && page <= 4096 && (page & (page - 1)) == 0, op,
                    ": page_size must be a power of two up to 4096, got ", page);
  TORCH_CHECK_VALUE(k_cache.size(0) >= 1 && k_cache.size(0) <= INT32_MAX, op,
                    ": the cache must hold 1 to 2**31 - 1 pages, got ", k_cache.size(0));
  TORCH_CHECK_VALUE(k_cache.size(1) == kv_heads && k_cache.size(3) == dim, op,
                    ": the cache holds ", k_cache.size(1), " heads of dim ", k_cache.size(3),
                    ", expected ", kv_heads, " of ", dim);
  TORCH_CHECK_VALUE(dim >= 8 && dim <= 256 && dim % 8 == 0, op,
                    ": dim must be a multiple of 8 up to 256, got ", dim);
  const int64_t wide = 16 / k_cache.element_size();
  for (const Tensor* t : {&k_cache, &v_cache}) {
    TORCH_CHECK_VALUE(t->stride(3) == 1, op, ": a cache's last dim must be dense");
    bool aligned = reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0;
    for (int d = 0; d < 3; ++d) aligned = aligned && (t->size(d) == 1 || t->stride(d) % wide == 0);
    TORCH_CHECK_VALUE(aligned, op, ": a cache's rows must be aligned to 16 bytes");
  }
  TORCH_CHECK_TYPE(page_table.scalar_type() == torch::kInt32, op, ": page_table must be int32, got ",
                   page_table.scalar_type());
  TORCH_CHECK_VALUE(page_table.dim() == 2 && page_table.size(0) == batch, op,
                    ": page_table must be [batch, pages] with batch ", batch, ", got ",
                    page_table.sizes());
  TORCH_CHECK_VALUE(page_table.size(1) <= (int64_t(1) << 30) / page, op,
                    ": page_table must span at most 2**30 positions, got ", page_table.size(1),
                    " pages of ", page);
}

void per_sequence(const char* op, const Tensor& t, const char* name, int64_t batch,
                  const Tensor& cache) {
  TORCH_CHECK_TYPE(index_type(t), op, ": ", name, " must be int32 or int64, got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == batch, op, ": ", name, " must be [batch] with batch ",
                    batch, ", got ", t.sizes());
  same_device(cache, t, op, name);
}

void no_grad(const char* op, const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(!(at::GradMode::is_enabled() && t.requires_grad()), op, ": ", name,
                    " requires a gradient, and this operator has none: call it under torch.no_grad()");
  TORCH_CHECK_VALUE(!t._fw_grad(0).defined(), op, ": ", name,
                    " carries a forward derivative, and this operator has none");
}

using Rope = std::optional<std::tuple<Tensor, Tensor>>;

void paged_kv_append_check(const Tensor& k, const Tensor& v, const Tensor& k_cache,
                           const Tensor& v_cache, const Tensor& page_table, const Tensor& start,
                           const OptTensor& lengths, const OptTensor& q, const Rope& rope) {
  const char* op = "paged_kv_append";
  TORCH_CHECK_VALUE(k.dim() == 4 && v.sizes() == k.sizes(), op,
                    ": k and v must be [batch, tokens, kv_heads, dim] alike, got ", k.sizes(),
                    " and ", v.sizes());
  const int64_t batch = k.size(0), kv_heads = k.size(2), dim = k.size(3);
  TORCH_CHECK_VALUE(kv_heads >= 1, op, ": k has no heads");
  cache_check(op, k_cache, v_cache, page_table, batch, kv_heads, dim);
  for (const Tensor* t : {&k, &v}) {
    TORCH_CHECK_TYPE(t->scalar_type() == k_cache.scalar_type(), op, ": k and v must have the cache's dtype ",
                     k_cache.scalar_type(), ", got ", t->scalar_type());
    same_device(k_cache, *t, op, "k or v");
    no_grad(op, *t, "k or v");
  }
  no_grad(op, k_cache, "k_cache");
  no_grad(op, v_cache, "v_cache");
  TORCH_CHECK_VALUE(k_cache.data_ptr() != v_cache.data_ptr() || k_cache.data_ptr() == nullptr, op,
                    ": k_cache and v_cache are the same memory");
  for (const Tensor* t : {&k_cache, &v_cache})
    for (int d = 0; d < 3; ++d)
      TORCH_CHECK_VALUE(t->size(d) == 1 || t->stride(d) != 0, op,
                        ": a cache that is written must not be expanded");
  TORCH_CHECK_VALUE(batch * k.size(1) <= kMostBlocks, op, ": at most ", kMostBlocks,
                    " tokens in one call, got ", batch * k.size(1));
  per_sequence(op, start, "start", batch, k_cache);
  if (lengths) per_sequence(op, *lengths, "lengths", batch, k_cache);
  if (q) {
    TORCH_CHECK_VALUE(q->dim() == 4 && q->size(0) == batch && q->size(1) == k.size(1) &&
                          q->size(2) >= 1 && q->size(3) == dim,
                      op, ": q must be [batch, tokens, heads, dim] with k's batch, tokens and dim, got ",
                      q->sizes());
    TORCH_CHECK_TYPE(q->scalar_type() == k.scalar_type(), op, ": q must have the cache's dtype ",
                     k.scalar_type(), ", got ", q->scalar_type());
    same_device(k_cache, *q, op, "q");
    no_grad(op, *q, "q");
  }
  if (rope) {
    const Tensor &cos = std::get<0>(*rope), &sin = std::get<1>(*rope);
    TORCH_CHECK_VALUE(cos.dim() == 2 && sin.sizes() == cos.sizes() && cos.size(1) >= 1 &&
                          2 * cos.size(1) <= dim,
                      op, ": rope must be (cos, sin), each [positions, rotary_dim / 2] with rotary_dim "
                          "up to dim, got ", cos.sizes(), " and ", sin.sizes());
    for (const Tensor* t : {&cos, &sin}) {
      TORCH_CHECK_TYPE(t->scalar_type() == torch::kFloat32, op, ": rope must be float32, got ",
                       t->scalar_type());
      TORCH_CHECK_VALUE(t->is_contiguous(), op, ": rope must be contiguous");
      same_device(k_cache, *t, op, "rope");
      no_grad(op, *t, "rope");
    }
  } else {
    TORCH_CHECK_VALUE(!q, op, ": q is taken to be rotated, and there is no rope");
  }
}

void paged_attention_check(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache,
                           const Tensor& page_table, const Tensor& lengths, double scale) {
  const char* op = "paged_attention_decode";
  TORCH_CHECK_VALUE(q.dim() == 3 && q.size(1) >= 1, op, ": q must be [batch, heads, dim], got ",
                    q.sizes());
  TORCH_CHECK_VALUE(k_cache.dim() == 4 && k_cache.size(1) >= 1 && q.size(1) % k_cache.size(1) == 0, op,
                    ": the cache must be [pages, kv_heads, page_size, dim] with kv_heads a divisor of q's ",
                    q.size(1), " heads, got ", k_cache.sizes());
  cache_check(op, k_cache, v_cache, page_table, q.size(0), k_cache.size(1), q.size(2));
  TORCH_CHECK_TYPE(q.scalar_type() == k_cache.scalar_type(), op, ": q must have the cache's dtype ",
                   k_cache.scalar_type(), ", got ", q.scalar_type());
  same_device(k_cache, q, op, "q");
  per_sequence(op, lengths, "lengths", q.size(0), k_cache);
  TORCH_CHECK_VALUE(q.size(0) * q.size(1) <= kMostBlocks, op, ": at most ", kMostBlocks,
                    " (sequence, head) pairs in one call, got ", q.size(0) * q.size(1));
  TORCH_CHECK_VALUE(std::isfinite(scale), op, ": scale must be finite, got ", scale);
  no_grad(op, q, "q");
  no_grad(op, k_cache, "k_cache");
  no_grad(op, v_cache, "v_cache");
}

#ifdef RL_AMD_WITH_HIP

void* stream_of() { return (void*)c10::hip::getCurrentHIPStream().stream(); }

void launched(int status, const char* op) {
  TORCH_CHECK(status == 0, op, ": launch failed: ", hipGetErrorString((hipError_t)status));
}

// ------------------------------ log-probs -------------------------------- //
TokenLogProbArgs log_prob_args(const Tensor& logits, const Tensor& tokens, double temperature,
                               int64_t ignore_index) {
  TokenLogProbArgs a{};
  a.logits = logits.data_ptr();
  a.stride_batch = logits.stride(0);
  a.stride_row = logits.stride(1);
  a.width = logits.size(1);
  a.rows = logits.size(0) * a.width;
  a.vocab = (int)logits.size(2);
  a.dtype = code_of(logits, "token_log_probs");
  a.tokens = tokens.data_ptr();
  a.tokens_i32 = tokens.scalar_type() == torch::kInt32;
  a.ignore_index = ignore_index;
  a.inv_temperature = (float)(1.0 / temperature);
  return a;
}

// [.., V] as [batch, width, V] with a dense last dim; a copy only where the
// strides have no such form.
Tensor rows_of(const Tensor& logits) {
  Tensor x = logits;
  if (x.dim() == 1) x = x.view({1, 1, x.size(0)});
  if (x.dim() == 2) x = x.unsqueeze(0);
  if (x.dim() > 3) x = x.flatten(0, -3);
  return x.stride(2) == 1 || x.size(2) == 1 ? x : x.contiguous();
}

Tensor log_probs_raw(const Tensor& logits, const Tensor& tokens, double temperature,
                     int64_t ignore_index, Tensor* stats) {
  c10::DeviceGuard guard(logits.device());
  const auto f32 = logits.options().dtype(torch::kFloat32);
  Tensor lp = torch::empty(tokens.sizes(), f32);
  const Tensor x = rows_of(logits), t = tokens.contiguous();
  TokenLogProbArgs a = log_prob_args(x, t, temperature, ignore_index);
  a.log_probs = lp.data_ptr<float>();
  if (stats) {
    *stats = torch::empty({tokens.numel(), 2}, f32);
    a.stats = stats->data_ptr<float>();
  }
  if (!a.rows) return lp;
  Tensor parts;
  const int split = token_log_probs_parts(&a);
  if (split > 1) {
    parts = torch::empty({a.rows * split * 2}, f32);
    a.parts = parts.data_ptr<float>();
  }
  launched(launch_token_log_probs_fwd(&a, stream_of()), "token_log_probs");
  return lp;
}

// Whether a backward pass is left to elementary operations: where it is
// differentiated in turn (create_graph), and where upstream gradients are many at
// once (is_grads_batched), wrappers without memory of their own.
bool plain_backward(const torch::autograd::variable_list& grads) {
  return at::GradMode::is_enabled() ||
         std::any_of(grads.begin(), grads.end(),
                     [](const Tensor& g) { return g.defined() && !g.has_storage(); });
}

// The gradient (one-hot - softmax) * upstream / temperature in elementary
// operations.
Tensor log_probs_grad_plain(const Tensor& logits, const Tensor& tokens, const Tensor& upstream,
                            double temperature, int64_t ignore_index) {
  const Tensor gone = tokens.eq(ignore_index);
  const Tensor known = tokens.ge(0).logical_and(tokens.lt(logits.size(-1)));
  const Tensor g = upstream.to(torch::kFloat32).masked_fill(gone, 0);
  Tensor x = logits.to(torch::kFloat32) / temperature;
  // rows that pass nothing back may hold anything, and no NaN comes through them
  const Tensor finite = x.detach().logsumexp(-1).isfinite();
  const Tensor out = gone.logical_or(g.eq(0).logical_and(finite.logical_not()));
  x = x.masked_fill(out.unsqueeze(-1), 0);
  const Tensor at = tokens.to(torch::kInt64).masked_fill(known.logical_not(), 0).unsqueeze(-1);
  const Tensor hot =
      torch::zeros(logits.sizes(), logits.options().dtype(torch::kFloat32)).scatter_(-1, at, 1);
  const Tensor row = known.logical_or(gone).logical_or(g.eq(0));
  const Tensor d = (hot - x.softmax(-1)) * (g.masked_fill(row.logical_not(), NAN) / temperature).unsqueeze(-1);
  return d.to(logits.scalar_type());
}

class TokenLogProbs : public torch::autograd::Function<TokenLogProbs> {
 public:
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& logits,
                        const Tensor& tokens, double temperature, int64_t ignore_index) {
    Tensor stats;
    Tensor lp = log_probs_raw(logits, tokens, temperature, ignore_index, &stats);
    ctx->save_for_backward({logits, tokens, stats});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->set_materialize_grads(false);
    return lp;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const Tensor &logits = saved[0], &stats = saved[2];
    c10::DeviceGuard guard(logits.device());
    if (plain_backward(grads))
      return {log_probs_grad_plain(logits, saved[1], grads[0],
                                   ctx->saved_data["temperature"].toDouble(),
                                   ctx->saved_data["ignore_index"].toInt()),
              Tensor(), Tensor(), Tensor()};
    const Tensor tokens = saved[1].contiguous();
    const Tensor g = grads[0].to(torch::kFloat32).contiguous();
    Tensor out = torch::empty(logits.sizes(), logits.options());
    const Tensor x = rows_of(logits);
    TokenLogProbArgs a = log_prob_args(x, tokens, ctx->saved_data["temperature"].toDouble(),
                                       ctx->saved_data["ignore_index"].toInt());
    a.stats = stats.data_ptr<float>();
    a.upstream = g.data_ptr<float>();
    a.grad = out.data_ptr();
    if (a.rows) launched(launch_token_log_probs_bwd(&a, stream_of()), "token_log_probs");
    return {out, Tensor(), Tensor(), Tensor()};
  }
};

Tensor token_log_probs(const Tensor& logits, const Tensor& tokens, double temperature,
                       int64_t ignore_index) {
  token_log_probs_check(logits, tokens, temperature);
  TORCH_CHECK_VALUE(logits.is_cuda(), "token_log_probs: expected tensors on the GPU");
  if (at::GradMode::is_enabled() && logits.requires_grad())
    return TokenLogProbs::apply(logits, tokens, temperature, ignore_index);
  return log_probs_raw(logits, tokens, temperature, ignore_index, nullptr);
}

// ----------------------------- policy loss ------------------------------- //
struct PolicyViews {
  Tensor log_probs, old_log_probs, advantage, mask, ref;  // [rows, cols]; may be undefined
};

Tensor matrix_of(const Tensor& t, at::IntArrayRef shape) {
  Tensor x = t.sizes() == shape ? t : t.expand(shape);
  if (x.dim() == 2) return x;
  if (x.dim() < 2) return x.reshape({1, -1});
  return x.reshape({-1, shape.back()});  // a view where the strides allow it
}

PolicyOperand operand_of(const Tensor& t) {
  if (!t.defined()) return PolicyOperand{};
  return PolicyOperand{t.data_ptr(), (long)t.stride(0), (long)t.stride(1),
                       code_of(t, "token_policy_loss")};
}

struct PolicyConfig {
  int64_t variant;
  double low, high, kl, entropy;
  bool mean;
};

PolicyLossArgs policy_args(const PolicyViews& v, const PolicyConfig& c) {
  PolicyLossArgs a{};
  a.log_probs = operand_of(v.log_probs);
  a.old_log_probs = operand_of(v.old_log_probs);
  a.advantage = operand_of(v.advantage);
  a.mask = operand_of(v.mask);
  a.ref = operand_of(v.ref);
  a.rows = v.log_probs.size(0);
  a.cols = v.log_probs.size(1);
  a.variant = (int)c.variant;
  a.log_high = std::log1p(c.high);
  a.log_low = c.low < 1 ? std::log1p(-c.low) : -INFINITY;
  a.log_off = std::log1p(c.low);
  a.low = 1 - c.low;
  a.high = 1 + c.high;
  a.kl_coeff = c.kl;
  a.entropy_coeff = c.entropy;
  a.mean = c.mean;
  return a;
}

// The seven scalars and the three numbers that the backward pass needs, in one buffer.
Tensor policy_raw(const PolicyViews& v, const PolicyConfig& c) {
  c10::DeviceGuard guard(v.log_probs.device());
  PolicyLossArgs a = policy_args(v, c);
  a.blocks = policy_loss_blocks(a.rows * a.cols);
  Tensor out = torch::empty({10}, v.log_probs.options().dtype(torch::kFloat32));
  Tensor partials;
  if (a.blocks > 1) {
    partials = torch::empty({a.blocks, 8}, v.log_probs.options().dtype(torch::kFloat64));
    a.partials = partials.data_ptr<double>();
  }
  a.out = out.data_ptr<float>();
  a.scale = a.out + 7;
  launched(launch_policy_loss_fwd(&a, stream_of()), "token_policy_loss");
  return out;
}

// The seven scalars as tensors of their own over one allocation: not views of
// each other for autograd, so that a caller may change one in place.
std::vector<Tensor> scalars_of(const Tensor& out, int first, int last) {
  std::vector<Tensor> s;
  s.reserve(7);
  for (int i = first; i < last; ++i) {
    Tensor x = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(out.storage()), out.key_set(),
                                                        out.dtype());
    x.unsafeGetTensorImpl()->set_sizes_and_strides(at::IntArrayRef(), at::IntArrayRef(),
                                                   out.storage_offset() + i);
    s.push_back(std::move(x));
  }
  return s;
}

// The gradient in elementary operations, in double, for the upstream gradients `g`
// (undefined: none) of the five scalars.  `factor` is the 1 / D of the means.
Tensor policy_grad_plain(const Tensor& log_probs, const Tensor& old_log_probs,
                         const Tensor& advantage, const Tensor& mask, const Tensor& ref,
                         const Tensor& factor, const PolicyConfig& c, const Tensor (&g)[5]) {
  const auto f64 = [](const Tensor& t) { return t.to(torch::kFloat64); };
  const auto options = log_probs.options().dtype(torch::kFloat64);
  const Tensor w = mask.defined() ? f64(mask) : torch::ones(log_probs.sizes(), options);
  const Tensor gone = w.eq(0);
  const auto kept = [&](const Tensor& t) { return t.masked_fill(gone, 0); };
  const auto up = [&](int i) { return g[i].defined() ? f64(g[i]) : torch::zeros({}, options); };
  const Tensor total = up(0), lp = kept(f64(log_probs));
  const Tensor adv = kept(f64(advantage).expand(log_probs.sizes()));
  const Tensor x = kept(lp - f64(old_log_probs)), ratio = x.exp();
  const Tensor above = x.detach().gt(std::log1p(c.high));
  const Tensor below = c.low < 1 ? x.detach().lt(std::log1p(-c.low)) : torch::zeros_like(above);
  const Tensor against = above.logical_and(adv.gt(0)).logical_or(below.logical_and(adv.lt(0)));
  const Tensor dgain =
      adv * (c.variant == 0
                 ? ratio.masked_fill(against, 0)
                 : ratio.detach().masked_fill(above, 1 + c.high).masked_fill(below, 1 - c.low));
  Tensor d = (total + up(3)) * c.entropy - (total + up(1)) * dgain;
  if (ref.defined() && c.kl != 0) d = d - (total + up(2)) * c.kl * kept(f64(ref) - lp).expm1();
  d = kept(d * w * f64(factor));
  if (g[4].defined()) {
    const Tensor r = (f64(log_probs) - f64(old_log_probs)).exp();
    const Tensor squares = r.square().sum();
    const Tensor t = r * (r.sum() / squares.clamp_min(1e-9));
    const Tensor live = squares.detach().ge(1e-9).to(torch::kFloat64);
    d = d + up(4) * (2.0 / (double)log_probs.numel()) * (t - live * t.square());
  }
  return d.to(log_probs.scalar_type());
}

// The node of the five differentiable scalars; what they are is in `out` already.
class TokenPolicyLoss : public torch::autograd::Function<TokenPolicyLoss> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx,
                                                const Tensor& log_probs, const Tensor& old_lp,
                                                const Tensor& advantage, const OptTensor& mask,
                                                const OptTensor& ref, const Tensor& out,
                                                const std::vector<double>& config) {
    ctx->save_for_backward({log_probs, old_lp, advantage, mask ? *mask : Tensor(),
                            ref ? *ref : Tensor(), out});
    ctx->saved_data["config"] = config;
    ctx->set_materialize_grads(false);
    std::vector<Tensor> s = scalars_of(out, 0, 4);
    for (Tensor& x : scalars_of(out, 6, 7)) s.push_back(std::move(x));
    return s;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    torch::autograd::variable_list none(7);
    if (std::none_of(grads.begin(), grads.end(), [](const Tensor& g) { return g.defined(); }))
      return none;
    const auto saved = ctx->get_saved_variables();
    const auto cfg = ctx->saved_data["config"].toDoubleVector();
    const PolicyConfig c{(int64_t)cfg[0], cfg[1], cfg[2], cfg[3], cfg[4], cfg[5] != 0.0};
    if (plain_backward(grads)) {
      c10::DeviceGuard guard(saved[0].device());
      none[0] = policy_grad_plain(saved[0], saved[1], saved[2], saved[3], saved[4],
                                  saved[5].select(0, 7), c,
                                  {grads[0], grads[1], grads[2], grads[3], grads[4]});
      return none;
    }
    const auto shape = saved[0].sizes();
    PolicyViews v;
    v.log_probs = matrix_of(saved[0], shape);
    v.old_log_probs = matrix_of(saved[1], shape);
    v.advantage = matrix_of(saved[2], shape);
    if (saved[3].defined()) v.mask = matrix_of(saved[3], shape);
    if (saved[4].defined()) v.ref = matrix_of(saved[4], shape);
    c10::DeviceGuard guard(saved[0].device());
    PolicyLossArgs a = policy_args(v, c);
    a.scale = saved[5].data_ptr<float>() + 7;
    Tensor g[5];
    const float* p[5] = {};
    for (int i = 0; i < 5; ++i)
      if (grads[i].defined()) {
        g[i] = grads[i].to(torch::kFloat32);
        p[i] = g[i].data_ptr<float>();
      }
    a.g_total = p[0];
    a.g_objective = p[1];
    a.g_kl = p[2];
    a.g_entropy = p[3];
    a.g_ess = p[4];
    Tensor out = torch::empty(shape, saved[0].options());
    a.grad = out.data_ptr();
    launched(launch_policy_loss_bwd(&a, stream_of()), "token_policy_loss");
    none[0] = out;
    return none;
  }
};

std::vector<Tensor> token_policy_loss(const Tensor& log_probs, const Tensor& old_log_probs,
                                      const Tensor& advantage, const OptTensor& mask,
                                      const OptTensor& ref, int64_t variant, double clip_low,
                                      double clip_high, double kl_coeff, double entropy_coeff,
                                      bool mean) {
  token_policy_loss_check(log_probs, old_log_probs, advantage, mask, ref, clip_low, clip_high,
                          kl_coeff, entropy_coeff);
  TORCH_CHECK_VALUE(log_probs.is_cuda(), "token_policy_loss: expected tensors on the GPU");
  const auto shape = log_probs.sizes();
  const PolicyViews v{matrix_of(log_probs, shape), matrix_of(old_log_probs, shape),
                      matrix_of(advantage, shape), mask ? matrix_of(*mask, shape) : Tensor(),
                      ref ? matrix_of(*ref, shape) : Tensor()};
  const Tensor out =
      policy_raw(v, PolicyConfig{variant, clip_low, clip_high, kl_coeff, entropy_coeff, mean});
  if (!(at::GradMode::is_enabled() && log_probs.requires_grad())) return scalars_of(out, 0, 7);
  std::vector<Tensor> s = TokenPolicyLoss::apply(
      log_probs, old_log_probs, advantage, mask, ref, out,
      std::vector<double>{(double)variant, clip_low, clip_high, kl_coeff, entropy_coeff,
                          mean ? 1.0 : 0.0});
  std::vector<Tensor> data = scalars_of(out, 4, 6);
  s.insert(s.begin() + 4, data.begin(), data.end());
  return s;
}

// ------------------------------ paged cache ------------------------------ //
PagedCache cache_of(const Tensor& k, const Tensor& v, const Tensor& table) {
  PagedCache c{};
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  c.k_page = k.stride(0);
  c.k_head = k.stride(1);
  c.k_slot = k.stride(2);
  c.v_page = v.stride(0);
  c.v_head = v.stride(1);
  c.v_slot = v.stride(2);
  c.pages = k.size(0);
  while ((int64_t(1) << c.page_shift) < k.size(2)) ++c.page_shift;
  c.table = table.data_ptr<int>();
  c.table_stride = table.stride(0);
  c.table_cols = (int)table.size(1);
  return c;
}

Tensor dense_last(const Tensor& t) { return t.stride(-1) == 1 ? t : t.contiguous(); }

bool aligned_rows(const Tensor& t, int64_t wide) {
  bool ok = reinterpret_cast<uintptr_t>(t.data_ptr()) % (wide * t.element_size()) == 0;
  for (int64_t d = 0; d + 1 < t.dim(); ++d) ok = ok && (t.size(d) == 1 || t.stride(d) % wide == 0);
  return ok;
}

OptTensor paged_kv_append(const Tensor& k_in, const Tensor& v_in, const Tensor& k_cache,
                          const Tensor& v_cache, const Tensor& page_table, const Tensor& start,
                          const OptTensor& lengths, const OptTensor& q_in, const Rope& rope,
                          bool interleaved) {
  paged_kv_append_check(k_in, v_in, k_cache, v_cache, page_table, start, lengths, q_in, rope);
  TORCH_CHECK_VALUE(k_cache.is_cuda(), "paged_kv_append: expected tensors on the GPU");
  c10::DeviceGuard guard(k_cache.device());
  const Tensor k = dense_last(k_in), v = dense_last(v_in);
  const Tensor table = page_table.stride(1) == 1 ? page_table : page_table.contiguous();
  const Tensor first = start.contiguous();
  Tensor count, q, q_out;
  PagedAppendArgs a{};
  a.cache = cache_of(k_cache, v_cache, table);
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.k_batch = k.stride(0), a.k_token = k.stride(1), a.k_head = k.stride(2);
  a.v_batch = v.stride(0), a.v_token = v.stride(1), a.v_head = v.stride(2);
  a.start = first.data_ptr();
  a.start_i64 = first.scalar_type() == torch::kInt64;
  if (lengths) {
    count = lengths->contiguous();
    a.lengths = count.data_ptr();
    a.lengths_i64 = count.scalar_type() == torch::kInt64;
  }
  a.batch = k.size(0);
  a.width = (int)k.size(1);
  a.kv_heads = (int)k.size(2);
  a.dim = (int)k.size(3);
  a.dtype = code_of(k, "paged_kv_append");
  a.interleaved = interleaved;
  if (rope) {
    const Tensor& cos = std::get<0>(*rope);
    a.cos = cos.data_ptr<float>();
    a.sin = std::get<1>(*rope).data_ptr<float>();
    a.positions = cos.size(0);
    a.rotary = 2 * (int)cos.size(1);
  }
  if (q_in) {
    q = dense_last(*q_in);
    a.q = q.data_ptr();
    a.q_batch = q.stride(0), a.q_token = q.stride(1), a.q_head = q.stride(2);
    a.heads = (int)q.size(2);
    q_out = torch::empty(q.sizes(), q.options());
    a.q_out = q_out.data_ptr();
  }
  // the widest access, up to 16 bytes, that addresses and rotation halves allow
  a.vec = (int)(16 / k.element_size());
  auto fits = [&](int64_t wide) {
    return aligned_rows(k, wide) && aligned_rows(v, wide) && (!q_in || aligned_rows(q, wide)) &&
           a.rotary / 2 % wide == 0;
  };
  while (a.vec > 1 && !fits(a.vec)) a.vec = a.vec > 4 ? 4 : 1;
  if (a.batch * a.width) {
    launched(launch_paged_append(&a, stream_of()), "paged_kv_append");
    // what autograd has saved of the caches is no longer what it was
    for (const Tensor* t : {&k_cache, &v_cache})
      if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  }
  return q_in ? OptTensor(q_out) : std::nullopt;
}

Tensor paged_attention_decode(const Tensor& q_in, const Tensor& k_cache, const Tensor& v_cache,
                              const Tensor& page_table, const Tensor& lengths,
                              std::optional<double> scale_in) {
  const double scale =
      scale_in ? *scale_in : 1.0 / std::sqrt((double)std::max<int64_t>(1, q_in.size(-1)));
  paged_attention_check(q_in, k_cache, v_cache, page_table, lengths, scale);
  TORCH_CHECK_VALUE(q_in.is_cuda(), "paged_attention_decode: expected tensors on the GPU");
  c10::DeviceGuard guard(k_cache.device());
  Tensor q = dense_last(q_in);
  if (!aligned_rows(q, 16 / q.element_size())) q = q.clone(at::MemoryFormat::Contiguous);
  const Tensor table = page_table.stride(1) == 1 ? page_table : page_table.contiguous();
  const Tensor count = lengths.contiguous();
  Tensor out = torch::empty(q.sizes(), q.options());
  PagedAttendArgs a{};
  a.cache = cache_of(k_cache, v_cache, table);
  a.q = q.data_ptr();
  a.q_batch = q.stride(0);
  a.q_head = q.stride(1);
  a.out = out.data_ptr();
  a.lengths = count.data_ptr();
  a.lengths_i64 = count.scalar_type() == torch::kInt64;
  a.batch = q.size(0);
  a.heads = (int)q.size(1);
  a.kv_heads = (int)k_cache.size(1);
  a.dim = (int)q.size(2);
  a.dtype = code_of(q, "paged_attention_decode");
  a.scale = (float)(scale * 1.4426950408889634);
  if (!a.batch) return out;
  plan_paged_attend(&a, at::cuda::getCurrentDeviceProperties()->multiProcessorCount);
  Tensor part;
  if (a.workers) {
    const int64_t rows = 2 * (int64_t)a.workers * std::min(16, a.heads / a.kv_heads);
    const int64_t notes = a.workers * paged_attend_note_bytes() / 4;
    part = torch::empty({rows * (a.dim + 2) + notes}, q.options().dtype(torch::kFloat32));
    // widest accesses first: rows is even and dim a multiple of 8, so all are aligned
    a.part = part.data_ptr<float>();
    a.part_ms = a.part + rows * a.dim;
    a.notes = a.part_ms + rows * 2;
  }
  launched(launch_paged_attend(&a, stream_of()), "paged_attention_decode");
  return out;
}

#endif  // RL_AMD_WITH_HIP

}  // namespace

void define_language_ops(py::module& m) {
  m.def("token_log_probs_check", &token_log_probs_check, "argument checks of token_log_probs");
  m.def("token_policy_loss_check", &token_policy_loss_check, "argument checks of token_policy_loss");
  m.def("paged_kv_append_check", &paged_kv_append_check, "argument checks of paged_kv_append");
  m.def("paged_attention_check", &paged_attention_check,
        "argument checks of paged_attention_decode");
#ifdef RL_AMD_WITH_HIP
  m.def("token_log_probs", &token_log_probs, "log-probabilities of tokens under logits (HIP)");
  m.def("token_policy_loss", &token_policy_loss, "clipped token policy loss with KL (HIP)");
  m.def("paged_kv_append", &paged_kv_append, "paged key-value append with rotation (HIP)");
  m.def("paged_attention_decode", &paged_attention_decode,
        "single-token attention over a paged cache (HIP)");
#endif
}

}  // namespace rl_amd
