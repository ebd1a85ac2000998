// Python bindings of the token-policy operators and the multi-tensor AdamW step. Every entry point checks devices,
// types, shapes and strides, then launches on the current stream of the tensors' device; scratch memory comes from the
// caching allocator of that stream, call by call.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <tuple>
#include <vector>

#include "adamw_kernels.cuh"
#include "kernels.cuh"
#include "token_kernels.cuh"

namespace {

using torch::Tensor;
using OptT = c10::optional<Tensor>;

void ok(cudaError_t e, const char* what) { TORCH_CHECK(e == cudaSuccess, what, " failed: ", cudaGetErrorString(e)); }

// Numbers in messages are formatted here: where the extension is linked against a libstdc++ of its own, a number streamed
// into a message (c10::str) meets the locale of the other one and crashes.
std::string text(int64_t x) { return std::to_string(x); }
std::string text(double x) { return std::to_string(x); }
std::string text(c10::IntArrayRef x) {
  std::string s = "[";
  for (size_t i = 0; i < x.size(); ++i) s += (i ? ", " : "") + std::to_string(x[i]);
  return s + "]";
}

bool given(const OptT& t) { return t.has_value() && t->defined(); }

int token_dtype(const Tensor& t) {
  switch (t.scalar_type()) {
    case torch::kFloat32: return rlb::kTokF32;
    case torch::kBFloat16: return rlb::kTokBF16;
    case torch::kFloat16: return rlb::kTokF16;
    default: TORCH_CHECK_TYPE(false, "logits must be float32, bfloat16 or float16, got ", t.scalar_type());
  }
}

// Logits [rows, V] or [batch, rows, V] with any row strides and contiguous columns.
struct Logits {
  const Tensor& t;
  int dtype;
  int64_t rows, vocab;
  rlb::TokenRows z;
  explicit Logits(const Tensor& x) : t(x), dtype(token_dtype(x)) {
    TORCH_CHECK_VALUE(x.is_cuda(), "logits must be a CUDA tensor");
    TORCH_CHECK_NOT_IMPLEMENTED(!x._fw_grad(0).defined(), "the kernels have no forward-mode derivative by the logits");
    TORCH_CHECK_VALUE(x.dim() == 2 || x.dim() == 3, "logits must be [rows, V] or [batch, rows, V], got ", text(x.sizes()));
    vocab = x.size(-1);
    TORCH_CHECK_VALUE(vocab > 0, "logits need at least one column");
    TORCH_CHECK_VALUE(vocab == 1 || x.stride(-1) == 1, "the columns of logits must be contiguous");
    rows = x.numel() / vocab;
    TORCH_CHECK_VALUE(rows < (int64_t{1} << 31) && vocab < (int64_t{1} << 31), "logits have too many rows or columns");
    z = rows_of(x);
  }
  static rlb::TokenRows rows_of(const Tensor& x) {
    const int64_t inner = std::max<int64_t>(1, x.size(-2));
    return {x.data_ptr(), inner, x.dim() == 3 ? x.stride(0) : 0, x.stride(-2)};
  }
  std::vector<int64_t> lead() const { return {t.sizes().begin(), t.sizes().end() - 1}; }
  torch::TensorOptions f32() const { return t.options().dtype(torch::kFloat32).requires_grad(false); }
  // A contiguous tensor of the logits' leading shape.
  Tensor row_input(const Tensor& x, const char* name, c10::ScalarType dt) const {
    TORCH_CHECK_TYPE(x.scalar_type() == dt, name, " must be ", dt, ", got ", x.scalar_type());
    TORCH_CHECK_VALUE(x.device() == t.device(), name, " must be on the device of the logits");
    TORCH_CHECK_VALUE(x.sizes() == t.sizes().slice(0, t.dim() - 1), name, " must have the shape ",
                      text(t.sizes().slice(0, t.dim() - 1)), ", got ", text(x.sizes()));
    return x.contiguous();
  }
  // Whether every row of a gradient starts at the same place within 16 bytes as its logits.
  bool same_phase(const Tensor& grad) const {
    const int64_t size = t.element_size();
    auto same = [&](int64_t x, int64_t y) { return (x - y) * size % 16 == 0; };
    return (reinterpret_cast<uintptr_t>(t.data_ptr()) - reinterpret_cast<uintptr_t>(grad.data_ptr())) % 16 == 0 &&
           same(t.stride(-2), grad.stride(-2)) && (t.dim() == 2 || same(t.stride(0), grad.stride(0)));
  }
  // Where rows start at different places within 16 bytes, the gradient takes the logits' strides (if that costs at most
  // a quarter more memory), so that both can be accessed 16 bytes at a time. A whole number of 16 bytes in rows that are
  // padded to another pitch (a slice of a padded vocabulary) is left contiguous: its rows take the slower kernels.
  Tensor gradient() const {
    const int64_t size = t.element_size();
    bool wide = (vocab * size) % 16 == 0;
    if (!wide && !t.is_contiguous() && rows > 0) {
      int64_t span = vocab;
      bool plain = t.stride(-2) >= vocab;
      span += (t.size(-2) - 1) * t.stride(-2);
      if (t.dim() == 3) {
        plain = plain && t.stride(0) >= span;
        span += (t.size(0) - 1) * t.stride(0);
      }
      if (plain && span <= t.numel() + t.numel() / 4) {
        return torch::empty({span}, t.options().requires_grad(false)).as_strided(t.sizes(), t.strides());
      }
    }
    return torch::empty(t.sizes(), t.options().requires_grad(false));
  }
};

// Tokens and mask of the rows; holds contiguous copies where the caller's are not contiguous.
struct Index {
  Tensor tokens, mask;
  rlb::TokenIndex idx{};
  Index(const Logits& l, const Tensor& tok, const OptT& m) {
    TORCH_CHECK_TYPE(tok.scalar_type() == torch::kInt64 || tok.scalar_type() == torch::kInt32,
                     "tokens must be int64 or int32, got ", tok.scalar_type());
    tokens = l.row_input(tok, "tokens", tok.scalar_type());
    idx.tokens = tokens.data_ptr();
    idx.tokens_i64 = tokens.scalar_type() == torch::kInt64;
    if (given(m)) {
      const auto dt = m->scalar_type();
      TORCH_CHECK_TYPE(dt == torch::kBool || dt == torch::kUInt8 || dt == torch::kFloat32,
                       "mask must be bool, uint8 or float32, got ", dt);
      mask = l.row_input(*m, "mask", dt);
      idx.mask = mask.data_ptr();
      idx.mask_kind = dt == torch::kFloat32 ? 2 : 1;
    }
  }
};

double inverse(double temperature) {
  TORCH_CHECK_VALUE(temperature >= 1e-6 && temperature <= 1e6, "temperature must lie in [1e-6, 1e6], got ",
                    text(temperature));
  return 1.0 / temperature;
}

const float* scale_ptr(const Logits& l, const OptT& s) {
  if (!given(s)) return nullptr;
  TORCH_CHECK_VALUE(s->device() == l.t.device() && s->scalar_type() == torch::kFloat32 && s->numel() == 1,
                    "a gradient scale on the device must be one float32 there");
  return s->data_ptr<float>();
}

// ---- log-probabilities ----------------------------------------------------------------------------------------------
std::vector<Tensor> token_logprobs(const Tensor& logits, const Tensor& tokens, const OptT& mask, double temperature) {
  const Logits l(logits);
  const c10::cuda::CUDAGuard guard(logits.device());
  const Index ix(l, tokens, mask);
  Tensor logp = torch::empty(l.lead(), l.f32()), entropy = torch::empty(l.lead(), l.f32());
  Tensor ml = torch::empty({l.rows, 2}, l.f32());
  rlb::TokenStatsArgs a{};
  a.dtype = l.dtype, a.rows = l.rows, a.vocab = l.vocab, a.z = l.z, a.idx = ix.idx, a.inv_temp = inverse(temperature);
  a.logp = logp.data_ptr<float>();
  a.entropy = entropy.data_ptr<float>();
  a.ml = reinterpret_cast<float2*>(ml.data_ptr<float>());
  ok(rlb::token_stats(a, at::cuda::getCurrentCUDAStream()), "token_logprobs");
  return {logp, entropy, ml};
}

Tensor token_logprobs_backward(const Tensor& logits, const Tensor& tokens, const OptT& mask, double temperature,
                               const Tensor& ml, const Tensor& entropy, const Tensor& d_logp, const OptT& d_entropy) {
  const Logits l(logits);
  const c10::cuda::CUDAGuard guard(logits.device());
  const Index ix(l, tokens, mask);
  const Tensor da = l.row_input(d_logp, "d_logp", torch::kFloat32);
  Tensor db;
  TORCH_CHECK_VALUE(ml.is_contiguous() && ml.numel() == 2 * l.rows && entropy.numel() == l.rows,
                    "token_logprobs_backward: statistics of other logits");
  Tensor grad = l.gradient();
  rlb::TokenGradArgs a{};
  a.dtype = l.dtype, a.rows = l.rows, a.vocab = l.vocab, a.z = l.z, a.idx = ix.idx, a.inv_temp = inverse(temperature);
  a.out = Logits::rows_of(grad);
  a.ml = reinterpret_cast<const float2*>(ml.data_ptr<float>());
  a.entropy = entropy.data_ptr<float>();
  a.a = da.data_ptr<float>(), a.a_stride = 1;
  if (given(d_entropy)) {
    db = l.row_input(*d_entropy, "d_entropy", torch::kFloat32);
    a.b = db.data_ptr<float>(), a.b_stride = 1;
  }
  a.scale = 1.f;
  ok(rlb::token_grad(a, at::cuda::getCurrentCUDAStream()), "token_logprobs_backward");
  return grad;
}

// ---- policy loss ------------------------------------------------------------------------------------------------------
// Returns loss, surrogate, kl, entropy mean, clip fraction, factor, logp, then [grad] with want_grad, [entropy, ml, coef]
// without.
std::vector<Tensor> token_policy_loss(const Tensor& logits, const Tensor& tokens, const Tensor& old_logp,
                                      const Tensor& advantages, const OptT& ref_logp, const OptT& mask, double clip_lo,
                                      double clip_hi, double kl_coef, int64_t kl_kind, double entropy_coef,
                                      double temperature, bool mean, bool want_grad, double grad_scale,
                                      const OptT& grad_scale_device) {
  const Logits l(logits);
  const c10::cuda::CUDAGuard guard(logits.device());
  const auto stream = at::cuda::getCurrentCUDAStream();
  const Index ix(l, tokens, mask);
  const Tensor old = l.row_input(old_logp, "old_logp", torch::kFloat32);
  const Tensor adv = l.row_input(advantages, "advantages", torch::kFloat32);
  Tensor ref;
  rlb::PolicyTerms q{};
  q.old_logp = old.data_ptr<float>();
  q.adv = adv.data_ptr<float>();
  if (given(ref_logp)) {
    ref = l.row_input(*ref_logp, "ref_logp", torch::kFloat32);
    q.ref_logp = ref.data_ptr<float>();
  }
  q.clip_lo = static_cast<float>(clip_lo), q.clip_hi = static_cast<float>(clip_hi);
  q.kl_coef = static_cast<float>(kl_coef), q.entropy_coef = static_cast<float>(entropy_coef);
  q.kl_kind = static_cast<int>(kl_kind);
  // the loss is a tensor of its own where autograd takes it, else (one allocation less) a view like the means
  Tensor out = torch::empty({6}, l.f32()), logp = torch::empty(l.lead(), l.f32()), loss;
  if (!want_grad) loss = torch::empty({}, l.f32());
  // one row more than terms: the sum of the weights
  Tensor terms = torch::empty({l.rows + 1, 4}, l.f32()), entropy, ml, coef, grad;
  if (want_grad) grad = l.gradient();
  const bool one_pass = want_grad && l.same_phase(grad);
  rlb::TokenStatsArgs a{};
  a.dtype = l.dtype, a.rows = l.rows, a.vocab = l.vocab, a.z = l.z, a.idx = ix.idx, a.inv_temp = inverse(temperature);
  a.logp = logp.data_ptr<float>();
  a.policy = &q;
  a.terms = reinterpret_cast<float4*>(terms.data_ptr<float>());
  const float* scale_device = scale_ptr(l, grad_scale_device);
  if (one_pass) {
    ok(rlb::token_policy(a, Logits::rows_of(grad), static_cast<float>(grad_scale), scale_device, mean,
                         reinterpret_cast<double*>(terms.data_ptr<float>() + 4 * l.rows), stream),
       "token_policy_loss");
  } else {
    entropy = torch::empty(l.lead(), l.f32()), ml = torch::empty({l.rows, 2}, l.f32());
    coef = torch::empty({l.rows, 2}, l.f32());
    a.entropy = entropy.data_ptr<float>();
    a.ml = reinterpret_cast<float2*>(ml.data_ptr<float>());
    a.coef = reinterpret_cast<float2*>(coef.data_ptr<float>());
    ok(rlb::token_stats(a, stream), "token_policy_loss");
  }
  rlb::PolicyFinishArgs f{};
  f.rows = l.rows, f.terms = a.terms, f.idx = ix.idx, f.vocab = l.vocab, f.kl_coef = q.kl_coef;
  f.entropy_coef = q.entropy_coef, f.mean = mean;
  f.loss = want_grad ? out.data_ptr<float>() : loss.data_ptr<float>(), f.out = out.data_ptr<float>() + 1;
  ok(rlb::policy_finish(f, stream), "token_policy_loss");
  std::vector<Tensor> result = out.unbind();
  if (!want_grad) result[0] = loss;
  result.push_back(logp);
  if (!want_grad) {
    result.insert(result.end(), {entropy, ml, coef});
    return result;
  }
  if (!one_pass) {
    rlb::TokenGradArgs g{};
    g.dtype = l.dtype, g.rows = l.rows, g.vocab = l.vocab, g.z = l.z, g.idx = ix.idx, g.inv_temp = a.inv_temp;
    g.out = Logits::rows_of(grad);
    g.ml = a.ml, g.entropy = a.entropy;
    g.a = coef.data_ptr<float>(), g.a_stride = 2;
    if (q.entropy_coef != 0.f) g.b = coef.data_ptr<float>() + 1, g.b_stride = 2;
      g.scale = static_cast<float>(grad_scale), g.scale_a = scale_device;
    g.scale_b = out.data_ptr<float>() + 5;
    ok(rlb::token_grad(g, stream), "token_policy_loss");
  }
  result.push_back(grad);
  return result;
}

// Gradient from what token_policy_loss returned without its gradient (or preference_loss, with factor and entropy unset).
Tensor token_loss_backward(const Tensor& logits, const Tensor& tokens, const OptT& mask, double temperature,
                           const Tensor& ml, const OptT& entropy, const Tensor& coef, const OptT& factor,
                           const Tensor& grad_output) {
  const Logits l(logits);
  const c10::cuda::CUDAGuard guard(logits.device());
  const Index ix(l, tokens, mask);
  const int64_t width = coef.dim() == 2 ? coef.size(1) : 1;  // there may be no rows
  TORCH_CHECK_VALUE(ml.numel() == 2 * l.rows && coef.numel() == width * l.rows && (width == 1 || width == 2),
                    "token_loss_backward: statistics of other logits");
  Tensor grad = l.gradient();
  rlb::TokenGradArgs g{};
  g.dtype = l.dtype, g.rows = l.rows, g.vocab = l.vocab, g.z = l.z, g.idx = ix.idx, g.inv_temp = inverse(temperature);
  g.out = Logits::rows_of(grad);
  g.ml = reinterpret_cast<const float2*>(ml.data_ptr<float>());
  g.a = coef.data_ptr<float>(), g.a_stride = width;
  if (given(entropy)) {
    TORCH_CHECK_VALUE(entropy->numel() == l.rows && width == 2, "token_loss_backward: statistics of other logits");
    g.entropy = entropy->data_ptr<float>();
    g.b = g.a + 1, g.b_stride = width;
  }
  g.scale = 1.f, g.scale_a = scale_ptr(l, grad_output), g.scale_b = scale_ptr(l, factor);
  ok(rlb::token_grad(g, at::cuda::getCurrentCUDAStream()), "token_loss_backward");
  return grad;
}

// ---- preference loss ----------------------------------------------------------------------------------------------------
// Returns loss, chosen rewards, rejected rewards, seq_logp, logp, then [grad] with want_grad, [ml, coef] without.
std::vector<Tensor> preference_loss(const Tensor& logits, const Tensor& tokens, const OptT& ref, const OptT& offsets,
                                    const OptT& mask, double beta, double smoothing, int64_t kind, bool average,
                                    double temperature, bool want_grad, double grad_scale,
                                    const OptT& grad_scale_device) {
  const Logits l(logits);
  const c10::cuda::CUDAGuard guard(logits.device());
  const auto stream = at::cuda::getCurrentCUDAStream();
  const Index ix(l, tokens, mask);
  rlb::PreferenceArgs p{};
  Tensor off;
  if (logits.dim() == 3) {
    TORCH_CHECK_VALUE(!given(offsets), "offsets belong to packed logits [rows, V]; [sequences, rows, V] has none");
    p.seqs = logits.size(0), p.length = logits.size(1);
  } else {
    TORCH_CHECK_VALUE(given(offsets), "packed logits [rows, V] need the offsets of their sequences");
    TORCH_CHECK_TYPE(offsets->scalar_type() == torch::kInt64 || offsets->scalar_type() == torch::kInt32,
                     "offsets must be int64 or int32, got ", offsets->scalar_type());
    TORCH_CHECK_VALUE(offsets->device() == logits.device(), "offsets must be on the device of the logits");
    TORCH_CHECK_VALUE(offsets->dim() == 1 && offsets->numel() >= 1, "offsets must be [sequences + 1]");
    off = offsets->contiguous();
    p.seqs = off.numel() - 1;
    p.offsets = off.data_ptr(), p.offsets_i64 = off.scalar_type() == torch::kInt64;
  }
  TORCH_CHECK_VALUE(p.seqs % 2 == 0, "sequences 2 k and 2 k + 1 form a pair: their number must be even, got ",
                    text(p.seqs));
  Tensor r;
  if (given(ref)) {
    TORCH_CHECK_TYPE(ref->scalar_type() == torch::kFloat32, "ref_logps must be float32, got ", ref->scalar_type());
    TORCH_CHECK_VALUE(ref->device() == logits.device() && ref->dim() == 1 && ref->numel() == p.seqs,
                      "ref_logps must be [sequences] on the device of the logits");
    r = ref->contiguous();
    p.ref = r.data_ptr<float>();
  }
  Tensor loss = torch::empty({}, l.f32()), seq = torch::empty({p.seqs}, l.f32()), rew = torch::empty({2, p.seqs / 2}, l.f32());
  Tensor logp = torch::empty(l.lead(), l.f32()), ml = torch::empty({l.rows, 2}, l.f32());
  Tensor coef = torch::empty({l.rows}, l.f32());
  std::vector<Tensor> result = rew.unbind();
  result.insert(result.begin(), loss);
  result.insert(result.end(), {seq, logp});
  rlb::TokenStatsArgs a{};
  a.dtype = l.dtype, a.rows = l.rows, a.vocab = l.vocab, a.z = l.z, a.idx = ix.idx, a.inv_temp = inverse(temperature);
  a.logp = logp.data_ptr<float>();
  a.ml = reinterpret_cast<float2*>(ml.data_ptr<float>());
  ok(rlb::token_stats(a, stream), "preference_loss");
  p.rows = l.rows, p.vocab = l.vocab, p.idx = ix.idx, p.logp = a.logp;
  p.beta = static_cast<float>(beta), p.smoothing = static_cast<float>(smoothing), p.kind = static_cast<int>(kind);
  p.average = average;
  p.loss = loss.data_ptr<float>(), p.seq_logp = seq.data_ptr<float>(), p.rewards = rew.data_ptr<float>();
  p.coef = coef.data_ptr<float>();
  ok(rlb::preference_pairs(p, stream), "preference_loss");
  if (!want_grad) {
    result.insert(result.end(), {ml, coef});
    return result;
  }
  Tensor grad = l.gradient();
  rlb::TokenGradArgs g{};
  g.dtype = l.dtype, g.rows = l.rows, g.vocab = l.vocab, g.z = l.z, g.idx = ix.idx, g.inv_temp = a.inv_temp;
  g.out = Logits::rows_of(grad);
  g.ml = a.ml;
  g.a = p.coef, g.a_stride = 1;
  g.scale = static_cast<float>(grad_scale), g.scale_a = scale_ptr(l, grad_scale_device);
  ok(rlb::token_grad(g, stream), "preference_loss");
  result.push_back(grad);
  return result;
}

// ---- differentiable forms -----------------------------------------------------------------------------------------------
// Autograd in C++: a backward pass in Python waits for the interpreter (log-probabilities and their gradient for a few rows
// took 84 us, these 61). They keep the logits and a few numbers per row.
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void backward_checks(const char* name) {
  TORCH_CHECK(c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None, name,
              ": a backward pass cannot be captured in a CUDA graph; capture a form that returns the gradient");
  TORCH_CHECK(!at::GradMode::is_enabled(), name, " is differentiable once (create_graph is not supported)");
}

Tensor or_none(const OptT& t) { return given(t) ? *t : Tensor(); }
OptT optional(const Tensor& t) { return t.defined() ? OptT(t) : OptT(); }

struct LogProbs : torch::autograd::Function<LogProbs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, const OptT& mask,
                               double temperature) {
    const std::vector<Tensor> x = token_logprobs(logits, tokens, mask, temperature);  // logp, entropy, ml
    ctx->save_for_backward({logits, tokens, or_none(mask), x[2], x[1]});
    ctx->saved_data["temperature"] = temperature;
    ctx->set_materialize_grads(false);
    return {x[0], x[1]};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& d) {
    backward_checks("token_logprobs");
    if (!d[0].defined() && !d[1].defined()) return variable_list(4);
    const variable_list s = ctx->get_saved_variables();
    const Tensor d_logp = d[0].defined() ? d[0] : torch::zeros_like(d[1]);
    return {token_logprobs_backward(s[0], s[1], optional(s[2]), ctx->saved_data["temperature"].toDouble(), s[3], s[4],
                                    d_logp, optional(d[1])),
            Tensor(), Tensor(), Tensor()};
  }
};

struct PolicySettings {
  double clip_lo, clip_hi, kl_coef;
  int64_t kl_kind;
  double entropy_coef, temperature;
  bool mean;
};

struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, const Tensor& old,
                               const Tensor& adv, const OptT& ref, const OptT& mask, const PolicySettings& p) {
    // loss, four means, factor, logp, entropy, ml, coef
    const std::vector<Tensor> x =
        token_policy_loss(logits, tokens, old, adv, ref, mask, p.clip_lo, p.clip_hi, p.kl_coef, p.kl_kind,
                          p.entropy_coef, p.temperature, p.mean, false, 1.0, OptT());
    ctx->save_for_backward(
        {logits, tokens, or_none(mask), x[8], p.entropy_coef != 0.0 ? x[7] : Tensor(), x[9], x[5]});
    ctx->saved_data["temperature"] = p.temperature;
    ctx->mark_non_differentiable({x[1], x[2], x[3], x[4], x[6]});
    ctx->set_materialize_grads(false);
    return {x[0], x[1], x[2], x[3], x[4], x[6]};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& d) {
    backward_checks("token_policy_loss");
    if (!d[0].defined()) return variable_list(7);
    const variable_list s = ctx->get_saved_variables();
    variable_list grads(7);
    grads[0] = token_loss_backward(s[0], s[1], optional(s[2]), ctx->saved_data["temperature"].toDouble(), s[3],
                                   optional(s[4]), s[5], s[6], d[0]);
    return grads;
  }
};

struct PreferenceSettings {
  double beta, smoothing;
  int64_t kind;
  bool average;
  double temperature;
};

struct PreferenceLoss : torch::autograd::Function<PreferenceLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, const OptT& ref,
                               const OptT& offsets, const OptT& mask, const PreferenceSettings& p) {
    // loss, two rewards, seq_logp, logp, ml, coef
    const std::vector<Tensor> x = preference_loss(logits, tokens, ref, offsets, mask, p.beta, p.smoothing, p.kind,
                                                  p.average, p.temperature, false, 1.0, OptT());
    ctx->save_for_backward({logits, tokens, or_none(mask), x[5], x[6]});
    ctx->saved_data["temperature"] = p.temperature;
    ctx->mark_non_differentiable({x[1], x[2], x[3], x[4]});
    ctx->set_materialize_grads(false);
    return {x[0], x[1], x[2], x[3], x[4]};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& d) {
    backward_checks("preference_loss");
    if (!d[0].defined()) return variable_list(6);
    const variable_list s = ctx->get_saved_variables();
    variable_list grads(6);
    grads[0] = token_loss_backward(s[0], s[1], optional(s[2]), ctx->saved_data["temperature"].toDouble(), s[3], OptT(),
                                   s[4], OptT(), d[0]);
    return grads;
  }
};

// ---- AdamW ------------------------------------------------------------------------------------------------------------
// The parameters and states of one step over many tensors. Holds the tensors; pointers are read at every step.
class AdamWPlan {
 public:
  AdamWPlan(std::vector<Tensor> params, std::vector<Tensor> m, std::vector<Tensor> v, Tensor steps,
            std::vector<Tensor> m_scales, std::vector<Tensor> v_scales, std::vector<Tensor> low, int64_t first_stream)
      : p_(std::move(params)), m_(std::move(m)), v_(std::move(v)), ms_(std::move(m_scales)), vs_(std::move(v_scales)),
        low_(std::move(low)), steps_(std::move(steps)), first_stream_(first_stream) {
    const size_t n = p_.size();
    TORCH_CHECK_VALUE(n > 0, "AdamWPlan: no parameters");
    TORCH_CHECK_VALUE(n < 65536, "AdamWPlan: at most 65,535 parameters");
    TORCH_CHECK_VALUE(m_.size() == n && v_.size() == n, "AdamWPlan: one exp_avg and one exp_avg_sq per parameter");
    const auto dt = p_[0].scalar_type();
    TORCH_CHECK_TYPE(dt == torch::kFloat32 || dt == torch::kBFloat16,
                     "AdamWPlan: parameters must be float32 or bfloat16, got ", dt);
    bf16_ = dt == torch::kBFloat16;
    const auto state = m_[0].scalar_type();
    TORCH_CHECK_TYPE(state == torch::kFloat32 || state == torch::kFloat8_e4m3fn,
                     "AdamWPlan: states must be float32 or float8_e4m3fn, got ", state);
    bits8_ = state == torch::kFloat8_e4m3fn;
    TORCH_CHECK_VALUE(!bits8_ || (ms_.size() == n && vs_.size() == n),
                      "AdamWPlan: 8-bit states need their scales (exp_avg_scales, exp_avg_sq_scales)");
    TORCH_CHECK_VALUE(!bf16_ || low_.size() == n, "AdamWPlan: bfloat16 parameters need low_bits");
    TORCH_CHECK_VALUE(bits8_ || (ms_.empty() && vs_.empty()), "AdamWPlan: float32 states have no scales");
    TORCH_CHECK_VALUE(bf16_ || low_.empty(), "AdamWPlan: low_bits belong to bfloat16 parameters");
    const auto dev = p_[0].device();
    TORCH_CHECK_VALUE(dev.is_cuda(), "AdamWPlan: parameters must be CUDA tensors");
    TORCH_CHECK_VALUE(steps_.device() == dev && steps_.scalar_type() == torch::kFloat32 && steps_.is_contiguous() &&
                          steps_.numel() == static_cast<int64_t>(n),
                      "AdamWPlan: steps must be a contiguous float32 tensor, one element per parameter");
    for (size_t i = 0; i < n; ++i) {
      const Tensor& p = p_[i];
      TORCH_CHECK_TYPE(p.scalar_type() == dt, "AdamWPlan: parameters of one plan share a type");
      TORCH_CHECK_VALUE(p.device() == dev && p.layout() == torch::kStrided, "AdamWPlan: parameters of one plan share a device");
      TORCH_CHECK_VALUE(p.is_non_overlapping_and_dense(), "AdamWPlan: parameter ", number(i),
                        " has gaps or overlaps in memory (strides ", text(p.strides()), ")");
      check_state(m_[i], p, state, "exp_avg", i);
      check_state(v_[i], p, state, "exp_avg_sq", i);
      if (bf16_) check_state(low_[i], p, torch::kInt16, "low_bits", i);
      if (bits8_) {
        check_scale(ms_[i], p, "exp_avg_scales", i);
        check_scale(vs_[i], p, "exp_avg_sq_scales", i);
      }
    }
    check_apart();
  }

  // The list of this step: every parameter that has a gradient. The list lives until the next call.
  rlb::AdamLaunch list() {
    const auto dev = device();
    table_.clear();
    copies_.clear();
    for (size_t i = 0; i < p_.size(); ++i) {
      const Tensor& p = p_[i];
      const Tensor& grad = p.grad();
      if (!grad.defined()) continue;
      TORCH_CHECK_VALUE(p.device() == dev && p.scalar_type() == (bf16_ ? torch::kBFloat16 : torch::kFloat32) &&
                            p.sizes() == m_[i].sizes() && same_order(p, m_[i]),
                        "AdamW: parameter ", number(i), " has changed its device, type, shape or strides");
      TORCH_CHECK_TYPE(grad.layout() == torch::kStrided, "AdamW: sparse gradients are not supported");
      TORCH_CHECK_TYPE(grad.scalar_type() == p.scalar_type(), "AdamW: the gradient of parameter ", number(i), " is ",
                       grad.scalar_type(), ", the parameter ", p.scalar_type());
      TORCH_CHECK_VALUE(grad.device() == dev && grad.sizes() == p.sizes(), "AdamW: gradient ", number(i),
                        " has another shape or device than its parameter");
      // memory is walked in the parameter's order (strides of single elements do not matter)
      const Tensor* g = &grad;
      if (!same_order(grad, p)) {
        copies_.push_back(torch::empty_strided(p.sizes(), p.strides(), p.options().requires_grad(false)).copy_(grad));
        g = &copies_.back();
      }
      rlb::AdamTensor t{};
      t.p = p.data_ptr(), t.g = g->data_ptr(), t.m = m_[i].data_ptr(), t.v = v_[i].data_ptr();
      if (bits8_) t.m_scale = ms_[i].data_ptr<float>(), t.v_scale = vs_[i].data_ptr<float>();
      if (bf16_) t.low = low_[i].data_ptr<int16_t>();
      t.n = p.numel();
      t.id = static_cast<uint32_t>(i);
      table_.push_back(t);
    }
    rlb::AdamLaunch a{};
    a.tensors = table_.data(), a.count = static_cast<int>(table_.size());
    a.bf16 = bf16_, a.bits8 = bits8_;
    a.steps = steps_.data_ptr<float>();
    a.first_stream = static_cast<uint32_t>(first_stream_);
    return a;
  }

  // The step writes behind autograd's back: a graph that saved a parameter must notice.
  void stepped() {
    for (const auto& t : table_) {
      const Tensor& p = p_[t.id];
      if (!p.is_inference()) p.unsafeGetTensorImpl()->bump_version();
    }
    copies_.clear();
  }

  c10::Device device() const { return steps_.device(); }

 private:
  // All tensors are dense: each is one range of memory, and no two of them share any.
  void check_apart() const {
    std::vector<std::pair<uintptr_t, uintptr_t>> ranges;
    for (const auto* list : {&p_, &m_, &v_, &ms_, &vs_, &low_}) {
      for (const Tensor& t : *list) {
        const auto at = reinterpret_cast<uintptr_t>(t.data_ptr());
        if (t.numel()) ranges.emplace_back(at, at + t.numel() * t.element_size());
      }
    }
    std::sort(ranges.begin(), ranges.end());
    for (size_t i = 1; i < ranges.size(); ++i) {
      TORCH_CHECK_VALUE(ranges[i].first >= ranges[i - 1].second, "AdamWPlan: two tensors share memory");
    }
  }
  static std::string number(size_t i) { return text(static_cast<int64_t>(i)); }
  static bool same_order(const Tensor& a, const Tensor& b) {
    for (int64_t d = 0; d < a.dim(); ++d) {
      if (a.size(d) != 1 && a.stride(d) != b.stride(d)) return a.numel() == 0;
    }
    return true;
  }
  static void check_state(const Tensor& s, const Tensor& p, c10::ScalarType dt, const char* name, size_t i) {
    TORCH_CHECK_TYPE(s.scalar_type() == dt, "AdamWPlan: ", name, " ", number(i), " must be ", dt, ", got ", s.scalar_type());
    TORCH_CHECK_VALUE(s.device() == p.device() && s.sizes() == p.sizes() && same_order(s, p), "AdamWPlan: ", name, " ",
                      number(i), " must have the parameter's device, shape and strides");
  }
  static void check_scale(const Tensor& s, const Tensor& p, const char* name, size_t i) {
    TORCH_CHECK_TYPE(s.scalar_type() == torch::kFloat32, "AdamWPlan: ", name, " must be float32");
    TORCH_CHECK_VALUE(s.device() == p.device() && s.is_contiguous() &&
                          s.numel() == (p.numel() + rlb::kAdamBlock - 1) / rlb::kAdamBlock,
                      "AdamWPlan: ", name, " ", number(i), " must hold one element per ",
                      number(rlb::kAdamBlock), " elements of the parameter");
  }
  std::vector<Tensor> p_, m_, v_, ms_, vs_, low_, copies_;
  Tensor steps_;
  int64_t first_stream_;
  bool bf16_ = false, bits8_ = false;
  std::vector<rlb::AdamTensor> table_;
};

struct AdamSettings {  // of one plan
  double lr;
  OptT lr_device;
  double beta1, beta2, eps, weight_decay;
  bool maximize;
  int64_t seed;
};

// One step of every parameter of the plans that has a gradient. Returns the gradients' norm with max_norm > 0.
OptT adamw_step(const std::vector<AdamWPlan*>& plans, const std::vector<AdamSettings>& settings, double max_norm) {
  TORCH_CHECK_VALUE(!plans.empty() && settings.size() == plans.size(), "adamw_step: one set of settings per plan");
  const auto dev = plans[0]->device();
  const c10::cuda::CUDAGuard guard(dev);
  std::vector<rlb::AdamLaunch> lists;
  for (size_t i = 0; i < plans.size(); ++i) {
    for (size_t j = 0; j < i; ++j) TORCH_CHECK_VALUE(plans[i] != plans[j], "adamw_step: a plan is given twice");
    TORCH_CHECK_VALUE(plans[i]->device() == dev, "adamw_step: plans of one step share a device");
    rlb::AdamLaunch a = plans[i]->list();
    const AdamSettings& s = settings[i];
    if (s.lr_device.has_value() && s.lr_device->defined()) {
      TORCH_CHECK_VALUE(s.lr_device->device() == dev && s.lr_device->numel() == 1,
                        "AdamW: a learning rate tensor must be one element on the parameters' device");
      TORCH_CHECK_TYPE(s.lr_device->scalar_type() == torch::kFloat32 || s.lr_device->scalar_type() == torch::kFloat64,
                       "AdamW: a learning rate tensor must be float32 or float64");
      a.h.lr_device = s.lr_device->data_ptr();
      a.h.lr_f64 = s.lr_device->scalar_type() == torch::kFloat64;
    }
    a.h.lr = s.lr, a.h.beta1 = s.beta1, a.h.beta2 = s.beta2, a.h.eps = s.eps, a.h.weight_decay = s.weight_decay;
    a.h.maximize = s.maximize, a.h.seed = static_cast<uint64_t>(s.seed);
    if (a.count) lists.push_back(a);
  }
  const auto f32 = torch::TensorOptions().device(dev).dtype(torch::kFloat32);
  OptT norm;
  if (max_norm > 0.0) norm = torch::empty({}, f32);
  if (lists.empty()) {
    if (norm) norm->zero_();
    return norm;
  }
  const int n = static_cast<int>(lists.size());
  const Tensor work = torch::empty({rlb::adamw_workspace_bytes(lists.data(), n)}, f32.dtype(torch::kUInt8));
  ok(rlb::adamw_step(lists.data(), n, max_norm, work.data_ptr(), norm ? norm->data_ptr<float>() : nullptr,
                     at::cuda::getCurrentCUDAStream()),
     "adamw_step");
  for (AdamWPlan* p : plans) p->stepped();
  return norm;
}

}  // namespace

void rlb_register_token(pybind11::module& m) {
  m.def("token_logprobs", &token_logprobs);
  m.def("token_policy_loss", &token_policy_loss);
  m.def("token_logprobs_autograd", [](const Tensor& logits, const Tensor& tokens, const OptT& mask, double temperature) {
    return LogProbs::apply(logits, tokens, mask, temperature);
  });
  m.def("token_policy_loss_autograd",
        [](const Tensor& logits, const Tensor& tokens, const Tensor& old, const Tensor& adv, const OptT& ref,
           const OptT& mask, double clip_lo, double clip_hi, double kl_coef, int64_t kl_kind, double entropy_coef,
           double temperature, bool mean) {
          return PolicyLoss::apply(logits, tokens, old, adv, ref, mask,
                                   PolicySettings{clip_lo, clip_hi, kl_coef, kl_kind, entropy_coef, temperature, mean});
        });
  m.def("preference_loss_autograd",
        [](const Tensor& logits, const Tensor& tokens, const OptT& ref, const OptT& offsets, const OptT& mask, double beta,
           double smoothing, int64_t kind, bool average, double temperature) {
          return PreferenceLoss::apply(logits, tokens, ref, offsets, mask,
                                       PreferenceSettings{beta, smoothing, kind, average, temperature});
        });
  m.def("preference_loss", &preference_loss);
  pybind11::class_<AdamWPlan>(m, "AdamWPlan")
      .def(pybind11::init<std::vector<Tensor>, std::vector<Tensor>, std::vector<Tensor>, Tensor, std::vector<Tensor>,
                          std::vector<Tensor>, std::vector<Tensor>, int64_t>());
  // settings: (lr, lr tensor or None, beta1, beta2, eps, weight decay, maximize, seed) of each plan
  m.def("adamw_step", [](const std::vector<AdamWPlan*>& plans,
                         const std::vector<std::tuple<double, OptT, double, double, double, double, bool, int64_t>>& s,
                         double max_norm) {
    std::vector<AdamSettings> settings;
    for (const auto& [lr, lr_device, b1, b2, eps, wd, maximize, seed] : s) {
      settings.push_back({lr, lr_device, b1, b2, eps, wd, maximize, seed});
    }
    return adamw_step(plans, settings, max_norm);
  });
}
