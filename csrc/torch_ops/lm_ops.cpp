// Registrations of the language-model operators (vocab_rows.hip, layer_norm.hip): shape and type checks on
// the host, then the launchers on the current stream of the tensors' device.  Workspaces come from the
// caching allocator, call by call: no two streams or captured graphs share one.
//
// Their autograd nodes are C++ (torch::autograd::Function): a backward pass through them takes no Python
// interpreter lock in the engine's thread.  A training step of 6400 rows of 65 logits, bound by the host,
// takes 57 us with them and took 83 us with nodes in Python.
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/custom_class.h>
#include <torch/library.h>

#include <cmath>
#include <memory>
#include <mutex>
#include <stdexcept>
#include <tuple>
#include <unordered_map>

#include "tfx_kernels.h"

using at::Tensor;
using c10::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

// A launch that the runtime refuses leaves no result
template <typename F>
void launching(const char* what, F f) {
  try {
    f();
  } catch (const std::runtime_error& e) {
    TORCH_CHECK(false, what, ": ", e.what());
  }
}

// the backward kernels leave no graph of their own: create_graph=True would give gradients without one
void first_order(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, ": its gradient cannot be differentiated again (create_graph=True)");
}

// ... and the passes write into tensors of their own, in which a forward-mode derivative would end
void no_tangent(const Tensor& t, const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), what, ": forward-mode derivatives are not implemented");
}

bool is_bf16(const Tensor& t, const char* what) {
  const bool b = t.scalar_type() == at::kBFloat16;
  TORCH_CHECK_TYPE(b || t.scalar_type() == at::kFloat, what, ": float32 or bfloat16 expected, got ", t.scalar_type());
  return b;
}

bool is_int64(const Tensor& t, const char* what) {
  const bool b = t.scalar_type() == at::kLong;
  TORCH_CHECK_TYPE(b || t.scalar_type() == at::kInt, what, ": int64 or int32 expected, got ", t.scalar_type());
  return b;
}

bool has(const optional<Tensor>& t) { return t.has_value() && t->defined(); }

void check_matrix(const Tensor& t, int64_t most, const char* what) {
  TORCH_CHECK_VALUE(t.is_cuda(), what, " must be a GPU tensor");
  TORCH_CHECK_VALUE(t.dim() >= 2 && t.size(-1) >= 1 && t.size(-1) <= most, what,
                    ": at least two dimensions, the last between 1 and ", most, ", expected; got ", t.sizes());
}

// `t` [..., width] as [rows, width]: its own memory wherever the elements of a row are next to each other
Tensor rows_of(const Tensor& t, int64_t most, const char* what) {
  check_matrix(t, most, what);
  const Tensor c = t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous();
  return c.dim() == 2 ? c : c.reshape({c.numel() / c.size(-1), c.size(-1)});
}

// `t`, of the shape [lead..., last] (last < 0: [lead...]), on x's device
void check_side(const Tensor& t, const Tensor& x, at::IntArrayRef lead, int64_t last, const char* what) {
  TORCH_CHECK_VALUE(t.device() == x.device(), what, ": on ", t.device(), ", the matrix is on ", x.device());
  bool same = t.dim() == (int64_t)lead.size() + (last >= 0);
  for (size_t i = 0; same && i < lead.size(); ++i) same = t.size(i) == lead[i];
  TORCH_CHECK_VALUE(same && (last < 0 || t.size(-1) == last), what, ": shape ", t.sizes(), " for a matrix of ", x.sizes());
}

// n contiguous f32 elements on x's device, or null
float* f32_or_null(const optional<Tensor>& t, const Tensor& x, int64_t n, const char* what) {
  if (!has(t)) return nullptr;
  TORCH_CHECK_VALUE(t->device() == x.device(), what, ": on ", t->device(), ", the matrix is on ", x.device());
  TORCH_CHECK_TYPE(t->scalar_type() == at::kFloat, what, ": float32 expected, got ", t->scalar_type());
  TORCH_CHECK_VALUE(t->is_contiguous() && t->numel() == n, what, ": ", n, " contiguous elements expected");
  return t->data_ptr<float>();
}

// of an upstream gradient of any layout (undefined: none)
Tensor flat_f32(const Tensor& g) {
  return !g.defined() || (g.scalar_type() == at::kFloat && g.is_contiguous()) ? g : g.to(at::kFloat).contiguous();
}

// What a node keeps beside its saved tensors: one entry of its context, found once
template <typename S>
void keep(AutogradContext* ctx, c10::intrusive_ptr<S> s) {
  ctx->saved_data["s"] = c10::IValue::make_capsule(std::move(s));
}
template <typename S>
c10::intrusive_ptr<S> kept(AutogradContext* ctx) {
  return c10::static_intrusive_pointer_cast<S>(ctx->saved_data["s"].toCapsule());
}

struct LogitsKept : torch::CustomClassHolder {
  double temperature = 1.;
  std::vector<int64_t> shape;  // of the logits
  bool fused = false;
  Tensor dx;                   // fused: the gradient, until it is taken
};

tfx::VocabArgs logits_args(const Tensor& x, double temperature) {
  TORCH_CHECK_VALUE(temperature >= 1e-6 && temperature <= 1e6,
                    "temperature: a number between 1e-6 and 1e6 expected, got ", temperature);
  tfx::VocabArgs a;
  a.bf16 = is_bf16(x, "logits");
  // the passes count rows and [row, part] pairs (parts of 1024 elements at least) in 31 bits, and up to a grid further
  TORCH_CHECK_VALUE(x.size(0) * ((x.size(1) + 1023) / 1024) <= (int64_t(1) << 30), "logits: too many rows for their length");
  a.x = x.data_ptr();
  a.stride = x.stride(0);
  a.rows = (int)x.size(0);
  a.V = (int)x.size(1);
  a.scale = (float)(1.0 / temperature);
  a.c = (float)(1.4426950408889634 / temperature);
  return a;
}

// the pieces of split rows
void with_parts(tfx::VocabArgs& a, const Tensor& x, Tensor& ws, Tensor& keys) {
  a.nparts = tfx::vocab_parts(a.bf16, a.rows, a.V, a.K);
  if (a.nparts == 1) return;
  const int64_t items = (int64_t)a.rows * a.nparts;
  ws = at::empty({items, 4}, x.options().dtype(at::kFloat));
  a.ws = ws.data_ptr<float>();
  if (a.K) {
    keys = at::empty({items, a.K}, x.options().dtype(at::kLong));
    a.ws_keys = reinterpret_cast<uint64_t*>(keys.data_ptr<int64_t>());
  }
}

std::vector<int64_t> with_last(at::IntArrayRef lead, int64_t last) {
  std::vector<int64_t> v(lead.begin(), lead.end());
  v.push_back(last);
  return v;
}

// ------------------------------------------------------------------ token log probabilities
struct TokenResult {
  Tensor logp, entropy, top_logp, top_ids;  // of the leading shape; undefined unless asked for
  Tensor stats;                             // [rows, 4]
};

// x: logits as rows; tokens: flat
TokenResult token_pass(const Tensor& x, const Tensor& tokens, at::IntArrayRef lead, int64_t top_k, bool entropy, bool stats,
                       double temperature) {
  auto a = logits_args(x, temperature);
  a.tok64 = is_int64(tokens, "tokens");
  a.tok = tokens.data_ptr();
  c10::DeviceGuard guard(x.device());
  const auto f32 = x.options().dtype(at::kFloat);
  TokenResult r;
  Tensor ws, keys;
  r.logp = at::empty(lead, f32);
  a.logp = r.logp.data_ptr<float>();
  if (entropy) {
    r.entropy = at::empty(lead, f32);
    a.ent = r.entropy.data_ptr<float>();
  }
  if (stats) {
    r.stats = at::empty({a.rows, 4}, f32);
    a.stats = r.stats.data_ptr<float>();
  }
  if (top_k) {
    a.K = (int)top_k;
    r.top_logp = at::empty(with_last(lead, top_k), f32);
    r.top_ids = at::empty(with_last(lead, top_k), x.options().dtype(at::kLong));
    a.top_logp = r.top_logp.data_ptr<float>();
    a.top_ids = r.top_ids.data_ptr<int64_t>();
  }
  if (a.rows) {
    with_parts(a, x, ws, keys);
    launching("token_log_probs", [&] {
      tfx::vocab_stats(a, stream_of(x));
    });
  }
  return r;
}

Tensor token_pass_bwd(const Tensor& x, const Tensor& tokens, const Tensor& stats, const Tensor& g_logp, const Tensor& g_ent,
                      const LogitsKept& s) {
  auto a = logits_args(x, s.temperature);
  a.tok64 = is_int64(tokens, "tokens");
  a.tok = tokens.data_ptr();
  a.stats = f32_or_null(stats, x, (int64_t)a.rows * 4, "stats");
  const Tensor g = flat_f32(g_logp), h = flat_f32(g_ent);
  const float* gp = f32_or_null(g, x, a.rows, "the log probabilities' gradient");
  const float* hp = f32_or_null(h, x, a.rows, "the entropies' gradient");
  c10::DeviceGuard guard(x.device());
  Tensor dx = at::empty(s.shape, x.options());
  if (a.rows) {
    launching("token_log_probs backward", [&] {
      tfx::vocab_bwd(a, gp, hp, dx.data_ptr(), stream_of(x));
    });
  }
  return dx;
}

struct TokenLogProbsFn : torch::autograd::Function<TokenLogProbsFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, int64_t top_k,
                               bool entropy, double temperature) {
    const Tensor x = rows_of(logits, tfx::kVocabMax, "logits");
    auto r = token_pass(x, tokens, logits.sizes().slice(0, logits.dim() - 1), top_k, entropy, true, temperature);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, tokens, r.stats});
    auto s = c10::make_intrusive<LogitsKept>();
    s->temperature = temperature;
    s->shape = logits.sizes().vec();
    keep(ctx, s);
    variable_list out{r.logp};
    if (entropy) out.push_back(r.entropy);
    if (top_k) {
      out.push_back(r.top_logp);
      out.push_back(r.top_ids);
      ctx->mark_non_differentiable({r.top_logp, r.top_ids});
    }
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    first_order("token_log_probs");
    variable_list out(5);
    const Tensor h = g.size() % 2 == 0 ? g[1] : Tensor();  // logp, entropy if asked for, the alternatives' two
    if (!g[0].defined() && !h.defined()) return out;
    const auto saved = ctx->get_saved_variables();
    out[0] = token_pass_bwd(saved[0], saved[1], saved[2], g[0], h, *kept<LogitsKept>(ctx));
    return out;
  }
};

// (logp [...], entropy [...]?, top_logp [..., K]?, top_ids [..., K]?)
std::tuple<Tensor, Tensor, Tensor, Tensor> token_log_probs(const Tensor& logits, const Tensor& tokens, int64_t top_k,
                                                           bool entropy, double temperature) {
  no_tangent(logits, "token_log_probs");
  check_matrix(logits, tfx::kVocabMax, "logits");
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  check_side(tokens, logits, lead, -1, "tokens");
  TORCH_CHECK_VALUE(top_k >= 0 && top_k <= tfx::kVocabMaxTop, "top_k between 0 and ", tfx::kVocabMaxTop, " expected, got ",
                    top_k);
  const Tensor t = tokens.contiguous();
  if (at::GradMode::is_enabled() && logits.requires_grad()) {
    const auto out = TokenLogProbsFn::apply(logits, t, top_k, entropy, temperature);
    Tensor none;
    return {out[0], entropy ? out[1] : none, top_k ? out[1 + entropy] : none, top_k ? out[2 + entropy] : none};
  }
  const Tensor x = rows_of(logits.detach(), tfx::kVocabMax, "logits");
  const auto r = token_pass(x, t, lead, top_k, entropy, false, temperature);
  return {r.logp, r.entropy, r.top_logp, r.top_ids};
}

// ------------------------------------------------------------------ distillation
tfx::DistillArgs distill_args(const Tensor& x, const Tensor& ids, double temperature) {
  tfx::DistillArgs a;
  a.v = logits_args(x, temperature);
  a.K = (int)ids.size(-1);
  a.ids64 = is_int64(ids, "teacher_ids");
  a.ids = ids.data_ptr();
  a.temp = (float)temperature;
  return a;
}

struct DistillResult {
  Tensor loss;
  Tensor dx;              // the gradient, formed with the loss; or, where that is not possible or asked for,
  Tensor stats, q, coef;  // what the backward pass forms it from: [rows, 4], [rows, K], [rows]
};

DistillResult distill_pass(const Tensor& x, const Tensor& teacher, const Tensor& ids, const optional<Tensor>& weight,
                           double temperature, bool want_grad, bool fuse) {
  auto a = distill_args(x, ids, temperature);
  a.teacher_bf16 = is_bf16(teacher, "teacher_logits");
  a.teacher = teacher.data_ptr();
  a.v.weight = f32_or_null(weight, x, a.v.rows, "row_weight");
  a.w = a.v.rows ? 1.f / (float)a.v.rows : 0.f;
  c10::DeviceGuard guard(x.device());
  const auto f32 = x.options().dtype(at::kFloat);
  DistillResult r;
  r.loss = at::empty({}, f32);
  if (!a.v.rows) {
    r.loss.zero_();
    if (want_grad) r.dx = at::empty({0, a.v.V}, x.options());
    return r;
  }
  const hipStream_t s = stream_of(x);
  Tensor rows = at::empty({a.v.rows}, f32), ws, keys;
  a.loss_rows = rows.data_ptr<float>();
  if (want_grad && fuse && tfx::distill_fits(a.v.bf16, a.v.V)) {
    r.dx = at::empty({a.v.rows, a.v.V}, x.options());
    launching("distillation_loss", [&] {
      tfx::distill_fused(a, r.dx.data_ptr(), r.loss.data_ptr<float>(), s);
    });
    return r;
  }
  r.stats = at::empty({a.v.rows, 4}, f32);
  a.v.stats = r.stats.data_ptr<float>();
  if (want_grad) {
    r.q = at::empty({a.v.rows, a.K}, f32);
    r.coef = at::empty({a.v.rows}, f32);
    a.q = r.q.data_ptr<float>();
    a.coef = r.coef.data_ptr<float>();
  }
  with_parts(a.v, x, ws, keys);
  launching("distillation_loss", [&] {
    tfx::vocab_stats(a.v, s);
    tfx::distill_loss(a, r.loss.data_ptr<float>(), s);
  });
  return r;
}

struct DistillationFn : torch::autograd::Function<DistillationFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& teacher, const Tensor& ids,
                        const optional<Tensor>& weight, double temperature, bool fuse) {
    const Tensor x = rows_of(logits, tfx::kVocabMax, "logits");
    auto r = distill_pass(x, teacher, ids, weight, temperature, true, fuse);
    auto s = c10::make_intrusive<LogitsKept>();
    s->temperature = temperature;
    s->shape = logits.sizes().vec();
    s->fused = r.dx.defined();
    s->dx = r.dx;
    keep(ctx, s);
    if (!s->fused) ctx->save_for_backward({x, ids, r.stats, r.q, r.coef});
    return r.loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    first_order("distillation_loss");
    variable_list out(6);
    const Tensor seed = flat_f32(g[0]);
    const auto k = kept<LogitsKept>(ctx);
    if (k->fused) {
      // the gradient left the forward pass: it is handed over, not kept
      TORCH_CHECK(k->dx.defined(), "distillation_loss: with unit_seed=True its gradient can be taken once");
      Tensor dx = std::move(k->dx);
      k->dx = Tensor();
      const float* s = f32_or_null(seed, dx, 1, "the loss's gradient");
      if (dx.numel()) {
        c10::DeviceGuard guard(dx.device());
        launching("distillation_loss backward", [&] {
          tfx::scale_unless_one(dx.data_ptr(), is_bf16(dx, "dx"), dx.numel(), s, stream_of(dx));
        });
      }
      out[0] = k->shape.size() == 2 ? std::move(dx) : dx.view(k->shape);
      return out;
    }
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &ids = saved[1];
    auto a = distill_args(x, ids, k->temperature);
    a.v.stats = f32_or_null(saved[2], x, (int64_t)a.v.rows * 4, "stats");
    a.q = f32_or_null(saved[3], x, (int64_t)a.v.rows * a.K, "q");
    a.coef = f32_or_null(saved[4], x, a.v.rows, "coef");
    const float* s = f32_or_null(seed, x, 1, "the loss's gradient");
    c10::DeviceGuard guard(x.device());
    out[0] = at::empty(k->shape, x.options());
    if (a.v.rows) {
      launching("distillation_loss backward", [&] {
        tfx::distill_bwd(a, s, out[0].data_ptr(), stream_of(x));
      });
    }
    return out;
  }
};

Tensor distillation_loss(const Tensor& logits, const Tensor& teacher, const Tensor& ids, double temperature,
                         const optional<Tensor>& weight, bool fuse) {
  no_tangent(logits, "distillation_loss");
  check_matrix(logits, tfx::kVocabMax, "logits");
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  TORCH_CHECK_VALUE(ids.dim() == logits.dim() && ids.size(-1) >= 1 && ids.size(-1) <= tfx::kDistillMaxTop,
                    "teacher_ids [..., K] with K between 1 and ", tfx::kDistillMaxTop, " expected, got ", ids.sizes());
  check_side(ids, logits, lead, ids.size(-1), "teacher_ids");
  check_side(teacher, logits, lead, ids.size(-1), "teacher_logits");
  const Tensor t = teacher.detach().contiguous(), i = ids.contiguous();
  optional<Tensor> w;
  if (has(weight)) {
    check_side(*weight, logits, lead, -1, "row_weight");
    w = weight->detach().contiguous();
  }
  if (at::GradMode::is_enabled() && logits.requires_grad())
    return DistillationFn::apply(logits, t, i, w, temperature, fuse);
  const Tensor x = rows_of(logits.detach(), tfx::kVocabMax, "logits");
  return distill_pass(x, t, i, w, temperature, false, false).loss;
}

// ------------------------------------------------------------------ layer norm
tfx::LayerNormArgs norm_args(const Tensor& x, const float* gamma) {
  tfx::LayerNormArgs a;
  a.bf16 = is_bf16(x, "layer_norm");
  a.x = x.data_ptr();
  a.stride = x.stride(0);
  a.rows = x.size(0);
  a.C = (int)x.size(1);
  a.gamma = gamma;
  return a;
}

// What a backward pass asks of a variable store when it runs: its gradients' buffer then, and whether it wants to hear of
// each gradient that is there (variables.py tells; the store's number is its key).
struct Store {
  int64_t number = 0;
  Tensor grad;
  bool hooked = false;
};
std::mutex stores_lock;
std::unordered_map<int64_t, std::shared_ptr<Store>>& stores() {
  static std::unordered_map<int64_t, std::shared_ptr<Store>> s;
  return s;
}

std::shared_ptr<Store> store_of(int64_t number) {  // below 0: none
  if (number < 0) return nullptr;
  const std::lock_guard<std::mutex> l(stores_lock);
  const auto it = stores().find(number);
  TORCH_CHECK(it != stores().end(), "no variable store of number ", number);
  return it->second;
}

int64_t store_new() {
  static int64_t next = 0;
  const std::lock_guard<std::mutex> l(stores_lock);
  auto s = std::make_shared<Store>();
  s->number = next;
  stores()[next] = std::move(s);
  return next++;
}

void store_set(int64_t number, const optional<Tensor>& grad, bool hooked) {
  const auto s = store_of(number);
  Tensor g = has(grad) ? *grad : Tensor();  // the former one goes behind the lock
  const std::lock_guard<std::mutex> l(stores_lock);
  std::swap(s->grad, g);
  s->hooked = hooked;
}

void store_free(int64_t number) {
  std::shared_ptr<Store> s;
  const std::lock_guard<std::mutex> l(stores_lock);
  const auto it = stores().find(number);
  if (it == stores().end()) return;
  s = std::move(it->second);
  stores().erase(it);
}

optional<Tensor> grad_of(const std::shared_ptr<Store>& s) {
  if (!s) return c10::nullopt;
  const std::lock_guard<std::mutex> l(stores_lock);
  TORCH_CHECK(s->grad.defined(), "layer_norm: the variable store has no gradients");
  return s->grad;
}

// The store's hook, in Python (ops/lm.py), for the variable at element `at`
void tell_ready(const std::shared_ptr<Store>& s, int64_t at) {
  if (!s) return;
  {
    const std::lock_guard<std::mutex> l(stores_lock);
    if (!s->hooked) return;
  }
  static const auto ready =
      c10::Dispatcher::singleton().findSchemaOrThrow("tfx::grad_ready", "").typed<void(int64_t, int64_t)>();
  ready.call(s->number, at);
}

// C elements of a variable store's flat f32 buffer
float* var_or_null(const optional<Tensor>& flat, int64_t offset, const Tensor& x, const char* what) {
  if (!has(flat)) return nullptr;
  TORCH_CHECK_VALUE(flat->device() == x.device(), what, ": on ", flat->device(), ", the input is on ", x.device());
  TORCH_CHECK_TYPE(flat->scalar_type() == at::kFloat, what, ": float32 expected");
  TORCH_CHECK_VALUE(flat->is_contiguous() && offset >= 0 && offset + x.size(-1) <= flat->numel(), what,
                    ": outside its buffer");
  return flat->data_ptr<float>() + offset;
}

std::tuple<Tensor, Tensor> norm_pass(const Tensor& x, at::IntArrayRef shape, const float* gamma, const float* beta,
                                     double eps, bool stats) {
  auto a = norm_args(x, gamma);
  a.beta = beta;
  a.eps = (float)eps;
  c10::DeviceGuard guard(x.device());
  Tensor y = at::empty(shape, x.options()), st;
  a.y = y.data_ptr();
  if (stats) {
    st = at::empty({a.rows, 2}, x.options().dtype(at::kFloat));
    a.stats = st.data_ptr<float>();
  }
  if (a.rows) {
    launching("layer_norm", [&] {
      tfx::layer_norm_fwd(a, stream_of(x));
    });
  }
  return {y, st};
}

// dx (undefined unless wanted); dgamma, dbeta [C] are added to
Tensor norm_pass_bwd(const Tensor& x, const Tensor& gy, const Tensor& stats, const float* gamma, float* dgamma,
                     float* dbeta, bool want_dx) {
  auto a = norm_args(x, gamma);
  const Tensor dy = rows_of(gy, tfx::kLayerNormMax, "layer_norm gradient");
  TORCH_CHECK(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type() && dy.device() == x.device(),
              "layer_norm gradient: shape, type and device of the input");
  a.dy = dy.data_ptr();
  a.dy_stride = dy.stride(0);
  a.stats = f32_or_null(stats, x, a.rows * 2, "stats");
  a.dgamma = dgamma;
  a.dbeta = dbeta;
  c10::DeviceGuard guard(x.device());
  Tensor dx, part;
  if (want_dx) {
    dx = at::empty(gy.sizes(), x.options());
    a.dx = dx.data_ptr();
  }
  if (!a.rows || (!want_dx && !dgamma && !dbeta)) return dx;
  if (dgamma || dbeta) {
    part = at::empty({tfx::layer_norm_parts(a.bf16, a.rows, a.C), 2, a.C}, x.options().dtype(at::kFloat));
    a.part = part.data_ptr<float>();
  }
  launching("layer_norm backward", [&] {
    tfx::layer_norm_bwd(a, stream_of(x));
  });
  return dx;
}

struct NormKept : torch::CustomClassHolder {
  optional<Tensor> gamma;                   // flat buffer
  std::shared_ptr<Store> gammas, betas;     // whose gradients are wanted
  int64_t gamma_at = 0, beta_at = 0;
  bool want_dx = false;
};

// The weights are slices of their stores' flat buffers (variables.py), whose gradients the backward pass adds
// to (those of gamma_store and beta_store; below 0: not wanted); `anchor` is the leaf that records a call whose input needs no gradient.
struct LayerNormFn : torch::autograd::Function<LayerNormFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& input, const optional<Tensor>& anchor,
                        const optional<Tensor>& gamma, int64_t gamma_at, const optional<Tensor>& beta, int64_t beta_at,
                        int64_t gamma_store, int64_t beta_store, double eps) {
    const Tensor x = rows_of(input, tfx::kLayerNormMax, "layer_norm");
    auto [y, stats] = norm_pass(x, input.sizes(), var_or_null(gamma, gamma_at, x, "gamma"),
                                var_or_null(beta, beta_at, x, "beta"), eps, true);
    ctx->save_for_backward({x, stats});
    // (not saved variables: an optimizer may write them before a later backward pass, as with every other op)
    auto k = c10::make_intrusive<NormKept>();
    k->gamma = gamma;
    k->gammas = store_of(gamma_store);
    k->betas = store_of(beta_store);
    k->gamma_at = gamma_at;
    k->beta_at = beta_at;
    k->want_dx = input.requires_grad();
    keep(ctx, k);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    first_order("layer_norm");
    variable_list out(9);
    const auto saved = ctx->get_saved_variables();
    const Tensor& x = saved[0];
    const auto k = kept<NormKept>(ctx);
    out[0] = norm_pass_bwd(x, g[0], saved[1], var_or_null(k->gamma, k->gamma_at, x, "gamma"),
                           var_or_null(grad_of(k->gammas), k->gamma_at, x, "gamma"),
                           var_or_null(grad_of(k->betas), k->beta_at, x, "beta"), k->want_dx);
    tell_ready(k->gammas, k->gamma_at);
    tell_ready(k->betas, k->beta_at);
    return out;
  }
};

Tensor layer_norm(const Tensor& input, const optional<Tensor>& anchor, const optional<Tensor>& gamma, int64_t gamma_at,
                  const optional<Tensor>& beta, int64_t beta_at, int64_t gamma_store, int64_t beta_store, double eps) {
  TORCH_CHECK_VALUE(eps >= 1e-30 && std::isfinite(eps), "layer_norm: eps of at least 1e-30 expected, got ", eps);
  no_tangent(input, "layer_norm");
  if (at::GradMode::is_enabled() && (input.requires_grad() || has(anchor)))
    return LayerNormFn::apply(input, anchor, gamma, gamma_at, beta, beta_at, gamma_store, beta_store, eps);
  const Tensor x = rows_of(input, tfx::kLayerNormMax, "layer_norm");
  return std::get<0>(norm_pass(x, input.sizes(), var_or_null(gamma, gamma_at, x, "gamma"),
                               var_or_null(beta, beta_at, x, "beta"), eps, false));
}

// The two passes by themselves (for a caller that has to run code of its own after the backward pass):
// (y, stats [rows, 2]), and dx (undefined unless wanted), with dgamma, dbeta [C] added to
std::tuple<Tensor, Tensor> layer_norm_fwd(const Tensor& input, const optional<Tensor>& gamma, const optional<Tensor>& beta,
                                          double eps) {
  TORCH_CHECK_VALUE(eps >= 1e-30 && std::isfinite(eps), "layer_norm: eps of at least 1e-30 expected, got ", eps);
  const Tensor x = rows_of(input, tfx::kLayerNormMax, "layer_norm");
  return norm_pass(x, input.sizes(), f32_or_null(gamma, x, x.size(1), "gamma"), f32_or_null(beta, x, x.size(1), "beta"), eps,
                   true);
}

Tensor layer_norm_bwd(const Tensor& input, const Tensor& dy, const Tensor& stats, const optional<Tensor>& gamma,
                      const optional<Tensor>& dgamma, const optional<Tensor>& dbeta, bool want_dx) {
  const Tensor x = rows_of(input, tfx::kLayerNormMax, "layer_norm");
  return norm_pass_bwd(x, dy, stats, f32_or_null(gamma, x, x.size(1), "gamma"), f32_or_null(dgamma, x, x.size(1), "dgamma"),
                       f32_or_null(dbeta, x, x.size(1), "dbeta"), want_dx);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(tfx, m) {
  m.def("token_log_probs", &token_log_probs);
  m.def("distillation_loss", &distillation_loss);
  m.def("layer_norm(Tensor x, Tensor? anchor, Tensor? gamma, int gamma_at, Tensor? beta, int beta_at, int gamma_store, "
        "int beta_store, float eps) -> Tensor", &layer_norm);
  m.def("store_new", &store_new);
  m.def("store_set", &store_set);
  m.def("store_free", &store_free);
  m.def("layer_norm_fwd", &layer_norm_fwd);
  m.def("layer_norm_bwd(Tensor x, Tensor dy, Tensor stats, Tensor? gamma, Tensor(a!)? dgamma, Tensor(b!)? dbeta, "
        "bool want_dx) -> Tensor", &layer_norm_bwd);
}
