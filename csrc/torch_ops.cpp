// torch operators kfac_hip::layer_norm, ::token_logprobs and ::topk_distill over
// the kernels of csrc/ln.hip and csrc/vocab.hip, with their autograd nodes.
//
// The nodes are C++ because a language model's step is bound by the host: a
// backward node in Python runs under the interpreter's lock on the engine's
// device thread.  The 6 x 512 Transformer LM (700 tokens, 13 norms, eager SGD
// step): 4.5 .. 4.9 ms with these, 7.25 ms with Python nodes, 5.55 ms with
// torch's own layer norm.
//
// ops/ln.py and ops/vocab.py check the arguments; what is checked here again is
// what the kernels' addressing rests on.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <cmath>

#include "records.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int code(at::ScalarType t) {
  TORCH_CHECK(t == at::kFloat || t == at::kBFloat16 || t == at::kHalf,
              "kfac_hip: fp32, bf16 or fp16 expected, got ", t);
  return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : 2;
}

ihipStream_t* stream_of(const Tensor& t) {
  return (ihipStream_t*)c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

void check(int err, const char* name) {
  TORCH_CHECK(err == 0, name, " failed with HIP error ", err);
}

template <class T = void> T* ptr(const Tensor& t) {
  return t.defined() ? (T*)t.data_ptr() : nullptr;
}

Tensor contiguous_like(const Tensor& t, at::ScalarType dtype) {
  return at::empty_like(t, t.options().dtype(dtype), at::MemoryFormat::Contiguous);
}

// t as (rows, n) with contiguous rows (a copy where no view has them) and the
// distance between them
struct Rows {
  Tensor t;
  int64_t ld = 0;
  Rows(const Tensor& x, int64_t rows, int64_t n) : t(x), ld(n) {
    if (!x.defined() || x.is_contiguous()) return;
    t = x.reshape({rows, n});
    if (n > 1 && t.stride(1) != 1) t = t.contiguous();
    ld = t.stride(0);
  }
};

// ------------------------------------------------------------------ layer norm
struct Norm {
  Tensor y, s, stats;
};

int64_t width(const Tensor& x, int64_t dims) {
  int64_t n = 1;
  for (int64_t i = x.dim() - dims; i < x.dim(); ++i) n *= x.size(i);
  return n;
}

Norm norm_forward(Tensor x, Tensor z, Tensor weight, Tensor bias, int64_t dims, double eps,
                  bool wide, bool keep) {
  at::AutoDispatchBelowADInplaceOrView below;
  c10::DeviceGuard guard(x.device());
  const int64_t D = width(x, dims), rows = x.numel() / D;
  if (z.defined() && x.scalar_type() != z.scalar_type() && x.scalar_type() != at::kFloat) {
    std::swap(x, z);                                    // the sum has the wider type: fp32 ...
    if (x.scalar_type() != at::kFloat) x = x.to(at::kFloat);      // ... of bf16 + fp16, too
  }
  Norm r;
  r.y = contiguous_like(x, wide ? at::kFloat : x.scalar_type());
  r.s = z.defined() ? contiguous_like(x, x.scalar_type()) : x;
  if (keep) r.stats = at::empty({2 * rows}, x.options().dtype(at::kFloat));
  const Rows xr(x, rows, D), zr(z, rows, D);
  if (weight.defined()) weight = weight.contiguous();
  if (bias.defined()) bias = bias.contiguous();
  KfacLnFwd a = {};
  a.x = xr.t.data_ptr();
  a.z = ptr(zr.t);
  a.w = ptr(weight);
  a.b = ptr(bias);
  a.y = r.y.data_ptr();
  a.s = z.defined() ? r.s.data_ptr() : nullptr;
  a.mean = ptr<float>(r.stats);
  a.rstd = keep ? a.mean + rows : nullptr;
  a.ldx = xr.ld;
  a.ldz = zr.ld;
  a.rows = rows;
  a.D = D;
  a.sdt = code(x.scalar_type());
  a.zdt = z.defined() ? code(z.scalar_type()) : 0;
  a.wdt = weight.defined() ? code(weight.scalar_type()) : 0;
  a.bdt = bias.defined() ? code(bias.scalar_type()) : 0;
  a.ydt = code(r.y.scalar_type());
  a.eps = (float)eps;
  check(kfac_ln_forward(&a, stream_of(x)), "kfac_ln_forward");
  return r;
}

struct NormGrad {
  Tensor d, low, dw, db;        // of s; the same in the narrower type of x and z; of the weights
};

NormGrad norm_backward(const Tensor& dy, const Tensor& ds, const Tensor& s, Tensor weight,
                       const Tensor& bias, const Tensor& stats, int64_t dims,
                       optional<at::ScalarType> low, bool need_s, bool need_w, bool need_b) {
  at::AutoDispatchBelowADInplaceOrView below;
  c10::DeviceGuard guard(s.device());
  const int64_t D = width(s, dims), rows = s.numel() / D;
  NormGrad r;
  Tensor part;
  if (need_s) r.d = contiguous_like(s, s.scalar_type());
  if (need_s && low) r.low = contiguous_like(s, *low);
  if (need_w) r.dw = contiguous_like(weight, weight.scalar_type());
  if (need_b) r.db = contiguous_like(bias, bias.scalar_type());
  if (need_w || need_b)
    part = at::empty({(int64_t)kfac_ln_ws_floats(rows, D, code(s.scalar_type()))}, s.options().dtype(at::kFloat));
  const Rows gr(dy, rows, D), er(ds, rows, D), sr(s, rows, D);
  if (weight.defined()) weight = weight.contiguous();
  KfacLnBwd a = {};
  a.dy = gr.t.data_ptr();
  a.ds = ptr(er.t);
  a.s = sr.t.data_ptr();
  a.w = ptr(weight);
  a.mean = ptr<float>(stats);
  a.rstd = a.mean + rows;
  a.dx = ptr(r.d);
  a.dz = ptr(r.low);
  a.dw = ptr(r.dw);
  a.db = ptr(r.db);
  a.part = ptr<float>(part);
  a.lddy = gr.ld;
  a.ldds = er.ld;
  a.lds = sr.ld;
  a.rows = rows;
  a.D = D;
  a.sdt = code(s.scalar_type());
  a.zdt = r.low.defined() ? code(*low) : 0;
  a.wdt = weight.defined() ? code(weight.scalar_type()) : 0;
  a.bdt = bias.defined() ? code(bias.scalar_type()) : 0;
  a.ydt = code(dy.scalar_type());
  check(kfac_ln_backward(&a, stream_of(s)), "kfac_ln_backward");
  return r;
}

// the same by operations that autograd follows (create_graph); the formulas of
// csrc/ln.hip, since a node that calls the engine again can wait for itself
NormGrad norm_backward_graph(const Tensor& dy, const Tensor& ds, const Tensor& s,
                             const Tensor& weight, const Tensor& bias, int64_t dims, double eps) {
  std::vector<int64_t> row, over;                    // the normalised dimensions, the others
  for (int64_t i = 0; i < s.dim(); ++i) (i < s.dim() - dims ? over : row).push_back(i);
  const Tensor x = s.to(at::kFloat), gy = dy.to(at::kFloat);
  // as csrc/ln.hip sums: scaled, so that a sum of the type's lowest values is finite
  const double D = (double)width(s, dims), scale = std::ldexp(1.0, -1 - std::ilogb(D));
  const Tensor c = x - (x * scale).sum(row, true) / (D * scale);
  const Tensor r = (c.square().mean(row, true) + eps).rsqrt(), h = c * r;
  const Tensor g = weight.defined() ? gy * weight.to(at::kFloat) : gy;
  NormGrad out;
  out.d = (r * (g - g.mean(row, true) - h * (g * h).mean(row, true))).to(s.scalar_type());
  if (ds.defined()) out.d = out.d + ds;
  auto columns = [&](const Tensor& t, const Tensor& like) {
    return (over.empty() ? t : t.sum(over)).to(like.scalar_type());
  };
  if (weight.defined()) out.dw = columns(gy * h, weight);
  if (bias.defined()) out.db = columns(gy, bias);
  return out;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& z,
                               const optional<Tensor>& weight, const optional<Tensor>& bias,
                               int64_t dims, double eps, bool wide) {
    const Tensor none;
    const bool sum = z.has_value();
    const Norm r = norm_forward(x, z.value_or(none), weight.value_or(none), bias.value_or(none),
                                dims, eps, wide, true);
    ctx->save_for_backward({r.s, weight.value_or(none), bias.value_or(none), r.stats});
    ctx->saved_data["dims"] = dims;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["x"] = (int64_t)x.scalar_type();
    ctx->saved_data["z"] = sum ? (int64_t)z->scalar_type() : (int64_t)-1;
    ctx->set_materialize_grads(false);
    return sum ? variable_list{r.y, r.s} : variable_list{r.y};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &s = saved[0], &weight = saved[1], &bias = saved[2], &stats = saved[3];
    const int64_t dims = ctx->saved_data["dims"].toInt();
    const auto xt = (at::ScalarType)ctx->saved_data["x"].toInt();
    const int64_t zcode = ctx->saved_data["z"].toInt();
    const bool sum = zcode >= 0;
    const auto zt = sum ? (at::ScalarType)zcode : xt;
    // edges are those of the tensors that were given
    const bool need_x = ctx->needs_input_grad(0), need_z = sum && ctx->needs_input_grad(1);
    const bool need_w = weight.defined() && ctx->needs_input_grad(1 + sum);
    const bool need_b = bias.defined() && ctx->needs_input_grad(1 + sum + weight.defined());
    const Tensor dy = grads[0], ds = sum ? grads[1] : Tensor();
    variable_list out(7);
    if (!dy.defined() && !ds.defined()) return out;
    NormGrad r;
    if (!dy.defined()) {
      r.d = ds;
    } else if (at::GradMode::is_enabled()) {
      r = norm_backward_graph(dy, ds, s, weight, bias, dims, ctx->saved_data["eps"].toDouble());
    } else {
      optional<at::ScalarType> low;
      if (xt != s.scalar_type()) low = xt;
      else if (zt != s.scalar_type()) low = zt;
      r = norm_backward(dy, ds, s, weight, bias, stats, dims, low, need_x || need_z, need_w,
                        need_b);
    }
    auto as = [&](at::ScalarType t) {
      return t == r.d.scalar_type() ? r.d
             : r.low.defined() && t == r.low.scalar_type() ? r.low : r.d.to(t);
    };
    if (need_x) out[0] = as(xt);
    if (need_z) out[1] = as(zt);
    if (need_w) out[2] = r.dw;
    if (need_b) out[3] = r.db;
    return out;
  }
};

bool wants(const optional<Tensor>& t) { return t && t->requires_grad(); }

// (y, s): s undefined without z
std::tuple<Tensor, Tensor> layer_norm(const Tensor& x, const optional<Tensor>& z,
                                      const optional<Tensor>& weight, const optional<Tensor>& bias,
                                      int64_t dims, double eps, bool wide) {
  TORCH_CHECK(x.is_cuda() && dims >= 1 && dims <= x.dim() && x.numel() > 0,
              "kfac_hip::layer_norm: a GPU tensor with elements expected");
  const int64_t D = width(x, dims);
  TORCH_CHECK(!z || (z->sizes() == x.sizes() && z->device() == x.device()),
              "kfac_hip::layer_norm: z must have x's shape and device");
  for (const auto* p : {&weight, &bias})
    TORCH_CHECK(!*p || ((*p)->numel() == D && (*p)->device() == x.device()),
                "kfac_hip::layer_norm: weight and bias must fit x's last dimensions and device");
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || wants(z) || wants(weight) || wants(bias))) {
    const variable_list r = LayerNorm::apply(x, z, weight, bias, dims, eps, wide);
    return {r[0], z ? r[1] : Tensor()};
  }
  const Tensor none;
  const Norm r = norm_forward(x, z.value_or(none), weight.value_or(none), bias.value_or(none),
                              dims, eps, wide, false);
  return {r.y, z ? r.s : Tensor()};
}

// -------------------------------------------------------- behind the vocabulary
void check_logits(const Tensor& x) {
  TORCH_CHECK(x.is_cuda() && x.dim() >= 1 && x.size(-1) >= 1,
              "kfac_hip: GPU logits (..., V) expected");
}

// g or a copy of it and the distance between its rows: the gradient of a mean or
// sum is one number expanded (distance 0)
struct RowGrad {
  Tensor t;
  int64_t step = 0;
  explicit RowGrad(const Tensor& g) : t(g), step(1) {
    if (!g.defined() || g.is_contiguous()) return;
    for (const int64_t s : g.strides())
      if (s != 0) {
        t = g.contiguous();
        return;
      }
    step = 0;
  }
};

// a gradient whose own derivative is an error, not silently zero
Tensor once(const Tensor& dx) {
  if (!at::GradMode::is_enabled()) return dx;
  const auto node = std::make_shared<torch::autograd::DelayedError>(
      "kfac_hip: the operators on logits have no second derivative", 1);
  return node->apply({dx.requires_grad_(true)})[0];
}

KfacVocabFwd vocab_args(const Rows& x, int64_t rows, int64_t V, double inv_t) {
  KfacVocabFwd a = {};
  a.x = x.t.data_ptr();
  a.ld = x.ld;
  a.rows = rows;
  a.V = V;
  a.dt = code(x.t.scalar_type());
  a.inv_t = (float)inv_t;
  return a;
}

Tensor workspace(const KfacVocabFwd& a, const Tensor& x) {
  const int64_t n = kfac_vocab_ws_bytes(a.dt, a.rows, a.V, a.k);
  return n ? at::empty({n}, x.options().dtype(at::kByte)) : Tensor();
}

Tensor vocab_backward(const Tensor& x, const Tensor& stats, KfacVocabBwd a, const Tensor& g,
                      const Tensor& gh, double inv_t) {
  const int64_t V = x.size(-1), rows = x.numel() / V;
  Tensor dx = contiguous_like(x, x.scalar_type());
  if (rows == 0) return dx;
  const Rows xr(x, rows, V);
  const RowGrad gr(g), hr(gh);
  a.x = xr.t.data_ptr();
  a.stats = ptr<float>(stats);
  a.g = ptr<float>(gr.t);
  a.gh = ptr<float>(hr.t);
  a.dx = dx.data_ptr();
  a.ld = xr.ld;
  a.rows = rows;
  a.V = V;
  a.gs = gr.step;
  a.ghs = hr.step;
  a.dt = code(x.scalar_type());
  a.inv_t = (float)inv_t;
  check(kfac_vocab_backward(&a, stream_of(x)), "kfac_vocab_backward");
  return dx;
}

struct Scores {
  Tensor lp, entropy, top_lp, top_ids, targets, stats;
};

Scores scores_forward(const Tensor& x, const Tensor& targets, int64_t k, bool entropy,
                      double inv_t, int64_t ignore, bool keep) {
  at::AutoDispatchBelowADInplaceOrView below;
  c10::DeviceGuard guard(x.device());
  const int64_t V = x.size(-1), rows = x.numel() / V;
  const auto f32 = x.options().dtype(at::kFloat);
  const auto shape = x.sizes().slice(0, x.dim() - 1);
  Scores r;
  if (targets.defined()) {
    r.lp = at::empty(shape, f32);
    r.targets = targets.to(at::kLong).contiguous();
  }
  if (entropy) r.entropy = at::empty(shape, f32);
  if (k) {
    auto more = shape.vec();
    more.push_back(k);
    r.top_lp = at::empty(more, f32);
    r.top_ids = at::empty(more, f32.dtype(at::kLong));
  }
  if (rows == 0) return r;
  if (keep) r.stats = at::empty({2 * rows}, f32);
  const Rows xr(x, rows, V);
  KfacVocabFwd a = vocab_args(xr, rows, V, inv_t);
  a.targets = (const long long*)ptr(r.targets);
  a.logprob = ptr<float>(r.lp);
  a.entropy = ptr<float>(r.entropy);
  a.top_lp = ptr<float>(r.top_lp);
  a.top_ids = (long long*)ptr(r.top_ids);
  a.stats = ptr<float>(r.stats);
  a.ignore = ignore;
  a.k = (int)k;
  const Tensor ws = workspace(a, x);
  a.ws = ptr(ws);
  check(kfac_vocab_forward(&a, stream_of(x)), "kfac_vocab_forward");
  return r;
}

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
  // the outputs that are asked for, in the order logprobs, entropy, alternatives
  static variable_list forward(AutogradContext* ctx, const Tensor& logits,
                               const optional<Tensor>& targets, int64_t k, bool entropy,
                               double inv_t, int64_t ignore) {
    const Scores r = scores_forward(logits, targets.value_or(Tensor()), k, entropy, inv_t, ignore,
                                    true);
    ctx->save_for_backward({logits, r.targets, r.entropy, r.stats});
    ctx->saved_data["inv_t"] = inv_t;
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["inputs"] = (int64_t)targets.has_value();
    ctx->set_materialize_grads(false);
    variable_list out;
    if (r.lp.defined()) out.push_back(r.lp);
    if (entropy) out.push_back(r.entropy);
    if (k) {
      out.push_back(r.top_lp);
      out.push_back(r.top_ids);
      ctx->mark_non_differentiable({r.top_lp, r.top_ids});
    }
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &logits = saved[0], &targets = saved[1], &entropy = saved[2], &stats = saved[3];
    const bool scored = ctx->saved_data["inputs"].toInt() != 0;
    const Tensor g = scored ? grads[0] : Tensor();
    const Tensor gh = entropy.defined() ? grads[scored ? 1 : 0] : Tensor();
    variable_list out(6);
    if (!g.defined() && !gh.defined()) return out;
    Tensor dx;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      c10::DeviceGuard guard(logits.device());
      KfacVocabBwd a = {};
      a.entropy = ptr<float>(entropy);
      a.targets = (const long long*)ptr(targets);
      a.ignore = ctx->saved_data["ignore"].toInt();
      dx = vocab_backward(logits, stats, a, g, gh, ctx->saved_data["inv_t"].toDouble());
    }
    out[0] = once(dx);
    return out;
  }
};

std::tuple<Tensor, Tensor, Tensor, Tensor> token_logprobs(const Tensor& logits,
                                                          const optional<Tensor>& targets,
                                                          int64_t k, bool entropy, double inv_t,
                                                          int64_t ignore) {
  check_logits(logits);
  TORCH_CHECK(!targets || (targets->sizes() == logits.sizes().slice(0, logits.dim() - 1) &&
                           targets->device() == logits.device()),
              "kfac_hip::token_logprobs: targets must fit the logits' rows and device");
  Tensor lp, h, tl, ti;
  if (at::GradMode::is_enabled() && logits.requires_grad()) {
    const variable_list r = TokenLogprobs::apply(logits, targets, k, entropy, inv_t, ignore);
    size_t i = 0;
    if (targets) lp = r[i++];
    if (entropy) h = r[i++];
    if (k) {
      tl = r[i++];
      ti = r[i++];
    }
  } else {
    const Scores r = scores_forward(logits, targets.value_or(Tensor()), k, entropy, inv_t, ignore,
                                    false);
    lp = r.lp;
    h = r.entropy;
    tl = r.top_lp;
    ti = r.top_ids;
  }
  return {lp, h, tl, ti};
}

struct Divergence {
  Tensor loss, stats, ids, mass;      // for the backward pass: (M, L), each id once and its mass
};

Divergence distill_forward(const Tensor& x, const Tensor& ids_, const Tensor& teacher_,
                           double inv_t, bool keep) {
  at::AutoDispatchBelowADInplaceOrView below;
  c10::DeviceGuard guard(x.device());
  const int64_t V = x.size(-1), rows = x.numel() / V, K = ids_.size(-1);
  const auto f32 = x.options().dtype(at::kFloat);
  Divergence r;
  r.loss = at::empty(x.sizes().slice(0, x.dim() - 1), f32);
  if (rows == 0) return r;
  const Tensor ids = ids_.to(at::kLong).contiguous(), teacher = teacher_.contiguous();
  if (keep) {
    r.stats = at::empty({2 * rows}, f32);
    r.ids = at::empty({rows * K}, f32.dtype(at::kInt));
    r.mass = at::empty({rows * K}, f32);
  }
  const Rows xr(x, rows, V);
  KfacVocabFwd a = vocab_args(xr, rows, V, inv_t);
  a.stats = ptr<float>(r.stats);
  a.ids = (const long long*)ptr(ids);
  a.teacher = teacher.data_ptr();
  a.loss = ptr<float>(r.loss);
  a.keep_ids = ptr<int>(r.ids);
  a.keep_q = ptr<float>(r.mass);
  a.K = (int)K;
  a.tdt = code(teacher.scalar_type());
  const Tensor ws = workspace(a, x);
  a.ws = ptr(ws);
  check(kfac_vocab_forward(&a, stream_of(x)), "kfac_vocab_forward");
  return r;
}

struct TopkDistill : torch::autograd::Function<TopkDistill> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& ids,
                        const Tensor& teacher, double inv_t) {
    const Divergence r = distill_forward(logits, ids, teacher, inv_t, true);
    ctx->save_for_backward({logits, r.stats, r.ids, r.mass});
    ctx->saved_data["inv_t"] = inv_t;
    ctx->saved_data["K"] = ids.size(-1);
    return r.loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    variable_list out(4);
    Tensor dx;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      c10::DeviceGuard guard(saved[0].device());
      KfacVocabBwd a = {};
      a.keep_ids = ptr<int>(saved[2]);
      a.keep_q = ptr<float>(saved[3]);
      a.K = (int)ctx->saved_data["K"].toInt();
      dx = vocab_backward(saved[0], saved[1], a, grads[0], Tensor(),
                          ctx->saved_data["inv_t"].toDouble());
    }
    out[0] = once(dx);
    return out;
  }
};

Tensor topk_distill(const Tensor& logits, const Tensor& ids, const Tensor& teacher, double inv_t) {
  check_logits(logits);
  TORCH_CHECK(ids.dim() == logits.dim() && ids.sizes() == teacher.sizes() &&
                  ids.sizes().slice(0, ids.dim() - 1) ==
                      logits.sizes().slice(0, logits.dim() - 1) &&
                  ids.device() == logits.device() && teacher.device() == logits.device(),
              "kfac_hip::topk_distill: ids and teacher must fit the logits' rows and device");
  if (at::GradMode::is_enabled() && logits.requires_grad())
    return TopkDistill::apply(logits, ids, teacher, inv_t);
  return distill_forward(logits, ids, teacher, inv_t, false).loss;
}

}  // namespace

TORCH_LIBRARY(kfac_hip, m) {
  m.def("layer_norm(Tensor x, Tensor? z, Tensor? weight, Tensor? bias, int dims, float eps, "
        "bool wide) -> (Tensor, Tensor)", &layer_norm);
  m.def("token_logprobs(Tensor logits, Tensor? targets, int k, bool entropy, float inv_t, "
        "int ignore) -> (Tensor, Tensor, Tensor, Tensor)", &token_logprobs);
  m.def("topk_distill(Tensor logits, Tensor ids, Tensor teacher, float inv_t) -> Tensor",
        &topk_distill);
}
