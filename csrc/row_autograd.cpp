// The differentiable forms of the row-wise operators (embedding, layer norm, activations kept
// in 8 bits, token log probabilities): allocation, layout and the autograd nodes, so that one
// call from Python is one call here and a backward needs no interpreter.
#include <torch/extension.h>

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = c10::optional<at::Tensor>;

// embedding.cu
void embedding_fwd(at::Tensor ids, at::Tensor w, at::Tensor y, double scale);
void embedding_bwd(at::Tensor ids, at::Tensor dy, at::Tensor dw, double scale);
// layernorm.cu
void layernorm_fwd(at::Tensor x, OptTensor delta, OptTensor w, OptTensor b, OptTensor h, at::Tensor y, OptTensor stats,
                   OptTensor codes, OptTensor steps, double eps);
void layernorm_bwd(at::Tensor dy, OptTensor dh, OptTensor x, OptTensor codes, OptTensor steps, OptTensor w, at::Tensor stats,
                   at::Tensor dx, OptTensor dw, OptTensor db);
// act8.cu
void act8_keep(at::Tensor x, at::Tensor codes, at::Tensor steps);
void act8_read(at::Tensor codes, at::Tensor steps, at::Tensor x);
void gelu8_fwd(at::Tensor x, at::Tensor y, at::Tensor codes, at::Tensor steps);
void gelu8_bwd(at::Tensor dy, at::Tensor codes, at::Tensor steps, at::Tensor dx);
void swiglu8_fwd(at::Tensor g, at::Tensor u, at::Tensor y, at::Tensor gcodes, at::Tensor gsteps, at::Tensor ucodes,
                 at::Tensor usteps);
void swiglu8_bwd(at::Tensor dy, at::Tensor gcodes, at::Tensor gsteps, at::Tensor ucodes, at::Tensor usteps, at::Tensor dg,
                 at::Tensor du);
// logprobs.cu
void logprob_fwd(at::Tensor z, OptTensor targets, OptTensor logp, at::Tensor entropy, at::Tensor top, at::Tensor ids,
                 at::Tensor stats, int64_t vocab, double temperature);
void logprob_bwd(at::Tensor z, OptTensor targets, at::Tensor top, at::Tensor ids, at::Tensor stats, OptTensor gp, OptTensor gh,
                 OptTensor gt, at::Tensor dz, int64_t vocab, double temperature);

namespace {

// Whether a call goes through its autograd node.  A forward-mode tangent is refused here: a
// call past the node would give a result without one, and no error.
bool wants_grad(std::initializer_list<const at::Tensor*> ts, const char* name) {
  for (const at::Tensor* t : ts)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), name, ": no forward-mode derivative");
  if (!at::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

void once_only(const char* name) {
  TORCH_CHECK(!at::GradMode::is_enabled(), name, ": its backward is not differentiable");
}

// [..., D] as [M, D] with unit column stride
at::Tensor rows2(const at::Tensor& x) {
  at::Tensor r = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
  return r.stride(1) == 1 || r.size(1) == 1 ? r : r.contiguous();
}

at::Tensor dense(const at::Tensor& like) { return at::empty(like.sizes(), like.options()); }

at::Tensor opt(const OptTensor& t) { return t.has_value() ? *t : at::Tensor(); }
OptTensor opt(const at::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

// ---------------------------------------------------------------------------
// embedding
// ---------------------------------------------------------------------------
at::Tensor embedding_call(const at::Tensor& ids, const at::Tensor& w, double scale) {
  std::vector<int64_t> shape = ids.sizes().vec();
  shape.push_back(w.size(1));
  at::Tensor y = at::empty(shape, w.options());
  embedding_fwd(ids.reshape({-1}), w.stride(1) == 1 || w.size(1) == 1 ? w : w.contiguous(), y.view({-1, w.size(1)}), scale);
  return y;
}

struct Embedding : public torch::autograd::Function<Embedding> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& w, const at::Tensor& ids, double scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({ids});
    ctx->saved_data["rows"] = w.size(0);
    ctx->saved_data["scale"] = scale;
    return embedding_call(ids, w, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once_only("embedding");
    const at::Tensor ids = ctx->get_saved_variables()[0], dy = rows2(g[0]);
    at::Tensor dw = at::empty({ctx->saved_data["rows"].toInt(), dy.size(1)}, dy.options());
    embedding_bwd(ids.reshape({-1}), dy, dw, ctx->saved_data["scale"].toDouble());
    return {dw, at::Tensor(), at::Tensor()};
  }
};

// ---------------------------------------------------------------------------
// 8 bits
// ---------------------------------------------------------------------------
struct Kept {
  at::Tensor codes, steps;
};
Kept kept_for(int64_t M, int64_t D, const at::Tensor& like) {
  return {at::empty({M, (D + 15) / 16 * 16}, like.options().dtype(at::kChar)),
          at::empty({M, (D + 127) / 128}, like.options().dtype(at::kFloat))};
}

struct Gelu8 : public torch::autograd::Function<Gelu8> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x) {
    at::AutoDispatchBelowADInplaceOrView below;
    const at::Tensor r = rows2(x);
    at::Tensor y = dense(x);
    const Kept k = kept_for(r.size(0), r.size(1), r);
    gelu8_fwd(r, y.view(r.sizes()), k.codes, k.steps);
    ctx->save_for_backward({k.codes, k.steps});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once_only("gelu");
    const auto s = ctx->get_saved_variables();
    const at::Tensor r = rows2(g[0]);
    at::Tensor dx = dense(g[0]);
    gelu8_bwd(r, s[0], s[1], dx.view(r.sizes()));
    return {dx};
  }
};

struct Swiglu8 : public torch::autograd::Function<Swiglu8> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& gate, const at::Tensor& up) {
    at::AutoDispatchBelowADInplaceOrView below;
    const at::Tensor a = rows2(gate), b = rows2(up);
    at::Tensor y = dense(gate);
    const Kept ka = kept_for(a.size(0), a.size(1), a), kb = kept_for(a.size(0), a.size(1), a);
    swiglu8_fwd(a, b, y.view(a.sizes()), ka.codes, ka.steps, kb.codes, kb.steps);
    ctx->save_for_backward({ka.codes, ka.steps, kb.codes, kb.steps});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once_only("swiglu");
    const auto s = ctx->get_saved_variables();
    const at::Tensor r = rows2(g[0]);
    at::Tensor da = dense(g[0]), db = dense(g[0]);
    swiglu8_bwd(r, s[0], s[1], s[2], s[3], da.view(r.sizes()), db.view(r.sizes()));
    return {da, db};
  }
};

// ---------------------------------------------------------------------------
// layer norm
// ---------------------------------------------------------------------------
// (h, y), or (y) without delta
struct LayerNorm : public torch::autograd::Function<LayerNorm> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const OptTensor& delta, const OptTensor& w,
                               const OptTensor& b, double eps, bool keep8) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->set_materialize_grads(false);
    const at::Tensor r = rows2(x);
    at::Tensor y = dense(x), stats = at::empty({2, r.size(0)}, r.options().dtype(at::kFloat)), h;
    OptTensor d, hr, codes, steps;
    if (delta.has_value()) {
      d = rows2(*delta);
      h = dense(x);
      hr = h.view(r.sizes());
    }
    if (keep8) {
      const Kept k = kept_for(r.size(0), r.size(1), r);
      codes = k.codes;
      steps = k.steps;
    }
    layernorm_fwd(r, d, w, b, hr, y.view(r.sizes()), stats, codes, steps, eps);
    at::Tensor input;
    if (!keep8) input = delta.has_value() ? h : x;
    ctx->save_for_backward({input, opt(codes), opt(steps), opt(w), stats});
    ctx->saved_data["residual"] = delta.has_value();
    ctx->saved_data["dw"] = w.has_value() && w->requires_grad();
    ctx->saved_data["db"] = b.has_value() && b->requires_grad();
    ctx->saved_data["type"] = w.has_value() ? w->scalar_type() : b.has_value() ? b->scalar_type() : at::kFloat;
    if (delta.has_value()) return {h, y};
    return {y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once_only("layer_norm");
    const bool residual = ctx->saved_data["residual"].toBool();
    const at::Tensor gh = residual ? g[0] : at::Tensor(), gy = residual ? g[1] : g[0];
    variable_list out(6);
    if (!gy.defined()) {
      out[0] = gh;
      if (residual) out[1] = gh;
      return out;
    }
    const auto s = ctx->get_saved_variables();
    const at::Tensor r = rows2(gy);
    at::Tensor dx = dense(gy);
    OptTensor dw, db, x, codes, steps, dh;
    const auto type = r.options().dtype(ctx->saved_data["type"].toScalarType());
    if (ctx->saved_data["dw"].toBool()) dw = at::empty({r.size(1)}, type);
    if (ctx->saved_data["db"].toBool()) db = at::empty({r.size(1)}, type);
    if (s[0].defined()) x = rows2(s[0]);
    else codes = s[1], steps = s[2];
    if (gh.defined()) dh = rows2(gh);
    layernorm_bwd(r, dh, x, codes, steps, opt(s[3]), s[4], dx.view(r.sizes()), dw, db);
    out[0] = dx;
    if (residual) out[1] = dx;
    out[2] = opt(dw);
    out[3] = opt(db);
    return out;
  }
};

// ---------------------------------------------------------------------------
// token log probabilities
// ---------------------------------------------------------------------------
// an empty gradient with the logits' row pitch and alignment
at::Tensor like_logits(const at::Tensor& z) {
  const int64_t M = z.size(0), W = z.size(1), pitch = M > 1 ? z.stride(0) : W, es = z.element_size();
  const int64_t lead = (int64_t)((reinterpret_cast<uintptr_t>(z.data_ptr()) & 15) / es);
  if (pitch == W && lead == 0) return at::empty({M, W}, z.options());
  return at::empty({(M - 1) * pitch + W + lead}, z.options()).as_strided({M, W}, {pitch, 1}, lead);
}

variable_list logprobs_call(const at::Tensor& z, const OptTensor& targets, int64_t K, int64_t vocab, double temperature,
                            at::Tensor& stats) {
  const auto f32 = z.options().dtype(at::kFloat);
  const int64_t M = z.size(0);
  at::Tensor top = at::empty({M, K}, f32), ids = at::empty({M, K}, z.options().dtype(at::kLong));
  at::Tensor entropy = at::empty({M}, f32);
  OptTensor logp;
  if (targets.has_value()) logp = at::empty({M}, f32);
  stats = at::empty({M, 3}, f32);
  logprob_fwd(z, targets, logp, entropy, top, ids, stats, vocab, temperature);
  return {logp.has_value() ? *logp : at::empty({0}, f32), entropy, top, ids};
}

struct Logprobs : public torch::autograd::Function<Logprobs> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& z, const OptTensor& targets, int64_t K, int64_t vocab,
                               double temperature) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->set_materialize_grads(false);
    at::Tensor stats;
    variable_list out = logprobs_call(z, targets, K, vocab, temperature, stats);
    ctx->mark_non_differentiable({out[3]});
    ctx->save_for_backward({z, opt(targets), out[3], stats});
    ctx->saved_data["vocab"] = vocab;
    ctx->saved_data["temperature"] = temperature;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once_only("token_logprobs");
    variable_list out(5);
    if (!g[0].defined() && !g[1].defined() && !g[2].defined()) return out;
    const auto s = ctx->get_saved_variables();
    const at::Tensor z = s[0], ids = s[2];
    auto grad = [](const at::Tensor& t) { return t.defined() ? OptTensor(t.contiguous()) : OptTensor(); };
    const at::Tensor top = at::empty({ids.size(0), ids.size(1)}, z.options().dtype(at::kFloat));
    at::Tensor dz = like_logits(z);
    logprob_bwd(z, opt(s[1]), top, ids, s[3], s[1].defined() ? grad(g[0]) : OptTensor(), grad(g[1]), grad(g[2]), dz,
                ctx->saved_data["vocab"].toInt(), ctx->saved_data["temperature"].toDouble());
    out[0] = dz;
    return out;
  }
};

}  // namespace

at::Tensor embedding_lookup(at::Tensor ids, at::Tensor w, double scale) {
  ids = ids.contiguous();
  if (wants_grad({&w}, "embedding")) return Embedding::apply(w, ids, scale);
  return embedding_call(ids, w, scale);
}

// (h, y) with delta, (y) without
std::vector<at::Tensor> layer_norm(at::Tensor x, OptTensor delta, OptTensor w, OptTensor b, double eps, bool keep8) {
  if (w.has_value()) w = w->contiguous();
  if (b.has_value()) b = b->contiguous();
  const at::Tensor d = opt(delta), wt = opt(w), bt = opt(b);
  if (wants_grad({&x, &d, &wt, &bt}, "layer_norm")) return LayerNorm::apply(x, delta, w, b, eps, keep8);
  const at::Tensor r = rows2(x);
  at::Tensor y = dense(x);
  OptTensor dr, hr;
  at::Tensor h;
  if (delta.has_value()) {
    dr = rows2(*delta);
    h = dense(x);
    hr = h.view(r.sizes());
  }
  layernorm_fwd(r, dr, w, b, hr, y.view(r.sizes()), c10::nullopt, c10::nullopt, c10::nullopt, eps);
  if (delta.has_value()) return {h, y};
  return {y};
}

// (codes, steps)
std::vector<at::Tensor> act8_quantize(at::Tensor x) {
  at::AutoDispatchBelowADInplaceOrView below;
  const at::Tensor r = rows2(x);
  const Kept k = kept_for(r.size(0), r.size(1), r);
  act8_keep(r, k.codes, k.steps);
  return {k.codes, k.steps};
}

at::Tensor act8_dequantize(at::Tensor codes, at::Tensor steps, std::vector<int64_t> shape, at::ScalarType dtype) {
  at::Tensor x = at::empty(shape, codes.options().dtype(dtype));
  act8_read(codes, steps, x.view({codes.size(0), shape.back()}));
  return x;
}

at::Tensor gelu8(at::Tensor x) { return Gelu8::apply(x); }

at::Tensor swiglu8(at::Tensor gate, at::Tensor up) { return Swiglu8::apply(gate, up); }

// (logp [M] or [0] without targets, entropy [M], top [M, K], ids [M, K])
std::vector<at::Tensor> token_logprobs(at::Tensor z, OptTensor targets, int64_t K, int64_t vocab, double temperature) {
  if (targets.has_value()) targets = targets->to(at::kLong).contiguous();
  if (wants_grad({&z}, "token_logprobs")) return Logprobs::apply(z, targets, K, vocab, temperature);
  at::Tensor stats;
  return logprobs_call(z, targets, K, vocab, temperature, stats);
}
