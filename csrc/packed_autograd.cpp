// The differentiable forms of the packed-row operators (rotary positions, attention
// over packed sequences, distillation): allocation, layout and the autograd nodes, so
// that one call from Python is one call here and a backward needs no interpreter.
#include <torch/extension.h>

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = c10::optional<at::Tensor>;

// rotary.cu
void rotary_turns(const at::Tensor& q, const OptTensor& k, const at::Tensor& positions, const void* turns, int64_t pairs,
                  const at::Tensor& qo, const OptTensor& ko, bool interleaved, double factor, double sign);
// attention_varlen_sm100.cu
int64_t packed_plan_words(int64_t T, int64_t n);
void packed_plan(at::Tensor cu, int64_t T, at::Tensor plan, OptTensor positions);
void attn_varlen_fwd(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor plan, int64_t n, at::Tensor o, at::Tensor lse,
                     OptTensor low, bool causal, double scale);
void attn_varlen_bwd(at::Tensor dout, at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor o, at::Tensor lse, at::Tensor low,
                     at::Tensor plan, int64_t n, at::Tensor dq, at::Tensor dk, at::Tensor dv, bool causal, double scale);
// distill.cu
void distill(at::Tensor logits, at::Tensor ids, at::Tensor teacher, OptTensor targets, at::Tensor rows, at::Tensor sums,
             OptTensor grad, OptTensor loss, int64_t vocab, int64_t ignore_index, double temperature, double alpha);
void distill_grad(at::Tensor logits, at::Tensor ids, at::Tensor teacher, OptTensor targets, at::Tensor sums, at::Tensor g,
                  at::Tensor grad, int64_t vocab, int64_t ignore_index, double temperature, double alpha, bool mean);
void scale_by_scalar(at::Tensor x, at::Tensor g);

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

at::Tensor fresh(const at::Tensor& like) { return at::empty(like.sizes(), like.options()); }

// ---------------------------------------------------------------------------
// rotary positions
// ---------------------------------------------------------------------------
at::Tensor rows3(const at::Tensor& x) {   // [..., H, D] as [T, H, D], unit stride inside a head
  at::Tensor r = x.dim() == 3 ? x : x.flatten(0, -3);
  return r.stride(2) == 1 ? r : r.contiguous();
}

// turns: the bytes of 64-bit numbers
variable_list rotary_call(const at::Tensor& a, const at::Tensor& b, const at::Tensor& positions, const std::string& turns,
                          bool interleaved, double factor, double sign) {
  TORCH_CHECK(turns.size() % sizeof(double) == 0, "rotary: turns are 64-bit numbers");
  at::Tensor ya = fresh(a), yb = b.defined() ? fresh(b) : at::Tensor();
  OptTensor rb, ryb;
  if (b.defined()) {
    rb = rows3(b);
    ryb = yb.dim() == 3 ? yb : yb.flatten(0, -3);
  }
  rotary_turns(rows3(a), rb, positions, turns.data(), (int64_t)(turns.size() / sizeof(double)),
               ya.dim() == 3 ? ya : ya.flatten(0, -3), ryb, interleaved, factor, sign);
  return {ya, yb};
}

struct Rotary : public torch::autograd::Function<Rotary> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const OptTensor& k, const at::Tensor& positions,
                               const std::string& turns, bool interleaved, double factor) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({positions});
    ctx->saved_data["turns"] = turns;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["factor"] = factor;
    variable_list y = rotary_call(q, k.has_value() ? *k : at::Tensor(), positions, turns, interleaved, factor, 1.0);
    if (!k.has_value()) y.pop_back();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "rotary_embedding: its backward is not differentiable");
    const at::Tensor gq = g[0], gk = g.size() > 1 ? g[1] : at::Tensor();
    variable_list out(6);
    if (!gq.defined() && !gk.defined()) return out;
    const bool first = gq.defined();
    variable_list d = rotary_call(first ? gq : gk, first ? gk : at::Tensor(), ctx->get_saved_variables()[0],
                                  ctx->saved_data["turns"].toStringRef(), ctx->saved_data["interleaved"].toBool(),
                                  ctx->saved_data["factor"].toDouble(), -1.0);
    out[first ? 0 : 1] = d[0];
    if (first && gk.defined()) out[1] = d[1];
    return out;
  }
};

// ---------------------------------------------------------------------------
// attention over packed sequences
// ---------------------------------------------------------------------------
// Readable through a tensor map as it is: aligned, unit stride, no repeated rows or heads.
at::Tensor mapped(const at::Tensor& t) {
  bool ok = t.stride(2) == 1 && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
  for (int i = 0; i < 2; ++i) ok = ok && (t.size(i) == 1 || (t.stride(i) > 0 && t.stride(i) % 8 == 0));
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

struct VarlenAttention : public torch::autograd::Function<VarlenAttention> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& v_,
                            const at::Tensor& plan, int64_t n, bool causal, double scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    const at::Tensor q = mapped(q_), k = mapped(k_), v = mapped(v_);
    at::Tensor o = fresh(q), low = at::empty(q.sizes(), q.options().dtype(at::kChar));
    at::Tensor lse = at::empty({q.size(1), q.size(0)}, q.options().dtype(at::kFloat));
    attn_varlen_fwd(q, k, v, plan, n, o, lse, low, causal, scale);
    ctx->save_for_backward({q, k, v, o, lse, low, plan});
    ctx->saved_data["n"] = n;
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "flash_attention_varlen: its backward is not differentiable");
    const auto s = ctx->get_saved_variables();
    at::Tensor dq = fresh(s[0]), dk = fresh(s[1]), dv = fresh(s[2]);
    attn_varlen_bwd(mapped(g[0]), s[0], s[1], s[2], s[3], s[4], s[5], s[6], ctx->saved_data["n"].toInt(), dq, dk, dv,
                    ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble());
    return {dq, dk, dv, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// ---------------------------------------------------------------------------
// distillation
// ---------------------------------------------------------------------------
// an empty gradient with the logits' row pitch
at::Tensor like_rows(const at::Tensor& z) {
  const int64_t M = z.size(0), W = z.size(1), pitch = M > 1 ? z.stride(0) : W;
  if (pitch == W) return at::empty({M, W}, z.options());
  return at::empty({M * pitch}, z.options()).as_strided({M, W}, {pitch, 1});
}

struct DistillArgs {
  int64_t vocab, ignore_index;
  double temperature, alpha;
};

void save_args(AutogradContext* ctx, const DistillArgs& a) {
  ctx->saved_data["vocab"] = a.vocab;
  ctx->saved_data["ignore_index"] = a.ignore_index;
  ctx->saved_data["temperature"] = a.temperature;
  ctx->saved_data["alpha"] = a.alpha;
}

// The mean of the rows, and in the same pass over the logits its gradient for an
// upstream gradient of 1.  The gradient is kept, the logits are not; the backward
// multiplies it by another upstream gradient in place (one more rounding) and hands
// it over, so it runs once.
struct DistillMean : public torch::autograd::Function<DistillMean> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& z, const at::Tensor& ids, const at::Tensor& teacher,
                            const OptTensor& targets, int64_t vocab, int64_t ignore_index, double temperature, double alpha) {
    at::AutoDispatchBelowADInplaceOrView below;
    const auto f32 = z.options().dtype(at::kFloat);
    at::Tensor rows = at::empty({4 * z.size(0)}, f32), loss = at::empty({}, f32), grad = like_rows(z);
    const int64_t M = z.size(0);
    distill(z, ids, teacher, targets, rows.narrow(0, 0, M), rows.narrow(0, M, 3 * M), grad, loss, vocab, ignore_index,
            temperature, alpha);
    ctx->saved_data["grad"] = grad;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "distillation_loss: its backward is not differentiable");
    c10::IValue& kept = ctx->saved_data["grad"];
    TORCH_CHECK(kept.isTensor(), "distillation_loss: its gradient was handed over by the first backward; "
                                 "call it again for another one");
    at::Tensor grad = kept.toTensor();
    kept = c10::IValue();
    scale_by_scalar(grad.is_contiguous() ? grad : grad.as_strided({grad.size(0) * grad.stride(0)}, {1}), g[0].to(at::kFloat));
    return {grad, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// The rows' losses, or their mean; the backward reads the logits again with the upstream
// gradient in 32 bits.
struct DistillRows : public torch::autograd::Function<DistillRows> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& z, const at::Tensor& ids, const at::Tensor& teacher,
                            const OptTensor& targets, int64_t vocab, int64_t ignore_index, double temperature, double alpha,
                            bool mean) {
    at::AutoDispatchBelowADInplaceOrView below;
    const auto f32 = z.options().dtype(at::kFloat);
    at::Tensor rows = at::empty({z.size(0)}, f32), sums = at::empty({3 * z.size(0)}, f32);
    OptTensor loss;
    if (mean) loss = at::empty({}, f32);
    distill(z, ids, teacher, targets, rows, sums, c10::nullopt, loss, vocab, ignore_index, temperature, alpha);
    ctx->saved_data["mean"] = mean;
    ctx->save_for_backward({z, ids, teacher, targets.has_value() ? *targets : at::Tensor(), sums});
    save_args(ctx, {vocab, ignore_index, temperature, alpha});
    return mean ? *loss : rows;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "distillation_loss: its backward is not differentiable");
    const auto s = ctx->get_saved_variables();
    at::Tensor grad = like_rows(s[0]);
    OptTensor targets;
    if (s[3].defined()) targets = s[3];
    distill_grad(s[0], s[1], s[2], targets, s[4], g[0].to(at::kFloat).contiguous(), grad, ctx->saved_data["vocab"].toInt(),
                 ctx->saved_data["ignore_index"].toInt(), ctx->saved_data["temperature"].toDouble(),
                 ctx->saved_data["alpha"].toDouble(), ctx->saved_data["mean"].toBool());
    variable_list out(9);
    out[0] = grad;
    return out;
  }
};

}  // namespace

// (q', k') for [..., H, D] tensors; positions 1-D
std::vector<at::Tensor> rotary_embedding(at::Tensor q, OptTensor k, at::Tensor positions, std::string turns, bool interleaved,
                                         double factor) {
  const at::Tensor kt = k.has_value() ? *k : at::Tensor();
  variable_list y;
  if (wants_grad({&q, &kt}, "rotary_embedding")) {
    y = Rotary::apply(q, k, positions, turns, interleaved, factor);
  } else {
    y = rotary_call(q, kt, positions, turns, interleaved, factor, 1.0);
    if (!k.has_value()) y.pop_back();
  }
  return y;
}

// (plan, positions) of packed sequences
std::vector<at::Tensor> packed_sequences(at::Tensor cu, int64_t T) {
  const int64_t words = packed_plan_words(T, cu.numel() - 1);
  at::Tensor buf = at::empty({words + T}, cu.options().dtype(at::kInt));
  at::Tensor plan = buf.narrow(0, 0, words), positions = buf.narrow(0, words, T);
  packed_plan(cu, T, plan, positions);
  return {plan, positions};
}

at::Tensor attn_varlen(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor plan, int64_t n, bool causal, double scale) {
  if (wants_grad({&q, &k, &v}, "flash_attention_varlen")) return VarlenAttention::apply(q, k, v, plan, n, causal, scale);
  q = mapped(q);
  at::Tensor o = fresh(q), lse = at::empty({q.size(1), q.size(0)}, q.options().dtype(at::kFloat));
  attn_varlen_fwd(q, mapped(k), mapped(v), plan, n, o, lse, c10::nullopt, causal, scale);
  return o;
}

// with the sequences as cu_seqlens (int32, on q's device): the plan is built for this call
at::Tensor attn_varlen_cu(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor cu, bool causal, double scale) {
  at::Tensor plan = at::empty({packed_plan_words(q.size(0), cu.numel() - 1)}, cu.options());
  packed_plan(cu, q.size(0), plan, c10::nullopt);
  return attn_varlen(q, k, v, plan, cu.numel() - 1, causal, scale);
}

// The mean (`fused`: with its gradient in the same pass, where one is wanted) or the rows
at::Tensor distill_loss(at::Tensor z, at::Tensor ids, at::Tensor teacher, OptTensor targets, int64_t vocab,
                        int64_t ignore_index, double temperature, double alpha, bool mean, bool fused) {
  ids = ids.contiguous();
  teacher = teacher.contiguous();
  if (targets.has_value()) targets = targets->to(at::kLong).contiguous();
  if (wants_grad({&z}, "distillation_loss")) {
    if (mean && fused) return DistillMean::apply(z, ids, teacher, targets, vocab, ignore_index, temperature, alpha);
    return DistillRows::apply(z, ids, teacher, targets, vocab, ignore_index, temperature, alpha, mean);
  }
  const auto f32 = z.options().dtype(at::kFloat);
  at::Tensor rows = at::empty({z.size(0)}, f32), sums = at::empty({3 * z.size(0)}, f32);
  OptTensor loss;
  if (mean) loss = at::empty({}, f32);
  distill(z, ids, teacher, targets, rows, sums, c10::nullopt, loss, vocab, ignore_index, temperature, alpha);
  return mean ? *loss : rows;
}
