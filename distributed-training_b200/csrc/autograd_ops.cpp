// Autograd of the router and the experts' products as C++ functions.
//
// The kernels of a small call take a few microseconds.  A forward and backward pass of the
// router (16384 x 16) took 131 us through a Python autograd.Function (its frames, the zero
// gradients it makes for integer outputs) and takes 62 through this one, of which the
// engine's own share is about 40.
#include <torch/extension.h>

#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>

namespace dtb {

// route.cu
std::vector<torch::Tensor> route_fwd(torch::Tensor logits, int64_t k, bool softmax, c10::optional<torch::Tensor> bias,
                                     int64_t groups, int64_t keep, int64_t top, bool renorm, double scale);
torch::Tensor route_bwd(torch::Tensor logits, torch::Tensor idx, torch::Tensor dgates, bool softmax, bool renorm,
                        double scale);
// moe.cu
std::vector<torch::Tensor> experts_fwd(torch::Tensor x, torch::Tensor w1, c10::optional<torch::Tensor> b1,
                                       torch::Tensor w2, c10::optional<torch::Tensor> b2, torch::Tensor idx,
                                       torch::Tensor gates, bool save);
std::vector<torch::Tensor> experts_bwd(torch::Tensor dy, torch::Tensor x, torch::Tensor w1, torch::Tensor w2,
                                       c10::optional<torch::Tensor> b2, torch::Tensor gates,
                                       std::vector<torch::Tensor> saved, torch::Tensor dw1,
                                       c10::optional<torch::Tensor> db1, torch::Tensor dw2,
                                       c10::optional<torch::Tensor> db2);

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

// Whether a tensor carries a forward-mode derivative.  The kernels have none, so the callers compute such inputs
// with torch ops, which do.
static bool is_dual(const torch::Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
static void check_not_dual(const torch::Tensor& dy, const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(!is_dual(dy), what, ": a forward-mode derivative through the kernels' backward is not implemented");
}

// The kernels' gradients have no graph of their own.  Where one is asked for (create_graph), they hang on a node that
// raises, and whose edges lead to what they were made from: no derivative passes it by.
static variable_list once_differentiable(variable_list grads, const variable_list& from, const char* what) {
  if (!torch::GradMode::is_enabled()) return grads;
  auto node = std::make_shared<torch::autograd::Error>(
      std::string(what) + ": the gradient of the kernels' gradient is not implemented",
      torch::autograd::collect_next_edges(from));
  for (auto& g : grads)
    if (g.defined()) torch::autograd::set_history(g, node);
  return grads;
}

struct RouteFn : public torch::autograd::Function<RouteFn> {
  static variable_list forward(AutogradContext* ctx, Variable logits, int64_t k, bool softmax,
                               c10::optional<torch::Tensor> bias, int64_t groups, int64_t keep, int64_t top,
                               bool renorm, double scale) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto out = route_fwd(logits, k, softmax, bias, groups, keep, top, renorm, scale);
    ctx->save_for_backward({logits, out[1]});
    ctx->saved_data["softmax"] = softmax;
    ctx->saved_data["renorm"] = renorm;
    ctx->saved_data["scale"] = scale;
    ctx->mark_non_differentiable({out[1], out[2]});
    ctx->set_materialize_grads(false);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(9);
    if (!grads[0].defined()) return out;
    check_not_dual(grads[0], "route");
    const auto saved = ctx->get_saved_variables();
    {
      at::AutoDispatchBelowADInplaceOrView guard;
      out[0] = route_bwd(saved[0], saved[1], grads[0].contiguous(), ctx->saved_data["softmax"].toBool(),
                         ctx->saved_data["renorm"].toBool(), ctx->saved_data["scale"].toDouble());
    }
    return once_differentiable(std::move(out), {saved[0], grads[0]}, "route");
  }
};

// route on logits of any leading shape and layout; nothing where the kernels do not take them (other types or
// devices, more than 512 experts, 32 slots or 32 groups, forward-mode derivatives).
c10::optional<std::tuple<torch::Tensor, torch::Tensor, torch::Tensor>> route_autograd(
    torch::Tensor logits, int64_t k, const std::string& score, c10::optional<torch::Tensor> bias, int64_t groups,
    int64_t keep, int64_t top, bool renorm, double scale) {
  TORCH_CHECK_VALUE(score == "softmax" || score == "sigmoid", "route: score must be 'softmax' or 'sigmoid', got '", score,
                    "'");
  TORCH_CHECK_VALUE(logits.dim() >= 1, "route: logits (..., experts) expected");
  const int64_t e = logits.size(-1);
  TORCH_CHECK_VALUE(k >= 1 && k <= e, "route: k must be in [1, ", e, "], got ", k);
  TORCH_CHECK_VALUE(groups >= 1 && e % groups == 0 && keep >= 1 && keep <= groups && keep * (e / groups) >= k, "route: ", e,
                    " experts in ", groups, " groups, ", keep, " kept, do not give ", k, " experts a token");
  TORCH_CHECK_VALUE(top == 1 || (top == 2 && e / groups >= 2), "route: group_top must be 1, or 2 with groups of at least 2, got ",
                    top);
  const bool biased = bias && bias->defined();
  TORCH_CHECK_VALUE(!biased || (bias->dim() == 1 && bias->size(0) == e && bias->device() == logits.device()),
                    "route: bias must be [", e, "] on the logits' device");
  const auto t = logits.scalar_type();
  if (!logits.is_cuda() || (t != at::kFloat && t != at::kBFloat16) || e > 512 || k > 32 || groups > 32 ||
      is_dual(logits))
    return c10::nullopt;
  if (biased) bias = bias->detach().to(at::kFloat).contiguous();
  const bool two = logits.dim() == 2;
  auto shape = logits.sizes().vec();
  shape.back() = k;
  const auto z = (two ? logits : logits.reshape({-1, e})).contiguous();
  const auto out = torch::GradMode::is_enabled() && z.requires_grad()
                       ? RouteFn::apply(z, k, score == "softmax", bias, groups, keep, top, renorm, scale)
                       : route_fwd(z, k, score == "softmax", bias, groups, keep, top, renorm, scale);
  if (two) return std::make_tuple(out[0], out[1], out[2]);
  return std::make_tuple(out[0].view(shape), out[1].view(shape), out[2]);
}

// Contiguous, and at a 16-byte boundary as the experts' loads need it: views of a flat buffer may start anywhere.
static torch::Tensor aligned(const torch::Tensor& t) {
  auto c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.const_data_ptr()) % 16 ? c.clone() : c;
}

struct ExpertsFn : public torch::autograd::Function<ExpertsFn> {
  static Variable forward(AutogradContext* ctx, Variable x, Variable w1, c10::optional<Variable> b1, Variable w2,
                          c10::optional<Variable> b2, Variable idx, Variable gates) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto out = experts_fwd(x, w1, b1, w2, b2, idx, gates, true);
    variable_list keep{x, w1, w2, gates, b2.value_or(torch::Tensor()), b1.value_or(torch::Tensor())};
    keep.insert(keep.end(), out.begin() + 1, out.end());
    ctx->save_for_backward(keep);
    ctx->set_materialize_grads(false);
    return out[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(7);
    if (!grads[0].defined()) return out;
    check_not_dual(grads[0], "expert_mlp");
    const auto saved = ctx->get_saved_variables();
    compute(ctx, saved, grads[0], out);
    variable_list from(saved.begin(), saved.begin() + 6);  // x, w1, w2, gates, b2, b1
    from.push_back(grads[0]);
    return once_differentiable(std::move(out), from, "expert_mlp");
  }
  static void compute(AutogradContext* ctx, const variable_list& saved, const Variable& dy, variable_list& out) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const auto &x = saved[0], &w1 = saved[1], &w2 = saved[2], &gates = saved[3];
    auto dw1 = torch::empty_like(w1), dw2 = torch::empty_like(w2);
    c10::optional<torch::Tensor> db1, db2;
    if (saved[5].defined()) db1 = torch::empty_like(saved[5]);
    c10::optional<torch::Tensor> b2;
    if (saved[4].defined()) {
      b2 = saved[4];
      db2 = torch::empty_like(*b2);
    }
    auto d = experts_bwd(aligned(dy), x, w1, w2, b2, gates, std::vector<torch::Tensor>(saved.begin() + 6, saved.end()),
                         dw1, db1, dw2, db2);
    out[0] = d[0];
    out[1] = dw1;
    if (db1) out[2] = *db1;
    out[3] = dw2;
    if (db2) out[4] = *db2;
    out[6] = d[1];
  }
};

// expert_mlp on inputs of any leading shape and layout; nothing where the kernels do not take them (other
// types or devices, widths that are not multiples of 8, forward-mode derivatives).
c10::optional<torch::Tensor> experts_autograd(torch::Tensor x, torch::Tensor w1, c10::optional<torch::Tensor> b1,
                                              torch::Tensor w2, c10::optional<torch::Tensor> b2, torch::Tensor idx,
                                              torch::Tensor gates) {
  TORCH_CHECK_VALUE(x.dim() >= 1 && w1.dim() == 3 && w2.dim() == 3 && w1.size(1) == x.size(-1) &&
                        w2.size(0) == w1.size(0) && w2.size(1) == w1.size(2),
                    "expert_mlp: x ", x.sizes(), ", w1 ", w1.sizes(), " and w2 ", w2.sizes(), " do not fit");
  TORCH_CHECK_VALUE(idx.dim() == x.dim() && idx.sizes() == gates.sizes() &&
                        idx.sizes().slice(0, idx.dim() - 1) == x.sizes().slice(0, x.dim() - 1),
                    "expert_mlp: idx ", idx.sizes(), " and gates ", gates.sizes(), " must be x's rows by slots");
  const auto it = idx.scalar_type(), gt = gates.scalar_type();
  TORCH_CHECK_VALUE(it == at::kInt || it == at::kLong, "expert_mlp: idx must be int32 or int64, got ", it);
  const auto there = [](const c10::optional<torch::Tensor>& t) { return t && t->defined(); };
  const auto fast = [](const torch::Tensor& t) { return t.is_cuda() && t.scalar_type() == at::kBFloat16; };
  const int64_t c = x.size(-1), k = idx.size(-1);
  if (!fast(x) || !fast(w1) || !fast(w2) || (there(b1) && !fast(*b1)) || (there(b2) && !fast(*b2)) ||
      !gates.is_cuda() || (gt != at::kFloat && gt != at::kBFloat16) || c % 8 || w1.size(2) % 8 || w2.size(2) % 8 ||
      w1.size(0) > 512 || k > 32 || is_dual(x) || is_dual(w1) || is_dual(w2) || is_dual(gates) ||
      (there(b1) && is_dual(*b1)) || (there(b2) && is_dual(*b2)))
    return c10::nullopt;
  const bool two = x.dim() == 2;
  auto shape = x.sizes().vec();
  shape.back() = w2.size(2);
  const auto flat = [two](const torch::Tensor& t, int64_t n) { return two ? t : t.reshape({-1, n}); };
  x = aligned(flat(x, c));
  idx = flat(idx, k).contiguous();
  gates = flat(gates, k).contiguous();
  w1 = aligned(w1);
  w2 = aligned(w2);
  if (there(b1)) b1 = aligned(*b1);
  if (there(b2)) b2 = aligned(*b2);
  const auto wants = [&](const c10::optional<torch::Tensor>& t) { return there(t) && t->requires_grad(); };
  torch::Tensor y;
  if (!torch::GradMode::is_enabled() || !(x.requires_grad() || w1.requires_grad() || w2.requires_grad() ||
                                          gates.requires_grad() || wants(b1) || wants(b2)))
    y = experts_fwd(x, w1, b1, w2, b2, idx, gates, false)[0];
  else
    y = ExpertsFn::apply(x, w1, b1, w2, b2, idx, gates);
  return two ? y : y.view(shape);
}

}  // namespace dtb
