// LayerNorm as one autograd node: no Python between the kernels in either direction (a handful of
// rows is bound by the host: a module's forward and backward of 37 x 64 fp32 take 80 us, 96 with a
// node in Python, its forward without a graph 11.6, 17 before).
//
// Reference counterpart: torch LayerNorm's autograd (model/layer.py:219-230).
#include <torch/extension.h>

#include "plain.h"

namespace nori {

std::vector<torch::Tensor> layer_norm_fwd(const torch::Tensor& x, const c10::optional<torch::Tensor>& w,
                                          const c10::optional<torch::Tensor>& b, double eps, bool out_f32);
std::vector<torch::Tensor> layer_norm_bwd(const torch::Tensor& dy, const torch::Tensor& x, const torch::Tensor& mean,
                                          const torch::Tensor& rstd, const c10::optional<torch::Tensor>& w,
                                          bool weight_grad, bool bias_grad, c10::ScalarType grad_type);

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

// t [.., C] as [R, C] with contiguous columns (a view where the strides allow it)
Tensor rows_of(const Tensor& t) {
  if (t.dim() == 2 && t.size(1) > 0 && t.stride(1) == 1) return t;
  const Tensor r = t.size(-1) > 0 ? t.reshape({-1, t.size(-1)}) : t.reshape({0, 0});
  return r.size(1) <= 1 || r.stride(1) == 1 ? r : r.contiguous();
}
Tensor shaped(const Tensor& rows, const Tensor& like) { return like.dim() == 2 ? rows : rows.view(like.sizes()); }

// The backward in differentiable operations (for gradients of gradients).
std::vector<Tensor> backward_plain(const Tensor& dy, const Tensor& x, const Tensor& w, double eps, bool want_w,
                                   bool want_b) {
  const Tensor xf = x.to(at::kFloat), d = dy.to(at::kFloat);
  const Tensor xc = xf - xf.mean(-1, true);
  const Tensor rstd = (xc.square().mean(-1, true) + eps).rsqrt();
  const Tensor h = xc * rstd;
  const Tensor q = w.defined() ? d * w.to(at::kFloat).reshape(-1) : d;
  const Tensor dx = rstd * (q - q.mean(-1, true) - h * (q * h).mean(-1, true));
  const int64_t C = x.size(-1);
  return {dx.to(x.scalar_type()), want_w ? (d * h).reshape({-1, C}).sum(0) : Tensor(),
          want_b ? d.reshape({-1, C}).sum(0) : Tensor()};
}

struct LayerNormNode : public torch::autograd::Function<LayerNormNode> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const OptTensor& w, const OptTensor& b,
                        double eps, bool out_f32) {
    const auto r = layer_norm_fwd(rows_of(x), w, b, eps, out_f32);
    const bool has_w = w.has_value() && w->defined(), has_b = b.has_value() && b->defined();
    ctx->save_for_backward({x, r[1], r[2], has_w ? *w : Tensor()});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["bias"] = has_b;
    if (has_b) {
      ctx->saved_data["bias_type"] = static_cast<int64_t>(b->scalar_type());
      ctx->saved_data["bias_shape"] = b->sizes().vec();
    }
    return shaped(r[0], x);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 const torch::autograd::variable_list& grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[3];
    const double eps = ctx->saved_data["eps"].toDouble();
    const bool has_b = ctx->saved_data["bias"].toBool();
    // edges of the tensor arguments that are there: x, then the weight, then the bias
    const bool want_x = ctx->needs_input_grad(0), want_w = w.defined() && ctx->needs_input_grad(1);
    const bool want_b = has_b && ctx->needs_input_grad(w.defined() ? 2 : 1);
    Tensor dy = grads[0], dx, dw, db;
    const auto bias_type = has_b ? static_cast<c10::ScalarType>(ctx->saved_data["bias_type"].toInt()) : at::kFloat;
    if (torch::GradMode::is_enabled()) {  // a second derivative is wanted
      const auto r = backward_plain(dy, x, w, eps, want_w, want_b);
      dx = r[0], dw = r[1], db = r[2];
    } else {
      if (dy.scalar_type() != x.scalar_type()) dy = dy.to(at::kFloat);
      auto own = [&](bool want, c10::ScalarType t) { return !want || t == x.scalar_type(); };
      const bool typed = own(want_w, want_w ? w.scalar_type() : at::kFloat) && own(want_b, bias_type);
      const auto r = layer_norm_bwd(rows_of(dy), rows_of(x), saved[1], saved[2], w.defined() ? OptTensor(w) : OptTensor(),
                                    want_w, want_b, typed ? x.scalar_type() : at::kFloat);
      if (want_x) dx = shaped(r[0], x);
      if (want_w) dw = r[1];
      if (want_b) db = r[2];
    }
    if (want_w) dw = dw.to(w.scalar_type()).view(w.sizes());
    if (want_b) db = db.to(bias_type).view(ctx->saved_data["bias_shape"].toIntVector());
    return {dx, dw, db, Tensor(), Tensor()};
  }
};

}  // namespace

// LayerNorm of x [.., C], differentiable where a gradient is wanted; `dual` where inputs may carry
// forward-mode tangents (which the node refuses).
torch::Tensor layer_norm(const torch::Tensor& x, const c10::optional<torch::Tensor>& w,
                         const c10::optional<torch::Tensor>& b, double eps, bool out_f32, bool dual) {
  check_plain(x, "layer_norm: x");
  check_plain(w, "layer_norm: weight");
  check_plain(b, "layer_norm: bias");
  const bool grad = torch::GradMode::is_enabled() &&
                    (x.requires_grad() || (w.has_value() && w->requires_grad()) || (b.has_value() && b->requires_grad()));
  if (!grad && !dual) return shaped(layer_norm_fwd(rows_of(x), w, b, eps, out_f32)[0], x);
  return LayerNormNode::apply(x, w, b, eps, out_f32);
}

}  // namespace nori
