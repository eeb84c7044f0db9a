// Autograd node of the query / key norm + rotation.
//
// The same forward and backward as a Python function of two operator calls, without the interpreter between them.  A forward
// and backward of 8 tokens takes 126 us of host time through the Python function and 103 us through this node (55 us of it
// for any operator and its gradient), more than the kernels of a short sequence (17 us for 1023 tokens, 16 + 8 heads of
// 64).  Weights with a `main_grad` (the sharded engine's) take the Python function.  Only the projection output is kept;
// the backward recomputes each head's rsqrt from it.
#include <torch/csrc/autograd/custom_function.h>

#include <ATen/ATen.h>

namespace tb200 {

using OptTensor = c10::optional<at::Tensor>;

std::tuple<at::Tensor, at::Tensor> qk_norm_rope_fwd(const at::Tensor& x, int64_t hq, int64_t hkv, const OptTensor& qw, const OptTensor& kw,
                                                    const OptTensor& table, const OptTensor& positions, const OptTensor& axes,
                                                    bool interleaved, double eps, double gain, double q_scale);
std::tuple<at::Tensor, at::Tensor> qk_norm_rope_bwd(const at::Tensor& dq, const at::Tensor& dk, const OptTensor& dv, const at::Tensor& x,
                                                    int64_t hq, int64_t hkv, const OptTensor& qw, const OptTensor& kw,
                                                    const OptTensor& table, const OptTensor& positions, const OptTensor& axes,
                                                    bool interleaved, double eps, double gain, double q_scale, bool fp32_dw);

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct QKNormRope : public torch::autograd::Function<QKNormRope> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const OptTensor& qw, const OptTensor& kw, const OptTensor& table,
                               const OptTensor& positions, const OptTensor& axes, int64_t hq, int64_t hkv, bool interleaved,
                               double eps, double gain, double q_scale) {
    auto [q, k] = qk_norm_rope_fwd(x, hq, hkv, qw, kw, table, positions, axes, interleaved, eps, gain, q_scale);
    auto tensor = [](const OptTensor& t) { return t.has_value() ? *t : at::Tensor(); };
    ctx->save_for_backward({x, tensor(qw), tensor(kw), tensor(table), tensor(positions), tensor(axes)});
    ctx->saved_data["heads"] = std::vector<int64_t>{hq, hkv, interleaved};
    ctx->saved_data["scales"] = std::vector<double>{eps, gain, q_scale};
    ctx->set_materialize_grads(false);
    return {q, k, x.slice(1, hq + hkv)};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    auto optional = [](const at::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    const at::Tensor& x = saved[0];
    const auto heads = ctx->saved_data["heads"].toIntVector();
    const auto scales = ctx->saved_data["scales"].toDoubleVector();
    auto given = [&](const at::Tensor& g, int64_t n) { return g.defined() ? g : at::zeros({x.size(0), n, x.size(2)}, x.options()); };
    auto [dx, dw] = qk_norm_rope_bwd(given(grads[0], heads[0]), given(grads[1], heads[1]), optional(grads[2]), x, heads[0], heads[1],
                                     optional(saved[1]), optional(saved[2]), optional(saved[3]), optional(saved[4]), optional(saved[5]),
                                     heads[2] != 0, scales[0], scales[1], scales[2], false);
    variable_list out(12);
    out[0] = dx;
    if (saved[1].defined()) out[1] = dw.select(0, 0);
    if (saved[2].defined()) out[2] = dw.select(0, 1);
    return out;
  }
};

}  // namespace

// (q, k, v) of the projection output, v a view of it; gradients for it and for the weights, in their own types.
std::tuple<at::Tensor, at::Tensor, at::Tensor> qk_norm_rope(const at::Tensor& x, int64_t hq, int64_t hkv, const OptTensor& qw,
                                                            const OptTensor& kw, const OptTensor& table, const OptTensor& positions,
                                                            const OptTensor& axes, bool interleaved, double eps, double gain, double q_scale) {
  auto o = QKNormRope::apply(x, qw, kw, table, positions, axes, hq, hkv, interleaved, eps, gain, q_scale);
  return {o[0], o[1], o[2]};
}

}  // namespace tb200
