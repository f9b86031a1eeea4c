// LayerNormNode: every column normalised to mean 0 and variance 1 (ginn/node/layernorm.h), with a gain and
// a bias per row where they are given.
//   forward   y_j = gain (.) (x_j - mean) / sqrt(var + eps) + bias; mean and 1 / sqrt(var + eps) are kept
//   backward  gradients of x, gain and bias, each only if that input has_grad()
// One kernel each way, and one more for the weights' gradients.
#ifndef GINN_B200_HOST_NODE_LAYERNORM_H
#define GINN_B200_HOST_NODE_LAYERNORM_H

#include <ginn/node/data.h>
#include <ginn/prod.h>

namespace ginn {

template <typename Scalar = Real>
class LayerNormNode : public BaseDataNode<Scalar> {
  NodePtr<Scalar> in_, gain_, bias_;  // gain_ and bias_ may be null
  float eps_;
  Tensor<Real> mean_, rstd_;

  void forward_() override {
    GINN_ASSERT(this->dev()->kind() == GPU, "ginn_b200 serves GPU devices only");
    auto& x = in_->value();
    for (auto& w : {gain_, bias_})
      GINN_ASSERT(!w || w->value().size() == x.rows(), "LayerNorm expects one gain and one bias per row!");
    this->value().resize(x.shape());
    mean_.resize({x.cols()});
    rstd_.resize({x.cols()});
    internal::b200_check(ginn_b200_layer_norm_forward(
        internal::b200_device(this->dev()), stream_of(*this->dev()), internal::b200_dtype<Scalar>(), x.rows(), x.cols(),
        x.data(), x.rows(), gain_ ? gain_->value().data() : nullptr, bias_ ? bias_->value().data() : nullptr, eps_,
        this->value().data(), x.rows(), mean_.data(), rstd_.data()));
  }

  void backward_() override {
    auto& x = in_->value();
    auto grad_of = [](const NodePtr<Scalar>& n) { return n && n->has_grad() ? n->grad().data() : nullptr; };
    internal::b200_check(ginn_b200_layer_norm_backward(
        internal::b200_device(this->dev()), stream_of(*this->dev()), internal::b200_dtype<Scalar>(), x.rows(), x.cols(),
        x.data(), x.rows(), gain_ ? gain_->value().data() : nullptr, mean_.data(), rstd_.data(), this->grad().data(),
        x.rows(), grad_of(in_), x.rows(), grad_of(gain_), grad_of(bias_), 1));
  }

  static std::vector<BaseNodePtr> inputs(const NodePtr<Scalar>& in, const NodePtr<Scalar>& gain, const NodePtr<Scalar>& bias) {
    std::vector<BaseNodePtr> v{in};
    if (gain) v.push_back(gain);
    if (bias) v.push_back(bias);
    return v;
  }

 public:
  LayerNormNode(const NodePtr<Scalar>& in, const NodePtr<Scalar>& gain, const NodePtr<Scalar>& bias, float eps)
      : BaseDataNode<Scalar>(inputs(in, gain, bias)), in_(in), gain_(gain), bias_(bias), eps_(eps),
        mean_(this->value_.dev()), rstd_(this->value_.dev()) {
    // one tensor as two operands would have both gradients added to one place by one call
    GINN_ASSERT(!gain || gain != bias, "LayerNorm expects gain and bias to be different nodes!");
  }
  std::string name() const override { return "LayerNorm"; }
};

template <typename In>
auto LayerNorm(const Ptr<In>& in, float eps = 1e-5f) {
  using Scalar = typename In::Scalar;
  return make_ptr<LayerNormNode<Scalar>>(NodePtr<Scalar>(in), nullptr, nullptr, eps);
}
template <typename In, typename Gain, typename Bias>
auto LayerNorm(const Ptr<In>& in, const Ptr<Gain>& gain, const Ptr<Bias>& bias, float eps = 1e-5f) {
  using Scalar = typename In::Scalar;
  return make_ptr<LayerNormNode<Scalar>>(NodePtr<Scalar>(in), NodePtr<Scalar>(gain), NodePtr<Scalar>(bias), eps);
}

}  // namespace ginn
#endif
