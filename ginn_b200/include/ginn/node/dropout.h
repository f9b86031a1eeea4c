// DropoutNode: elements are zeroed with probability p and the others scaled by 1 / (1 - p) (the Dropout node of
// ginn/node/common.h), with a residual added in the same pass where one is given.  No mask is stored: it is a
// function of the node's seed, the number of the forward pass and the element, which the backward pass forms
// again.  Every forward pass of a node draws a new mask.  A pass that is captured into a CUDA graph is recorded with one
// number, so there the node needs `step`, a counter on the device which is added to it and which whoever replays
// the graph advances; without it the capture is refused.
#ifndef GINN_B200_HOST_NODE_DROPOUT_H
#define GINN_B200_HOST_NODE_DROPOUT_H

#include <atomic>

#include <ginn/node/data.h>
#include <ginn/prod.h>

namespace ginn {

namespace internal {
// Seeds of nodes that are not given one: different for every node of a process.
inline uint64_t next_dropout_seed() {
  static std::atomic<uint64_t> next{0x9E3779B97F4A7C15ull};
  return next.fetch_add(1);
}
}  // namespace internal

template <typename Scalar = Real>
class DropoutNode : public BaseDataNode<Scalar> {
  NodePtr<Scalar> in_, residual_;  // residual_ may be null
  ginn_b200_dropout drop_;

  void forward_() override {
    GINN_ASSERT(this->dev()->kind() == GPU, "ginn_b200 serves GPU devices only");
    auto& x = in_->value();
    GINN_ASSERT(!residual_ || residual_->value().size() == x.size(), "Dropout expects a residual of its input's size!");
    this->value().resize(x.shape());
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    GINN_CUDA_CALL(cudaStreamIsCapturing(stream_of(*this->dev()), &capture));
    GINN_ASSERT(capture == cudaStreamCaptureStatusNone || drop_.step != nullptr || drop_.p == 0.f,
                "Dropout needs a step counter in a captured pass: every replay would draw the same mask!");
    ++drop_.offset;
    internal::b200_check(ginn_b200_dropout_forward(
        internal::b200_device(this->dev()), stream_of(*this->dev()), internal::b200_dtype<Scalar>(), x.rows(), x.cols(),
        x.data(), x.rows(), residual_ ? residual_->value().data() : nullptr, x.rows(), &drop_, this->value().data(), x.rows()));
  }

  void backward_() override {
    const Size rows = this->value().rows(), cols = this->value().cols();
    auto add = [&](const NodePtr<Scalar>& to, const ginn_b200_dropout& d) {
      if (!to || !to->has_grad()) return;
      internal::b200_check(ginn_b200_dropout_backward(internal::b200_device(this->dev()), stream_of(*this->dev()),
                                                      internal::b200_dtype<Scalar>(), rows, cols, this->grad().data(), rows, &d,
                                                      to->grad().data(), rows, 1));
    };
    add(in_, drop_);
    ginn_b200_dropout all = drop_;
    all.p = 0.f;  // the residual's gradient passes whole
    add(residual_, all);
  }

  static std::vector<BaseNodePtr> inputs(const NodePtr<Scalar>& in, const NodePtr<Scalar>& residual) {
    std::vector<BaseNodePtr> v{in};
    if (residual) v.push_back(residual);
    return v;
  }

 public:
  DropoutNode(const NodePtr<Scalar>& in, const NodePtr<Scalar>& residual, float p, uint64_t seed, const uint64_t* step)
      : BaseDataNode<Scalar>(inputs(in, residual)), in_(in), residual_(residual), drop_{p, seed, 0, step} {}
  std::string name() const override { return "Dropout"; }
};

template <typename In>
auto Dropout(const Ptr<In>& in, float p, uint64_t seed = internal::next_dropout_seed(), const uint64_t* step = nullptr) {
  using Scalar = typename In::Scalar;
  return make_ptr<DropoutNode<Scalar>>(NodePtr<Scalar>(in), nullptr, p, seed, step);
}
// residual + dropout(in)
template <typename In, typename Res>
auto DropoutAdd(const Ptr<In>& in, const Ptr<Res>& residual, float p, uint64_t seed = internal::next_dropout_seed(),
                const uint64_t* step = nullptr) {
  using Scalar = typename In::Scalar;
  return make_ptr<DropoutNode<Scalar>>(NodePtr<Scalar>(in), NodePtr<Scalar>(residual), p, seed, step);
}

}  // namespace ginn
#endif
