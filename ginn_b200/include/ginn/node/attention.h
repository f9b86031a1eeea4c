// RelativeAttentionNode: attention whose scores get a learned bias by the distance of key and query.
//   q       (head size, queries, heads, sequences)       k, v  (head size, keys, kv heads, sequences)
//   table   (buckets, heads), a column per head; may be null: no bias
//   value   like q
// The distances' buckets are those of ginn_b200_relative_buckets; the scores are never stored, the statistics
// of the softmax are kept for the backward pass.
#ifndef GINN_B200_HOST_NODE_ATTENTION_H
#define GINN_B200_HOST_NODE_ATTENTION_H

#include <cmath>

#include <ginn/node/data.h>
#include <ginn/prod.h>

namespace ginn {

struct RelativeAttentionOptions {
  float scale = 0;              // 0: 1 / sqrt(head size)
  bool causal = false;          // then buckets look backwards only
  int max_distance = 128;       // distances from here on share a bucket
  Size offset = 0;              // position of the first query among the keys
};

template <typename Scalar = Real>
class RelativeAttentionNode : public BaseDataNode<Scalar> {
  NodePtr<Scalar> q_, k_, v_, table_;
  RelativeAttentionOptions opt_;
  Tensor<Real> lse_;
  Tensor<Int> map_;
  Size mapped_ = 0;  // rows of the table that map_ was made for

  ginn_b200_relative_attention describe() {
    const Shape q = Tensor<Scalar>::reduce(q_->shape(), 4), k = Tensor<Scalar>::reduce(k_->shape(), 4);
    GINN_ASSERT(Tensor<Scalar>::reduce(v_->shape(), 4) == k, "RelativeAttention expects keys and values of one shape!");
    GINN_ASSERT(q[0] == k[0] && q[3] == k[3], "Mismatching head sizes or sequences in RelativeAttention!");
    GINN_ASSERT(!table_ || table_->value().cols() == q[2], "RelativeAttention expects a table column per head!");
    ginn_b200_relative_attention a = {};
    a.tq = q[1]; a.tk = k[1]; a.head_size = q[0]; a.heads = q[2]; a.kv_heads = k[2]; a.batch = q[3];
    a.q = q_->value().data(); a.ldq = q[0]; a.stride_q_head = q[0] * q[1]; a.stride_q_batch = q[0] * q[1] * q[2];
    a.k = k_->value().data(); a.ldk = k[0]; a.stride_k_head = k[0] * k[1]; a.stride_k_batch = k[0] * k[1] * k[2];
    a.v = v_->value().data(); a.ldv = a.ldk; a.stride_v_head = a.stride_k_head; a.stride_v_batch = a.stride_k_batch;
    a.o = this->value().data(); a.ldo = a.ldq; a.stride_o_head = a.stride_q_head; a.stride_o_batch = a.stride_q_batch;
    a.scale = opt_.scale != 0 ? opt_.scale : 1.f / std::sqrt(static_cast<float>(q[0]));
    a.causal = opt_.causal;
    a.q_offset = opt_.offset;
    a.lse = lse_.data();
    if (table_) {
      a.table = table_->value().data(); a.ldt = a.buckets = table_->value().rows();
      a.reach = opt_.max_distance;
      a.map = map_.data();
    }
    return a;
  }

  void forward_() override {
    GINN_ASSERT(this->dev()->kind() == GPU, "ginn_b200 serves GPU devices only");
    this->value().resize(q_->shape());
    lse_.resize({this->value().size() / this->value().rows()});
    if (table_ && mapped_ != table_->value().rows()) {
      std::vector<Int> map(2 * opt_.max_distance + 1);
      internal::b200_check(ginn_b200_relative_buckets(static_cast<int>(table_->value().rows()), opt_.max_distance,
                                                      !opt_.causal, opt_.max_distance, map.data()));
      map_.resize({static_cast<Size>(map.size())});
      map_.set(map);
      mapped_ = table_->value().rows();
    }
    const ginn_b200_relative_attention a = describe();
    internal::b200_check(ginn_b200_relative_attention_forward(internal::b200_device(this->dev()), stream_of(*this->dev()),
                                                              internal::b200_dtype<Scalar>(), &a));
  }

  void backward_() override {
    const ginn_b200_relative_attention a = describe();
    auto grad_of = [](const NodePtr<Scalar>& n) { return n && n->has_grad() ? n->grad().data() : nullptr; };
    ginn_b200_relative_attention_grad g = {};
    g.d_o = this->grad().data(); g.lddo = a.ldo; g.stride_do_head = a.stride_o_head; g.stride_do_batch = a.stride_o_batch;
    g.dq = grad_of(q_); g.lddq = a.ldq; g.stride_dq_head = a.stride_q_head; g.stride_dq_batch = a.stride_q_batch;
    g.dk = grad_of(k_); g.lddk = a.ldk; g.stride_dk_head = a.stride_k_head; g.stride_dk_batch = a.stride_k_batch;
    g.dv = grad_of(v_); g.lddv = a.ldv; g.stride_dv_head = a.stride_v_head; g.stride_dv_batch = a.stride_v_batch;
    g.dtable = grad_of(table_); g.lddt = a.ldt;
    g.accumulate = 1;
    internal::b200_check(ginn_b200_relative_attention_backward(internal::b200_device(this->dev()), stream_of(*this->dev()),
                                                               internal::b200_dtype<Scalar>(), &a, &g));
  }

  static std::vector<BaseNodePtr> inputs(const NodePtr<Scalar>& q, const NodePtr<Scalar>& k, const NodePtr<Scalar>& v,
                                         const NodePtr<Scalar>& table) {
    std::vector<BaseNodePtr> in{q, k, v};
    if (table) in.push_back(table);
    return in;
  }

 public:
  RelativeAttentionNode(const NodePtr<Scalar>& q, const NodePtr<Scalar>& k, const NodePtr<Scalar>& v,
                        const NodePtr<Scalar>& table, const RelativeAttentionOptions& opt)
      : BaseDataNode<Scalar>(inputs(q, k, v, table)), q_(q), k_(k), v_(v), table_(table), opt_(opt),
        lse_(this->value_.dev()), map_(this->value_.dev()) {
    // one tensor as two operands would have both gradients added to one place by one call
    GINN_ASSERT(q != k && q != v && k != v, "RelativeAttention expects q, k and v to be different nodes!");
  }
  std::string name() const override { return "RelativeAttention"; }
};

template <typename Q, typename K, typename V>
auto RelativeAttention(const Ptr<Q>& q, const Ptr<K>& k, const Ptr<V>& v, const RelativeAttentionOptions& opt = {}) {
  using Scalar = typename Q::Scalar;
  return make_ptr<RelativeAttentionNode<Scalar>>(NodePtr<Scalar>(q), NodePtr<Scalar>(k), NodePtr<Scalar>(v), nullptr, opt);
}
template <typename Q, typename K, typename V, typename T>
auto RelativeAttention(const Ptr<Q>& q, const Ptr<K>& k, const Ptr<V>& v, const Ptr<T>& table,
                       const RelativeAttentionOptions& opt = {}) {
  using Scalar = typename Q::Scalar;
  return make_ptr<RelativeAttentionNode<Scalar>>(NodePtr<Scalar>(q), NodePtr<Scalar>(k), NodePtr<Scalar>(v),
                                                 NodePtr<Scalar>(table), opt);
}

}  // namespace ginn
#endif
