// The nodes of a transformer block (layer norm, dropout with a residual, attention with a relative position
// bias) on a GPU, one by one and as a graph, against their formulas in double precision on the host.
#include <cmath>
#include <cstdio>

#include <ginn/ginn.h>

using namespace ginn;

static int g_failed = 0, g_checks = 0;
#define CHECK(cond)                                                          \
  do {                                                                       \
    ++g_checks;                                                              \
    if (!(cond)) {                                                           \
      ++g_failed;                                                            \
      std::printf("FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond);          \
    }                                                                        \
  } while (0)

using Vec = std::vector<double>;
static double f(float x) { return x; }
static double f(Half x) { return __half2float(x); }
template <typename S>
static Vec values(Tensor<S>& t) {
  Vec out;
  for (auto x : t.vector()) out.push_back(f(x));
  return out;
}
// Largest difference relative to the largest magnitude of what is expected.
static double off(const Vec& got, const Vec& want) {
  if (got.size() != want.size()) return INFINITY;
  double most = 0, worst = 0;
  for (double x : want) most = std::max(most, std::fabs(x));
  for (size_t i = 0; i < got.size(); ++i) {
    const double d = std::fabs(got[i] - want[i]);
    worst = d <= worst ? worst : d;  // not a number: the worst
  }
  return worst / std::max(most, 1e-30);
}

struct NormResult {
  Vec y, dx, dgain, dbias;
};
static NormResult norm(const Vec& x, const Vec& gain, const Vec& bias, const Vec& dy, size_t rows, double eps) {
  NormResult r{Vec(x.size()), Vec(x.size()), Vec(rows), Vec(rows)};
  for (size_t c = 0; c < x.size() / rows; ++c) {
    const double* xc = &x[c * rows];
    double mean = 0, var = 0, s0 = 0, s1 = 0;
    for (size_t i = 0; i < rows; ++i) mean += xc[i] / rows;
    for (size_t i = 0; i < rows; ++i) var += (xc[i] - mean) * (xc[i] - mean) / rows;
    const double rstd = 1 / std::sqrt(var + eps);
    for (size_t i = 0; i < rows; ++i) {
      const double xh = (xc[i] - mean) * rstd, g = gain[i] * dy[c * rows + i];
      r.y[c * rows + i] = xh * gain[i] + bias[i];
      r.dgain[i] += dy[c * rows + i] * xh;
      r.dbias[i] += dy[c * rows + i];
      s0 += g / rows;
      s1 += g * xh / rows;
    }
    for (size_t i = 0; i < rows; ++i) {
      const double xh = (xc[i] - mean) * rstd, g = gain[i] * dy[c * rows + i];
      r.dx[c * rows + i] = rstd * (g - s0 - xh * s1);
    }
  }
  return r;
}

template <typename S>
static void test_layer_norm(double eps) {
  const size_t rows = 72, cols = 9;
  auto x = Random<S>(gpu(), {72, 3, 3}, 1), gain = Random<S>(gpu(), {72}, 2), bias = Random<S>(gpu(), {72}, 3);
  auto y = LayerNorm(x, gain, bias);
  Graph g(y);
  g.forward();
  CHECK((y->shape() == Shape{72, 3, 3}));
  g.reset_grad().backward(0.5);
  auto ref = norm(values(x->value()), values(gain->value()), values(bias->value()), Vec(rows * cols, 0.5), rows, 1e-5);
  CHECK(off(values(y->value()), ref.y) < eps);
  CHECK(off(values(x->grad()), ref.dx) < eps);
  CHECK(off(values(gain->grad()), ref.dgain) < eps);
  CHECK(off(values(bias->grad()), ref.dbias) < eps);
  // without weights; the input's gradient adds up
  auto z = LayerNorm(x);
  Graph h(z);
  h.forward().init_grad();
  z->reset_grad();
  h.backward(0.5);
  auto bare = norm(values(x->value()), Vec(rows, 1.), Vec(rows, 0.), Vec(rows * cols, 0.5), rows, 1e-5);
  for (size_t i = 0; i < bare.dx.size(); ++i) bare.dx[i] += ref.dx[i];
  CHECK(off(values(z->value()), bare.y) < eps);
  CHECK(off(values(x->grad()), bare.dx) < eps);
}

template <typename S>
static void test_dropout(double eps) {
  const double p = 0.25;
  auto x = Random<S>(gpu(), {40, 100}, 4), res = Random<S>(gpu(), {40, 100}, 5);
  auto y = DropoutAdd(x, res, 0.25f, 7);
  Graph g(y);
  g.forward().reset_grad().backward(1.);
  const Vec xv = values(x->value()), rv = values(res->value()), yv = values(y->value()), dx = values(x->grad());
  Vec want(xv.size());
  int kept = 0;
  for (size_t i = 0; i < xv.size(); ++i) {
    want[i] = rv[i] + xv[i] * dx[i];  // the gradient is the mask
    CHECK(dx[i] == 0 || std::fabs(dx[i] - 1 / (1 - p)) < eps);
    kept += dx[i] != 0;
  }
  CHECK(off(yv, want) < eps);
  CHECK(off(values(res->grad()), Vec(xv.size(), 1.)) == 0);
  CHECK(std::fabs(kept / 4000. - (1 - p)) < 5 * std::sqrt(p * (1 - p) / 4000));  // five standard deviations
  // the next pass draws another mask; a node of another seed as well; the same seed the same one
  g.reset_forwarded().forward().reset_grad().backward(1.);
  CHECK(values(x->grad()) != dx);
  auto same = DropoutAdd(x, res, 0.25f, 7);
  Graph(same).forward();
  CHECK(values(same->value()) == yv);
  auto a = Dropout(x, 0.25f), b = Dropout(x, 0.25f);
  Graph(a).forward();
  Graph(b).forward();
  CHECK(values(a->value()) != values(b->value()));
}

template <typename S>
static void test_attention(double eps, bool causal) {
  const size_t hs = 24, tq = 10, tk = 13, heads = 4, kv = 2, batch = 2, buckets = 8, off0 = 3;
  auto q = Random<S>(gpu(), {24, 10, 4, 2}, 8), k = Random<S>(gpu(), {24, 13, 2, 2}, 9), v = Random<S>(gpu(), {24, 13, 2, 2}, 10);
  auto table = Random<S>(gpu(), {8, 4}, 11);
  RelativeAttentionOptions opt;
  opt.causal = causal;
  opt.max_distance = 6;
  opt.offset = off0;
  opt.scale = 0.4f;
  auto o = RelativeAttention(q, k, v, table, opt);
  Graph g(o);
  g.forward().reset_grad().backward(1.);
  std::vector<int> map(13);
  CHECK(ginn_b200_relative_buckets(buckets, 6, !causal, 6, map.data()) == GINN_B200_OK);
  const Vec Q = values(q->value()), K = values(k->value()), V = values(v->value()), T = values(table->value());
  Vec O(Q.size()), dQ(Q.size()), dK(K.size()), dV(V.size()), dT(T.size());
  for (size_t b = 0; b < batch; ++b)
    for (size_t h = 0; h < heads; ++h) {
      const size_t n = h * kv / heads;
      for (size_t i = 0; i < tq; ++i) {
        const size_t qi = hs * (i + tq * (h + heads * b));
        auto at = [&](size_t j) { return hs * (j + tk * (n + kv * b)); };
        Vec p(tk), dp(tk);
        std::vector<int> bucket(tk);
        double sum = 0, delta = 0;
        const size_t seen = causal ? std::min(tk, i + off0 + 1) : tk;
        for (size_t j = 0; j < seen; ++j) {
          const int d = static_cast<int>(j) - static_cast<int>(i + off0);
          bucket[j] = map[6 + std::max(-6, std::min(6, d))];
          double s = 0;
          for (size_t e = 0; e < hs; ++e) s += Q[qi + e] * K[at(j) + e];
          sum += p[j] = std::exp(static_cast<double>(opt.scale) * s + T[bucket[j] + buckets * h]);
        }
        for (size_t j = 0; j < seen; ++j) {
          p[j] /= sum;
          for (size_t e = 0; e < hs; ++e) {
            O[qi + e] += p[j] * V[at(j) + e];
            dV[at(j) + e] += p[j];
            dp[j] += V[at(j) + e];
          }
          delta += p[j] * dp[j];
        }
        for (size_t j = 0; j < seen; ++j) {
          const double ds = p[j] * (dp[j] - delta);
          dT[bucket[j] + buckets * h] += ds;
          for (size_t e = 0; e < hs; ++e) {
            dQ[qi + e] += opt.scale * ds * K[at(j) + e];
            dK[at(j) + e] += opt.scale * ds * Q[qi + e];
          }
        }
      }
    }
  CHECK(off(values(o->value()), O) < eps);
  CHECK(off(values(q->grad()), dQ) < eps);
  CHECK(off(values(k->grad()), dK) < eps);
  CHECK(off(values(v->grad()), dV) < eps);
  CHECK(off(values(table->grad()), dT) < eps);
}

// norm -> attention -> dropout with the residual -> norm, as one graph: its directional derivative along its
// own gradient is the gradient's squared norm.
static void test_graph() {
  auto x = Random<Real>(gpu(), {32, 12, 2, 2}, 12), k = Random<Real>(gpu(), {32, 12, 2, 2}, 13), v = Random<Real>(gpu(), {32, 12, 2, 2}, 14);
  auto gain = Random<Real>(gpu(), {32}, 15), bias = Random<Real>(gpu(), {32}, 16), table = Random<Real>(gpu(), {8, 2}, 17);
  auto w = Random<Real>(gpu(), {1, 32}, 18);
  auto build = [&](const DataPtr<Real>& in) {
    auto a = RelativeAttention(LayerNorm(in, gain, bias), k, v, table, RelativeAttentionOptions{0, true, 5, 0});
    return w * LayerNorm(DropoutAdd(a, in, 0.3f, 21), gain, bias);
  };
  auto loss = build(x);
  Graph g(loss);
  g.forward().reset_grad().backward(1.);
  const Vec grad = values(x->grad());
  double square = 0;
  for (double d : grad) square += d * d;
  CHECK(square > 1e-3);
  const double step = 1e-2 / std::sqrt(square);
  const auto x0 = x->value().vector();
  double side[2] = {0, 0}, moved = 0;
  for (int s = 0; s < 2; ++s) {
    auto xs = x0;
    for (size_t i = 0; i < xs.size(); ++i) xs[i] += static_cast<float>((s ? -1 : 1) * step * grad[i]);
    for (size_t i = 0; i < xs.size(); ++i) moved += (s ? -1 : 1) * (static_cast<double>(xs[i]) - x0[i]) * grad[i];
    auto y = Data<Real>(gpu(), {32, 12, 2, 2});
    y->value().set(xs);
    auto l = build(y);  // the same seed: the same mask
    Graph(l).forward();
    for (double d : values(l->value())) side[s] += d;
  }
  // central difference: truncation ~ step^2 (1e-4 of the derivative's own scale), rounding of 48 sums of
  // 32 products each ~ 1e-5 against a difference of 2e-2 |gradient|
  CHECK(std::fabs((side[0] - side[1]) / moved - 1) < 5e-3);
}

static void test_errors() {
  auto x = Random<Real>(gpu(), {8, 4}, 30), short_gain = Random<Real>(gpu(), {7}, 31);
  auto throws = [](auto make) {
    try {
      make();
    } catch (const RuntimeError&) {
      return true;
    }
    return false;
  };
  CHECK(throws([&] { Graph(LayerNorm(x, short_gain, short_gain)).forward(); }));
  CHECK(throws([&] { Graph(Dropout(x, 1.5f)).forward(); }));
  CHECK(throws([&] { Graph(DropoutAdd(x, short_gain, 0.5f)).forward(); }));
  auto q = Random<Real>(gpu(), {8, 4, 3, 1}, 32), k = Random<Real>(gpu(), {8, 5, 2, 1}, 33), v = Random<Real>(gpu(), {8, 5, 2, 1}, 34);
  CHECK(throws([&] { Graph(RelativeAttention(q, k, v)).forward(); }));  // 3 heads cannot share 2
  CHECK(throws([&] { RelativeAttention(q, k, k); }));
  auto c = Random<Real>(cpu(), {8, 4}, 35);
  CHECK(throws([&] { Graph(LayerNorm(c)).forward(); }));
}

int main() {
  test_layer_norm<Real>(1e-5);
  test_layer_norm<Half>(3e-3);
  test_dropout<Real>(1e-6);
  test_dropout<Half>(2e-3);
  for (bool causal : {false, true}) {
    test_attention<Real>(1e-5, causal);
    test_attention<Half>(5e-3, causal);
  }
  test_graph();
  test_errors();
  cudaDeviceSynchronize();
  CHECK(ginn_b200_device_status(0, 1) == 0);
  std::printf("%d checks, %d failed\n", g_checks, g_failed);
  return g_failed == 0 ? 0 : 1;
}
