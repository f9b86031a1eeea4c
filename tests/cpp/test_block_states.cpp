// What the nodes of a transformer block keep from one pass to the next: a bucket map, and the number of the pass in a
// dropout's mask.
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

// A table whose number of buckets changes between passes: the node gives what a new one gives.
static void test_table_of_another_size() {
  auto q = Random<Real>(gpu(), {16, 20, 2, 1}, 1), k = Random<Real>(gpu(), {16, 20, 2, 1}, 2), v = Random<Real>(gpu(), {16, 20, 2, 1}, 3);
  RelativeAttentionOptions opt;
  opt.max_distance = 10;
  auto table = Random<Real>(gpu(), {8, 2}, 4);
  auto o = RelativeAttention(q, k, v, table, opt);
  Graph g(o);
  g.forward().reset_grad().backward(1.);
  for (Size rows : {4, 12, 8}) {
    auto other = Random<Real>(gpu(), {rows, 2}, 4 + rows);
    table->value().resize({rows, 2});
    table->value().set(other->value().vector());
    g.reset_forwarded().forward().reset_grad().backward(1.);
    auto fresh = RelativeAttention(q, k, v, other, opt);
    Graph h(fresh);
    h.forward();
    CHECK(o->value().vector() == fresh->value().vector());
    const auto d = table->grad().vector();
    h.reset_grad().backward(1.);
    CHECK(d.size() == static_cast<size_t>(2 * rows));
    CHECK(d == other->grad().vector());
  }
}

// A captured pass: refused without a counter, whose absence would freeze the mask, and the graph runs on afterwards;
// with one, every replay draws the mask of its number, the same in both directions.
static void test_captured_dropout() {
  auto x = Random<Real>(gpu(), {40, 50}, 20), res = Random<Real>(gpu(), {40, 50}, 21);
  for (bool residual : {false, true}) {
    auto plain = residual ? DropoutAdd(x, res, 0.4f, 9) : Dropout(x, 0.4f, 9);
    Graph g(plain);
    auto bg = Autobatch(g);
    bool refused = false;
    try {
      bg.capture_pass(1.);
    } catch (const RuntimeError&) {
      refused = true;
    }
    CHECK(refused);
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusActive;
    CHECK(cudaStreamIsCapturing(stream_of(*x->dev()), &capture) == cudaSuccess && capture == cudaStreamCaptureStatusNone);
    bg.reset_forwarded().forward().reset_grad().backward(1.);
    CHECK(cudaDeviceSynchronize() == cudaSuccess);

    uint64_t* step = nullptr;
    GINN_CUDA_CALL(cudaMalloc(&step, sizeof(uint64_t)));
    GINN_CUDA_CALL(cudaMemset(step, 0, sizeof(uint64_t)));
    auto y = residual ? DropoutAdd(x, res, 0.4f, 9, step) : Dropout(x, 0.4f, 9, step);
    Graph h(y);
    auto bh = Autobatch(h);
    bh.capture_pass(1.);  // two passes: the recorded one has number 2
    std::vector<std::vector<Real>> seen;
    for (uint64_t turn = 0; turn < 3; ++turn) {
      GINN_CUDA_CALL(cudaMemcpy(step, &turn, sizeof(uint64_t), cudaMemcpyHostToDevice));
      bh.replay_pass();
      GINN_CUDA_CALL(cudaDeviceSynchronize());
      const auto dx = x->grad().vector(), xv = x->value().vector(), rv = res->value().vector(), yv = y->value().vector();
      for (size_t i = 0; i < dx.size(); ++i) CHECK(std::fabs(yv[i] - (xv[i] * dx[i] + (residual ? rv[i] : 0.f))) < 1e-6f);
      for (auto& other : seen) CHECK(dx != other);
      seen.push_back(dx);
      auto eager = Dropout(x, 0.4f, 9);  // its pass number turn + 2 has this mask
      Graph e(eager);
      for (uint64_t n = 0; n < turn + 2; ++n) e.reset_forwarded().forward();
      e.reset_grad().backward(1.);
      CHECK(x->grad().vector() == dx);
    }
    GINN_CUDA_CALL(cudaFree(step));
  }
  auto none = Dropout(x, 0.f, 9);  // nothing is drawn
  Graph g(none);
  auto bg = Autobatch(g);
  bg.capture_pass(1.).replay_pass();
  GINN_CUDA_CALL(cudaDeviceSynchronize());
  CHECK(none->value().vector() == x->value().vector());
}

static void test_one_node_as_two_weights() {
  auto x = Random<Real>(gpu(), {8, 4}, 30), w = Random<Real>(gpu(), {8}, 31);
  bool refused = false;
  try {
    LayerNorm(x, w, w);
  } catch (const RuntimeError&) {
    refused = true;
  }
  CHECK(refused);
}

int main() {
  test_table_of_another_size();
  test_one_node_as_two_weights();
  test_captured_dropout();
  cudaDeviceSynchronize();
  CHECK(ginn_b200_device_status(0, 1) == 0);
  std::printf("%d checks, %d failed\n", g_checks, g_failed);
  return g_failed == 0 ? 0 : 1;
}
