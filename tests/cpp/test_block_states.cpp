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

int main() {
  test_table_of_another_size();
  cudaDeviceSynchronize();
  CHECK(ginn_b200_device_status(0, 1) == 0);
  std::printf("%d checks, %d failed\n", g_checks, g_failed);
  return g_failed == 0 ? 0 : 1;
}
