// CPU checks of where the state space scan keeps what the pieces of a cut sequence hand on to each other
// (engine-mlx_amd/csrc/packed.hpp), and that a workspace of the size that is told for some bounds is as
// good as any for every call within them (engine-mlx_amd/csrc/ssm_plan.hpp).
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "packed.hpp"
#include "ssm_plan.hpp"

using namespace ema;

static long checks = 0;
#define CHECK(c)                                                        \
  do {                                                                  \
    ++checks;                                                           \
    if (!(c)) {                                                         \
      std::printf("failed: %s (line %d)\n", #c, __LINE__);              \
      std::exit(1);                                                     \
    }                                                                   \
  } while (0)

// The places of the sequences of more than one piece: each its own, all below packed_places.
static void places(const std::vector<int>& lens, int tail, int L) {
  const int B = (int)lens.size();
  int rows = tail;
  for (int n : lens) rows += n;
  const int64_t all = packed_places(rows, B, L);
  int s = 0;
  int64_t free = 0;
  for (int b = 0; b < B; s += lens[b++]) {
    const int first = packed_first_place(s, b, L), n = (lens[b] + L - 1) / L;
    if (lens[b] <= L) continue;
    CHECK(first >= free);
    free = first + n;
    CHECK(free <= all);
  }
}

static int log_pick(std::mt19937& rng, int most) {  // 1 .. most, over its logarithm
  return (int)std::exp(std::uniform_real_distribution<double>(0, std::log(most + 0.99))(rng));
}

static void within_bounds(std::mt19937& rng) {
  const int G = 1 << (rng() % 4), heads = G * log_pick(rng, 24), P = rng() % 3 ? 32 * (1 + (int)(rng() % 5)) : log_pick(rng, 200);
  const int N = rng() % 3 ? 64 << (rng() % 3) : 4 * (1 + (int)(rng() % 64)), cus = rng() % 4 ? 256 : 32;
  const int batch = log_pick(rng, 4096), rows = log_pick(rng, 1 << 30), longest = log_pick(rng, rows);
  const bool bf16 = rng() % 2;
  const uint64_t told = ssm_workspace_bytes(batch, rows, longest, heads, P, N, G, bf16, cus);
  for (int k = 0; k < 60; ++k) {
    const int b = rng() % 3 ? log_pick(rng, batch) : batch, n = rng() % 3 ? log_pick(rng, rows) : rows;
    int most = rng() % 3 ? log_pick(rng, longest) : longest;
    if (most > n) most = n;
    for (int vectors = 0; vectors <= (bf16 ? 1 : 0); ++vectors) {
      const SsmPlan best = plan_ssm(b, n, most, heads, P, N, G, vectors, cus, UINT64_MAX);
      const SsmPlan p = plan_ssm(b, n, most, heads, P, N, G, vectors, cus, told);
      CHECK(best.bytes <= told);
      CHECK(p.piece == best.piece && p.chunks == best.chunks && p.bytes == best.bytes);
    }
  }
}

int main() {
  std::mt19937 rng(11);
  auto pick = [&](int n) { return (int)(rng() % n); };
  for (int L : {1, 2, 16, 32, 128, 512}) {
    places({1}, 0, L);
    places({L + 1}, 0, L);
    places({0, L + 1, L, L + 1, 2 * L, 2 * L + 1, 0}, 0, L);
    for (int k = 0; k < 400; ++k) {
      std::vector<int> lens(1 + pick(30));
      for (int& n : lens) {
        const int kind = pick(4);
        n = kind == 0 ? pick(3) : kind == 1 ? L + pick(2) : kind == 2 ? pick(6 * L) : (1 + pick(4)) * L + pick(3) - 1;
        if (n < 0) n = 0;
      }
      places(lens, pick(2) * pick(3 * L), L);
    }
    // row starts that are none, taken inside the rows
    for (int k = 0; k < 2000; ++k) {
      const int rows = 1 + pick(10 * L), B = 1 + pick(8), b = pick(B);
      const PackedRows r = packed_rows(pick(14 * L) - 2 * L, pick(14 * L) - 2 * L, rows);
      if (r.n > L) CHECK(packed_first_place(r.begin, b, L) + (r.n + L - 1) / L <= packed_places(rows, B, L));
    }
  }
  for (int k = 0; k < 20000; ++k) within_bounds(rng);
  std::printf("%ld checks passed\n", checks);
  return 0;
}
