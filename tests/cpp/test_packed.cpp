// CPU checks of the mixer calls' integer parts (engine-mlx_amd/csrc/packed.hpp): the piece numbers of
// a batch are distinct, a search over the sequences' first numbers finds each one's sequence, and
// every row is in one piece.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <set>
#include <vector>

#include "packed.hpp"

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

static void batch_of(const std::vector<int>& lens, int L) {
  const int B = (int)lens.size();
  std::vector<int> s(B + 1, 0);
  for (int b = 0; b < B; ++b) s[b + 1] = s[b] + lens[b];
  const int rows = s[B];
  const int64_t pieces = packed_pieces(rows, B, L);
  std::vector<int> seen(rows, 0);
  for (int64_t i = 0; i < pieces; ++i) {
    int b = 0;  // the last sequence whose first number is at most i
    for (int j = 0; j < B; ++j)
      if (packed_first_piece(s[j], j, L) <= i) b = j;
    const int64_t at = (i - packed_first_piece(s[b], b, L)) * L;
    for (int64_t r = at; r < at + L && r < lens[b]; ++r) ++seen[s[b] + r];
  }
  for (int v : seen) CHECK(v == 1);
  for (int b = 0; b + 1 < B; ++b) CHECK(packed_first_piece(s[b], b, L) < packed_first_piece(s[b + 1], b + 1, L));
}

static void uniform(int B, int T, int L) {
  const int64_t pieces = packed_pieces(B * T, B, L);
  for (int64_t i = 0; i < pieces; ++i) {
    int b = 0;
    for (int j = 0; j < B; ++j)
      if (packed_first_piece(j * T, j, L) <= i) b = j;
    CHECK(packed_uniform_sequence((int)i, T, L, B) == b);
  }
}

int main() {
  std::mt19937 rng(7);
  auto pick = [&](int n) { return (int)(rng() % n); };
  for (int L : {1, 16, 32, 64, 512, 1 << 30}) {
    batch_of({1}, L);
    batch_of({0, 0, 5, 0}, L);
    for (int k = 0; k < 60; ++k) {
      std::vector<int> lens(1 + pick(20));
      for (int& n : lens) n = pick(3) ? pick(200) : pick(3);
      batch_of(lens, L);
      uniform(1 + pick(9), pick(150), L);
    }
  }
  // starts that are no row starts stay inside the rows
  for (int s0 : {-5, 0, 7, 100, 1 << 30})
    for (int s1 : {-7, 0, 3, 7, 99, 1 << 30}) {
      const PackedRows r = packed_rows(s0, s1, 100);
      CHECK(r.begin >= 0 && r.n >= 0 && r.begin + r.n <= 100);
    }
  std::printf("%ld checks passed\n", checks);
  return 0;
}
