// CPU checks of the paged kernels' integer parts (engine-mlx_amd/csrc/paged.hpp): the split's
// slices cover every unit once, worker_of inverts them, and the partial-state slots and arrival
// counters of pieces that are alive together are distinct.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <set>
#include <vector>

#include "paged.hpp"

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

static void split_of(const std::vector<int>& segs, int plan) {
  int total = 0;
  for (int n : segs) total += n;
  if (!total) return;
  const int W = paged_active_workers(total, plan);
  CHECK(W >= 1 && W <= plan && W <= total);
  const PagedSplit s = paged_split(total, W);
  CHECK(paged_begin(s, 0) == 0 && paged_begin(s, W) == total);
  for (int w = 0; w < W; ++w) {
    CHECK(paged_begin(s, w) < paged_begin(s, w + 1));
    CHECK(paged_worker_of(s, paged_begin(s, w)) == w && paged_worker_of(s, paged_begin(s, w + 1) - 1) == w);
  }
  std::set<int> slots, counters;
  int t = 0;
  for (int n : segs) {
    if (!n) continue;
    const int w0 = paged_worker_of(s, t), w1 = paged_worker_of(s, t + n - 1);
    if (w0 != w1) {
      CHECK(counters.insert(w0).second);
      for (int w = w0; w <= w1; ++w) {
        const int slot = paged_slot(w, w0);
        CHECK(slot >= 0 && slot < 2 * plan);
        CHECK(slots.insert(slot).second);
      }
    }
    t += n;
  }
}

int main() {
  std::mt19937 rng(1);
  for (int i = 0; i < 4000; ++i) {
    std::vector<int> segs(1 + rng() % 300);
    const int top = 1 << (rng() % 12);
    for (int& n : segs) n = (int)(rng() % (unsigned)top);
    split_of(segs, 1 + (int)(rng() % kPagedMaxWorkers));
  }
  for (int n = 1; n < 3000; n += 7) split_of({n}, kPagedMaxWorkers);
  {  // the largest totals: no overflow in 32 bits
    const int total = 2147483646;
    for (int W : {1, 2, 511, 512}) {
      const PagedSplit s = paged_split(total, W);
      CHECK(paged_begin(s, W) == total && paged_begin(s, W - 1) < total);
      CHECK(paged_worker_of(s, total - 1) == W - 1 && paged_worker_of(s, 0) == 0);
      for (int w = 1; w < W; ++w) CHECK(paged_worker_of(s, paged_begin(s, w)) == w && paged_worker_of(s, paged_begin(s, w) - 1) == w - 1);
    }
  }
  for (int s0 : {-5, 0, 3, 10, 99}) for (int s1 : {-7, 0, 2, 10, 11, 99}) {
    const PagedRows r = paged_rows(s0, s1, 10);
    CHECK(r.begin >= 0 && r.n >= 0 && r.begin + r.n <= 10);
  }
  CHECK(paged_rows(3, 7, 10).begin == 3 && paged_rows(3, 7, 10).n == 4);
  for (int i = 0; i < 4000; ++i) {  // the bound of the row blocks holds for any batch
    const int B = 1 + rng() % 50, G = 1 + rng() % 16;
    int64_t rows = 0, most = 0, blocks = 0;
    for (int b = 0; b < B; ++b) {
      const int n = rng() % 40;
      rows += n;
      most = n > most ? n : most;
      blocks += ((int64_t)n * G + kPagedRows - 1) / kPagedRows;
    }
    CHECK(blocks <= paged_row_blocks(B, rows, most, G));
  }
  for (int G = 1; G <= kPagedMaxGroup; ++G) {  // the product for r / G
    const uint32_t m = paged_magic(G);
    for (int i = 0; i < 3000; ++i) {
      const int r = (int)(rng() & ((1u << 23) - 1));
      CHECK(paged_div(r, m) == r / G);
      CHECK(paged_div(r / G * G, m) == r / G && (r < G || paged_div(r / G * G - 1, m) == r / G - 1));
    }
    CHECK(paged_div((1 << 23) - 1, m) == ((1 << 23) - 1) / G && paged_div(0, m) == 0);
  }
  for (int64_t rows : {0, 1, 33, 128, 129, 5000}) for (int n : {1, 63, 64, 65, 8001, 32768, 2000000000}) for (int hkv : {1, 8, 40}) {
    const PagedChunks c = paged_chunks(rows, hkv, n, 256);  // the chunks cover the prefix, none empty
    CHECK(c.n >= 1 && c.blocks >= 1 && (int64_t)c.n * c.blocks * 64 >= n && ((int64_t)c.n - 1) * c.blocks * 64 < n);
  }
  std::printf("%ld checks passed\n", checks);
}
