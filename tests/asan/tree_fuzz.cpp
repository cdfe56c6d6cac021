// Fuzz driver of the drafted-tree planner for a sanitizer build (AddressSanitizer and
// UndefinedBehaviorSanitizer, g++ on the host): random trees through hy_tree_lines, and
// their requests, up to the longest caches, through hy_plan_tree with buffers of the
// documented capacity, of exactly the counts it reported, and one record short of each
// (HY_ENOSPACE). Guard words behind every buffer must stay untouched.
// Usage: tree_fuzz <seed> <ticks>; prints "ok <ticks>" and exits 0.
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>

#include <algorithm>
#include <random>
#include <vector>

#include "../../include/hayate_attn.h"

namespace hy {
void set_error(const char *, ...) {}
void clear_error() {}
}  // namespace hy

namespace {

constexpr int32_t kPoison = 0x5a5a5a5a;
constexpr size_t kMargin = 64;

#define CHECK(cond)                                                               \
  do {                                                                            \
    if (!(cond)) {                                                                \
      fprintf(stderr, "check failed (%s:%d): %s\n", __FILE__, __LINE__, #cond);   \
      exit(1);                                                                    \
    }                                                                             \
  } while (0)

template <typename T>
struct Guarded {
  std::vector<T> v;
  size_t used;
  explicit Guarded(size_t n) : v(n + kMargin, static_cast<T>(kPoison)), used(n) {}
  ~Guarded() {
    for (size_t i = used; i < v.size(); ++i) CHECK(v[i] == static_cast<T>(kPoison));
  }
  T *data() { return v.data(); }
};

int plan(const std::vector<int32_t> &q, const std::vector<int32_t> &kv, int hq, int hkv, int cus,
         int items, int merges, int32_t *counts) {
  Guarded<int32_t> a(8 * static_cast<size_t>(items)), b(8 * static_cast<size_t>(merges));
  const int rc = hy_plan_tree(q.data(), kv.data(), static_cast<int32_t>(q.size()), hq, hkv, cus,
                              a.data(), items, b.data(), merges, counts);
  if (rc != HY_OK) return rc;
  // every node in one tile, and every key of every tile once
  int64_t keys = 0, want = 0, nodes = 0;
  for (int p = 0; p < counts[1]; ++p) {
    const int32_t *r = a.data() + 16 * static_cast<size_t>(counts[0]) + 8 * static_cast<size_t>(p);
    CHECK(r[0] >= 0 && r[0] < static_cast<int32_t>(q.size()) && r[1] < r[2] && r[3] < r[4]);
    CHECK(r[3] % 64 == 0 && r[4] <= kv[r[0]] && (r[2] - r[1]) * (hq / hkv) <= counts[4]);
    CHECK(r[5] < counts[3]);
    keys += r[4] - r[3];
    if (r[3] > 0) continue;
    nodes += r[2] - r[1];
    want += kv[r[0]] - q[r[0]] + r[2];
  }
  for (int32_t n : q) nodes -= n;
  CHECK(keys == want && nodes == 0);
  return rc;
}

}  // namespace

int main(int argc, char **argv) {
  if (argc != 3) return 2;
  std::mt19937 rng(static_cast<unsigned>(atoi(argv[1])));
  auto pick = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
  const int ticks = atoi(argv[2]);
  for (int tick = 0; tick < ticks; ++tick) {
    const int n = pick(1, 40), group = 1 << pick(0, 4), hkv = 1 << pick(0, 5), cus = pick(0, 304);
    const int nodes = pick(0, 2) ? pick(1, 40) : 256;
    const int longest = pick(0, 3) ? pick(0, 70000) : INT32_MAX - 128 - nodes;
    std::vector<int32_t> q, kv, parents;
    for (int b = 0; b < n; ++b) {
      q.push_back(pick(1, nodes));
      kv.push_back(q.back() + pick(0, longest));
      for (int i = 0; i < q.back(); ++i) parents.push_back(pick(-1, i - 1));
    }
    const int words = *std::max_element(q.begin(), q.end()) > 128 ? 8 : 4;
    {
      Guarded<uint32_t> lines(parents.size() * words);
      Guarded<int32_t> depths(parents.size());
      CHECK(hy_tree_lines(parents.data(), q.data(), n, words, lines.data(), depths.data()) == HY_OK);
      for (size_t i = 0; i < parents.size(); ++i) {
        int bits = 0;
        for (int w = 0; w < words; ++w) bits += __builtin_popcount(lines.data()[i * words + w]);
        CHECK(bits == depths.data()[i] + 1);
      }
      const size_t at = static_cast<size_t>(pick(0, static_cast<int>(parents.size()) - 1));
      parents[at] = 300;
      CHECK(hy_tree_lines(parents.data(), q.data(), n, words, lines.data(), depths.data()) == HY_EINVAL);
    }
    const int tiles = 32 * n, chunks = (cus > 0 ? cus : 256) / hkv + 1;
    int32_t counts[5], again[5];
    CHECK(plan(q, kv, hkv * group, hkv, cus, 3 * (chunks + tiles), tiles, counts) == HY_OK);
    const int items = 2 * counts[0] + counts[1];
    CHECK(plan(q, kv, hkv * group, hkv, cus, items, counts[2], again) == HY_OK);
    CHECK(std::equal(counts, counts + 5, again));
    CHECK(plan(q, kv, hkv * group, hkv, cus, items - 1, counts[2], again) == HY_ENOSPACE);
    if (counts[2] > 0)
      CHECK(plan(q, kv, hkv * group, hkv, cus, items, counts[2] - 1, again) == HY_ENOSPACE);
    kv[static_cast<size_t>(pick(0, n - 1))] = INT32_MAX - pick(0, 127);
    CHECK(plan(q, kv, hkv * group, hkv, cus, items, counts[2], again) == HY_EUNSUPPORTED);
  }
  printf("ok %d\n", ticks);
  return 0;
}
