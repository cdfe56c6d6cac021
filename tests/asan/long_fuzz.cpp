// Fuzz driver of the planners of windowed and weighed attention for a sanitizer build
// (AddressSanitizer and UndefinedBehaviorSanitizer, g++ on the host): random ticks, up to the longest
// caches, windows and sinks, with buffers of exactly the counts that a first call reported and one
// record short of each (HY_ENOSPACE). Guard words behind every buffer must stay untouched.
// Usage: long_fuzz <seed> <ticks>; prints "ok <ticks>" and exits 0.
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>

#include <algorithm>
#include <random>
#include <vector>

#include "../../hayate-exp_amd/csrc/window.h"
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

struct Guarded {
  std::vector<int32_t> v;
  size_t used;
  explicit Guarded(int64_t n) : v(static_cast<size_t>(n) + kMargin, kPoison), used(static_cast<size_t>(n)) {}
  ~Guarded() {
    for (size_t i = used; i < v.size(); ++i) CHECK(v[i] == kPoison);
  }
  int32_t *data() { return v.data(); }
};

struct Tick {
  std::vector<int32_t> q, kv, rows;
  int hq, hkv, cus, window, sinks;
};

int plan(const Tick &t, int dec, int mrg, int pre, int pmrg, int32_t *counts,
         std::vector<int32_t> &merge) {
  Guarded a(8 * static_cast<int64_t>(dec)), b(4 * static_cast<int64_t>(mrg)),
      c(8 * static_cast<int64_t>(pre)), d(8 * static_cast<int64_t>(pmrg));
  const int n = static_cast<int>(t.q.size());
  const int rc =
      t.window > 0
          ? hy_plan_tick_window(t.q.data(), t.kv.data(), n, t.hq, t.hkv, 128, t.cus, 0, t.window,
                                t.sinks, a.data(), dec, b.data(), mrg, c.data(), pre, d.data(), pmrg,
                                counts)
          : hy_plan_tick(t.q.data(), t.kv.data(), n, t.hq, t.hkv, 128, t.cus, 0, a.data(), dec,
                         b.data(), mrg, c.data(), pre, d.data(), pmrg, counts);
  if (rc != HY_OK) return rc;
  // every number of every decode token once
  int64_t keys = 0, want = 0;
  for (int p = 0; p < counts[6]; ++p) {
    const int32_t *r = a.data() + 8 * (static_cast<size_t>(counts[0]) + static_cast<size_t>(p));
    CHECK(r[0] >= 0 && r[0] < n && r[1] < r[2] && r[1] % 32 == 0);
    keys += r[2] - r[1];
  }
  for (int i = 0; i < n; ++i)
    if (t.q[i] == 1)
      want += t.kv[i] - (t.window > 0 ? hy::window_keys(t.kv[i] - 1, t.window, t.sinks).gap : 0);
  CHECK(keys == want);
  merge.assign(b.data(), b.data() + 4 * counts[1]);
  return rc;
}

int weigh(const Tick &t, const std::vector<int32_t> &merge, int items, int adds, int64_t *counts) {
  Guarded starts(static_cast<int64_t>(t.q.size())), a(8 * static_cast<int64_t>(items)),
      b(8 * static_cast<int64_t>(adds));
  const int rc = hy_plan_weigh(t.q.data(), t.kv.data(), t.rows.data(),
                               static_cast<int32_t>(t.q.size()), t.hq, t.hkv, t.cus, merge.data(),
                               static_cast<int32_t>(merge.size() / 4), starts.data(), a.data(), items,
                               b.data(), adds, counts);
  if (rc != HY_OK) return rc;
  int64_t tokens = 0;
  for (int64_t i = 0; i < counts[1]; ++i) {
    const int32_t *x = b.data() + 8 * i;
    CHECK(x[1] < x[2] && x[2] - x[1] <= 256 && x[3] > 0 && x[4] >= 0 && x[6] >= 0);
    CHECK(x[6] + x[1] + (x[2] - x[1] + 3) / 4 * 4 <= (x[5] ? counts[2] : counts[3]));
    if (!x[5]) CHECK(x[4] + x[3] <= counts[4] * t.hkv);
    tokens += x[2] - x[1];
  }
  for (int32_t n : t.kv) tokens -= n;
  CHECK(tokens == 0);
  for (int64_t i = 0; i < counts[0]; ++i) {
    const int32_t *x = a.data() + 8 * i;
    CHECK(x[0] >= 0 && x[0] < static_cast<int32_t>(t.q.size()) && x[2] < x[3] && x[3] <= t.q[x[0]]);
    CHECK(x[4] < counts[4] && x[7] + x[1] + 256 <= counts[3] && x[1] < t.kv[x[0]]);
  }
  return rc;
}

}  // namespace

int main(int argc, char **argv) {
  if (argc != 3) return 2;
  std::mt19937 rng(static_cast<unsigned>(atoi(argv[1])));
  auto pick = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
  const int ticks = atoi(argv[2]);
  for (int tick = 0; tick < ticks; ++tick) {
    Tick t;
    const int n = pick(1, 40), longest = pick(0, 3) ? pick(0, 3000) : 70000;
    t.hkv = 1 << pick(0, 5);
    t.hq = t.hkv << pick(0, 4);
    t.cus = pick(0, 304);
    t.window = pick(0, 3) ? pick(1, pick(0, 1) ? 2000 : INT32_MAX) : 0;
    t.sinks = t.window ? pick(0, pick(0, 2) ? 300 : hy::kMaxSinks) : 0;
    for (int b = 0; b < n; ++b) {
      t.q.push_back(pick(0, 1) ? 1 : pick(2, 600));
      t.kv.push_back(t.q.back() + pick(0, longest));
      t.rows.push_back(pick(0, 1000));
    }
    int32_t counts[7], again[7];
    std::vector<int32_t> merge, other;
    int roomy = 40000;
    CHECK(plan(t, roomy, n + 1, roomy, roomy, counts, merge) == HY_OK);
    const int dec = counts[0] + counts[6];
    CHECK(plan(t, dec, counts[1], counts[3], counts[4], again, other) == HY_OK);
    CHECK(std::equal(counts, counts + 7, again) && merge == other);
    if (dec > 0) CHECK(plan(t, dec - 1, counts[1], counts[3], counts[4], again, other) == HY_ENOSPACE);
    if (counts[1] > 0)
      CHECK(plan(t, dec, counts[1] - 1, counts[3], counts[4], again, other) == HY_ENOSPACE);
    if (counts[3] > 0)
      CHECK(plan(t, dec, counts[1], counts[3] - 1, counts[4], again, other) == HY_ENOSPACE);
    if (t.window) {
      // one long cache in sight of a window: keys in sight only are planned
      Tick l = t;
      l.kv[0] = INT32_MAX - 1024;
      l.sinks = std::min(l.sinks, 300);
      l.window = std::min(l.window, 100000);
      CHECK(plan(l, roomy, n + 1, roomy, roomy, again, other) == HY_OK);
      continue;
    }
    int64_t sizes[5], same[5];
    int64_t blocks = 0, chunk_blocks = 0;
    for (int b = 0; b < n; ++b) {
      blocks += (t.kv[b] + 255) / 256;
      if (t.q[b] > 1) chunk_blocks += (t.kv[b] + 255) / 256;
    }
    CHECK(weigh(t, merge, static_cast<int>(32 * chunk_blocks), static_cast<int>(blocks), sizes) == HY_OK);
    CHECK(sizes[1] == blocks);
    const int items = static_cast<int>(sizes[0]), adds = static_cast<int>(sizes[1]);
    CHECK(weigh(t, merge, items, adds, same) == HY_OK);
    CHECK(std::equal(sizes, sizes + 5, same));
    CHECK(weigh(t, merge, items, adds - 1, same) == HY_ENOSPACE);
    if (items > 0) CHECK(weigh(t, merge, items - 1, adds, same) == HY_ENOSPACE);
    if (!merge.empty()) {
      merge[0] = n;
      CHECK(weigh(t, merge, items, adds, same) == HY_EINVAL);
      merge.erase(merge.begin(), merge.begin() + 4);  // a decode token without its slots
      CHECK(weigh(t, merge, items, adds, same) == HY_EINVAL);
    }
    if (tick % 50 == 0) {
      Tick l = t;
      l.kv[0] = 20000000;
      l.q[0] = 2;
      CHECK(weigh(l, merge, items, adds, same) != HY_OK);
    }
  }
  printf("ok %d\n", ticks);
  return 0;
}
