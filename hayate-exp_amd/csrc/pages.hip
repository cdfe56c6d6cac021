// Token moves and page copies inside the K/V pool, over every layer at once.
//
// Both take their lists from host memory and pass them to the kernel as
// arguments, kRuns records a launch: no device list to build, copy or keep
// alive, and every index has been checked against the pool before the launch.
// A (layer, K or V, kv head) is a unit: 256-byte rows of its own, which no other
// unit reads or writes.

#include <stdlib.h>

#include <algorithm>

#include "hy_common.h"

namespace hy {
namespace {

constexpr int kThreads = 256;
constexpr int kRowsPerPass = kThreads / 16;  // a row is 16 lanes x 16 bytes
constexpr int kRuns = 320;                   // records a launch: 3,840 of the 4,096 argument bytes

// Consecutive rows from dst on take the values of those from src on. n: in a
// move, the rows of the launch before this run (the next run's n ends it); in a
// copy, the number of rows.
struct Run {
  int32_t src, dst, n;
};
struct Runs {
  Run r[kRuns];
};

// Base of unit u = (layer * 2 + (0: K, 1: V)) * num_kv_heads + head.
__device__ __forceinline__ uint16_t *unit_base(uint16_t *k_pool, uint16_t *v_pool, int64_t ls,
                                               int64_t hs, int u, int num_kv_heads) {
  const int h = u % num_kv_heads;
  const int lk = u / num_kv_heads;
  return ((lk & 1) ? v_pool : k_pool) + (lk >> 1) * ls + h * hs;
}

// Moves. One workgroup per unit walks the launch's rows in order, kMovePasses *
// kRowsPerPass rows a step: a step's rows are all loaded before the first of them is
// stored (a row may be the target of a later row of the same step), and the
// host has checked that no row is read after it was written, so the next step's
// loads go out before this step's stores. 5,999 tokens of 36 layers of 8 heads (1.77 GB): 376
// us, 4.7 TB/s, 95 % of what a large copy reaches; 2 or 8 passes a step 394 and 415 us. That
// is 576 units; with fewer than the GPU has compute units the steps' latency bounds it (1 us
// each): 93 us for 1 layer of 8 heads (0.5 TB/s), 96 for 36 layers of one (2.3 TB/s).
constexpr int kMovePasses = 4;
constexpr int kStepRows = kMovePasses * kRowsPerPass;

__global__ __launch_bounds__(kThreads) void move_kernel(uint16_t *k_pool, uint16_t *v_pool,
                                                        int64_t ls, int64_t hs, int num_kv_heads,
                                                        int n_runs, int n_rows, Runs runs) {
  __shared__ Run run[kRuns];
  for (int i = threadIdx.x; i < n_runs; i += kThreads) run[i] = runs.r[i];
  __syncthreads();
  uint16_t *base = unit_base(k_pool, v_pool, ls, hs, blockIdx.x, num_kv_heads) +
                   8 * (threadIdx.x & 15);
  const int group = threadIdx.x >> 4;
  // Run of a row: the last one that begins at or before it, by bisection (single tokens make
  // as many runs as rows).
  auto run_of = [&](int row) {
    int lo = 0, hi = n_runs;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (run[mid].n <= row)
        lo = mid;
      else
        hi = mid;
    }
    return run[lo];
  };
  u32x4 cur[kMovePasses], nxt[kMovePasses];
  int64_t cur_dst[kMovePasses], nxt_dst[kMovePasses];
  auto load = [&](int row0, u32x4(&x)[kMovePasses], int64_t(&dst)[kMovePasses]) {
#pragma unroll
    for (int j = 0; j < kMovePasses; ++j) {
      const int row = row0 + j * kRowsPerPass + group;
      dst[j] = -1;
      if (row >= n_rows) continue;
      const Run at = run_of(row);
      dst[j] = static_cast<int64_t>(at.dst + row - at.n) * kHeadDim;
      x[j] = load16(base + static_cast<int64_t>(at.src + row - at.n) * kHeadDim);
    }
  };
  load(0, cur, cur_dst);
  for (int row0 = 0; row0 < n_rows; row0 += kStepRows) {
    if (row0 + kStepRows < n_rows) load(row0 + kStepRows, nxt, nxt_dst);
    // this step's rows have arrived in every wave before one of them is stored
#pragma unroll
    for (int j = 0; j < kMovePasses; ++j) __asm__ volatile("" ::"v"(cur[j]) : "memory");
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kMovePasses; ++j)
      if (cur_dst[j] >= 0) store16(base + cur_dst[j], cur[j]);
#pragma unroll
    for (int j = 0; j < kMovePasses; ++j) {
      cur[j] = nxt[j];
      cur_dst[j] = nxt_dst[j];
    }
  }
}

// Copies. Sources and targets are distinct pages, so nothing is ordered: one
// workgroup per (unit, record), 128 rows (32 KiB) in flight. Nontemporal on both
// sides: 15 pages of 77 tokens in 36 layers (341 MB read and written) 65.9 us against 70.4, 32
// pages 232 against 238; a large torch copy moves 4.93 TB/s, these 5.1 to 5.2. (In the moves it
// gave nothing.)
constexpr int kCopyPasses = 8;

__global__ __launch_bounds__(kThreads) void copy_kernel(uint16_t *k_pool, uint16_t *v_pool,
                                                        int64_t ls, int64_t hs, int num_kv_heads,
                                                        Runs runs) {
  const Run r = runs.r[blockIdx.y];
  uint16_t *base = unit_base(k_pool, v_pool, ls, hs, blockIdx.x, num_kv_heads) +
                   8 * (threadIdx.x & 15);
  const uint16_t *src = base + static_cast<int64_t>(r.src) * kHeadDim;
  uint16_t *dst = base + static_cast<int64_t>(r.dst) * kHeadDim;
  for (int row0 = threadIdx.x >> 4; row0 < r.n; row0 += kCopyPasses * kRowsPerPass) {
    u32x4 x[kCopyPasses];
#pragma unroll
    for (int j = 0; j < kCopyPasses; ++j)
      if (row0 + j * kRowsPerPass < r.n)
        x[j] = load16_stream(src + static_cast<int64_t>(row0 + j * kRowsPerPass) * kHeadDim);
#pragma unroll
    for (int j = 0; j < kCopyPasses; ++j)
      if (row0 + j * kRowsPerPass < r.n)
        __builtin_nontemporal_store(
            x[j], reinterpret_cast<u32x4 *>(
                      dst + static_cast<int64_t>(row0 + j * kRowsPerPass) * kHeadDim));
  }
}

// A set of indexes below a limit, in memory that may be refused (no exception
// leaves a C entry).
class Marks {
 public:
  explicit Marks(int64_t limit)
      : bits_(static_cast<uint64_t *>(calloc(static_cast<size_t>((limit + 63) / 64), 8))) {}
  ~Marks() { free(bits_); }
  Marks(const Marks &) = delete;
  Marks &operator=(const Marks &) = delete;
  bool ok() const { return bits_ != nullptr; }
  bool has(int64_t i) const { return bits_[i >> 6] >> (i & 63) & 1; }
  void set(int64_t i) { bits_[i >> 6] |= uint64_t{1} << (i & 63); }

 private:
  uint64_t *bits_;
};

int check_pool(const void *k_pool, const void *v_pool, int64_t layer_stride, int64_t head_stride,
               int32_t num_layers, int32_t num_kv_heads, int32_t head_dim, int64_t tokens,
               const char *name) {
  HY_REQUIRE(num_layers >= 1 && num_kv_heads >= 1, "%s: layers and kv heads must be positive",
             name);
  HY_REQUIRE(static_cast<int64_t>(num_layers) * num_kv_heads <= (1 << 22),
             "%s: %d layers of %d kv heads exceed the grid", name, num_layers, num_kv_heads);
  HY_REQUIRE_SUPPORTED(head_dim == kHeadDim, "head_dim %d unsupported (kernels are built for %d)",
                       head_dim, kHeadDim);
  HY_REQUIRE(tokens >= 1 && tokens <= INT32_MAX, "%s: a pool of %lld tokens is out of range", name,
             static_cast<long long>(tokens));
  HY_REQUIRE(k_pool && v_pool, "%s: null pointer argument", name);
  // units do not overlap, and rows start on 16 bytes
  const int64_t unit = tokens * kHeadDim;
  HY_REQUIRE(num_kv_heads == 1 || head_stride >= unit, "%s: heads %lld elements apart overlap",
             name, static_cast<long long>(head_stride));
  HY_REQUIRE(num_layers == 1 || layer_stride >= (num_kv_heads - 1) * head_stride + unit,
             "%s: layers %lld elements apart overlap", name, static_cast<long long>(layer_stride));
  HY_REQUIRE((layer_stride & 7) == 0 && (head_stride & 7) == 0 &&
                 ((reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool)) & 15) == 0,
             "%s: the pools must be 16-byte aligned with strides that are multiples of 8", name);
  return HY_OK;
}

}  // namespace
}  // namespace hy

using hy::kHeadDim;

extern "C" int hy_kv_move(void *k_pool, void *v_pool, int64_t pool_layer_stride,
                          int64_t pool_head_stride, int32_t num_pages, const int32_t *pages,
                          const int32_t *page_start, const int32_t *first_page, const int32_t *src,
                          const int32_t *src_start, const int32_t *first, int32_t num_seqs,
                          int32_t num_layers, int32_t num_kv_heads, int32_t head_dim,
                          int32_t page_size, void *stream) {
  hy::clear_error();
  HY_REQUIRE(num_seqs >= 0, "hy_kv_move: num_seqs must be non-negative");
  HY_REQUIRE(num_pages >= 1 && page_size >= 1, "hy_kv_move: pages must be positive");
  const int64_t tokens = static_cast<int64_t>(num_pages) * page_size;
  if (int rc = hy::check_pool(k_pool, v_pool, pool_layer_stride, pool_head_stride, num_layers,
                              num_kv_heads, head_dim, tokens, "hy_kv_move"))
    return rc;
  if (num_seqs == 0) return HY_OK;
  HY_REQUIRE(pages && page_start && first_page && src && src_start && first,
             "hy_kv_move: null pointer argument");
  // Of the tokens: moved to; filled by a token that stays; read for a move; read for moves of
  // two sequences. (Only other sequences' reads matter, so the last two go with several.)
  hy::Marks written(tokens), stays(tokens), read(num_seqs > 1 ? tokens : 1),
      shared(num_seqs > 1 ? tokens : 1);
  if (!written.ok() || !stays.ok() || !read.ok() || !shared.ok()) {
    hy::set_error("hy_kv_move: no host memory to check %lld tokens", static_cast<long long>(tokens));
    return HY_ENOSPACE;
  }
  hy::Runs runs;
  int n_runs = 0, n_rows = 0;
  auto launch = [&]() {
    hipLaunchKernelGGL(hy::move_kernel, dim3(2 * num_layers * num_kv_heads), dim3(hy::kThreads), 0,
                       static_cast<hipStream_t>(stream), static_cast<uint16_t *>(k_pool),
                       static_cast<uint16_t *>(v_pool), pool_layer_stride, pool_head_stride,
                       num_kv_heads, n_runs, n_rows, runs);
    n_runs = n_rows = 0;
    return hy::launch_status("hy_kv_move");
  };
  // Every move is checked before the first launch: once to check, once to enqueue.
  for (int pass = 0; pass < 2; ++pass) {
    int64_t last_src = -1, last_dst = -1;  // of the run being built
    for (int32_t b = 0; b < num_seqs; ++b) {
      const int64_t held = static_cast<int64_t>(page_start[b + 1]) - page_start[b];
      const int64_t base = static_cast<int64_t>(first_page[b]) * page_size;
      if (pass == 0) {
        HY_REQUIRE(held >= 0 && first_page[b] >= 0 && src_start[b + 1] >= src_start[b] &&
                       page_start[b] >= 0 && src_start[b] >= 0,
                   "hy_kv_move: sequence %d has a negative start or count", b);
        for (int32_t i = page_start[b]; i < page_start[b + 1]; ++i)
          HY_REQUIRE(pages[i] >= 0 && pages[i] < num_pages,
                     "hy_kv_move: page %d is not in the pool of %d", pages[i], num_pages);
      }
      int32_t own = src_start[b];  // the first source not before the position being filled
      for (int32_t i = src_start[b]; i < src_start[b + 1]; ++i) {
        const int64_t from = src[i] - base;
        const int64_t to = static_cast<int64_t>(first[b]) + (i - src_start[b]) - base;
        if (pass == 0)
          HY_REQUIRE(to >= 0 && from >= to && from < held * page_size &&
                         (i == src_start[b] || src[i] > src[i - 1]),
                     "hy_kv_move: sequence %d cannot take its token %d to position %lld (sources "
                     "ascend, none before the position it fills, all in the given pages)",
                     b, src[i], static_cast<long long>(to + base));
        if (from == to && pass == 1) continue;
        const int32_t *list = pages + page_start[b];
        const int64_t d = static_cast<int64_t>(list[to / page_size]) * page_size + to % page_size;
        if (from == to) {
          HY_REQUIRE(!written.has(d), "hy_kv_move: sequence %d shares pages that are written", b);
          stays.set(d);
          continue;
        }
        const int64_t s = static_cast<int64_t>(list[from / page_size]) * page_size + from % page_size;
        if (pass == 0) {
          bool clash = written.has(s) || written.has(d) || stays.has(d);
          if (num_seqs > 1) {
            (read.has(s) ? shared : read).set(s);
            while (src[own] - base < to) ++own;  // ends at i at the latest
            clash = clash || shared.has(d) || (read.has(d) && src[own] - base != to);
          }
          HY_REQUIRE(!clash, "hy_kv_move: sequence %d shares pages that are written", b);
          written.set(d);
          continue;
        }
        if (n_runs > 0 && s == last_src + 1 && d == last_dst + 1) {
          ++n_rows;
        } else {
          if (n_runs == hy::kRuns)
            if (int rc = launch()) return rc;
          runs.r[n_runs++] = {static_cast<int32_t>(s), static_cast<int32_t>(d), n_rows++};
        }
        last_src = s;
        last_dst = d;
      }
    }
  }
  return n_runs ? launch() : HY_OK;
}

extern "C" int hy_page_copy(void *k_pool, void *v_pool, int64_t pool_layer_stride,
                            int64_t pool_head_stride, int32_t num_pages, const int32_t *src_pages,
                            const int32_t *dst_pages, const int32_t *tokens, int32_t n,
                            int32_t num_layers, int32_t num_kv_heads, int32_t head_dim,
                            int32_t page_size, void *stream) {
  hy::clear_error();
  HY_REQUIRE(n >= 0, "hy_page_copy: n must be non-negative");
  HY_REQUIRE(num_pages >= 1 && page_size >= 1, "hy_page_copy: pages must be positive");
  if (int rc = hy::check_pool(k_pool, v_pool, pool_layer_stride, pool_head_stride, num_layers,
                              num_kv_heads, head_dim, static_cast<int64_t>(num_pages) * page_size,
                              "hy_page_copy"))
    return rc;
  if (n == 0) return HY_OK;
  HY_REQUIRE(src_pages && dst_pages, "hy_page_copy: null pointer argument");
  hy::Marks written(num_pages);
  if (!written.ok()) {
    hy::set_error("hy_page_copy: no host memory to check %d pages", num_pages);
    return HY_ENOSPACE;
  }
  for (int32_t i = 0; i < n; ++i) {
    HY_REQUIRE(src_pages[i] >= 0 && src_pages[i] < num_pages && dst_pages[i] >= 0 &&
                   dst_pages[i] < num_pages,
               "hy_page_copy: copy %d (page %d to %d) leaves the pool of %d pages", i, src_pages[i],
               dst_pages[i], num_pages);
    HY_REQUIRE(tokens == nullptr || (tokens[i] >= 0 && tokens[i] <= page_size),
               "hy_page_copy: copy %d of %d tokens, pages hold %d", i, tokens ? tokens[i] : 0,
               page_size);
    HY_REQUIRE(!written.has(dst_pages[i]), "hy_page_copy: two copies write page %d", dst_pages[i]);
    written.set(dst_pages[i]);
  }
  for (int32_t i = 0; i < n; ++i)
    HY_REQUIRE(!written.has(src_pages[i]), "hy_page_copy: page %d is read and written",
               src_pages[i]);
  hy::Runs runs;
  for (int32_t i = 0; i < n;) {
    int n_runs = 0;
    for (; i < n && n_runs < hy::kRuns; ++i) {
      const int32_t len = tokens ? tokens[i] : page_size;
      if (len > 0) runs.r[n_runs++] = {src_pages[i] * page_size, dst_pages[i] * page_size, len};
    }
    if (n_runs == 0) break;
    hipLaunchKernelGGL(hy::copy_kernel, dim3(2 * num_layers * num_kv_heads, n_runs),
                       dim3(hy::kThreads), 0, static_cast<hipStream_t>(stream),
                       static_cast<uint16_t *>(k_pool), static_cast<uint16_t *>(v_pool),
                       pool_layer_stride, pool_head_stride, num_kv_heads, runs);
    if (int rc = hy::launch_status("hy_page_copy")) return rc;
  }
  return HY_OK;
}
