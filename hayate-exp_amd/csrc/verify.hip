// Verification of trees of drafted tokens against the target's probabilities (gfx950).
//
// Node 0 of a request is its last token; from there the walk takes, node by node, the first
// child (in index order) that passes its test, and draws the next token where none does. With
// p the softmax of the node's logits over its temperature, cut by top-k and top-p, and u given
// uniform numbers:
//   drafts as given  child x is taken where u (1 - R) < p(x), R the p of its refused earlier
//                    siblings' tokens (a token that was refused already has p(x) = 0); the draw is
//                    from p without the refused tokens.
//   drafts drawn     (chains) from probabilities q: taken where u q(x) < p(x); the draw is from
//                    max(p - q, 0) where the child was refused.
//   greedy           taken where x is the largest logit's token, which is also the draw.
// Either way the tokens of path and draw are distributed as the target's own samples.
// The draw takes the smallest token whose cumulative mass exceeds u times the total; where
// nothing is left (all mass refused) it is from p.
//
//   cut_kernel    rows of requests with top-k or top-p only: where they are cut.
//   mass_kernel   many workgroups a row: the maximum and the sum of exponentials of each one's
//                 share of the logits (greedy: its largest logit).
//   walk_kernel   the walk, in every workgroup of the request: its tests need the shares of its
//                 rows and a logit a node, a few reads that all nodes make at once. Then the
//                 masses of its share of the last node's row, in 64 bits: a border between
//                 two of 151,936 tokens is met by one draw in thousands of 32-bit sums.
//   rest_kernel   (drafts drawn) the masses of max(p - q, 0).
//   pick_kernel   the share that holds the draw, then the token.

#include "logit_rows.h"

namespace hy {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kShare = kThreads * kVec * kAhead;  // logits of a workgroup
constexpr int kRequests = 64;                     // requests of one launch
constexpr int kMaxNodes = 256;

struct Request {
  float temp;
  int32_t k;
  float p;
  int32_t first;  // its first row
};
struct Requests {
  static constexpr bool kCutsOnly = true;
  Request r[kRequests];
  int32_t count, rows;

  __device__ __forceinline__ int of_row(int row) const {
    int lo = 0, hi = count;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (r[mid].first <= row)
        lo = mid;
      else
        hi = mid;
    }
    return lo;
  }
  __device__ __forceinline__ int nodes(int b) const {
    return (b + 1 < count ? r[b + 1].first : rows) - r[b].first;
  }
  __device__ __forceinline__ SampleRow row(int i) const {
    const Request &q = r[of_row(i)];
    return {q.temp, q.k, q.p, 0};
  }
  __device__ __forceinline__ bool cut(int b, int vocab) const {
    return r[b].temp != 0.f && (r[b].k < vocab || r[b].p < 1.f);
  }
};

// A workgroup's share of a row: the largest kept logit and the sum of exp((x - max) / temp); of a
// greedy row rank_of() of the largest.
struct Share {
  float max, sum;
  uint64_t best;
};
// Masses of a share of a request's last row: all of it, and what the draw is from.
struct Mass {
  double all, left;
};
struct State {
  int32_t last, child;  // the path's last node, and its refused child where drafts are drawn, or -1
  float max;            // largest kept logit of the last node's row
  int32_t bad;
};

struct Tree {
  const int32_t *parents;
  const int64_t *tokens;
  const float *uniforms;  // a number a node, of the launch's requests
  const float *draws;     // and a number a request
  const float *drafts;    // or null
  int64_t drafts_ld;
};

// This thread's logits of a share: kAhead loads of kVec, load a from index first + a * step on.
// Past the row's end the last logit is repeated.
__device__ __forceinline__ void load_share(const uint16_t *x, int vocab, int first, int step,
                                           u32x4 (&w)[kAhead]) {
#pragma unroll
  for (int a = 0; a < kAhead; ++a) {
    const int i = first + a * step;
    if (i + kVec <= vocab) {
      __builtin_memcpy(&w[a], x + i, sizeof(w[a]));
    } else {
      w[a] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        w[a][j >> 1] |= static_cast<uint32_t>(x[min(i + j, vocab - 1)]) << (16 * (j & 1));
    }
  }
}
__device__ __forceinline__ uint32_t key_in(const u32x4 &w, int j) {
  return merge_zero((keys_of(w[j >> 1]) >> (16 * (j & 1))) & 0xffffu);
}
__device__ __forceinline__ bool kept(const RowCut &cut, uint32_t key, int index) {
  return static_cast<int>(key) >= cut.low && !(static_cast<int>(key) == cut.cut && index > cut.last);
}
__device__ __forceinline__ RowCut no_cut(int vocab) { return {0, 0, vocab, 1, 0.f}; }

// Sums over the workgroup in a fixed order, in every thread.
__device__ __forceinline__ double block_sum(double v, double *box) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) box[threadIdx.x >> 6] = v;
  __syncthreads();
  v = box[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) v += box[i];
  return v;
}

// Grid (shares, rows).
template <bool kBf16>
__global__ __launch_bounds__(kThreads) void mass_kernel(
    const uint16_t *__restrict__ logits, int64_t ld, int vocab, Requests requests,
    const RowCut *__restrict__ cuts, Share *__restrict__ shares, uint8_t *__restrict__ valid,
    bool first_rows) {
  __shared__ uint64_t best[kWaves];
  __shared__ float maxes[kWaves];
  __shared__ double box[kWaves];
  if (first_rows && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *valid = 1;
  const int row = blockIdx.y;
  const int b = requests.of_row(row);
  const Request req = requests.r[b];
  const int i0 = blockIdx.x * kShare + kVec * threadIdx.x;
  constexpr int kRound = kThreads * kVec;
  u32x4 w[kAhead];
  load_share(logits + row * ld, vocab, i0, kRound, w);
  Share *out = shares + static_cast<int64_t>(row) * gridDim.x + blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  constexpr uint32_t kInf = kInfBits<kBf16>;
  if (req.temp == 0.f) {  // a NaN counts as the largest
    uint64_t top = 0;
#pragma unroll
    for (int a = 0; a < kAhead; ++a)
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        uint32_t key = key_in(w[a], j);
        if (key > (0x8000u | kInf) || key < 0x7fffu - kInf) key = 0xffffu;
        const int i = i0 + a * kRound + j;
        const uint64_t r = i < vocab ? rank_of(key, i) : 0;
        top = r > top ? r : top;
      }
    top = wave_best(top);
    if (lane == 0) best[wave] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
      for (int i = 1; i < kWaves; ++i) top = best[i] > top ? best[i] : top;
      out->best = top;
    }
    return;
  }
  const RowCut cut = requests.cut(b, vocab) ? cuts[row] : no_cut(vocab);
  bool nan = cut.ok != 1;
  float x[kAhead][kVec], m = -INFINITY;
#pragma unroll
  for (int a = 0; a < kAhead; ++a)
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const uint32_t key = key_in(w[a], j);
      const int i = i0 + a * kRound + j;
      nan = nan || key > (0x8000u | kInf) || key < 0x7fffu - kInf;
      x[a][j] = i < vocab && kept(cut, key, i) ? value_of<kBf16>(key) : -INFINITY;
      m = fmaxf(m, x[a][j]);
    }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  if (lane == 0) maxes[wave] = m;
  nan = __syncthreads_or(nan);
  m = maxes[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) m = fmaxf(m, maxes[i]);
  const float slope = 1.0f / req.temp * kLog2eS;
  float s = 0.f;
  if (m != -INFINITY) {
#pragma unroll
    for (int a = 0; a < kAhead; ++a)
#pragma unroll
      for (int j = 0; j < kVec; ++j) s += __builtin_amdgcn_exp2f((x[a][j] - m) * slope);
  }
  const double sum = block_sum(s, box);
  if (threadIdx.x == 0) {
    out->max = nan ? NAN : m;
    out->sum = static_cast<float>(sum);
  }
}

// exp((x - max) / temp) of this thread's kept logits of a share, 0 elsewhere: f(mass, index).
template <bool kBf16, class F>
__device__ __forceinline__ void each_mass(const u32x4 (&w)[kAhead], int first, int step, int vocab,
                                          const RowCut &cut, float max, float temp, F f) {
#pragma unroll
  for (int a = 0; a < kAhead; ++a) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const uint32_t key = key_in(w[a], j);
      const int i = first + a * step + j;
      if (i < vocab && kept(cut, key, i))
        f(exp((static_cast<double>(value_of<kBf16>(key)) - max) / static_cast<double>(temp)), i);
    }
  }
}

// Marks the tokens of a share that the draw leaves out: those of the last node's children.
__device__ __forceinline__ void mark_refused(uint32_t *bits, const int32_t *parents,
                                             const int64_t *tokens, int nodes, int last, int first) {
  for (int i = threadIdx.x; i < kShare / 32; i += kThreads) bits[i] = 0;
  __syncthreads();
  for (int j = threadIdx.x; j < nodes; j += kThreads) {
    const int64_t at = tokens[j] - first;
    if (j > 0 && parents[j] == last && at >= 0 && at < kShare)
      atomicOr(&bits[at >> 5], 1u << (at & 31));
  }
  __syncthreads();
}

// Grid (shares, requests).
template <bool kBf16>
__global__ __launch_bounds__(kThreads) void walk_kernel(
    const uint16_t *__restrict__ logits, int64_t ld, int vocab, Requests requests,
    const RowCut *__restrict__ cuts, const Share *__restrict__ shares, Tree tree,
    State *__restrict__ states, Mass *__restrict__ masses, int32_t *__restrict__ paths, int levels,
    int32_t *__restrict__ lengths, int64_t *__restrict__ next, uint8_t *__restrict__ valid) {
  __shared__ float max_of[kMaxNodes];
  __shared__ double sum_of[kMaxNodes];
  __shared__ double p_of[kMaxNodes];  // p(x) of a node's token under its parent; greedy: 1 or 0
  __shared__ double q_of[kMaxNodes];
  __shared__ float u_of[kMaxNodes];
  __shared__ int best_of[kMaxNodes], token_of[kMaxNodes], refused[kMaxNodes];
  __shared__ State sh;
  __shared__ uint32_t bits[kShare / 32];
  __shared__ double box[kWaves];
  const int b = blockIdx.y;
  const Request req = requests.r[b];
  const int nodes = requests.nodes(b), row0 = req.first;
  const bool greedy = req.temp == 0.f, cut_rows = requests.cut(b, vocab);
  const int32_t *parents = tree.parents + row0;
  const int64_t *tokens = tree.tokens + row0;
  const int tid = threadIdx.x, lane = tid & 63;
  const int n_shares = gridDim.x;

  int32_t up = 0;
  if (tid < nodes) {
    const int64_t x = tokens[tid];
    token_of[tid] = x >= 0 && x < vocab ? static_cast<int32_t>(x) : -1;
    u_of[tid] = tree.uniforms[row0 + tid];
    if (tid > 0) up = min(max(parents[tid], 0), tid - 1);
  }
  int par[kMaxNodes / 64];  // of nodes 64 i + lane
#pragma unroll
  for (int i = 0; i < kMaxNodes / 64; ++i)
    par[i] = 64 * i + lane < nodes && 64 * i + lane > 0 ? parents[64 * i + lane] : -1;
  // Every row's maximum and sum (or largest logit), from its shares: 32 lanes a row.
  const int l32 = tid & 31;
  const float slope = greedy ? 0.f : 1.0f / req.temp * kLog2eS;
#pragma unroll 2
  for (int r = tid >> 5; r < nodes; r += kThreads / 32) {
    const Share *s = shares + static_cast<int64_t>(row0 + r) * n_shares;
    if (greedy) {
      uint64_t top = 0;
      for (int i = l32; i < n_shares; i += 32) top = s[i].best > top ? s[i].best : top;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const uint64_t t = __shfl_xor(static_cast<unsigned long long>(top), o);
        top = t > top ? t : top;
      }
      if (l32 == 0) best_of[r] = index_of(top);
      continue;
    }
    float m = -INFINITY;
    double z = 0;
    bool nan = false;
    for (int i = l32; i < n_shares; i += 32) {
      const float sm = s[i].max, ss = s[i].sum;
      nan = nan || sm != sm;
      if (sm > m) {
        z *= __builtin_amdgcn_exp2f((m - sm) * slope);
        m = sm;
      }
      if (ss > 0.f) z += static_cast<double>(ss) * __builtin_amdgcn_exp2f((sm - m) * slope);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float om = __shfl_xor(m, o);
      const double oz = __shfl_xor(z, o);
      const float top = fmaxf(m, om);
      z = (z > 0 ? z * __builtin_amdgcn_exp2f((m - top) * slope) : 0) +
          (oz > 0 ? oz * __builtin_amdgcn_exp2f((om - top) * slope) : 0);
      m = top;
      nan = nan || __shfl_xor(static_cast<int>(nan), o);
    }
    if (l32 == 0) {
      max_of[r] = nan || isinf(m / req.temp) ? NAN : m;
      sum_of[r] = z;
    }
  }
  __syncthreads();
  if (tid > 0 && tid < nodes) {
    const int x = token_of[tid];
    double p = 0, q = 0;
    if (greedy) {
      p = x == best_of[up];
    } else if (x >= 0) {
      const uint32_t word = logits[(row0 + up) * ld + x];
      const uint32_t key = merge_zero(keys_of(word) & 0xffffu);
      const RowCut cut = cut_rows ? cuts[row0 + up] : no_cut(vocab);
      if (tree.drafts) q = tree.drafts[(row0 + tid) * tree.drafts_ld + x];
      if (kept(cut, key, x))
        p = exp((static_cast<double>(value_of<kBf16>(key)) - max_of[up]) /
                static_cast<double>(req.temp)) /
            sum_of[up];
    }
    p_of[tid] = p;
    q_of[tid] = q;
  }
  __syncthreads();
  // The walk, by one wave: a node's children come after it, in index order.
  if (tid < 64) {
    int last = 0, length = 1, child = -1;
    bool bad = false;
    int32_t *path = paths + static_cast<int64_t>(b) * levels;
    const bool tell = blockIdx.x == 0;
    if (tell && lane == 0 && levels > 0) path[0] = 0;
    while (true) {
      bad = !greedy && max_of[last] != max_of[last];
      if (bad) break;
      double gone = 0;
      int n_refused = 0, taken = -1;
#pragma unroll 1
      for (int i = 0; i < kMaxNodes / 64 && taken < 0; ++i) {
        int mine = par[0];
#pragma unroll
        for (int k = 1; k < kMaxNodes / 64; ++k) mine = i == k ? par[k] : mine;
        // (a child has a higher index, so the walk ends)
        uint64_t children = __ballot(mine == last && 64 * i + lane > last);
        while (children != 0) {
          const int j = 64 * i + __ffsll(static_cast<long long>(children)) - 1;
          children &= children - 1;
          const double u = u_of[j];
          bool took;
          double p = p_of[j];
          const int x = token_of[j];
          if (greedy) {
            took = p != 0;
          } else if (tree.drafts) {
            took = u * q_of[j] < p;
            child = j;
          } else {
            bool again = false;
            for (int k = lane; k < n_refused; k += 64) again = again || refused[k] == x;
            if (__any(again)) p = 0;
            took = u * (1 - gone) < p;
          }
          if (took) {
            taken = j;
            break;
          }
          gone += p;
          if (lane == 0) refused[n_refused] = x;
          ++n_refused;
          __builtin_amdgcn_s_waitcnt(0xc07f);  // (this wave alone reads it)
          __asm__ volatile("" ::: "memory");
        }
      }
      if (taken < 0) break;
      last = taken;
      child = -1;
      if (tell && lane == 0 && length < levels) path[length] = last;
      ++length;
    }
    if (lane == 0) {
      sh = {last, child, greedy ? 0.f : max_of[last], bad};
      if (tell) {
        lengths[b] = length;
        states[b] = sh;
        if (greedy) next[b] = best_of[last];
        if (bad) {
          next[b] = 0;
          *valid = 0;
        }
      }
    }
    if (tell)
      for (int i = length + lane; i < levels; i += 64) path[i] = -1;
  }
  __syncthreads();
  if (greedy || sh.bad) return;
  const int row = row0 + sh.last, first = blockIdx.x * kShare;
  if (!tree.drafts) mark_refused(bits, parents, tokens, nodes, sh.last, first);
  u32x4 w[kAhead];
  load_share(logits + row * ld, vocab, first + kVec * tid, kThreads * kVec, w);
  double all = 0, left = 0;
  each_mass<kBf16>(w, first + kVec * tid, kThreads * kVec, vocab,
                   cut_rows ? cuts[row] : no_cut(vocab), sh.max, req.temp, [&](double e, int i) {
                     all += e;
                     const int at = i - first;
                     if (tree.drafts || !(bits[at >> 5] >> (at & 31) & 1)) left += e;
                   });
  all = block_sum(all, box);
  left = block_sum(left, box);
  if (tid == 0) masses[static_cast<int64_t>(b) * n_shares + blockIdx.x] = {all, left};
}

// Grid (shares, requests): of requests whose drawn draft was refused, the masses of max(p - q, 0).
template <bool kBf16>
__global__ __launch_bounds__(kThreads) void rest_kernel(
    const uint16_t *__restrict__ logits, int64_t ld, int vocab, Requests requests,
    const RowCut *__restrict__ cuts, Tree tree, const State *__restrict__ states,
    const Mass *__restrict__ masses, double *__restrict__ rests) {
  __shared__ double box[kWaves];
  const int b = blockIdx.y;
  const Request req = requests.r[b];
  const State st = states[b];
  if (req.temp == 0.f || st.bad || st.child < 0) return;
  const Mass *m = masses + static_cast<int64_t>(b) * gridDim.x;
  double z = 0;
  for (int i = threadIdx.x; i < static_cast<int>(gridDim.x); i += kThreads) z += m[i].all;
  z = block_sum(z, box);
  const int row = req.first + st.last, first = blockIdx.x * kShare + kVec * threadIdx.x;
  u32x4 w[kAhead];
  load_share(logits + row * ld, vocab, first, kThreads * kVec, w);
  const float *q = tree.drafts + (req.first + st.child) * tree.drafts_ld;
  double left = 0;
  each_mass<kBf16>(w, first, kThreads * kVec, vocab,
                   requests.cut(b, vocab) ? cuts[row] : no_cut(vocab), st.max, req.temp,
                   [&](double e, int i) { left += fmax(e / z - q[i], 0.0); });
  left = block_sum(left, box);
  if (threadIdx.x == 0) rests[static_cast<int64_t>(b) * gridDim.x + blockIdx.x] = left;
}

// Grid (requests).
template <bool kBf16>
__global__ __launch_bounds__(kThreads) void pick_kernel(
    const uint16_t *__restrict__ logits, int64_t ld, int vocab, Requests requests,
    const RowCut *__restrict__ cuts, Tree tree, const State *__restrict__ states,
    const Mass *__restrict__ masses, const double *__restrict__ rests, int n_shares,
    int64_t *__restrict__ next) {
  __shared__ uint32_t bits[kShare / 32];
  __shared__ double box[kWaves];
  __shared__ struct {
    int share, found, tail;
    double before;
  } sh;
  const int b = blockIdx.x;
  const Request req = requests.r[b];
  const State st = states[b];
  if (req.temp == 0.f || st.bad) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const bool drawn = tree.drafts && st.child >= 0;  // the draw is from max(p - q, 0)
  const Mass *m = masses + static_cast<int64_t>(b) * n_shares;
  const double *rest = rests + static_cast<int64_t>(b) * n_shares;
  double z = 0, some = 0;
  for (int i = tid; i < n_shares; i += kThreads) {
    z += m[i].all;
    some += drawn ? rest[i] : m[i].left;
  }
  z = block_sum(z, box);
  some = block_sum(some, box);
  // where nothing is left, all of p
  const bool whole = !(some > 0);
  auto mass_at = [&](int i) { return whole ? m[i].all : drawn ? rest[i] : m[i].left; };
  // the share in which the running sum passes the target (a few hundred at most: one thread)
  if (tid == 0) {
    double total = 0;
    for (int i = 0; i < n_shares; ++i) total += mass_at(i);
    const double target = static_cast<double>(tree.draws[b]) * total;
    double sum = 0;
    sh.share = 0;
    sh.before = target;
    for (int i = 0; i < n_shares; ++i) {
      const double v = mass_at(i);
      if (v > 0) {
        sh.share = i;
        sh.before = target - sum;
        if (sum + v > target) break;
      }
      sum += v;
    }
    sh.found = vocab;
    sh.tail = -1;
  }
  __syncthreads();
  const int row = req.first + st.last, first = sh.share * kShare;
  const double target = sh.before;  // within the share
  if (!drawn)
    mark_refused(bits, tree.parents + req.first, tree.tokens + req.first, requests.nodes(b), st.last,
                 first);
  const float *q = drawn ? tree.drafts + (req.first + st.child) * tree.drafts_ld : nullptr;
  // a thread's logits lie in a row here
  const int own = first + kVec * kAhead * tid;
  u32x4 w[kAhead];
  load_share(logits + row * ld, vocab, own, kVec, w);
  const RowCut cut = requests.cut(b, vocab) ? cuts[row] : no_cut(vocab);
  auto mass = [&](double e, int i) {
    if (whole) return e;
    if (drawn) return fmax(e / z - q[i], 0.0);
    return bits[(i - first) >> 5] >> ((i - first) & 31) & 1 ? 0.0 : e;
  };
  double sum = 0;
  int tail = -1;
  each_mass<kBf16>(w, own, kVec, vocab, cut, st.max, req.temp, [&](double e, int i) {
    const double v = mass(e, i);
    sum += v;
    if (v > 0) tail = i;
  });
  double with = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double u = __shfl_up(with, o);
    if (lane >= o) with += u;
  }
  if (lane == 63) box[wave] = with;
  __syncthreads();
  double before = with - sum;
  for (int i = 0; i < wave; ++i) before += box[i];
  if (tail >= 0) atomicMax(&sh.tail, tail);
  if (sum > 0 && before + sum > target) {
    double at = before;
    int found = vocab;
    each_mass<kBf16>(w, own, kVec, vocab, cut, st.max, req.temp, [&](double e, int i) {
      const double v = mass(e, i);
      at += v;
      if (v > 0 && at > target && i < found) found = i;
    });
    atomicMin(&sh.found, found);
  }
  __syncthreads();
  // (a target that the share's own sum just misses by rounding takes its last token)
  if (tid == 0) next[b] = sh.found < vocab ? sh.found : max(sh.tail, 0);
}

int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }
int64_t share_count(int64_t vocab) { return (vocab + kShare - 1) / kShare; }

struct Room {
  int64_t cuts, shares, states, masses, rests, all;
};
Room room_of(int64_t rows, int64_t requests, int64_t vocab) {
  const int64_t n = share_count(vocab);
  requests = requests < kRequests ? requests : kRequests;
  Room r{};
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t from = at;
    at += align256(bytes);
    return from;
  };
  r.cuts = take(rows * static_cast<int64_t>(sizeof(RowCut)));
  r.shares = take(rows * n * static_cast<int64_t>(sizeof(Share)));
  r.states = take(requests * static_cast<int64_t>(sizeof(State)));
  r.masses = take(requests * n * static_cast<int64_t>(sizeof(Mass)));
  r.rests = take(requests * n * static_cast<int64_t>(sizeof(double)));
  r.all = at;
  return r;
}

template <bool kBf16>
void launch(hipStream_t st, const uint16_t *x, int64_t ld, int vocab, const Requests &req, bool cuts,
            const Tree &tree, char *ws, const Room &room, int32_t *paths, int levels,
            int32_t *lengths, int64_t *next, uint8_t *valid, bool first_rows) {
  const int n = static_cast<int>(share_count(vocab));
  auto *cut = reinterpret_cast<RowCut *>(ws + room.cuts);
  auto *shares = reinterpret_cast<Share *>(ws + room.shares);
  auto *states = reinterpret_cast<State *>(ws + room.states);
  auto *masses = reinterpret_cast<Mass *>(ws + room.masses);
  auto *rests = reinterpret_cast<double *>(ws + room.rests);
  if (cuts)
    hipLaunchKernelGGL((cut_kernel<kBf16, Requests>), dim3(req.rows), dim3(kCutThreads), 0, st, x,
                       ld, vocab, req, static_cast<int64_t *>(nullptr), cut);
  hipLaunchKernelGGL(mass_kernel<kBf16>, dim3(n, req.rows), dim3(kThreads), 0, st, x, ld, vocab, req,
                     cut, shares, valid, first_rows);
  hipLaunchKernelGGL(walk_kernel<kBf16>, dim3(n, req.count), dim3(kThreads), 0, st, x, ld, vocab,
                     req, cut, shares, tree, states, masses, paths, levels, lengths, next, valid);
  bool sampled = false;
  for (int b = 0; b < req.count; ++b) sampled = sampled || req.r[b].temp != 0.f;
  if (!sampled) return;
  if (tree.drafts)
    hipLaunchKernelGGL(rest_kernel<kBf16>, dim3(n, req.count), dim3(kThreads), 0, st, x, ld, vocab,
                       req, cut, tree, states, masses, rests);
  hipLaunchKernelGGL(pick_kernel<kBf16>, dim3(req.count), dim3(kThreads), 0, st, x, ld, vocab, req,
                     cut, tree, states, masses, rests, n, next);
}

}  // namespace
}  // namespace hy

extern "C" int64_t hy_verify_workspace_bytes(int32_t n_rows, int32_t num_seqs, int32_t vocab) {
  if (n_rows <= 0 || num_seqs <= 0 || vocab <= 0) return 0;
  return hy::room_of(n_rows, num_seqs, vocab).all;
}

extern "C" int hy_verify_tree(const void *logits, int64_t row_stride, int32_t dtype, int32_t vocab,
                              const int32_t *parents, const int64_t *tokens,
                              const int32_t *q_lens, int32_t num_seqs, const float *temperature,
                              const int32_t *top_k, const float *top_p, const float *uniforms,
                              const float *draft_probs, int64_t draft_stride, int32_t *paths,
                              int32_t levels, int32_t *lengths, int64_t *next_tokens,
                              uint8_t *valid, void *workspace, int64_t workspace_bytes,
                              void *stream) {
  hy::clear_error();
  HY_REQUIRE(num_seqs >= 0 && vocab >= 1 && levels >= 1, "hy_verify_tree: invalid sizes %d, %d, %d",
             num_seqs, vocab, levels);
  HY_REQUIRE(dtype == 0 || dtype == 1, "hy_verify_tree: dtype %d (0: bf16, 1: fp16)", dtype);
  HY_REQUIRE_SUPPORTED(vocab <= hy::kStep * hy::kMaxRounds, "hy_verify_tree: vocabulary %d too large",
                       vocab);
  if (num_seqs == 0) return HY_OK;
  HY_REQUIRE(logits && parents && tokens && q_lens && temperature && top_k && top_p && uniforms &&
                 paths && lengths && next_tokens && valid && workspace,
             "hy_verify_tree: null pointer argument");
  int64_t rows = 0;
  for (int32_t b = 0; b < num_seqs; ++b) {
    HY_REQUIRE(q_lens[b] >= 1 && q_lens[b] <= hy::kMaxNodes,
               "hy_verify_tree: tree %d has %d nodes, not 1 to %d", b, q_lens[b], hy::kMaxNodes);
    const float t = temperature[b];
    HY_REQUIRE_SUPPORTED(t == 0.f || (t >= 1e-30f && t <= 1e30f), "hy_verify_tree: temperature %g", t);
    HY_REQUIRE(top_k[b] >= 1 && top_p[b] > 0.f, "hy_verify_tree: request %d has top_k %d, top_p %g",
               b, top_k[b], top_p[b]);
    rows += q_lens[b];
  }
  HY_REQUIRE(rows <= INT32_MAX, "hy_verify_tree: too many rows");
  const hy::Room room = hy::room_of(rows, num_seqs, vocab);
  if (workspace_bytes < room.all) {
    hy::set_error("hy_verify_tree: workspace too small: need %lld bytes, got %lld",
                  static_cast<long long>(room.all), static_cast<long long>(workspace_bytes));
    return HY_ENOSPACE;
  }
  int64_t row0 = 0;
  for (int32_t b0 = 0; b0 < num_seqs; b0 += hy::kRequests) {
    hy::Requests req{};
    req.count = num_seqs - b0 < hy::kRequests ? num_seqs - b0 : hy::kRequests;
    bool cuts = false;
    for (int i = 0; i < req.count; ++i) {
      const int b = b0 + i;
      const int32_t k = top_k[b] < vocab ? top_k[b] : vocab;
      req.r[i] = {temperature[b], k, top_p[b], req.rows};
      req.rows += q_lens[b];
      cuts = cuts || (temperature[b] != 0.f && (k < vocab || top_p[b] < 1.f));
    }
    const hy::Tree tree{parents + row0, tokens + row0, uniforms + row0, uniforms + rows + b0,
                        draft_probs ? draft_probs + row0 * draft_stride : nullptr, draft_stride};
    (dtype == 0 ? hy::launch<true> : hy::launch<false>)(
        static_cast<hipStream_t>(stream), static_cast<const uint16_t *>(logits) + row0 * row_stride,
        row_stride, vocab, req, cuts, tree, static_cast<char *>(workspace), room,
        paths + static_cast<int64_t>(b0) * levels, levels, lengths + b0, next_tokens + b0, valid,
        b0 == 0);
    row0 += req.rows;
  }
  return hy::launch_status("hy_verify_tree");
}
