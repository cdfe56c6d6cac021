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
//   mass_kernel   many workgroups a row: the maximum and the sum of exponentials of each one's
//                 share of the logits (greedy: its largest logit).
//   cut_mass_kernel  instead, where a request has top-k or top-p: its rows are cut first (a
//                 workgroup each), and what the cut's counts sum up to is their mass, without a
//                 second read; the other rows' shares go to the CUs beside them. 16 trees of up
//                 to 26 nodes, half of them cut: 63.6 us a call with two launches and a second
//                 read, 60.0 without it, 47.3 in one launch (with two shares' loads in flight a
//                 workgroup 52.6: fewer, longer ones end later).
//   walk_kernel   the walk, in every workgroup of the request: its tests need the shares of its
//                 rows and a logit a node, a few reads that all nodes make at once. Then the
//                 masses of its part of the last node's row, in 64 bits: a border between
//                 two of 151,936 tokens is met by one draw in thousands of 32-bit sums. (Of
//                 max(p - q, 0) in the same pass, see Mass: in one of its own, once the row's sum
//                 was known, 32 chains of 5 took 46 us instead of 39.)
//   pick_kernel   the part that holds the draw, then the token; with few requests in the walk's
//                 last workgroup of each instead (see kPickers; with 32 requests, 20 us more).
//
// A call is bound by its chain of dependent launches: 8 nodes of 151,936 tokens take 3.9 us (mass)
// and 12.6 (walk and pick), less than the host's 23. With many rows the cuts lead (16 trees of up
// to 26 nodes: 30.4 with the masses, 10.9 and 6.8 us; a CU's reads and LDS counts), then the
// masses' exponentials (32 drawn chains of 5: 11, 17 and 8).

#include <algorithm>

#include "logit_rows.h"

namespace hy {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kShare = kThreads * kVec * kAhead;  // logits of a workgroup
constexpr int kRequests = 64;                     // requests of one launch
constexpr int kMaxNodes = 256;
// The last row of a path goes to more workgroups, a load of logits a thread: its masses in 64 bits
// take as long as one thread's chain of operations.
constexpr int kPart = kThreads * kVec;
// Workgroups of one walk launch, about: as many as run at once, so that none begins its walk when
// others end theirs. 32 drawn chains of 5 took 19.0, 19.2, 17.3 and 20.9 us at 768, 1024, 1536 and
// 2048, 16 trees of 26 nodes 11.9, 13.6, 10.8 and 10.8.
constexpr int kWalkers = 1536;

// A workgroup's share of a row: the largest kept logit and the sum of exp((x - max) / temp); of a
// greedy row rank_of() of the largest.
struct Share {
  float max, sum;
  uint64_t best;
};
// Workgroups of a walk up to which its last ones pick. In a row, without and with a launch for the
// picks (us, 151,936 tokens): 1 request 23.5 and 28.4, 4 (300 workgroups) 23.6 and 28.6, 16 chains
// of 32,000 tokens (256) 26.8 and 31.5; 16 trees of 26 (1,200) 50.6 and 47.3. In a graph, where the
// host does not count, 17.3 and 17.3, 20.4 and 18.8, 19.5 and 18.3: each workgroup's release, the
// count and the last one's acquire are dependent trips, which many workgroups wait for.
constexpr int kPickers = 320;

struct Request {
  float temp;
  int32_t k;
  float p;
  int32_t first;       // its first row
  int32_t cut_before;  // rows before it that are cut
};
struct Requests {
  static constexpr bool kCutsOnly = true;
  Request r[kRequests];
  int32_t count, rows;
  Share *shares;
  int32_t n_shares;  // of a row

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
  // The i-th row that is cut, or that is not.
  __device__ __forceinline__ int nth_row(bool is_cut, int i) const {
    auto before = [&](int b) { return is_cut ? r[b].cut_before : r[b].first - r[b].cut_before; };
    int lo = 0, hi = count;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (before(mid) <= i)
        lo = mid;
      else
        hi = mid;
    }
    return r[lo].first + i - before(lo);
  }
  __device__ __forceinline__ int nodes(int b) const {
    return (b + 1 < count ? r[b + 1].first : rows) - r[b].first;
  }
  __device__ __forceinline__ SampleRow row(int i) const {
    const Request &q = r[of_row(i)];
    return {q.temp, q.k, q.p, 0};
  }
  // Row i's shares, by the whole workgroup: the first has all of it.
  __device__ __forceinline__ void mass(int i, float max, float sum) const {
    for (int x = threadIdx.x; x < n_shares; x += blockDim.x) {
      Share *s = shares + static_cast<int64_t>(i) * n_shares + x;
      s->max = x == 0 ? max : -INFINITY;
      s->sum = x == 0 ? sum : 0.f;
    }
  }
  __device__ __forceinline__ bool cut(int b, int vocab) const {
    return r[b].temp != 0.f && (r[b].k < vocab || r[b].p < 1.f);
  }
};

// Masses of a part of a request's last row: all of it, and what the draw is from. Where that is
// max(p - q, 0), `left` and `drafts` are the sums of exp and of q over the tokens with p > q:
// left / sum - drafts, once all parts have told the row's sum. (Which tokens these are goes by the
// shares' sum; one on the wrong side differs from 0 by the error of that sum times q.)
struct Mass {
  double all, left, drafts;
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

// This thread's logits of a share: loads of kVec, load a from index first + a * step on.
// Past the row's end the last logit is repeated.
template <int kLoads>
__device__ __forceinline__ void load_share(const uint16_t *x, int vocab, int first, int step,
                                           u32x4 (&w)[kLoads]) {
#pragma unroll
  for (int a = 0; a < kLoads; ++a) {
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
// The j-th logit of a load.
template <bool kBf16>
__device__ __forceinline__ float value_in(const u32x4 &w, int j) {
  const uint32_t word = w[j >> 1];
  if (kBf16) return j & 1 ? bf16_hi(word) : bf16_lo(word);
  return static_cast<float>(
      __builtin_bit_cast(_Float16, static_cast<uint16_t>(j & 1 ? word >> 16 : word)));
}
// Where a row is cut, by value: logits of at least `low`, except those that are `at` and come
// after `last`.
struct Cut {
  float low, at;
  int last;
  bool ok;
  __device__ __forceinline__ bool keeps(float x, int index) const {
    return x >= low && !(x == at && index > last);
  }
};
__device__ __forceinline__ Cut no_cut() { return {-INFINITY, NAN, 0, true}; }
template <bool kBf16>
__device__ __forceinline__ Cut cut_of(const RowCut &c) {
  return {c.low > 0 ? value_of<kBf16>(c.low) : -INFINITY, c.cut > 0 ? value_of<kBf16>(c.cut) : NAN,
          c.last, c.ok == 1};
}

// Rotations within a row of 16 lanes, and the sums and maxima made of them: register moves, where
// a shuffle of 64 bits takes two trips through LDS.
template <int N>
__device__ __forceinline__ uint32_t ror(uint32_t x) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_mov_dpp(static_cast<int>(x), 0x120 + N, 0xf, 0xf, false));
}
template <int N>
__device__ __forceinline__ double ror(double x) {
  const uint64_t u = static_cast<uint64_t>(__double_as_longlong(x));
  const uint64_t hi = ror<N>(static_cast<uint32_t>(u >> 32)), lo = ror<N>(static_cast<uint32_t>(u));
  return __longlong_as_double(static_cast<long long>(hi << 32 | lo));
}
__device__ __forceinline__ double row_sum(double v) {
  v += ror<8>(v);
  v += ror<4>(v);
  v += ror<2>(v);
  return v + ror<1>(v);
}
__device__ __forceinline__ float row_max(float v) {
  v = fmaxf(v, __uint_as_float(ror<8>(__float_as_uint(v))));
  v = fmaxf(v, __uint_as_float(ror<4>(__float_as_uint(v))));
  v = fmaxf(v, __uint_as_float(ror<2>(__float_as_uint(v))));
  return fmaxf(v, __uint_as_float(ror<1>(__float_as_uint(v))));
}
__device__ __forceinline__ float lane_of(float v, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}
__device__ __forceinline__ double lane_of(double v, int lane) {
  const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v));
  const uint64_t hi = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(u >> 32), lane));
  const uint64_t lo = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(u), lane));
  return __longlong_as_double(static_cast<long long>(hi << 32 | lo));
}
// Over all 64 lanes, which take part.
__device__ __forceinline__ double wave_sum(double v) {
  v = row_sum(v);
  return (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
}
// Over each kThreads of the workgroup, in a fixed order and in every thread: of two values at once.
struct Pair {
  double a, b;
};
__device__ __forceinline__ Pair block_sums(double a, double b, Pair *box) {
  const Pair mine = {wave_sum(a), wave_sum(b)};
  __syncthreads();
  if ((threadIdx.x & 63) == 0) box[(threadIdx.x >> 6) % kWaves] = mine;
  __syncthreads();
  Pair all = box[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) {
    all.a += box[i].a;
    all.b += box[i].b;
  }
  return all;
}

// The first largest logit of a share as rank_of() has it; a NaN is the largest of all.
// Keys in pairs: of three operations a logit nothing but the maximum comes, and the threads
// that hold it look for its place.
template <bool kBf16>
__device__ __forceinline__ uint64_t best_of_share(const u32x4 (&w)[kAhead], int first, int step,
                                                  int vocab, uint32_t *top_box, int *first_box) {
  constexpr uint32_t kInf = kInfBits<kBf16>;
  const int lane = threadIdx.x & 63, wave = (threadIdx.x >> 6) % kWaves;
  u16x2 top2 = {0, 0}, mag2 = {0, 0};
#pragma unroll
  for (int a = 0; a < kAhead; ++a)
#pragma unroll
    for (int j = 0; j < kVec / 2; ++j) {
      const uint32_t word = keys_of(w[a][j]);
      const uint32_t mag = w[a][j] & 0x7fff7fffu;
      top2 = __builtin_elementwise_max(top2, __builtin_bit_cast(u16x2, word));
      mag2 = __builtin_elementwise_max(mag2, __builtin_bit_cast(u16x2, mag));
    }
  // (what a tail repeats past the row's end changes neither)
  uint32_t top = max(top2[0], top2[1]);
  const bool nan = max(mag2[0], mag2[1]) > kInf;
  if (top == 0x7fffu) top = 0x8000u;  // zeros are one value
  if (nan) top = 0x10000u;
  uint32_t t = top;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) t = max(t, static_cast<uint32_t>(__shfl_xor(static_cast<int>(t), o)));
  if (lane == 0) top_box[wave] = t;
  if (threadIdx.x % kThreads == 0) *first_box = vocab;
  __syncthreads();
  t = top_box[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) t = max(t, top_box[i]);
  if (top == t) {
    int at = vocab;
#pragma unroll
    for (int a = kAhead - 1; a >= 0; --a)
#pragma unroll
      for (int j = kVec - 1; j >= 0; --j) {
        const uint32_t bits = w[a][j >> 1] >> (16 * (j & 1)) & 0xffffu;
        const bool is = t == 0x10000u ? (bits & 0x7fffu) > kInf : merge_zero(keys_of(bits) & 0xffffu) == t;
        const int i = first + a * step + j;
        if (is && i < vocab) at = i;
      }
    atomicMin(first_box, at);
  }
  __syncthreads();
  return rank_of(t, *first_box);
}

struct MassRoom {
  float maxes[kWaves];
  uint32_t tops[kWaves];
  int place;
  double sums[kWaves];
};
// One share of a row that is not cut, by kThreads threads; the others of the workgroup have
// shares of the same row.
template <bool kBf16>
__device__ __forceinline__ void mass_of_share(const uint16_t *row, int vocab, float temp, int share,
                                              int n_shares, Share *shares, MassRoom &room) {
  const int tid = threadIdx.x % kThreads;
  constexpr int kRound = kThreads * kVec;
  const int i0 = min(share, n_shares - 1) * kShare + kVec * tid;
  u32x4 w[kAhead];
  load_share(row, vocab, i0, kRound, w);
  const bool tells = tid == 0 && share < n_shares;
  Share *out = shares + share;
  if (temp == 0.f) {
    const uint64_t best = best_of_share<kBf16>(w, i0, kRound, vocab, room.tops, &room.place);
    if (tells) out->best = best;
    return;
  }
  float x[kAhead][kVec], m = -INFINITY;
#pragma unroll
  for (int a = 0; a < kAhead; ++a)
#pragma unroll
    for (int j = 0; j < kVec; ++j) x[a][j] = value_in<kBf16>(w[a], j);
  if ((share + 1) * static_cast<int64_t>(kShare) > vocab) {
#pragma unroll
    for (int a = 0; a < kAhead; ++a)
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        if (i0 + a * kRound + j >= vocab) x[a][j] = -INFINITY;
  }
#pragma unroll
  for (int a = 0; a < kAhead; ++a)
#pragma unroll
    for (int j = 0; j < kVec; ++j) m = fmaxf(m, x[a][j]);
  m = row_max(m);
  m = fmaxf(fmaxf(lane_of(m, 0), lane_of(m, 16)), fmaxf(lane_of(m, 32), lane_of(m, 48)));
  if ((threadIdx.x & 63) == 0) room.maxes[tid >> 6] = m;
  __syncthreads();
  m = room.maxes[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) m = fmaxf(m, room.maxes[i]);
  const float slope = 1.0f / temp * kLog2eS;
  // The differences are scaled, not the terms: at small temperatures those are far apart. NaN,
  // and infinities less each other, make the sum NaN; a share without a finite logit is
  // measured from 0.
  const float from = m == -INFINITY ? 0.f : m;
  float s = 0.f;
#pragma unroll
  for (int a = 0; a < kAhead; ++a)
#pragma unroll
    for (int j = 0; j < kVec; ++j) s += __builtin_amdgcn_exp2f((x[a][j] - from) * slope);
  const double mine = wave_sum(static_cast<double>(s));
  if ((threadIdx.x & 63) == 0) room.sums[tid >> 6] = mine;
  __syncthreads();
  double sum = room.sums[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) sum += room.sums[i];
  if (tells) {
    out->max = sum == sum ? m : NAN;
    out->sum = static_cast<float>(sum);
  }
}

// What the walk starts from: no part is done, nothing is bad.
__device__ __forceinline__ void begin(const Requests &requests, int32_t *done, uint8_t *valid,
                                      bool first_rows) {
  if (static_cast<int>(threadIdx.x) < requests.count) done[threadIdx.x] = 0;
  if (first_rows && threadIdx.x == 0) *valid = 1;
}

// Grid (shares, rows): no row is cut.
template <bool kBf16>
__global__ __launch_bounds__(kThreads) void mass_kernel(const uint16_t *__restrict__ logits, int64_t ld,
                                                        int vocab, Requests requests,
                                                        int32_t *__restrict__ done,
                                                        uint8_t *__restrict__ valid, bool first_rows) {
  __shared__ MassRoom room;
  if (blockIdx.x == 0 && blockIdx.y == 0) begin(requests, done, valid, first_rows);
  const int row = blockIdx.y;
  mass_of_share<kBf16>(logits + row * ld, vocab, requests.r[requests.of_row(row)].temp, blockIdx.x,
                       gridDim.x, requests.shares + static_cast<int64_t>(row) * gridDim.x, room);
}

// The first n_cut workgroups find the cuts, a row each; the others, four shares each, fill the
// CUs beside them.
template <bool kBf16>
__global__ __launch_bounds__(kCutThreads) void cut_mass_kernel(
    const uint16_t *__restrict__ logits, int64_t ld, int vocab, Requests requests, int n_cut,
    RowCut *__restrict__ cuts, int32_t *__restrict__ done, uint8_t *__restrict__ valid,
    bool first_rows) {
  constexpr int kShares = kCutThreads / kThreads;
  __shared__ MassRoom rooms[kShares];
  if (blockIdx.x == 0) begin(requests, done, valid, first_rows);
  const int block = blockIdx.x;
  if (block < n_cut) {
    cut_row<kBf16>(logits, ld, vocab, requests, requests.nth_row(true, block), nullptr, cuts);
    return;
  }
  const int per_row = (requests.n_shares + kShares - 1) / kShares, group = threadIdx.x / kThreads;
  const int row = requests.nth_row(false, (block - n_cut) / per_row);
  mass_of_share<kBf16>(logits + row * ld, vocab, requests.r[requests.of_row(row)].temp,
                       (block - n_cut) % per_row * kShares + group, requests.n_shares,
                       requests.shares + static_cast<int64_t>(row) * requests.n_shares, rooms[group]);
}

// exp(x), x <= 0, to about 1e-12: 2^n times the Taylor series of the rest, |r| <= ln(2) / 2 and a
// little, its terms from the sixth on (r^6 / 720 < 3e-6) in 32 bits. Operations of 64 bits bound
// the kernels that call it: with the fourth and fifth term in 32 bits as well (1e-10, which one
// draw in ten thousand notices where little of p is left) 32 drawn chains take 0.8 us less.
__device__ __forceinline__ double exp_of(double x) {
  constexpr long double kLn2 = 0.693147180559945309417232L;
  constexpr double kHead = 45426.0 / 65536;  // n times it is exact
  constexpr double kTail = static_cast<double>(kLn2 - 45426.0L / 65536);
  const float n = rintf(static_cast<float>(x) * static_cast<float>(1 / kLn2));
  double r = fma(static_cast<double>(n), -kHead, x);
  r = fma(static_cast<double>(n), -kTail, r);
  const float s = static_cast<float>(r);
  float q = 1.0f / 39916800;
#pragma unroll
  for (const float c : {1.0f / 3628800, 1.0f / 362880, 1.0f / 40320, 1.0f / 5040, 1.0f / 720})
    q = __builtin_fmaf(q, s, c);
  double p = static_cast<double>(q);
#pragma unroll
  for (const double c : {1.0 / 120, 1.0 / 24, 1.0 / 6, 0.5, 1.0, 1.0}) p = fma(p, r, c);
  return x < -740.0 ? 0.0 : ldexp(p, static_cast<int>(n));
}

// exp((x - max) / temp) of kVec logits from index `first` on, 0 for those cut off. Without a
// branch, so that the eight chains of dependent operations run side by side.
template <bool kBf16>
__device__ __forceinline__ void masses_of(const u32x4 &w, int first, int vocab, const Cut &cut,
                                          double max, double inv_temp, double (&e)[kVec]) {
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    const float x = value_in<kBf16>(w, j);
    const double mass = exp_of((static_cast<double>(x) - max) * inv_temp);
    e[j] = first + j < vocab && cut.keeps(x, first + j) ? mass : 0.0;
  }
}

// kVec draft probabilities from index i on; past the row's end the last one.
__device__ __forceinline__ void load_drafts(const float *q, int i, int vocab, float (&v)[kVec]) {
  if (i + kVec <= vocab) {
    __builtin_memcpy(v, q + i, sizeof(v));
  } else {
#pragma unroll
    for (int j = 0; j < kVec; ++j) v[j] = q[min(i + j, vocab - 1)];
  }
}

// Marks the tokens of a part that the draw leaves out, those of the last node's children: every
// thread has a node (or -1 as its parent) and its token.
__device__ __forceinline__ void mark_refused(uint32_t *bits, int parent, int64_t token, int last,
                                             int first) {
  static_assert(kThreads >= kMaxNodes, "a node a thread");
  static_assert(kPart / 32 <= kThreads, "a word a thread");
  __syncthreads();  // earlier readers are done
  if (threadIdx.x < kPart / 32) bits[threadIdx.x] = 0;
  __syncthreads();
  const int64_t at = token - first;
  if (parent == last && at >= 0 && at < kPart) atomicOr(&bits[at >> 5], 1u << (at & 31));
  __syncthreads();
}

// What a wave has found of a place: the first one behind the target and the last with any mass,
// -1 where there is none, and what of the target is left at their start.
struct Found {
  int past, last;
  double past_rest, last_rest;
};
struct PickRoom {
  double all[kWaves], left[kWaves];
  Found parts[kWaves], tokens[kWaves];
};
// Neighbouring lanes hold neighbouring places. (Ballots: an LDS atomic of 64 lanes on one word
// is taken lane by lane, 2 us.)
__device__ __forceinline__ void tell_found(Found *of_wave, bool past, bool any, int place, double rest) {
  const uint64_t p = __ballot(past), a = __ballot(any);
  const int first = p ? __ffsll(static_cast<long long>(p)) - 1 : 0;
  const int last = a ? 63 - __clzll(static_cast<long long>(a)) : 0;
  const Found f = {p ? __shfl(place, first) : -1, a ? __shfl(place, last) : -1, __shfl(rest, first),
                   __shfl(rest, last)};
  if ((threadIdx.x & 63) == 0) of_wave[threadIdx.x >> 6] = f;
}
// The first place behind the target, else the last with any mass (0 if there is none).
__device__ __forceinline__ int take_found(const Found *of_waves, double &rest) {
  int place = -1, last = 0;
  double last_rest = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    if (place < 0 && of_waves[i].past >= 0) {
      place = of_waves[i].past;
      rest = of_waves[i].past_rest;
    }
    if (of_waves[i].last >= 0) {
      last = of_waves[i].last;
      last_rest = of_waves[i].last_rest;
    }
  }
  if (place >= 0) return place;
  rest = last_rest;
  return last;
}

// The draw of one request, by a whole workgroup: the smallest token whose running mass exceeds
// `number` times the total (where rounding leaves none, the last token with any). The masses are
// max(p - q, 0) with q (the row of draft probabilities), else those of p without the children of
// `last`, of which every thread has one's parent and token.
template <bool kBf16>
__device__ __forceinline__ int pick_token(const uint16_t *row, int vocab, const Cut &cut, float max,
                                          double inv_temp, double number, const Mass *masses,
                                          const float *q, int n_parts, int parent, int64_t token,
                                          int last, uint32_t *bits, PickRoom &room) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  auto scan = [&](double v) __attribute__((always_inline)) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double u = __shfl_up(v, o);
      if (lane >= o) v += u;
    }
    return v;
  };
  // A thread has neighbouring parts.
  const int per = (n_parts + kThreads - 1) / kThreads;
  const int from = min(tid * per, n_parts), to = min(from + per, n_parts);
  // The sum before this thread's own, and of all.
  auto sums = [&](double own, double *box, double &before) __attribute__((always_inline)) {
    const double with = scan(own);
    if (lane == 63) box[wave] = with;
    __syncthreads();
    double total = 0;
    before = with - own;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      if (i < wave) before += box[i];
      total += box[i];
    }
    return total;
  };
  double all = 0, left = 0, all_before, left_before;
  for (int i = from; i < to; ++i) all += masses[i].all;
  const double z = sums(all, room.all, all_before), inv_z = 1.0 / z;
  auto left_of = [&](const Mass &m) {
    return q ? fmax(fma(m.left, inv_z, -m.drafts), 0.0) : m.left;
  };
  for (int i = from; i < to; ++i) left += left_of(masses[i]);
  const double some = sums(left, room.left, left_before);
  const bool whole = !(some > 0);  // where nothing is left, all of p
  const double target = number * (whole ? z : some);
  const double own = whole ? all : left, before = whole ? all_before : left_before;
  int part = 0;  // of this thread's: where the sum passes the target, or the last with any mass
  double rest = 0;
  if (own > 0) {
    double at = before;
    for (int i = from; i < to; ++i) {
      const double v = whole ? masses[i].all : left_of(masses[i]);
      if (v > 0) {
        part = i;
        rest = target - at;
        if (at + v > target) break;
      }
      at += v;
    }
  }
  tell_found(room.parts, own > 0 && before + own > target, own > 0, part, rest);
  __syncthreads();
  const int chosen = take_found(room.parts, rest);
  const int first = chosen * kPart, at = kVec * tid, mine = first + at;
  u32x4 w[1];
  load_share(row, vocab, mine, 0, w);
  mark_refused(bits, whole || q ? -2 : parent, token, last, first);
  double e[kVec];
  masses_of<kBf16>(w[0], mine, vocab, cut, max, inv_temp, e);
  if (!whole && q) {
    float qv[kVec];
    load_drafts(q, mine, vocab, qv);
#pragma unroll
    for (int j = 0; j < kVec; ++j)
      e[j] = mine + j < vocab ? fmax(fma(e[j], inv_z, -static_cast<double>(qv[j])), 0.0) : 0.0;
  }
  const uint32_t out = bits[at >> 5] >> (at & 31);
  double sum = 0;
  int tail = -1;
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    e[j] = out >> j & 1 ? 0.0 : e[j];
    sum += e[j];
    if (e[j] > 0) tail = mine + j;
  }
  const double with = scan(sum);
  if (lane == 63) room.all[wave] = with;
  __syncthreads();
  double running = with - sum;
  for (int i = 0; i < wave; ++i) running += room.all[i];
  int found = -1;
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    running += e[j];
    if (found < 0 && e[j] > 0 && running > rest) found = mine + j;
  }
  tell_found(room.tokens, found >= 0, tail >= 0, found >= 0 ? found : tail, 0.0);
  __syncthreads();
  return take_found(room.tokens, rest);
}

// Grid (parts or fewer, requests). kPicks: the workgroup of a request that is done last picks.
template <bool kBf16, bool kPicks>
__global__ __launch_bounds__(kThreads) void walk_kernel(
    const uint16_t *__restrict__ logits, int64_t ld, int vocab, Requests requests,
    const RowCut *__restrict__ cuts, const Share *__restrict__ shares, int n_shares,
    int n_parts, Tree tree,
    State *__restrict__ states, Mass *__restrict__ masses, int32_t *__restrict__ done,
    int32_t *__restrict__ paths, int levels, int32_t *__restrict__ lengths,
    int64_t *__restrict__ next, uint8_t *__restrict__ valid) {
  __shared__ float max_of[kMaxNodes];
  __shared__ double sum_of[kMaxNodes];
  __shared__ double p_of[kMaxNodes];  // p(x) of a node's token under its parent; greedy: 1 or 0
  __shared__ double q_of[kMaxNodes];
  __shared__ float u_of[kMaxNodes];
  __shared__ int best_of[kMaxNodes], token_of[kMaxNodes], refused[kMaxNodes];
  __shared__ State sh;
  __shared__ uint32_t bits[kPart / 32];
  __shared__ Pair box[kWaves];
  __shared__ PickRoom room;
  __shared__ bool picks;
  const int b = blockIdx.y;
  const Request req = requests.r[b];
  const int nodes = requests.nodes(b), row0 = req.first;
  const bool greedy = req.temp == 0.f, cut_rows = requests.cut(b, vocab);
  const double inv_temp = greedy ? 0.0 : 1.0 / req.temp;
  const int32_t *parents = tree.parents + row0;
  const int64_t *tokens = tree.tokens + row0;
  const int tid = threadIdx.x, lane = tid & 63;

  // (all loads that depend on nothing go out before the first is waited for)
  const int mine = min(tid, nodes - 1);
  const int64_t my_token = tokens[mine];
  const int32_t up = min(max(parents[mine], 0), max(mine - 1, 0));
  const float my_u = tree.uniforms[row0 + mine];
  int par[kMaxNodes / 64];  // of nodes 64 i + lane
#pragma unroll
  for (int i = 0; i < kMaxNodes / 64; ++i) {
    par[i] = parents[min(64 * i + lane, nodes - 1)];
    if (64 * i + lane >= nodes || 64 * i + lane == 0) par[i] = -1;
  }
  // Every row's maximum and sum (or largest logit), from its shares: 16 lanes a row.
  const int l16 = tid & 15;
  const float slope = greedy ? 0.f : 1.0f / req.temp * kLog2eS;
  for (int r0 = 0; r0 < nodes; r0 += kThreads / 16) {
    const int r = r0 + (tid >> 4);
    const Share *s = shares + static_cast<int64_t>(row0 + min(r, nodes - 1)) * n_shares;
    if (greedy) {
      uint64_t top = 0;
      for (int i = l16; i < n_shares; i += 16) top = s[i].best > top ? s[i].best : top;
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) {
        const uint64_t t = __shfl_xor(static_cast<unsigned long long>(top), o);
        top = t > top ? t : top;
      }
      if (l16 == 0 && r < nodes) best_of[r] = index_of(top);
      continue;
    }
    float m = -INFINITY;
    for (int i = l16; i < n_shares; i += 16) m = fmaxf(m, s[i].max);
    m = row_max(m);
    const float from = m == -INFINITY ? 0.f : m;
    double z = 0;  // (a share's NaN makes it NaN)
    for (int i = l16; i < n_shares; i += 16)
      z += static_cast<double>(s[i].sum * __builtin_amdgcn_exp2f((s[i].max - from) * slope));
    z = row_sum(z);
    if (l16 == 0 && r < nodes) {
      max_of[r] = z != z || isinf(m / req.temp) ? NAN : m;
      sum_of[r] = z;
    }
  }
  const int x = my_token >= 0 && my_token < vocab ? static_cast<int>(my_token) : -1;
  if (tid < nodes) {
    token_of[tid] = x;
    u_of[tid] = my_u;
  }
  __syncthreads();
  if (tid > 0 && tid < nodes) {
    double p = 0, q = 0;
    if (greedy) {
      p = x == best_of[up];
    } else if (x >= 0) {
      const u32x4 word = {logits[(row0 + up) * ld + x], 0u, 0u, 0u};
      const Cut cut = cut_rows ? cut_of<kBf16>(cuts[row0 + up]) : no_cut();
      if (tree.drafts) q = tree.drafts[(row0 + tid) * tree.drafts_ld + x];
      const float v = value_in<kBf16>(word, 0);
      if (cut.keeps(v, x)) p = exp_of((static_cast<double>(v) - max_of[up]) * inv_temp) / sum_of[up];
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
        if (!kPicks) states[b] = sh;
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
  const int row = row0 + sh.last, at = kVec * tid;
  const uint16_t *x_row = logits + row * ld;
  const Cut cut = cut_rows ? cut_of<kBf16>(cuts[row]) : no_cut();
  const int my_parent = tree.drafts || tid == 0 || tid >= nodes ? -2 : up;
  const bool drawn = tree.drafts && sh.child >= 0;  // the draw is from max(p - q, 0)
  const float *q = drawn ? tree.drafts + (row0 + sh.child) * tree.drafts_ld : nullptr;
  const double inv_sum = 1.0 / sum_of[sh.last];
  u32x4 w[1];
  load_share(x_row, vocab, blockIdx.x * kPart + at, 0, w);
  for (int part = blockIdx.x; part < n_parts; part += gridDim.x) {
    const int first = part * kPart;
    mark_refused(bits, my_parent, my_token, sh.last, first);
    const uint32_t out = bits[at >> 5] >> (at & 31);
    double e[kVec], all = 0, left = 0, drafts = 0;
    float qv[kVec];
    if (drawn) load_drafts(q, first + at, vocab, qv);
    masses_of<kBf16>(w[0], first + at, vocab, cut, sh.max, inv_temp, e);
    if (part + static_cast<int>(gridDim.x) < n_parts)
      load_share(x_row, vocab, first + static_cast<int>(gridDim.x) * kPart + at, 0, w);
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      // (e is 0 past the row's end)
      const bool in = drawn ? e[j] * inv_sum > qv[j] : !(out >> j & 1);
      all += e[j];
      left += in ? e[j] : 0.0;
      if (drawn) drafts += in ? qv[j] : 0.0;
    }
    const Pair sums = block_sums(all, left, box);
    if (drawn) drafts = block_sums(drafts, 0.0, box).a;
    if (tid == 0) masses[static_cast<int64_t>(b) * n_parts + part] = {sums.a, sums.b, drafts};
  }
  if constexpr (!kPicks) return;
  if (tid == 0) {
    const int mine = (n_parts - 1 - static_cast<int>(blockIdx.x)) / static_cast<int>(gridDim.x) + 1;
    picks = __hip_atomic_fetch_add(done + b, mine, __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_AGENT) + mine ==
            n_parts;
  }
  __syncthreads();
  if (!picks) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
  const int got = pick_token<kBf16>(x_row, vocab, cut, sh.max, inv_temp, tree.draws[b],
                                    masses + static_cast<int64_t>(b) * n_parts, q, n_parts, my_parent,
                                    my_token, sh.last, bits, room);
  if (tid == 0) next[b] = got;
}

// Grid (requests).
template <bool kBf16>
__global__ __launch_bounds__(kThreads) void pick_kernel(
    const uint16_t *__restrict__ logits, int64_t ld, int vocab, Requests requests,
    const RowCut *__restrict__ cuts, Tree tree, const State *__restrict__ states,
    const Mass *__restrict__ masses, int n_parts, int64_t *__restrict__ next) {
  __shared__ uint32_t bits[kPart / 32];
  __shared__ PickRoom room;
  const int b = blockIdx.x, tid = threadIdx.x;
  const Request req = requests.r[b];
  if (req.temp == 0.f) return;
  // (loads that depend on nothing go out first)
  const int nodes = requests.nodes(b), mine = req.first + min(tid, nodes - 1);
  const int parent = tree.drafts || tid == 0 || tid >= nodes ? -2 : tree.parents[mine];
  const int64_t token = tree.tokens[mine];
  const double number = tree.draws[b];
  const State st = states[b];
  if (st.bad) return;
  const int row = req.first + st.last;
  const Cut cut = requests.cut(b, vocab) ? cut_of<kBf16>(cuts[row]) : no_cut();
  const bool drawn = tree.drafts && st.child >= 0;  // the draw is from max(p - q, 0)
  const int got = pick_token<kBf16>(
      logits + row * ld, vocab, cut, st.max, 1.0 / req.temp, number,
      masses + static_cast<int64_t>(b) * n_parts,
      drawn ? tree.drafts + (req.first + st.child) * tree.drafts_ld : nullptr, n_parts, parent, token,
      st.last, bits, room);
  if (tid == 0) next[b] = got;
}

int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }
int64_t share_count(int64_t vocab) { return (vocab + kShare - 1) / kShare; }
int64_t part_count(int64_t vocab) { return (vocab + kPart - 1) / kPart; }

struct Room {
  int64_t cuts, shares, states, done, masses, all;
};
Room room_of(int64_t rows, int64_t requests, int64_t vocab) {
  const int64_t n = share_count(vocab), parts = part_count(vocab);
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
  r.done = take(requests * static_cast<int64_t>(sizeof(int32_t)));
  r.masses = take(requests * parts * static_cast<int64_t>(sizeof(Mass)));
  r.all = at;
  return r;
}

template <bool kBf16>
void launch(hipStream_t st, const uint16_t *x, int64_t ld, int vocab, Requests &req, int n_cut,
            const Tree &tree, char *ws, const Room &room, int32_t *paths, int levels,
            int32_t *lengths, int64_t *next, uint8_t *valid, bool first_rows) {
  const int n = static_cast<int>(share_count(vocab)), parts = static_cast<int>(part_count(vocab));
  auto *cut = reinterpret_cast<RowCut *>(ws + room.cuts);
  auto *shares = reinterpret_cast<Share *>(ws + room.shares);
  auto *states = reinterpret_cast<State *>(ws + room.states);
  auto *done = reinterpret_cast<int32_t *>(ws + room.done);
  auto *masses = reinterpret_cast<Mass *>(ws + room.masses);
  req.shares = shares;
  req.n_shares = n;
  if (n_cut > 0) {
    constexpr int kShares = kCutThreads / kThreads;
    const int64_t blocks = n_cut + static_cast<int64_t>(req.rows - n_cut) * ((n + kShares - 1) / kShares);
    hipLaunchKernelGGL(cut_mass_kernel<kBf16>, dim3(static_cast<uint32_t>(blocks)), dim3(kCutThreads),
                       0, st, x, ld, vocab, req, n_cut, cut, done, valid, first_rows);
  } else {
    hipLaunchKernelGGL(mass_kernel<kBf16>, dim3(n, req.rows), dim3(kThreads), 0, st, x, ld, vocab, req,
                       done, valid, first_rows);
  }
  bool sampled = false;
  for (int b = 0; b < req.count; ++b) sampled = sampled || req.r[b].temp != 0.f;
  // Every workgroup of a request repeats its walk: no more of them than fill the GPU.
  const int walkers = sampled ? std::min(parts, std::max(1, kWalkers / req.count)) : 1;
  const bool picks = walkers * req.count <= kPickers;
  auto walk = picks ? walk_kernel<kBf16, true> : walk_kernel<kBf16, false>;
  hipLaunchKernelGGL(walk, dim3(walkers, req.count), dim3(kThreads), 0, st, x, ld, vocab, req, cut,
                     shares, n, parts, tree, states, masses, done, paths, levels, lengths, next, valid);
  if (!sampled || picks) return;
  hipLaunchKernelGGL(pick_kernel<kBf16>, dim3(req.count), dim3(kThreads), 0, st, x, ld, vocab, req,
                     cut, tree, states, masses, parts, next);
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
    int n_cut = 0;
    for (int i = 0; i < req.count; ++i) {
      const int b = b0 + i;
      const int32_t k = top_k[b] < vocab ? top_k[b] : vocab;
      req.r[i] = {temperature[b], k, top_p[b], req.rows, n_cut};
      req.rows += q_lens[b];
      if (temperature[b] != 0.f && (k < vocab || top_p[b] < 1.f)) n_cut += q_lens[b];
    }
    const hy::Tree tree{parents + row0, tokens + row0, uniforms + row0, uniforms + rows + b0,
                        draft_probs ? draft_probs + row0 * draft_stride : nullptr, draft_stride};
    (dtype == 0 ? hy::launch<true> : hy::launch<false>)(
        static_cast<hipStream_t>(stream), static_cast<const uint16_t *>(logits) + row0 * row_stride,
        row_stride, vocab, req, n_cut, tree, static_cast<char *>(workspace), room,
        paths + static_cast<int64_t>(b0) * levels, levels, lengths + b0, next_tokens + b0, valid,
        b0 == 0);
    row0 += req.rows;
  }
  return hy::launch_status("hy_verify_tree");
}
