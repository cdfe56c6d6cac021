// Rows of 16-bit logits, shared by sampling and by the verification of drafted tokens: ordered
// keys, scores, and the kernel that finds where top-k and top-p cut a row.
#pragma once

#include <math.h>

#include <type_traits>

#include "hy_common.h"

namespace hy {
namespace {

constexpr int kCutThreads = 1024;
constexpr int kCutWaves = kCutThreads / 64;
constexpr int kWords = 32768;                  // histogram words
constexpr int kVec = 8;                        // logits per load
constexpr int kAhead = 4;                      // loads in flight per thread
constexpr int kStep = kVec * kCutThreads;      // logits per round of the workgroup
constexpr int kMaxRounds = 512;                // rounds whose tie counts fit LDS
constexpr float kLog2eS = 1.4426950408889634f;

typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

struct SampleRow {
  float temp;     // 0: greedy
  int32_t k;      // of top-k, vocabulary size for none
  float p;        // of top-p, >= 1 for none
  int32_t noise;  // row of the noise
};
// What the cut leaves of a row: keys >= low, except those == cut past index last.
struct RowCut {
  int32_t low, cut, last, ok;
  float max;  // largest score
};

// Ordered keys of two 16-bit floats: larger key, larger value.
__device__ __forceinline__ uint32_t keys_of(uint32_t w) {
  const s16x2 sign = __builtin_bit_cast(s16x2, w) >> 15;
  return w ^ ((__builtin_bit_cast(uint32_t, sign) & 0x7fff7fffu) | 0x80008000u);
}
// -0 counts as +0.
__device__ __forceinline__ uint32_t merge_zero(uint32_t key) { return key == 0x7fffu ? 0x8000u : key; }
template <bool kBf16>
constexpr uint32_t kInfBits = kBf16 ? 0x7f80u : 0x7c00u;

template <bool kBf16>
__device__ __forceinline__ float value_of(uint32_t key) {
  const uint32_t u = (key & 0x8000u) ? key & 0x7fffu : 0xffffu & ~key;
  if (kBf16) return __uint_as_float(u << 16);
  return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(u)));
}

// v / t to within the last bit (t is in the range the entry accepts).
__device__ __forceinline__ float score_of(float v, float t, float rcp) {
  const float s = v * rcp;
  return isinf(s) ? s : __builtin_fmaf(__builtin_fmaf(-s, t, v), rcp, s);
}

// Larger value first, then smaller index.
__device__ __forceinline__ uint64_t rank_of(uint32_t value, int index) {
  return static_cast<uint64_t>(value) << 32 | (0xffffffffu - static_cast<uint32_t>(index));
}
__device__ __forceinline__ int index_of(uint64_t rank) {
  return static_cast<int>(0xffffffffu - static_cast<uint32_t>(rank));
}
__device__ __forceinline__ uint64_t wave_best(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t w = __shfl_xor(static_cast<unsigned long long>(v), o);
    v = w > v ? w : v;
  }
  return v;
}

__device__ __forceinline__ uint32_t wave_largest(uint32_t v) {
  auto turned = [](uint32_t x, auto by) __attribute__((always_inline)) {  // within 16 lanes
    return static_cast<uint32_t>(
        __builtin_amdgcn_mov_dpp(static_cast<int>(x), 0x120 + decltype(by)::value, 0xf, 0xf, false));
  };
  v = max(v, turned(v, std::integral_constant<int, 8>{}));
  v = max(v, turned(v, std::integral_constant<int, 4>{}));
  v = max(v, turned(v, std::integral_constant<int, 2>{}));
  v = max(v, turned(v, std::integral_constant<int, 1>{}));
  auto lane_of = [&](int i) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), i)); };
  return max(max(lane_of(0), lane_of(16)), max(lane_of(32), lane_of(48)));
}

// rows.row(i): row i's settings. With Rows::kCutsOnly only rows with a top-k or top-p are read, and
// rows.mass(i, largest logit or NaN, sum) gets the kept logits' sum of exp((x - largest) / temp),
// which the counts tell without another read of the row.
// A whole workgroup of kCutThreads takes row i.
template <bool kBf16, class Rows>
__device__ __forceinline__ void cut_row(const uint16_t *__restrict__ logits, int64_t ld, int vocab,
                                        const Rows &rows, int i_row, int64_t *__restrict__ out,
                                        RowCut *__restrict__ cuts) {
  __shared__ __attribute__((aligned(16))) uint32_t hist[kWords];
  __shared__ uint64_t best[kCutWaves];
  __shared__ uint32_t wave_cnt[kCutWaves];
  __shared__ float wave_mass[kCutWaves];
  __shared__ uint32_t tie_cnt[kMaxRounds];
  __shared__ struct {
    int kth;  // key of the k-th largest logit, -1 while unknown
    int cut;  // key that the top-p cut lies in, -1 while unknown
    uint32_t cut_keep, cut_count;  // its logits kept, and all of them
    int last;  // index of the last kept logit of the cut's value
  } sh;

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const SampleRow row = rows.row(i_row);
  const uint16_t *x = logits + i_row * ld;
  const bool greedy = row.temp == 0.f;
  const bool use_k = !greedy && row.k < vocab;
  const bool use_p = !greedy && row.p < 1.f;
  const float temp = greedy ? 1.f : row.temp;
  const float rcp = 1.0f / temp;

  // Calls f(keys, index of the first, how many) for this thread's logits, up to
  // kVec at a time (two keys a word), in index order.
  const int n_vec = vocab / kVec;
  auto each = [&](auto f) __attribute__((always_inline)) {
#pragma unroll 1
    for (int v = tid; v < n_vec; v += kAhead * kCutThreads) {
      u32x4 w[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a)  // rows may start at any logit
        __builtin_memcpy(&w[a], x + kVec * min(v + a * kCutThreads, n_vec - 1), sizeof(w[a]));
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const int va = v + a * kCutThreads;
        if (va >= n_vec) break;
#pragma unroll
        for (int j = 0; j < kVec / 2; ++j) w[a][j] = keys_of(w[a][j]);
        f(w[a], kVec * va, kVec);
      }
    }
    if (vocab % kVec && tid == n_vec % kCutThreads) {
      u32x4 w = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        w[j >> 1] |= static_cast<uint32_t>(x[min(kVec * n_vec + j, vocab - 1)]) << (16 * (j & 1));
#pragma unroll
      for (int j = 0; j < kVec / 2; ++j) w[j] = keys_of(w[j]);
      f(w, kVec * n_vec, vocab % kVec);
    }
  };
  auto key_at = [](const u32x4 &w, int j) { return (w[j >> 1] >> (16 * (j & 1))) & 0xffffu; };
  auto block_best = [&](uint64_t v) __attribute__((always_inline)) {
    v = wave_best(v);
    __syncthreads();  // earlier readers of best are done
    if (lane == 0) best[wave] = v;
    __syncthreads();
    v = best[0];
#pragma unroll
    for (int w = 1; w < kCutWaves; ++w) v = best[w] > v ? best[w] : v;
    return v;
  };

  const bool filter = use_k || use_p;
  if (Rows::kCutsOnly && !filter) return;
  auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kWords / 4; i += kCutThreads)
      reinterpret_cast<u32x4 *>(hist)[i + tid] = u32x4{0u, 0u, 0u, 0u};
  };
  if (filter) clear();
  if (tid == 0) {
    sh.kth = use_k ? -1 : 0;
    sh.cut = use_p ? -1 : 0;
    sh.cut_keep = sh.cut_count = 0;
    sh.last = vocab;
  }
  __syncthreads();

  // One read: the largest key and this thread's first load that holds it,
  // whether there is a NaN (a magnitude above infinity), and the histogram.
  // Past the end of the row a tail repeats its last logit, which changes
  // none of these.
  u16x2 mag2 = {0, 0};
  uint32_t my_key = 0;
  int my_load = 0;
  each([&](const u32x4 &w, int i0, int n) __attribute__((always_inline)) {
    u16x2 top2 = {0, 0};
#pragma unroll
    for (int j = 0; j < kVec / 2; ++j) {
      const uint32_t word = w[j];  // a bit cast of w[j] itself reads w[0]
      const u16x2 k2 = __builtin_bit_cast(u16x2, word);
      top2 = __builtin_elementwise_max(top2, k2);
      // a key or its complement is 0x8000 + the magnitude
      const u16x2 neg = __builtin_bit_cast(u16x2, ~word);
      mag2 = __builtin_elementwise_max(mag2, __builtin_elementwise_max(k2, neg));
    }
    const uint32_t top = max(top2[0], top2[1]);
    if (top > my_key) {
      my_key = top;
      my_load = i0;
    }
    if (filter) {
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        const uint32_t key = key_at(w, j);
        if (j < n) atomicAdd(&hist[key >> 1], 1u << (16 * (key & 1)));
      }
    }
  });
  const uint32_t mag = max(mag2[0], mag2[1]) & 0x7fffu;
  const bool my_nan = mag > kInfBits<kBf16>;
  uint64_t top = 0;
  uint32_t top_key;
  bool nan;
  if (greedy) {
    top = block_best(rank_of(my_key, my_load));
    top_key = merge_zero(static_cast<uint32_t>(top >> 32));
    nan = __syncthreads_or(my_nan);
  } else {
    top_key = wave_largest(my_nan ? 0x10000u : my_key);
    if (lane == 0) wave_cnt[wave] = top_key;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kCutWaves; ++w) top_key = max(top_key, wave_cnt[w]);
    nan = top_key == 0x10000u;
    top_key = merge_zero(top_key);
  }

  if (greedy) {
    // the first logit of the largest value; a NaN counts as the largest
    int first = vocab;
    if (nan || top_key == 0x8000u) {  // several keys count as the largest
      each([&](const u32x4 &w, int i0, int n) __attribute__((always_inline)) {
#pragma unroll
        for (int j = kVec - 1; j >= 0; --j) {
          const uint32_t key = key_at(w, j);
          const bool is_nan = key > (0x8000u | kInfBits<kBf16>) || key < 0x7fffu - kInfBits<kBf16>;
          if (j < n && (nan ? is_nan : merge_zero(key) == top_key)) first = min(first, i0 + j);
        }
      });
    } else if (tid < kVec) {
      const int i = index_of(top) + tid;
      if (i < vocab && (keys_of(x[i]) & 0xffffu) == top_key) first = i;
    }
    const uint64_t b = block_best(rank_of(1, first));
    if (tid == 0) {
      out[i_row] = index_of(b);
      cuts[i_row].ok = -1;
    }
    return;
  }
  const float mx = score_of(value_of<kBf16>(top_key), temp, rcp);
  // softmax of such a row has no probabilities
  if (nan || isinf(mx)) {
    if constexpr (Rows::kCutsOnly)
      rows.mass(i_row, NAN, NAN);
    else if (tid == 0)
      out[i_row] = 0;
    if (tid == 0) cuts[i_row].ok = 0;
    return;
  }
  auto finish = [&]() __attribute__((always_inline)) {
    if (tid == 0)
      cuts[i_row] = {max(sh.kth, sh.cut), sh.cut, sh.last, 1, mx};
  };
  if (!filter) {
    finish();
    return;
  }
  // exp(score - max), in the exp2 domain. The logits are subtracted before they
  // are scaled: of score * log2(e) and max * log2(e) the roundings alone are
  // hundreds apart at a temperature of 1e-8, and one fma of the two would leave
  // infinite or no mass.
  const float slope = rcp * kLog2eS, top_value = value_of<kBf16>(top_key);
  auto mass_of = [&](uint32_t key) __attribute__((always_inline)) {
    return __builtin_amdgcn_exp2f((value_of<kBf16>(key) - top_value) * slope);
  };

  // `wide`: 32-bit counters of the keys of one half (bit 15 `held`) at a time.
  bool wide = false;
  int held = 1;
  auto build = [&](int half) __attribute__((always_inline)) {
    held = half;
    __syncthreads();
    clear();
    __syncthreads();
    each([&](const u32x4 &w, int, int n) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        const uint32_t key = merge_zero(key_at(w, j));
        if (j < n && static_cast<int>(key >> 15) == half) atomicAdd(&hist[key & 0x7fff], 1u);
      }
    });
    __syncthreads();
  };
  // This thread's words, in an order that spreads a wave over the banks.
  constexpr int kSpan = kWords / kCutThreads, kBatch = 8;
  const int top_word = kWords - 1 - kSpan * tid;
  auto my_word = [&](int i) { return top_word - ((i + tid) & (kSpan - 1)); };
  // Keys and counts of a word: two in 16 bits, or one.
  auto key_of_word = [&](int w) { return wide ? held << 15 | w : 2 * w; };
  auto wave_scan = [&](auto v) __attribute__((always_inline)) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const auto u = __shfl_up(v, o);
      if (lane >= o) v += u;
    }
    return v;
  };
  // Counts above this thread's keys, and of all held keys after cnt0.
  uint32_t cnt, above;
  auto scan_counts = [&](uint32_t cnt0) __attribute__((always_inline)) {
    cnt = 0;
#pragma unroll 8
    for (int i = 0; i < kSpan; ++i) {
      const uint32_t c = hist[my_word(i)];
      cnt += wide ? c : (c >> 16) + (c & 0xffffu);
    }
    const uint32_t ci = lanes_up_to(cnt);
    __syncthreads();
    if (lane == 63) wave_cnt[wave] = ci;
    __syncthreads();
    uint32_t all = cnt0;
    above = cnt0 + ci - cnt;
    for (int w = 0; w < kCutWaves; ++w) {
      if (w < wave) above += wave_cnt[w];
      all += wave_cnt[w];
    }
    return all;
  };
  // The keys of lane `owner`'s words in descending order, one per lane of its
  // wave, with their counts.
  auto spread = [&](int owner, int &key, uint32_t &n) __attribute__((always_inline)) {
    const int w = __shfl(top_word, owner) - (wide ? lane & (kSpan - 1) : lane >> 1);
    const uint32_t c = hist[w];
    key = wide ? key_of_word(w) : 2 * w + 1 - (lane & 1);
    n = wide ? (lane < kSpan ? c : 0) : (key & 1 ? c >> 16 : c & 0xffffu);
  };
  auto find_kth = [&]() __attribute__((always_inline)) {
    const uint32_t k = static_cast<uint32_t>(row.k);
    const uint64_t owners = __ballot(above < k && k <= above + cnt);
    if (owners) {
      const int owner = __ffsll(static_cast<long long>(owners)) - 1;
      int key;
      uint32_t n;
      spread(owner, key, n);
      const uint32_t with = __shfl(above, owner) + wave_scan(n);
      if (with - n < k && k <= with) sh.kth = key;
    }
    __syncthreads();
  };
  // Masses of the kept keys above this thread's (and with them), after mass0.
  float mass_above, mass_with;
  auto scan_masses = [&](float mass0) __attribute__((always_inline)) {
    float s = 0.f;
    const int kth = sh.kth;
    if ((key_of_word(top_word) | 1) >= kth) {
#pragma unroll 1
      for (int i0 = 0; i0 < kSpan; i0 += kBatch) {
        uint32_t c[kBatch], some = 0;
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          c[j] = hist[my_word(i0 + j)];
          some |= c[j];
        }
        // (few of the keys occur; those that do, side by side and without a branch)
        if (!__any(some)) continue;
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          const int key = key_of_word(my_word(i0 + j));
          const uint32_t high = wide ? 0 : c[j] >> 16, low = wide ? c[j] : c[j] & 0xffffu;
          const float of_high = high * mass_of(key + 1), of_low = low * mass_of(key);
          s += high && key + 1 >= kth ? of_high : 0.f;
          s += low && key >= kth ? of_low : 0.f;
        }
      }
    }
    const float si = wave_scan(s);
    float se = __shfl_up(si, 1);  // the neighbour's own sum
    if (lane == 0) se = 0.f;
    __syncthreads();
    if (lane == 63) wave_mass[wave] = si;
    __syncthreads();
    float base = mass0, all = mass0;
    for (int w = 0; w < kCutWaves; ++w) {
      if (w < wave) base += wave_mass[w];
      all += wave_mass[w];
    }
    mass_above = base + se;
    mass_with = base + si;
    return all;
  };
  // A thread's range starts with the very sum its neighbour's ends with, so
  // some thread's straddles a target below the total; of several (the sums of
  // a scan need not grow) the first one is taken, and so for its keys.
  // Rounding can leave the keys' own sums short of the target: then it keeps
  // all of them.
  auto find_cut = [&](float target) __attribute__((always_inline)) {
    int my_cut = -1;
    uint32_t my_keep = 0, my_count = 0;
    const uint64_t owners = __ballot(mass_above <= target && target < mass_with);
    if (owners) {
      const int owner = __ffsll(static_cast<long long>(owners)) - 1;
      int key;
      uint32_t n;
      spread(owner, key, n);
      if (key < sh.kth) n = 0;
      const float e = n ? mass_of(key) : 0.f;
      const float base = __shfl(mass_above, owner);
      const float with = base + wave_scan(n * e);
      float before = __shfl_up(with, 1);
      if (lane == 0) before = base;
      const uint64_t at = __ballot(n && before <= target && target < with);
      const uint64_t some = __ballot(n != 0);
      const int pick = at ? __ffsll(static_cast<long long>(at)) - 1
                          : (some ? 63 - __clzll(static_cast<long long>(some)) : 0);
      if (lane == pick) {
        // logit j of the value stays if the mass before it is within the target
        const float over = (target - before) / e;
        my_cut = some ? key : key + 1;
        my_count = n;
        my_keep = at && over < static_cast<float>(n) ? min(n, static_cast<uint32_t>(over) + 1u) : n;
        atomicMax(&sh.cut, my_cut);
      }
    }
    __syncthreads();
    if (my_cut >= 0 && my_cut == sh.cut) {
      sh.cut_keep = my_keep;
      sh.cut_count = my_count;
    }
    __syncthreads();
  };

  // The two zeros become one value; then, did every counter hold its count?
  const uint32_t zeros = (hist[0x7fff >> 1] >> 16) + (hist[0x4000] & 0xffffu);
  __syncthreads();
  if (tid == 0 && zeros <= 0xffffu) {
    hist[0x4000] += hist[0x7fff >> 1] >> 16;
    hist[0x7fff >> 1] &= 0xffffu;
  }
  __syncthreads();
  uint32_t up_cnt = scan_counts(0);
  if (up_cnt != static_cast<uint32_t>(vocab) || zeros > 0xffffu) {
    wide = true;
    build(1);
    up_cnt = scan_counts(0);
  }
  if (use_k) {
    find_kth();
    if (wide && sh.kth < 0) {
      build(0);
      scan_counts(up_cnt);
      find_kth();
    }
  }
  if (use_p) {
    if (wide && !held) build(1);
    const float up_mass = scan_masses(0.f);
    float z = up_mass;
    if (wide && sh.kth < 0x8000) {
      build(0);
      z = scan_masses(up_mass);
    }
    const float target = row.p * z;
    if (wide && !held && target < up_mass) {
      build(1);
      scan_masses(0.f);
    }
    find_cut(target);
    if (sh.cut < 0) {  // the target is not reached: everything stays
      __syncthreads();
      if (tid == 0) sh.cut = 0;
      __syncthreads();
    }
  }
  if constexpr (Rows::kCutsOnly) {
    const int low = max(sh.kth, sh.cut);
    double sum = 0;
    // the held words from the largest key's down to `low`'s
    auto add = [&]() __attribute__((always_inline)) {
      const int base = wide ? held << 15 : 0, shift = wide ? 0 : 1;
      const int from = max(low - base, 0) >> shift;
      const int to = min(static_cast<int>(top_key) - base, (kWords << shift) - 1) >> shift;
      float s = 0.f;
      auto of = [&](int key, uint32_t n) __attribute__((always_inline)) {
        // (without a top-p `cut` is 0, which is no number's key)
        if (n && key >= low) s += (key == sh.cut ? sh.cut_keep : n) * mass_of(key);
      };
#pragma unroll 4
      for (int w = to - tid; w >= from; w -= kCutThreads) {
        const uint32_t c = hist[w];
        if (wide) {
          of(base + w, c);
        } else {
          of(2 * w + 1, c >> 16);
          of(2 * w, c & 0xffffu);
        }
      }
      sum += s;
    };
    __syncthreads();
    add();
    if (wide) {
      build(!held);
      add();
    }
    __shared__ double wave_sum[kCutWaves];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if (lane == 0) wave_sum[wave] = sum;
    __syncthreads();
    sum = 0;
    for (int w = 0; w < kCutWaves; ++w) sum += wave_sum[w];
    rows.mass(i_row, top_value, static_cast<float>(sum));
  }
  // A value that the cut splits keeps its first logits by index: count it by
  // rounds, then find the last kept one in its round.
  if (sh.cut_keep < sh.cut_count) {
    const uint32_t cut = sh.cut;
    for (int i = tid; i < kMaxRounds; i += kCutThreads) tie_cnt[i] = 0;
    __syncthreads();
    each([&](const u32x4 &w, int i0, int n) __attribute__((always_inline)) {
      // a word with the cut's key in either half (or, rarely, beside it)
      uint32_t any = 0;
#pragma unroll
      for (int j = 0; j < kVec / 2; ++j) {
        const uint32_t d = w[j] ^ (cut * 0x10001u);
        any |= (d - 0x10001u) & ~d & 0x80008000u;
      }
      if (!any && cut != 0x8000u) return;
      uint32_t c = 0;
#pragma unroll
      for (int j = 0; j < kVec; ++j) c += j < n && merge_zero(key_at(w, j)) == cut;
      if (c) atomicAdd(&tie_cnt[i0 / kStep], c);
    });
    __syncthreads();
    uint32_t before = 0;
    int round = 0;
    while (before + tie_cnt[round] < sh.cut_keep) before += tie_cnt[round++];
    const uint32_t want = sh.cut_keep - before;  // the want-th of this round, from 1
    const int i0 = round * kStep + kVec * tid;
    u32x4 mine = {0u, 0u, 0u, 0u};
    if (i0 + kVec <= vocab) {
      __builtin_memcpy(&mine, x + i0, sizeof(mine));
    } else {
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        mine[j >> 1] |= static_cast<uint32_t>(x[min(i0 + j, vocab - 1)]) << (16 * (j & 1));
    }
#pragma unroll
    for (int j = 0; j < kVec / 2; ++j) mine[j] = keys_of(mine[j]);
    auto is_cut = [&](int j) { return i0 + j < vocab && merge_zero(key_at(mine, j)) == cut; };
    uint32_t c = 0;
#pragma unroll
    for (int j = 0; j < kVec; ++j) c += is_cut(j);
    uint32_t ci = c;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t cu = __shfl_up(ci, o);
      if (lane >= o) ci += cu;
    }
    if (lane == 63) wave_cnt[wave] = ci;
    __syncthreads();
    for (int w = 0; w < wave; ++w) ci += wave_cnt[w];
    if (ci - c < want && want <= ci) {
      uint32_t at = ci - c;
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        if (is_cut(j) && ++at == want) sh.last = i0 + j;
    }
    __syncthreads();
  }
  finish();
}

}  // namespace
}  // namespace hy
