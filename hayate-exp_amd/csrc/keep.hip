// Which cached tokens stay when a cache is cut to a budget (gfx950): the first `sinks`, the
// last `recent`, and of those between the ones with the largest weights, equal ones by their
// position; positions in ascending order.
//
// One workgroup a request. The weights between become ordered 32-bit keys; a radix select (11,
// 11 and 10 bits) finds the key of the last one that stays and how many equal ones do. Each of
// the 16 waves holds a stretch of positions, 64 a round, so that the output's order is that of
// wave, round and lane and needs one exchange of counts. Up to 32,768 tokens the keys stay in
// registers between the passes; longer rows are read again.

#include "hy_common.h"

namespace hy {
namespace {

constexpr int kKeepThreads = 1024;
constexpr int kKeepWaves = kKeepThreads / 64;
constexpr int kKeepHeld = 32;   // keys of a lane in registers
constexpr int kKeepRows = 64;   // requests of one launch
constexpr int kBins = 2048;

struct KeepRow {
  int32_t row, len;
};
struct KeepRows {
  KeepRow r[kKeepRows];
};

// Ordered keys: larger key, larger weight; -0 is 0 and NaN the largest. No key is 0.
__device__ __forceinline__ uint32_t key_of(float w) {
  const uint32_t u = __float_as_uint(w);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if ((u & 0x7fffffffu) == 0) return 0x80000000u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <bool kHeld>
__device__ __forceinline__ void keep_row(const float *__restrict__ w, int n, int want,
                                         int32_t *__restrict__ out, int first_pos,
                                         uint32_t *hist, uint32_t *wave_cnt) {
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // wave's stretch: rounds of 64 positions
  const int rounds = ((n + 64 * kKeepWaves - 1) / (64 * kKeepWaves));
  const int from = wave * 64 * rounds;
  uint32_t held[kHeld ? kKeepHeld : 1];
  auto load = [&](int i) -> uint32_t {
    const int at = from + 64 * i + lane;
    return i < rounds && at < n ? key_of(w[at]) : 0u;
  };
  if constexpr (kHeld) {
#pragma unroll
    for (int i = 0; i < kKeepHeld; ++i) held[i] = load(i);
  }
  // f(key, round) for the lane's keys (0: none), in order
  auto each = [&](auto f) __attribute__((always_inline)) {
    if constexpr (kHeld) {
#pragma unroll
      for (int i = 0; i < kKeepHeld; ++i)
        if (i < rounds) f(held[i], i);
    } else {
#pragma unroll 4
      for (int i = 0; i < rounds; ++i) f(load(i), i);
    }
  };
  // Radix select of the want-th largest key, want of [1, n].
  uint32_t prefix = 0, left = static_cast<uint32_t>(want);
  int shift = 32;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int bits = pass < 2 ? 11 : 10;
    const int high = shift;  // key >> high equals the prefix
    shift -= bits;
    for (int i = tid; i < kBins; i += kKeepThreads) hist[i] = 0;
    __syncthreads();
    const uint32_t mask = (1u << bits) - 1;
    each([&](uint32_t key, int) __attribute__((always_inline)) {
      if (key != 0 && (pass == 0 || key >> high == prefix)) atomicAdd(&hist[key >> shift & mask], 1u);
    });
    __syncthreads();
    // thread t holds the bins 2047 - 2t and 2046 - 2t: a scan from the largest digit down
    const int top = kBins - 1 - 2 * tid;
    const uint32_t a = hist[top], b = hist[top - 1];
    uint32_t with = a + b;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t u = __shfl_up(with, o);
      if (lane >= o) with += u;
    }
    if (lane == 63) wave_cnt[wave] = with;
    __syncthreads();
    uint32_t before = with - a - b;
    for (int x = 0; x < wave; ++x) before += wave_cnt[x];
    if (before < left && left <= before + a) {
      wave_cnt[kKeepWaves] = top;
      wave_cnt[kKeepWaves + 1] = before;
    } else if (before + a < left && left <= before + a + b) {
      wave_cnt[kKeepWaves] = top - 1;
      wave_cnt[kKeepWaves + 1] = before + a;
    }
    __syncthreads();
    prefix = prefix << bits | wave_cnt[kKeepWaves];
    left -= wave_cnt[kKeepWaves + 1];
    __syncthreads();
  }
  // `prefix` is the last key that stays, `left` how many of its equals do, the first ones.
  uint32_t more = 0, same = 0;
  each([&](uint32_t key, int) __attribute__((always_inline)) {
    more += __popcll(__ballot(key > prefix));
    same += __popcll(__ballot(key == prefix));
  });
  if (lane == 0) {
    wave_cnt[wave] = more;
    wave_cnt[kKeepWaves + wave] = same;
  }
  __syncthreads();
  uint32_t more_before = 0, same_before = 0;
  for (int x = 0; x < wave; ++x) {
    more_before += wave_cnt[x];
    same_before += wave_cnt[kKeepWaves + x];
  }
  const uint64_t below = (1ull << lane) - 1;
  each([&](uint32_t key, int i) __attribute__((always_inline)) {
    const uint64_t gt = __ballot(key > prefix), eq = __ballot(key == prefix);
    const uint32_t eq_rank = same_before + __popcll(eq & below);
    const uint32_t at = more_before + __popcll(gt & below) + min(eq_rank, left);
    if (key > prefix || (key == prefix && eq_rank < left)) out[at] = first_pos + from + 64 * i + lane;
    more_before += __popcll(gt);
    same_before += __popcll(eq);
  });
}

__global__ __launch_bounds__(kKeepThreads) void keep_kernel(const float *__restrict__ weights,
                                                            int64_t stride, KeepRows rows,
                                                            int budget, int sinks, int recent,
                                                            int32_t *__restrict__ out) {
  __shared__ uint32_t hist[kBins];
  __shared__ uint32_t wave_cnt[2 * kKeepWaves];
  const KeepRow row = rows.r[blockIdx.x];
  int32_t *o = out + static_cast<int64_t>(blockIdx.x) * budget;
  const int n = row.len;
  if (n <= budget) {
    for (int i = threadIdx.x; i < budget; i += kKeepThreads) o[i] = i < n ? i : -1;
    return;
  }
  for (int i = threadIdx.x; i < sinks; i += kKeepThreads) o[i] = i;
  for (int i = threadIdx.x; i < recent; i += kKeepThreads) o[budget - recent + i] = n - recent + i;
  const int want = budget - sinks - recent;
  if (want == 0) return;
  const float *w = weights + row.row * stride + sinks;
  const int between = n - sinks - recent;
  if (between <= kKeepHeld * kKeepThreads)
    keep_row<true>(w, between, want, o + sinks, sinks, hist, wave_cnt);
  else
    keep_row<false>(w, between, want, o + sinks, sinks, hist, wave_cnt);
}

}  // namespace
}  // namespace hy

extern "C" int hy_keep_positions(const float *weights, int64_t weights_stride, const int32_t *rows,
                                 const int32_t *lens, int32_t num_seqs, int32_t budget,
                                 int32_t sinks, int32_t recent, int32_t *out, void *stream) {
  hy::clear_error();
  HY_REQUIRE(num_seqs >= 0, "hy_keep_positions: num_seqs must be non-negative");
  HY_REQUIRE(budget >= 1 && sinks >= 0 && recent >= 0 && sinks <= budget &&
                 recent <= budget - sinks,
             "hy_keep_positions: budget %d (at least 1) of %d first and %d last tokens", budget,
             sinks, recent);
  if (num_seqs == 0) return HY_OK;
  HY_REQUIRE(weights && rows && lens && out, "hy_keep_positions: null pointer argument");
  for (int32_t b = 0; b < num_seqs; ++b)
    HY_REQUIRE(rows[b] >= 0 && lens[b] >= 0 && lens[b] <= 1 << 30,
               "hy_keep_positions: sequence %d has row %d, length %d", b, rows[b], lens[b]);
  hipStream_t st = static_cast<hipStream_t>(stream);
  for (int32_t b0 = 0; b0 < num_seqs; b0 += hy::kKeepRows) {
    const int n = num_seqs - b0 < hy::kKeepRows ? num_seqs - b0 : hy::kKeepRows;
    hy::KeepRows r{};
    for (int i = 0; i < n; ++i) r.r[i] = {rows[b0 + i], lens[b0 + i]};
    hipLaunchKernelGGL(hy::keep_kernel, dim3(n), dim3(hy::kKeepThreads), 0, st, weights,
                       weights_stride, r, budget, sinks, recent,
                       out + static_cast<int64_t>(b0) * budget);
  }
  return hy::launch_status("hy_keep_positions");
}
