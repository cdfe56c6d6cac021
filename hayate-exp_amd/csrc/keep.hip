// Which cached tokens stay when a cache is cut to a budget (gfx950): the first `sinks`, the
// last `recent`, and of those between the ones with the largest weights, equal ones by their
// position; positions in ascending order.
//
// One workgroup a request. The weights between become ordered 32-bit keys; a radix select (11,
// 11 and 10 bits) finds the key of the last one that stays and how many equal ones do. Each of
// the 16 waves holds a stretch of positions, 64 a round, so that the output's order is that of
// wave, round and lane and needs one exchange of counts. Up to 32,768 tokens the keys stay in
// registers between the passes; longer rows are read again.
//
// Bound by one CU's instructions: five sweeps of about ten a key. 1,024 of 4,001 tokens take 5.1 us,
// 2,047 of 32,700 15.4 us (20 requests side by side the same). Several workgroups a row would
// meet three times in between, a launch of 2.5 us and more each.

#include "hy_common.h"

namespace hy {
namespace {

constexpr int kKeepThreads = 1024;
constexpr int kKeepWaves = kKeepThreads / 64;
constexpr int kKeepFew = 8;     // keys of a lane in registers, all loads in flight at once
constexpr int kKeepMost = 32;
constexpr int kKeepRows = 64;   // requests of one launch
constexpr int kKeepGroup = 4;   // rounds taken together
constexpr int kBins = 2048;
// Copies of the first pass's counts: weights share few exponents, and lanes that add to one
// word follow each other, so lane l adds to copy l % 4.
constexpr int kCopies = 4;

struct KeepShared {
  uint32_t first[kBins * kCopies];  // [bin][copy]
  uint32_t later[2][kBins];
  uint32_t sums[kKeepWaves], same[kKeepWaves];
  uint32_t found[2];
};

// Sum of the waves' values before `wave`.
__device__ __forceinline__ uint32_t waves_before(const uint32_t *of, int wave) {
  const int lane = threadIdx.x & 63;
  const uint32_t upto = lanes_up_to(of[lane & (kKeepWaves - 1)]);
  return wave == 0 ? 0 : __builtin_amdgcn_readlane(upto, wave - 1);
}

struct KeepRow {
  int32_t row, len;
};
struct KeepRows {
  KeepRow r[kKeepRows];
};

// Ordered keys: larger key, larger weight; -0 is 0 and NaN the largest. A number's key is at least
// that of -inf; 0 stands for none.
__device__ __forceinline__ uint32_t key_of(float w) {
  const uint32_t u = __float_as_uint(w + 0.0f);
  const uint32_t key = u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
  return w != w ? 0xffffffffu : key;
}

// kHeld: rounds whose keys are held, or 0.
template <int kHeld>
__device__ __forceinline__ void keep_row(const float *__restrict__ w, int n, int want,
                                         int32_t *__restrict__ out, int first_pos,
                                         KeepShared &sh) {
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // wave's stretch: rounds of 64 positions
  const int rounds = ((n + 64 * kKeepWaves - 1) / (64 * kKeepWaves));
  const int from = wave * 64 * rounds;
  uint32_t held[kHeld ? kHeld : 1];
  // (a load behind a branch would wait for the one before)
  auto value_at = [&](int i) { return w[min(from + 64 * i + lane, n - 1)]; };
  auto key_at = [&](int i, float v) {
    return i < rounds && from + 64 * i + lane < n ? key_of(v) : 0u;
  };
  if constexpr (kHeld) {
    float v[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) v[i] = value_at(i);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) held[i] = key_at(i, v[i]);
  }
  {
    uint4 *all = reinterpret_cast<uint4 *>(&sh);
    for (int i = tid; i < kBins * (kCopies + 2) / 4; i += kKeepThreads) all[i] = uint4{0, 0, 0, 0};
  }
  __syncthreads();
  // f(key, round) for the lane's keys (0: none), in order
  auto each = [&](auto f) __attribute__((always_inline)) {
    if constexpr (kHeld) {
#pragma unroll
      for (int i = 0; i < kHeld; i += kKeepGroup) {
        if (i >= rounds) break;
#pragma unroll
        for (int j = 0; j < kKeepGroup; ++j) f(held[i + j], i + j);
      }
    } else {
      for (int i = 0; i < rounds; i += kKeepFew) {
        float v[kKeepFew];
#pragma unroll
        for (int j = 0; j < kKeepFew; ++j) v[j] = value_at(i + j);
#pragma unroll
        for (int j = 0; j < kKeepFew; ++j) f(key_at(i + j, v[j]), i + j);
      }
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
    const uint32_t mask = (1u << bits) - 1;
    each([&](uint32_t key, int) __attribute__((always_inline)) {
      // (no number's key has the first digit 0, and no number is searched for behind them all)
      if (pass == 0)
        atomicAdd(&sh.first[(key >> shift) * kCopies + (lane & (kCopies - 1))], 1u);
      else if (key >> high == prefix)
        atomicAdd(&sh.later[pass - 1][key >> shift & mask], 1u);
    });
    __syncthreads();
    // thread t holds the bins 2047 - 2t and 2046 - 2t: a scan from the largest digit down
    const int top = kBins - 1 - 2 * tid;
    uint32_t a, b;
    if (pass == 0) {
      const uint4 *at = reinterpret_cast<const uint4 *>(sh.first + (top - 1) * kCopies);
      // (lanes whose counts lie 256 bytes apart start at different ones)
      constexpr int kReads = kCopies / 2;
      const int turn = lane / (32 / kCopies);
      a = b = 0;
#pragma unroll
      for (int j = 0; j < kReads; ++j) {
        const int i = (turn + j) & (kReads - 1);
        const uint4 v = at[i];
        const uint32_t sum = v.x + v.y + v.z + v.w;
        b += i < kReads / 2 ? sum : 0;
        a += i < kReads / 2 ? 0 : sum;
      }
    } else {
      const uint2 v = *reinterpret_cast<const uint2 *>(sh.later[pass - 1] + top - 1);
      b = v.x;
      a = v.y;
    }
    const uint32_t with = lanes_up_to(a + b);
    if (lane == 63) sh.sums[wave] = with;
    __syncthreads();
    const uint32_t before = waves_before(sh.sums, wave) + with - a - b;
    if (before < left && left <= before + a + b) {
      const bool second = left > before + a;
      sh.found[0] = top - second;
      sh.found[1] = before + (second ? a : 0);
    }
    __syncthreads();
    prefix = prefix << bits | __builtin_amdgcn_readfirstlane(sh.found[0]);
    left -= __builtin_amdgcn_readfirstlane(sh.found[1]);
  }
  // `prefix` is the last key that stays, `left` how many of its equals do, the first ones.
  uint32_t more = 0, same = 0;
  each([&](uint32_t key, int) __attribute__((always_inline)) {
    more += __popcll(__ballot(key > prefix));
    same += __popcll(__ballot(key == prefix));
  });
  // (sums was read before the last barrier)
  if (lane == 0) {
    sh.sums[wave] = more;
    sh.same[wave] = same;
  }
  __syncthreads();
  const uint32_t same_before = waves_before(sh.same, wave);
  uint32_t at = waves_before(sh.sums, wave) + min(same_before, left);
  left -= min(same_before, left);  // equals that stay from this wave on
  each([&](uint32_t key, int i) __attribute__((always_inline)) {
    uint64_t stay = __ballot(key > prefix);
    if (left > 0) {
      const uint64_t eq = __ballot(key == prefix);
      const uint32_t rank = __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(eq >> 32),
                                                      __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(eq), 0));
      stay |= __ballot(key == prefix && rank < left);
      left -= min(static_cast<uint32_t>(__popcll(eq)), left);
    }
    const uint32_t mine = __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(stay >> 32),
                                                    __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(stay), at));
    if (stay >> lane & 1) out[mine] = first_pos + from + 64 * i + lane;
    at += __popcll(stay);
  });
}

__global__ __launch_bounds__(kKeepThreads) void keep_kernel(const float *__restrict__ weights,
                                                            int64_t stride, KeepRows rows,
                                                            int budget, int sinks, int recent,
                                                            int32_t *__restrict__ out) {
  __shared__ __attribute__((aligned(16))) KeepShared sh;
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
  if (between <= kKeepFew * kKeepThreads)
    keep_row<kKeepFew>(w, between, want, o + sinks, sinks, sh);
  else if (between <= kKeepMost * kKeepThreads)
    keep_row<kKeepMost>(w, between, want, o + sinks, sinks, sh);
  else
    keep_row<0>(w, between, want, o + sinks, sinks, sh);
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
