// Batched sampling of 16-bit logits: greedy, temperature, top-k and top-p,
// without a sort.
//
// The reference sorts each row (hayate/engine/sampler.py:39-65); batched, the sort
// of 20 x 151,936 scores, the softmax and prefix sum over them and the scatter
// back took 1,040 us. What is needed of the order is only where top-k and top-p
// cut it. A 16-bit logit has 65,536 values, so a histogram of a row holds its
// whole order, and all logits of one value share one score and probability:
// counts times exp(score - max) are the cumulative masses.
//
//   cut_kernel   one workgroup per row: greedy rows end here; for the others
//                the histogram in LDS (65,536 16-bit counters; a value that
//                more than 65,535 logits share shows in the counters' sum,
//                and the row is done again with 32-bit counters, half of the
//                values at a time), the k-th value and the value in which the
//                mass passes top_p. A value that this cut splits keeps its
//                first logits by index, as a stable descending sort does.
//   draw_kernel  many workgroups per row: the largest p / q of each one's share
//                of the kept logits, q the exponential noise the caller made;
//                the draw of torch.multinomial.
//   pick_kernel  the largest of those per row.
//
// cut_kernel is bound by one CU's reads (304 KB a row of 151,936: 10 us, also
// of a greedy row), its LDS atomics (8 us), and for a top-p cut a walk over the
// counters and a second read for the ties (18 us); everything that needs an
// exponential per logit is in draw_kernel (9-11 us, 19 workgroups a row).
// Measured on MI355X, 20 rows of 151,936, noise and launches included, against
// the sort: greedy 35 -> 17 us, temperature alone 1,056 -> 38, top-k 1,060 -> 41,
// top-p 1,054 -> 62, a mix 1,020 -> 59.

#include "logit_rows.h"

namespace hy {
namespace {

constexpr int kDrawThreads = 256;
constexpr int kDrawShare = kDrawThreads * kVec * kAhead;  // logits per draw workgroup
constexpr int kSampleRows = 64;                // rows of one launch

struct SampleRows {
  static constexpr bool kCutsOnly = false;
  SampleRow r[kSampleRows];
  __device__ __forceinline__ SampleRow row(int i) const { return r[i]; }
};

// Grid (rows).
template <bool kBf16>
__global__ __launch_bounds__(kCutThreads) void cut_kernel(
    const uint16_t *__restrict__ logits, int64_t ld, int vocab, SampleRows rows,
    int64_t *__restrict__ out, RowCut *__restrict__ cuts) {
  cut_row<kBf16>(logits, ld, vocab, rows, blockIdx.x, out, cuts);
}

// Grid (shares of a row, rows): the best p / q of kDrawShare logits.
template <bool kBf16>
__global__ __launch_bounds__(kDrawThreads) void draw_kernel(
    const uint16_t *__restrict__ logits, int64_t ld, int vocab, SampleRows rows,
    const float *__restrict__ noise, const RowCut *__restrict__ cuts, uint64_t *__restrict__ bests) {
  __shared__ uint64_t best[kDrawThreads / 64];
  const SampleRow row = rows.r[blockIdx.y];
  if (row.temp == 0.f) return;
  const RowCut cut = cuts[blockIdx.y];
  if (cut.ok != 1) return;
  const uint16_t *x = logits + blockIdx.y * ld;
  const float *q = noise + static_cast<int64_t>(row.noise) * vocab;
  const float rcp = 1.0f / row.temp;
  const int i0 = blockIdx.x * kDrawShare + kVec * threadIdx.x;
  constexpr int kRound = kDrawThreads * kVec;

  u32x4 w[kAhead];
#pragma unroll
  for (int a = 0; a < kAhead; ++a) {
    const int i = i0 + a * kRound;
    if (i + kVec <= vocab) {
      __builtin_memcpy(&w[a], x + i, sizeof(w[a]));
    } else {
      w[a] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        w[a][j >> 1] |= static_cast<uint32_t>(x[min(i + j, vocab - 1)]) << (16 * (j & 1));
    }
  }
  float r_best = -1.f;
  int i_best = vocab;
#pragma unroll
  for (int a = 0; a < kAhead; ++a) {
    const int i = i0 + a * kRound;
    uint32_t key[kVec];
    bool keep[kVec], any = false;
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      key[j] = merge_zero((keys_of(w[a][j >> 1]) >> (16 * (j & 1))) & 0xffffu);
      keep[j] = i + j < vocab && static_cast<int>(key[j]) >= cut.low &&
                !(static_cast<int>(key[j]) == cut.cut && i + j > cut.last);
      any = any || keep[j];
    }
    if (!any) continue;  // no noise is read for these
    float qv[kVec];
    if (i + kVec <= vocab) {
      __builtin_memcpy(qv, q + i, sizeof(qv));
    } else {
#pragma unroll
      for (int j = 0; j < kVec; ++j) qv[j] = q[min(i + j, vocab - 1)];
    }
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const float s = score_of(value_of<kBf16>(key[j]), row.temp, rcp);
      const float p = exp2f((s - cut.max) * kLog2eS);  // up to the row's common factor
      const float r = p / qv[j];
      if (keep[j] && r > r_best) {
        r_best = r;
        i_best = i + j;
      }
    }
  }
  // r >= 0 orders as its bits; 0 marks "nothing kept"
  uint64_t b = wave_best(i_best < vocab ? rank_of(__float_as_uint(r_best) + 1u, i_best) : 0);
  if ((threadIdx.x & 63) == 0) best[threadIdx.x >> 6] = b;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int v = 1; v < kDrawThreads / 64; ++v) b = best[v] > b ? best[v] : b;
    bests[blockIdx.y * gridDim.x + blockIdx.x] = b;
  }
}

// One wave per row; `valid` collects whether every row had a distribution
// (the first launch of a call sets it, the following ones only clear it).
__global__ __launch_bounds__(1024) void pick_kernel(int rows, int shares, bool first_rows,
                                                    const RowCut *__restrict__ cuts,
                                                    const uint64_t *__restrict__ bests,
                                                    int64_t *__restrict__ out,
                                                    uint8_t *__restrict__ valid) {
  const int lane = threadIdx.x & 63;
  bool bad = false;
  for (int r = threadIdx.x >> 6; r < rows; r += 16) {
    const int ok = cuts[r].ok;
    bad = bad || ok == 0;
    if (ok != 1) continue;
    uint64_t b = 0;
    for (int s = lane; s < shares; s += 64) {
      const uint64_t v = bests[r * shares + s];
      b = v > b ? v : b;
    }
    b = wave_best(b);
    if (lane == 0) out[r] = index_of(b);
  }
  const bool any_bad = __syncthreads_or(bad);
  if (threadIdx.x == 0 && valid != nullptr && (first_rows || any_bad)) *valid = !any_bad;
}

int64_t cut_bytes(int rows) { return (static_cast<int64_t>(rows) * sizeof(RowCut) + 255) / 256 * 256; }

}  // namespace
}  // namespace hy

extern "C" int64_t hy_sample_workspace_bytes(int32_t n_rows, int32_t vocab) {
  if (n_rows <= 0 || vocab <= 0) return 0;
  const int rows = n_rows < hy::kSampleRows ? n_rows : hy::kSampleRows;
  const int64_t shares = (static_cast<int64_t>(vocab) + hy::kDrawShare - 1) / hy::kDrawShare;
  return hy::cut_bytes(rows) + rows * shares * static_cast<int64_t>(sizeof(uint64_t));
}

extern "C" int hy_sample(const void *logits, int64_t row_stride, int32_t dtype, int32_t n_rows,
                         int32_t vocab, const float *temperature, const int32_t *top_k,
                         const float *top_p, const float *noise, int64_t *out, uint8_t *valid,
                         void *workspace, int64_t workspace_bytes, void *stream) {
  hy::clear_error();
  HY_REQUIRE(n_rows >= 0 && vocab >= 1, "hy_sample: invalid sizes %d x %d", n_rows, vocab);
  HY_REQUIRE(dtype == 0 || dtype == 1, "hy_sample: dtype %d (0: bf16, 1: fp16)", dtype);
  HY_REQUIRE_SUPPORTED(vocab <= hy::kStep * hy::kMaxRounds, "hy_sample: vocabulary %d too large",
                       vocab);
  if (n_rows == 0) return HY_OK;
  HY_REQUIRE(logits && temperature && top_k && top_p && out && workspace,
             "hy_sample: null pointer argument");
  if (workspace_bytes < hy_sample_workspace_bytes(n_rows, vocab)) {
    hy::set_error("hy_sample: workspace too small: need %lld bytes, got %lld",
                  static_cast<long long>(hy_sample_workspace_bytes(n_rows, vocab)),
                  static_cast<long long>(workspace_bytes));
    return HY_ENOSPACE;
  }
  int sampled = 0;
  for (int r = 0; r < n_rows; ++r) {
    const float t = temperature[r];
    if (t == 0.f) continue;
    HY_REQUIRE_SUPPORTED(t >= 1e-30f && t <= 1e30f, "hy_sample: temperature %g", t);
    HY_REQUIRE(top_k[r] >= 1 && top_p[r] > 0.f, "hy_sample: row %d has top_k %d, top_p %g", r,
               top_k[r], top_p[r]);
    ++sampled;
  }
  HY_REQUIRE(sampled == 0 || (noise && valid), "hy_sample: null pointer argument");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int shares = (vocab + hy::kDrawShare - 1) / hy::kDrawShare;
  int noise_row = 0;
  for (int r0 = 0; r0 < n_rows; r0 += hy::kSampleRows) {
    const int n = n_rows - r0 < hy::kSampleRows ? n_rows - r0 : hy::kSampleRows;
    hy::SampleRows rows{};
    for (int i = 0; i < n; ++i) {
      const float t = temperature[r0 + i];
      rows.r[i] = {t, top_k[r0 + i] < vocab ? top_k[r0 + i] : vocab, top_p[r0 + i],
                   t == 0.f ? 0 : noise_row++};
    }
    const uint16_t *x = static_cast<const uint16_t *>(logits) + r0 * row_stride;
    auto *cuts = static_cast<hy::RowCut *>(workspace);
    auto *bests = reinterpret_cast<uint64_t *>(static_cast<char *>(workspace) + hy::cut_bytes(n));
    auto cut = dtype == 0 ? hy::cut_kernel<true> : hy::cut_kernel<false>;
    auto draw = dtype == 0 ? hy::draw_kernel<true> : hy::draw_kernel<false>;
    hipLaunchKernelGGL(cut, dim3(n), dim3(hy::kCutThreads), 0, st, x, row_stride, vocab, rows,
                       out + r0, cuts);
    if (sampled == 0) continue;
    hipLaunchKernelGGL(draw, dim3(shares, n), dim3(hy::kDrawThreads), 0, st, x, row_stride, vocab,
                       rows, noise, cuts, bests);
    hipLaunchKernelGGL(hy::pick_kernel, dim3(1), dim3(1024), 0, st, n, shares, r0 == 0, cuts,
                       bests, out + r0, valid);
  }
  return hy::launch_status("hy_sample");
}
