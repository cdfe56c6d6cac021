// What weight every cached token got from a tick's queries, added to a table (gfx950):
//   w[t] += sum over the sequence's rows i and query heads h of
//           exp(scale q_ih . k_t - max_ih) / sum_ih,   t <= position of i,
// with the row maxima and sums that the attention kernels leave (row_ml, exp2 domain).
//
// Single tokens: the decode kernel has stored its raw scores, 4 bytes a head and key where K and
// V take 512 bytes a kv head and key; add_kernel turns them into weights and sums the heads.
// Chunks: storing scores would cost more than the products (512 rows x 32 heads x 4 bytes a key),
// so weigh_kernel computes them again from K and Q, an item 256 keys by a range of rows, and
// leaves a sum per kv head, range and key; add_kernel adds those. Every sum has a fixed order.
//
// weigh_kernel: one workgroup of four waves per (kv head, item), each wave 64 keys whose K it
// keeps in registers; the rows go through LDS, 64 a stage, and meet them in
// v_mfma_f32_32x32x16_bf16 as S = K Q^T (lane l, c = l % 32, h = l / 32: row c's scores for keys
// 8 (i / 4) + 4 h + i % 4 of a 32-key block), so a lane adds up its row's weights key by key over
// the whole range and the 32 rows of a block are only joined at the end.

#include "hy_common.h"
#include "weigh_shape.h"

namespace hy {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kStageElems = kWeighRows * kHeadDim;

__device__ __forceinline__ void load_to_lds(const uint16_t *g, const uint16_t *lds) {
  const uint32_t m0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
      (const __attribute__((address_space(3))) uint16_t *)lds));
  // (a load that reads M0 must not directly follow its write)
  __asm__ volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
                   :
                   : "v"(g), "s"(__builtin_amdgcn_readfirstlane(m0))
                   : "memory");
}

// Every load of this wave done: vmcnt(0) lgkmcnt(0).
__device__ __forceinline__ void wait_all() {
  __builtin_amdgcn_s_waitcnt(0x0070);
  __asm__ volatile("" ::: "memory");
}

// Item = {seq, key0, token0, token1, part, q_row, cache_len, offset}: keys from key0 (a multiple
// of 256), the sequence's tokens [token0, token1) of this tick. Sums go to
// partials[(part * kv heads + kv head) * stride + offset + key].
template <int G>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2)))
void weigh_kernel(const uint16_t *__restrict__ q, int64_t q_ss, int64_t q_st, int64_t q_sh,
                  const uint16_t *__restrict__ k_pool, int64_t pool_hs,
                  const int32_t *__restrict__ page_table, int64_t pt_stride,
                  const int32_t *__restrict__ items, const float2 *__restrict__ row_ml,
                  float *__restrict__ partials, int64_t stride, int num_kv_heads, int page_shift,
                  float scale_log2, bool q_aligned) {
  __shared__ __attribute__((aligned(1024))) uint16_t smem[2 * kStageElems];
  const int32_t *it = items + 8 * blockIdx.y;
  const int kvh = blockIdx.x;
  const int seq = it[0], key0 = it[1], tok0 = it[2], tok1 = it[3];
  const int part = it[4], q_row = it[5], cache = it[6], off = it[7];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int c = lane & 31, h = lane >> 5;
  const int last_key = cache + tok1 - 1;  // the last one that some row sees
  const int n_rows = (tok1 - tok0) * G;
  const int n_stages = (n_rows + kWeighRows - 1) / kWeighRows;
  const int page_mask = (1 << page_shift) - 1;

  // Stage s: rows 64 s .. of the item, 16 rows x 4 chunks an instruction, laid out so that 16
  // lanes reading one chunk of 16 rows touch every bank once. Rows past the end repeat the
  // last one.
  const int chunk8 = 8 * ((lane & 3) ^ ((lane >> 4) & 3));
  const uint16_t *qb = q + seq * q_ss + static_cast<int64_t>(q_row) * q_st + kvh * G * q_sh;
  auto issue = [&](int s) {
    uint16_t *dst = smem + (s & 1) * kStageElems;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = 4 * wave + j;
      const int row = min(kWeighRows * s + 16 * (i >> 2) + (lane >> 2), n_rows - 1);
      const uint16_t *src =
          qb + static_cast<int64_t>(tok0 + row / G) * q_st + (row % G) * q_sh + 32 * (i & 3) + chunk8;
      if (q_aligned)
        load_to_lds(src, dst + i * 512);
      else
        *reinterpret_cast<u32x4 *>(dst + i * 512 + 8 * lane) = load16(src);
    }
  };
  issue(0);

  // K of the wave's two blocks (A operand: row c, dims 16 kk + 8 h ..).
  bf16x8 kop[2][8];
  const int first = key0 + 64 * wave;
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const int key = min(first + 32 * b + c, last_key);
    const int64_t p =
        (static_cast<int64_t>(page_table[seq * pt_stride + (key >> page_shift)]) << page_shift) +
        (key & page_mask);
    const uint16_t *src = k_pool + kvh * pool_hs + p * kHeadDim + 8 * h;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) kop[b][kk] = __builtin_bit_cast(bf16x8, load16(src + 16 * kk));
  }
  float sum[2][16];
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) sum[b][i] = 0.f;

  // This lane's row of row block r: its exponent base and the inverse of its sum.
  auto row_of = [&](int r) {
    const int row = 32 * r + c;
    if (row >= n_rows) return make_float2(INFINITY, 0.f);
    const int64_t tok = q_row + tok0 + row / G;
    const float2 ml = row_ml[tok * num_kv_heads * G + kvh * G + row % G];
    return make_float2(ml.x, 1.0f / ml.y);
  };
  int base[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    base[i] = (c >> 4) * 2048 + (c & 15) * 32 + 8 * ((2 * i + h) ^ ((c >> 2) & 3));

  wait_all();
  __syncthreads();
  for (int s = 0; s < n_stages; ++s) {
    if (s + 1 < n_stages) issue(s + 1);
    const uint16_t *stage = smem + (s & 1) * kStageElems;
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {
      const int r = 2 * s + rb;
      if (32 * r >= n_rows) break;
      // a block whose last row sees none of the wave's keys adds nothing
      const int end = min(tok1 - 1, tok0 + (32 * r + 31) / G) + cache;
      if (end < first) continue;
      const float2 ml = row_of(r);
      const int place = cache + tok0 + (32 * r + c) / G;
      const bool cut = cache + tok0 + 32 * r / G < first + 63;  // some row does not see all keys
      bf16x8 qop[8];
#pragma unroll
      for (int kk = 0; kk < 8; ++kk)
        qop[kk] = *reinterpret_cast<const bf16x8 *>(stage + 4096 * rb + base[kk & 1] + 512 * (kk >> 1));
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        f32x16 sc;
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[i] = 0.f;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kop[b][kk], qop[kk], sc, 0, 0, 0);
        if (cut) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (first + 32 * b + 8 * (i >> 2) + 4 * h + (i & 3) > place) sc[i] = -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i], scale_log2, -ml.x));
          sum[b][i] = __builtin_fmaf(p, ml.y, sum[b][i]);
        }
      }
    }
    wait_all();
    __syncthreads();
  }
  // Join the 32 rows; lane (0, h) has four keys in a row.
  float *dst = partials + (static_cast<int64_t>(part) * num_kv_heads + kvh) * stride + off + first;
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) sum[b][i] += __shfl_xor(sum[b][i], o);
  if (c == 0) {
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<f32x4 *>(dst + 32 * b + 8 * j + 4 * h) =
            f32x4{sum[b][4 * j], sum[b][4 * j + 1], sum[b][4 * j + 2], sum[b][4 * j + 3]};
  }
}

// Item = {row of the table, t0, t1, sources, first source, q_row or -1, offset, 0}: at most 256
// tokens [t0, t1). With q_row >= 0 the sources are the scores of the query heads, turned into
// weights by the row's maxima and sums; else partial sums. Source x of token t is at
// src[x * stride + offset + t]. Four waves take the sources in turn.
__global__ __launch_bounds__(256) void add_kernel(
    const int32_t *__restrict__ items, const float *__restrict__ scores, int64_t score_stride,
    const float *__restrict__ partials, int64_t partial_stride,
    const float2 *__restrict__ row_ml, int num_q_heads, float scale_log2,
    float *__restrict__ weights, int64_t weights_stride) {
  __shared__ f32x4 box[3][64];
  const int32_t *it = items + 8 * blockIdx.x;
  const int row = it[0], t0 = it[1], t1 = it[2], n = it[3], from = it[4], q_row = it[5];
  const int64_t off = it[6];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int t = t0 + 4 * lane;
  const bool live = t < t1;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  if (live) {
    if (q_row >= 0) {
      const float2 *ml = row_ml + static_cast<int64_t>(q_row) * num_q_heads;
#pragma unroll 4
      for (int x = wave; x < n; x += 4) {
        const f32x4 s = *reinterpret_cast<const f32x4 *>(scores + x * score_stride + off + t);
        const float2 r = ml[x];
        const float inv = 1.0f / r.y;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          sum[e] = __builtin_fmaf(
              __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], scale_log2, -r.x)), inv, sum[e]);
      }
    } else {
#pragma unroll 4
      for (int x = wave; x < n; x += 4)
        sum += *reinterpret_cast<const f32x4 *>(partials + (from + x) * partial_stride + off + t);
    }
  }
  if (wave > 0) box[wave - 1][lane] = sum;
  __syncthreads();
  if (wave != 0 || !live) return;
#pragma unroll
  for (int w = 0; w < 3; ++w) sum += box[w][lane];
  float *dst = weights + row * weights_stride + t;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (t + e < t1) dst[e] += sum[e];
}

}  // namespace
}  // namespace hy

using hy::kHeadDim;

extern "C" int hy_token_weights(
    const void *q, int64_t q_stride_seq, int64_t q_stride_tok, int64_t q_stride_head,
    const void *k_pool, int64_t pool_head_stride, const int32_t *page_table,
    int64_t page_table_stride, const int32_t *items, int32_t n_items, const int32_t *adds,
    int32_t n_adds, const float *scores, int64_t score_stride, float *partials,
    int64_t partial_stride, const float *row_ml, float *weights, int64_t weights_stride,
    int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t page_size, float scale,
    void *stream) {
  hy::clear_error();
  HY_REQUIRE(scale > 0.f, "softmax scale must be positive");
  HY_REQUIRE(num_kv_heads >= 1 && num_q_heads >= num_kv_heads &&
                 num_q_heads % num_kv_heads == 0,
             "num_q_heads (%d) must be a positive multiple of num_kv_heads (%d)",
             num_q_heads, num_kv_heads);
  HY_REQUIRE_SUPPORTED(head_dim == kHeadDim, "head_dim %d unsupported (need %d)", head_dim,
                       kHeadDim);
  HY_REQUIRE_SUPPORTED(page_size >= 32 && (page_size & (page_size - 1)) == 0,
                       "page_size %d unsupported (power of two >= 32 required)", page_size);
  HY_REQUIRE(n_items >= 0 && n_items <= 65535 && n_adds >= 0,
             "hy_token_weights: %d items (0 to 65535), %d additions", n_items, n_adds);
  if (n_adds == 0) return HY_OK;
  HY_REQUIRE(q && k_pool && page_table && adds && row_ml && weights && (n_items == 0 || items),
             "hy_token_weights: null pointer argument");
  HY_REQUIRE(scores || partials, "hy_token_weights: null pointer argument");
  HY_REQUIRE(n_items == 0 || partials, "hy_token_weights: null pointer argument");
  HY_REQUIRE(((reinterpret_cast<uintptr_t>(scores) | reinterpret_cast<uintptr_t>(partials)) & 15) ==
                     0 &&
                 score_stride % 4 == 0 && partial_stride % 4 == 0,
             "hy_token_weights: scores and partial sums lie on 16 bytes");
  const int G = num_q_heads / num_kv_heads;
  const float scale_log2 = scale * hy::kLog2e;
  const int page_shift = __builtin_ctz(static_cast<unsigned>(page_size));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const uint16_t *qq = static_cast<const uint16_t *>(q);
  const uint16_t *kp = static_cast<const uint16_t *>(k_pool);
  const float2 *ml = reinterpret_cast<const float2 *>(row_ml);
  const bool q_aligned = (reinterpret_cast<uintptr_t>(q) & 15) == 0 &&
                         ((q_stride_seq | q_stride_tok | q_stride_head) & 7) == 0;
  if (n_items > 0) {
    void (*kernel)(const uint16_t *, int64_t, int64_t, int64_t, const uint16_t *, int64_t,
                   const int32_t *, int64_t, const int32_t *, const float2 *, float *, int64_t, int,
                   int, float, bool) = nullptr;
    switch (G) {
      case 1: kernel = hy::weigh_kernel<1>; break;
      case 2: kernel = hy::weigh_kernel<2>; break;
      case 4: kernel = hy::weigh_kernel<4>; break;
      case 8: kernel = hy::weigh_kernel<8>; break;
      case 16: kernel = hy::weigh_kernel<16>; break;
      default:
        hy::set_error("GQA group size %d unsupported (1, 2, 4, 8, 16)", G);
        return HY_EUNSUPPORTED;
    }
    hipLaunchKernelGGL(kernel, dim3(num_kv_heads, n_items), dim3(256), 0, st, qq, q_stride_seq,
                       q_stride_tok, q_stride_head, kp, pool_head_stride, page_table,
                       page_table_stride, items, ml, partials, partial_stride, num_kv_heads,
                       page_shift, scale_log2, q_aligned);
  }
  hipLaunchKernelGGL(hy::add_kernel, dim3(n_adds), dim3(256), 0, st, adds, scores, score_stride,
                     partials, partial_stride, ml, num_q_heads, scale_log2, weights,
                     weights_stride);
  return hy::launch_status("hy_token_weights");
}
