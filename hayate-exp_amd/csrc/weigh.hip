// What weight every cached token got from a tick's queries, added to a table (gfx950):
//   w[t] += sum over the sequence's rows i and query heads h of
//           exp(scale q_ih . k_t - max_ih) / sum_ih,   t <= position of i,
// with the rows' maxima and sums that the attention kernels leave (exp2 domain).
//
// Single tokens: the decode kernel has stored its raw scores, 4 bytes a head and key where K and
// V take 512 bytes a kv head and key; finish_kernel turns them into weights and sums the heads,
// beside the workgroups that join the decode partials (18.1 -> 15.1 us a call for one token on 2,000
// against a launch behind the merge, 91 -> 89 for 32 on up to 8,000; 13.5 with the loads of up to 64
// partials, and of the first scores, in flight together: 6.0 us of its own instead of 9.1).
// Chunks: storing scores would cost more than the products (512 rows x 32 heads x 4 bytes a key),
// so weigh_kernel computes them again from K and Q, an item 256 keys by a range of rows, and
// leaves a sum per kv head, range and key; finish_kernel adds those. Every sum has a fixed order.
//
// weigh_kernel: one workgroup of four waves per (kv head, item), each wave 64 keys whose K it
// keeps in registers; the rows go through LDS, 64 a stage, and meet them in
// v_mfma_f32_32x32x16_bf16 as S = K Q^T (lane l, c = l % 32, h = l / 32: row c's scores for keys
// 8 (i / 4) + 4 h + i % 4 of a 32-key block), so a lane adds up its row's weights key by key over
// the whole range and the 32 rows of a block are only joined at the end. Bound by the exponentials
// and the products together (VALU and MFMA do not overlap within a wave's own chain: 0.32 us a
// 32 x 32 unit and head group for both): 2 chunks of 512 behind 1,000 to 3,584 tokens take 36 us for
// 19 GFLOP. K in registers and rows through LDS rather than the reverse: a wave's maxima and sums
// (row_ml) then change with the stage, but its 64 sums stay, where rows in registers would add
// across lanes for every block.

#include "attend.h"
#include "hy_common.h"
#include "weigh_shape.h"

namespace hy {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kStageElems = kWeighRows * kHeadDim;
constexpr int kStages = 3;
constexpr int kMaxHeads = 1024;  // query heads

__device__ __forceinline__ void load_to_lds(const uint16_t *g, const uint16_t *lds) {
  const uint32_t m0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
      (const __attribute__((address_space(3))) uint16_t *)lds));
  // (a load that reads M0 must not directly follow its write)
  __asm__ volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
                   :
                   : "v"(g), "s"(__builtin_amdgcn_readfirstlane(m0))
                   : "memory");
}

// At most N vector-memory loads of this wave outstanding (they return in order), and no LDS or
// scalar access.
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N >= 0 && N < 16, "the counter's low bits");
  __builtin_amdgcn_s_waitcnt(N | 7 << 4);
  __asm__ volatile("" ::: "memory");
}

template <int N>
__device__ __forceinline__ float ror16(float x) {
  return __int_as_float(
      __builtin_amdgcn_mov_dpp(__float_as_int(x), 0x120 + N, 0xf, 0xf, false));
}

constexpr int kSchedMfma = 0x008;
constexpr int kSchedValu = 0x002 | 0x400;  // VALU, transcendentals too

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
                  float scale_log2) {
  __shared__ __attribute__((aligned(1024))) uint16_t smem[kStages * kStageElems];
  const int32_t *it = items + 8 * blockIdx.y;
  const int kvh = blockIdx.x;
  const int seq = it[0], key0 = it[1], tok1 = it[3];
  const int part = it[4], q_row = it[5], cache = it[6], off = it[7];
  // tokens before the block's first key see none of it
  const int tok0 = max(it[2], key0 - cache);
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
  const uint16_t *qb =
      q + seq * q_ss + static_cast<int64_t>(q_row + tok0) * q_st + kvh * G * q_sh + chunk8;
  auto issue = [&](int s) __attribute__((always_inline)) {
    uint16_t *dst = smem + (s % kStages) * kStageElems + 2048 * wave;
    const int row = min(kWeighRows * s + 16 * wave + (lane >> 2), n_rows - 1);
    const uint16_t *src = qb + static_cast<int64_t>(row / G) * q_st + (row % G) * q_sh;
#pragma unroll
    for (int j = 0; j < 4; ++j) load_to_lds(src + 32 * j, dst + 512 * j);
  };
  // This lane's row of row block r: its exponent base and the inverse of its sum. Rows past the
  // end weigh nothing.
  const float2 *ml_rows = row_ml + static_cast<int64_t>(q_row + tok0) * num_kv_heads * G + kvh * G;
  auto load_ml = [&](int r) __attribute__((always_inline)) {
    const uint32_t row = min(32 * r + c, n_rows - 1);
    return ml_rows[row / G * (num_kv_heads * G) + row % G];
  };
  auto usable = [&](float2 ml, int r) __attribute__((always_inline)) {
    const bool live = 32 * r + c < n_rows;
    return make_float2(live ? ml.x : INFINITY, live ? __builtin_amdgcn_rcpf(ml.y) : 0.f);
  };

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
  float2 ml_next[2] = {load_ml(0), load_ml(1)};
  float sum[2][16];
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) sum[b][i] = 0.f;

  int base[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    base[i] = (c >> 4) * 2048 + (c & 15) * 32 + 8 * ((2 * i + h) ^ ((c >> 2) & 3));
  auto read_q = [&](bf16x8 (&op)[8], int s, int rb) __attribute__((always_inline)) {
    const uint16_t *at = smem + (s % kStages) * kStageElems + 4096 * rb;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk)
      op[kk] = *reinterpret_cast<const bf16x8 *>(at + base[kk & 1] + 512 * (kk >> 1));
  };
  auto scores = [&](const bf16x8 (&k)[8], const bf16x8 (&op)[8]) __attribute__((always_inline)) {
    f32x16 sc;
#pragma unroll
    for (int i = 0; i < 16; ++i) sc[i] = 0.f;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk)
      sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[kk], op[kk], sc, 0, 0, 0);
    return sc;
  };
  // Keys that a row of row block r does not see.
  auto mask = [&](f32x16 &sc, int b, int r) __attribute__((always_inline)) {
    const int last = cache + tok0 + (32 * r + c) / G - (first + 32 * b + 4 * h);
#pragma unroll
    for (int i = 0; i < 16; ++i) sc[i] = 8 * (i >> 2) + (i & 3) > last ? -INFINITY : sc[i];
  };
  auto add = [&](const f32x16 &sc, int b, const float2 &ml) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i], scale_log2, -ml.x));
      sum[b][i] = __builtin_fmaf(p, ml.y, sum[b][i]);
    }
  };
  // One product's matrix instructions among another's exponentials. The sums count as used here,
  // so that the compiler keeps what makes them in this straight piece of code.
  auto mix = [&](int b) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
      __builtin_amdgcn_sched_group_barrier(kSchedValu, 6, 0);
    }
    const float(&x)[16] = sum[b];
    __asm__ volatile("" ::"v"(x[0]), "v"(x[1]), "v"(x[2]), "v"(x[3]), "v"(x[4]), "v"(x[5]),
                     "v"(x[6]), "v"(x[7]), "v"(x[8]), "v"(x[9]), "v"(x[10]), "v"(x[11]),
                     "v"(x[12]), "v"(x[13]), "v"(x[14]), "v"(x[15]));
    __builtin_amdgcn_sched_barrier(0);
  };

  issue(0);
  if (n_stages > 1) issue(1);
  wait_loads<0>();  // K too, which no wait of the loop is to be for
  __syncthreads();
  bf16x8 qa[8], qc[8];
  read_q(qa, 0, 0);
  f32x16 sa = scores(kop[0], qa), sb;
  for (int s = 0; s < n_stages; ++s) {
    // (these were loaded a stage ago: waited for behind new loads, they would wait for those too)
    const float2 ml0 = usable(ml_next[0], 2 * s), ml1 = usable(ml_next[1], 2 * s + 1);
    __builtin_amdgcn_sched_barrier(0);
    if (s + 2 < n_stages) issue(s + 2);
    ml_next[0] = load_ml(2 * s + 2);
    ml_next[1] = load_ml(2 * s + 3);
    // whether some row of the row block does not see all keys of the wave
    const bool cut0 = cache + tok0 + 64 * s / G < first + 63;
    const bool cut1 = cache + tok0 + (64 * s + 32) / G < first + 63;
    // The scores of each (row block, key block) are made while the ones before are used: straight
    // code, which the scheduler can mix (a mask comes before it).
    if (cut0) mask(sa, 0, 2 * s);
    read_q(qc, s, 1);
    __builtin_amdgcn_sched_barrier(0);
    sb = scores(kop[1], qa);
    add(sa, 0, ml0);
    mix(0);
    if (cut0) mask(sb, 1, 2 * s);
    __builtin_amdgcn_sched_barrier(0);
    sa = scores(kop[0], qc);
    add(sb, 1, ml0);
    mix(1);
    if (cut1) mask(sa, 0, 2 * s + 1);
    // stage s + 1 has arrived in every wave (what is read of it past the last stage is unused)
    if (s + 2 < n_stages)
      wait_loads<4>();
    else
      wait_loads<0>();
    __syncthreads();
    read_q(qa, s + 1 < n_stages ? s + 1 : s, 0);
    __builtin_amdgcn_sched_barrier(0);
    sb = scores(kop[1], qc);
    add(sa, 0, ml1);
    mix(0);
    if (cut1) mask(sb, 1, 2 * s + 1);
    __builtin_amdgcn_sched_barrier(0);
    sa = scores(kop[0], qa);
    add(sb, 1, ml1);
    mix(1);
  }
  // Join the 32 rows; lane (0, h) has four keys in a row.
  float *dst = partials + (static_cast<int64_t>(part) * num_kv_heads + kvh) * stride + off + first;
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float x = sum[b][i];
      x += ror16<8>(x);
      x += ror16<4>(x);
      x += ror16<2>(x);
      x += ror16<1>(x);
      sum[b][i] = x + __shfl_xor(x, 16);
    }
  if (c == 0) {
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<f32x4 *>(dst + 32 * b + 8 * j + 4 * h) =
            f32x4{sum[b][4 * j], sum[b][4 * j + 1], sum[b][4 * j + 2], sum[b][4 * j + 3]};
  }
}

// One decode token's output from its partials, a dim a lane and a head two waves: the sums of
// decode_merge_kernel in its order (rounds of eight, each with the maximum so far as its base).
// 64 partials are in flight at a time; their factors are made a lane each. it = {seq, first
// slot, slots, q_row}.
__device__ __forceinline__ void join_partials(const int32_t *it, int head0, uint16_t *out,
                                              int64_t o_ss, int64_t o_st, int64_t o_sh,
                                              const float *ws_acc, const float *ws_ml,
                                              int num_q_heads) {
  const int seq = it[0], first = it[1], n = it[2];
  const int64_t q_row = it[3];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int hq = head0 + (wave >> 1);
  if (hq >= num_q_heads) return;
  const int d = 64 * (wave & 1) + lane;
  float mx = -INFINITY, lsum = 0.f, acc = 0.f;
  auto lane_of = [](float v, int i) __attribute__((always_inline)) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), i));
  };
  for (int s0 = 0; s0 < n; s0 += 64) {
    const int count = min(n - s0, 64);
    const int64_t slot0 = first + s0;
    float2 ml = *reinterpret_cast<const float2 *>(
        ws_ml + ((slot0 + min(lane, count - 1)) * num_q_heads + hq) * 2);
    float x[64];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      if (8 * r >= count) break;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        x[8 * r + j] = ws_acc[((slot0 + min(8 * r + j, count - 1)) * num_q_heads + hq) * kHeadDim + d];
    }
    if (lane >= count) ml = make_float2(-INFINITY, 0.f);
    // the maximum of the lane's eight, and of all before them
    float top = ml.x;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
    float base = mx, before = mx, after = mx;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const float next = fmaxf(after, lane_of(top, 8 * r));
      if (lane >> 3 == r) {
        before = after;
        base = next;
      }
      after = next;
    }
    mx = after;
    const float f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - base);
    const float fl = f * ml.y;
    const float rebase = before == -INFINITY ? 0.f : exp2f(before - base);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      if (8 * r >= count) break;
      const float old = lane_of(rebase, 8 * r);
      lsum *= old;
      acc *= old;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (8 * r + j >= count) break;
        lsum += lane_of(fl, 8 * r + j);
        acc += lane_of(f, 8 * r + j) * x[8 * r + j];
      }
    }
  }
  const float o = acc / lsum;
  out[seq * o_ss + q_row * o_st + hq * o_sh + d] = static_cast<uint16_t>(pack_bf16x2_rne(o, o));
}

// Slots of a decode token that one wave of the additions loads at a time, and scores.
constexpr int kSlotsAhead = 16;
constexpr int kScoresAhead = 8;

// The first n_adds workgroups add to the table, the others join the partials of two heads of a
// decode token each. Item = {row of the table, t0, t1, sources, first source, decode,
// offset, 0}: at most 256 tokens [t0, t1). Of a chunk the sources are rows of partial sums; of a
// decode token they are its partial slots, whose maxima and sums turn the scores of all query
// heads into weights. Source or head x of token t is at src[x * stride + offset + t]; four waves
// take them in turn.
__global__ __launch_bounds__(256) void finish_kernel(
    uint16_t *__restrict__ out, int64_t o_ss, int64_t o_st, int64_t o_sh,
    const int32_t *__restrict__ join_items, int groups,
    const float *__restrict__ ws_acc, const float *__restrict__ ws_ml,
    const int32_t *__restrict__ items, int n_adds, const float *__restrict__ scores,
    int64_t score_stride,
    const float *__restrict__ partials, int64_t partial_stride, int num_q_heads, float scale_log2,
    float *__restrict__ weights, int64_t weights_stride) {
  __shared__ f32x4 box[3][64];
  __shared__ float2 head_ml[kMaxHeads], part_ml[4][64];
  const int bid = blockIdx.x;
  if (bid >= n_adds) {
    join_partials(join_items + 4 * ((bid - n_adds) / groups), 2 * ((bid - n_adds) % groups), out,
                  o_ss, o_st, o_sh, ws_acc, ws_ml, num_q_heads);
    return;
  }
  const int32_t *it = items + 8 * bid;
  const int row = it[0], t0 = it[1], t1 = it[2], n = it[3], from = it[4];
  const bool decode = it[5] != 0;
  const int64_t off = it[6];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int t = t0 + 4 * lane;
  const bool live = t < t1;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  // (loads that depend on nothing go out first: what is in the table, and the first scores)
  float *dst = weights + row * weights_stride + t;
  float was[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) was[e] = wave == 0 && t + e < t1 ? dst[e] : 0.f;
  if (decode) {
    const int t_in = live ? t : t0;
    auto load_score = [&](int i) __attribute__((always_inline)) {
      return *reinterpret_cast<const f32x4 *>(scores + min(wave + 4 * i, num_q_heads - 1) * score_stride +
                                              off + t_in);
    };
    f32x4 sc[kScoresAhead];
#pragma unroll
    for (int i = 0; i < kScoresAhead; ++i) sc[i] = load_score(i);
    // every head's maximum and inverse sum: lanes are heads, waves take the slots in turn
    for (int h0 = 0; h0 < num_q_heads; h0 += 64) {
      const int h = min(h0 + lane, num_q_heads - 1);
      float m = -INFINITY, l = 0.f;
      for (int s0 = wave; s0 < n; s0 += 4 * kSlotsAhead) {
        float2 ml[kSlotsAhead];
        float top = m;
#pragma unroll
        for (int j = 0; j < kSlotsAhead; ++j) {
          ml[j] = make_float2(-INFINITY, 0.f);
          if (s0 + 4 * j >= n) continue;
          ml[j] = *reinterpret_cast<const float2 *>(
              ws_ml + (static_cast<int64_t>(from + s0 + 4 * j) * num_q_heads + h) * 2);
        }
#pragma unroll
        for (int j = 0; j < kSlotsAhead; ++j) top = fmaxf(top, ml[j].x);
        l = m == -INFINITY ? 0.f : l * exp2f(m - top);
#pragma unroll
        for (int j = 0; j < kSlotsAhead; ++j)
          if (ml[j].x != -INFINITY) l += ml[j].y * exp2f(ml[j].x - top);
        m = top;
      }
      part_ml[wave][lane] = make_float2(m, l);
      __syncthreads();
      if (wave == 0 && h0 + lane < num_q_heads) {
        float top = -INFINITY, all = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = fmaxf(top, part_ml[w][lane].x);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float2 p = part_ml[w][lane];
          if (p.x != -INFINITY) all += p.y * exp2f(p.x - top);
        }
        head_ml[h0 + lane] = make_float2(top, 1.0f / all);
      }
      __syncthreads();
    }
    for (int i0 = 0; wave + 4 * i0 < num_q_heads; i0 += kScoresAhead) {
#pragma unroll
      for (int i = 0; i < kScoresAhead; ++i) {
        const int x = wave + 4 * (i0 + i);
        if (x >= num_q_heads) break;
        const float2 r = head_ml[x];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          sum[e] = __builtin_fmaf(
              __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i][e], scale_log2, -r.x)), r.y, sum[e]);
      }
      if (wave + 4 * (i0 + kScoresAhead) >= num_q_heads) break;
#pragma unroll
      for (int i = 0; i < kScoresAhead; ++i) sc[i] = load_score(i0 + kScoresAhead + i);
    }
  } else if (live) {
#pragma unroll 4
    for (int x = wave; x < n; x += 4)
      sum += *reinterpret_cast<const f32x4 *>(partials + (from + x) * partial_stride + off + t);
  }
  if (wave > 0) box[wave - 1][lane] = sum;
  __syncthreads();
  if (wave != 0 || !live) return;
#pragma unroll
  for (int w = 0; w < 3; ++w) sum += box[w][lane];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (t + e < t1) dst[e] = was[e] + sum[e];
}

int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

}  // namespace
}  // namespace hy

int hy::check_weigh(const char *name, const Rows &q, const Shape &s, const Weigh &w) {
  HY_REQUIRE(w.n_items >= 0 && w.n_items <= 65535 && w.n_adds >= 0,
             "%s: %d items (0 to 65535), %d additions", name, w.n_items, w.n_adds);
  HY_REQUIRE_SUPPORTED(s.num_q_heads <= kMaxHeads, "%s: %d query heads (at most %d)", name,
                       s.num_q_heads, kMaxHeads);
  HY_REQUIRE(w.n_adds == 0 || (w.adds && w.weights && (w.scores.at || w.partials)),
             "%s: null pointer argument", name);
  HY_REQUIRE(w.n_items == 0 || (w.items && w.partials && w.row_ml), "%s: null pointer argument", name);
  HY_REQUIRE(((reinterpret_cast<uintptr_t>(w.scores.at) | reinterpret_cast<uintptr_t>(w.partials)) &
              15) == 0 &&
                 w.scores.stride % 4 == 0 && w.partial_stride % 4 == 0,
             "%s: scores and partial sums lie on 16 bytes", name);
  HY_REQUIRE((reinterpret_cast<uintptr_t>(w.row_ml) & 7) == 0, "%s: row_ml lies on 8 bytes", name);
  HY_REQUIRE((reinterpret_cast<uintptr_t>(q.at) & 15) == 0 && ((q.seq | q.tok | q.head) & 7) == 0,
             "%s: q rows lie on 16 bytes", name);
  return HY_OK;
}

int hy::weigh_chunks(const char *name, const Rows &q, const Pools &pools, const Shape &s,
                     const Weigh &w, void *stream) {
  if (w.n_items == 0) return HY_OK;
  const int G = s.num_q_heads / s.num_kv_heads;
  decltype(&weigh_kernel<1>) kernel = nullptr;
  switch (G) {
    case 1: kernel = weigh_kernel<1>; break;
    case 2: kernel = weigh_kernel<2>; break;
    case 4: kernel = weigh_kernel<4>; break;
    case 8: kernel = weigh_kernel<8>; break;
    case 16: kernel = weigh_kernel<16>; break;
    default:
      hy::set_error("GQA group size %d unsupported (1, 2, 4, 8, 16)", G);
      return HY_EUNSUPPORTED;
  }
  hipLaunchKernelGGL(kernel, dim3(s.num_kv_heads, w.n_items), dim3(256), 0,
                     static_cast<hipStream_t>(stream), static_cast<const uint16_t *>(q.at), q.seq,
                     q.tok, q.head, static_cast<const uint16_t *>(pools.k), pools.head_stride,
                     pools.page_table, pools.page_table_stride, w.items,
                     reinterpret_cast<const float2 *>(w.row_ml), w.partials, w.partial_stride,
                     s.num_kv_heads, __builtin_ctz(static_cast<unsigned>(s.page_size)),
                     s.scale * kLog2e);
  return hy::launch_status(name);
}

int hy::finish_weights(const char *name, const Rows &out, const Items &merge, const Workspace &ws,
                       const Shape &s, const Weigh &w, void *stream) {
  const int groups = (s.num_q_heads + 1) / 2;
  const int64_t blocks = static_cast<int64_t>(merge.count) * groups + w.n_adds;
  HY_REQUIRE(blocks <= INT32_MAX, "%s: too many records", name);
  if (blocks == 0) return HY_OK;
  HY_REQUIRE(merge.count == 0 || (out.at && merge.at && ws.at), "%s: null pointer argument", name);
  // (the decode call before has checked that the partials fit)
  const float *acc = static_cast<const float *>(ws.at);
  const float *ml = reinterpret_cast<const float *>(
      static_cast<const char *>(ws.at) +
      align256(static_cast<int64_t>(merge.slots) * s.num_q_heads * kHeadDim * 4));
  hipLaunchKernelGGL(finish_kernel, dim3(static_cast<uint32_t>(blocks)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), static_cast<uint16_t *>(out.at), out.seq,
                     out.tok, out.head, merge.at, groups, acc, ml, w.adds, w.n_adds, w.scores.at,
                     w.scores.stride, w.partials, w.partial_stride, s.num_q_heads, s.scale * kLog2e,
                     w.weights, w.weights_stride);
  return hy::launch_status(name);
}
