// Attention for trees of drafted tokens over a paged cache (gfx950).
//
// A request with c cached tokens and n drafted ones holds them in slots 0 ..
// c + n - 1. Node i's query sees every cached token, its ancestors and itself:
//   o_i = sum_j softmax_j(scale q_i k_j) v_j,  j < c  or  j - c in line(i).
// Slots of other branches may hold anything, infinities and NaN included.
//
// Work split: as in the decode kernel, the key steps (64 keys) of all requests, in
// order, form one stream per kv head that the planner cuts into one chunk per
// compute unit; a chunk holds pieces (the part of one request inside it). All
// rows (node, head of the group) of a request read each K/V row once: up to 256
// rows in W waves of 32. A piece that is not a request's whole stream leaves
// fp32 partials that tree_merge_kernel joins.
//
// A chunk's tiles (64 keys of K and V, 32 KiB) go through a ring of four LDS
// stages by direct-to-LDS loads, three tiles ahead of the one being used and
// across piece borders, so HBM stays busy while a piece is closed.
//
// The products are those of the prefill kernel: v_mfma_f32_32x32x16_bf16 with
// S^T = K Q^T and O^T += V^T P^T (lane l, c = l % 32, h = l / 32): a lane ends with
// row c's scores for keys 8 (i / 4) + 4 h + i % 4 of a 32-key block, which are, in
// its order, the probabilities the second product wants. Scores, the running
// maximum and sum and the accumulators are fp32; the probabilities are rounded
// to bf16 for the second product, the matrix core's input type.
//
// Only the blocks that hold drafted slots are masked: a node's line is a bit mask
// over the slots, kept in LDS per row.

#include "hy_common.h"
#include "tree_shape.h"

namespace hy {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazy = 8.0f;     // the exponent base moves when a score exceeds it by this (exp2)
constexpr float kLazyP = 256.0f;  // 2^kLazy
constexpr int kTile = kTreeTileKeys;
constexpr int kStage = 2 * kTile * kHeadDim;  // halfs per stage: K tile, then V tile
constexpr int kStages = 4;
constexpr int kMaskWords = kTreeMaxNodes / 32;
constexpr int kMaskStride = kMaskWords + 1;  // a zero word behind, and rows on other banks

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

__device__ __forceinline__ s16x4 tr_read(const uint16_t *p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(const_cast<uint16_t *>(p)));
}

// 16 bytes from base + off (bytes) straight into LDS: lane l's land at lds + 16 l
// (lds wave-uniform, through M0, with the wait state the ISA asks for between
// its write and the load). The caller waits (wait_loads) before it reads them.
__device__ __forceinline__ void load_to_lds(const uint16_t *base, uint32_t off,
                                            const uint16_t *lds) {
  const uint32_t m0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
      (const __attribute__((address_space(3))) uint16_t *)lds));
  __asm__ volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                   :
                   : "v"(off), "s"(base), "s"(__builtin_amdgcn_readfirstlane(m0))
                   : "memory");
}

// At most N vector-memory loads of this wave outstanding (they return in
// order), and no LDS or scalar read.
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N >= 0 && N < 64, "a six-bit counter");
  __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 7 << 4);
  __asm__ volatile("" ::: "memory");
}

__device__ __forceinline__ float halves_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

struct Piece {
  int seq, q0, q1, kv0, kv1, slot, q_row, cache;
  __device__ __forceinline__ int tiles() const { return (kv1 - kv0 + kTile - 1) / kTile; }
};

__device__ __forceinline__ Piece load_piece(const int32_t *r) {
  return Piece{r[0], r[1], r[2], r[3], r[4], r[5], r[6], r[7]};
}

template <int W>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(W > 4 ? 2 : 1, W > 4 ? 2 : 1)))
void tree_kernel(const uint16_t *__restrict__ q, int64_t q_ss, int64_t q_st, int64_t q_sh,
                 uint16_t *__restrict__ out, int64_t o_ss, int64_t o_st, int64_t o_sh,
                 const uint16_t *__restrict__ k_pool, const uint16_t *__restrict__ v_pool,
                 int64_t pool_hs, const int32_t *__restrict__ page_table, int64_t pt_stride,
                 const int32_t *__restrict__ items, int n_chunks,
                 const uint32_t *__restrict__ lines, int line_words, float *__restrict__ ws_acc,
                 float *__restrict__ ws_ml, int n_slots, int group_shift, int page_shift,
                 float scale_log2) {
  constexpr int kLoads = 32 / W;  // load instructions of a wave per tile
  __shared__ __attribute__((aligned(1024))) uint16_t ring[kStages * kStage];
  __shared__ uint32_t line[W * 32 * kMaskStride];

  const int32_t *ch = items + kTreeChunkInts * blockIdx.y;
  const int32_t *pieces = items + kTreeChunkInts * n_chunks;
  const int kvh = blockIdx.x;
  const int p_end = ch[1];
  const int n_tiles = ch[2];
  // an empty chunk record pads a list to a fixed launch size
  if (n_tiles <= 0) return;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int c = lane & 31;
  const int h = lane >> 5;
  const int h0 = kvh << group_shift;
  const int group_mask = (1 << group_shift) - 1;
  const int page_mask = (1 << page_shift) - 1;
  const uint16_t *kh = k_pool + kvh * pool_hs;
  const uint16_t *vh = v_pool + kvh * pool_hs;

  // ---- tile loads -------------------------------------------------------
  // Issue cursor: the piece holding the next tile to load. A tile's two
  // 32-key halves each lie in one page (pages hold at least 32 keys, pieces
  // start at multiples of 64). Keys past the piece are read from its last page:
  // in bounds, and masked.
  Piece ip = load_piece(ch + 8);
  int ip_index = ch[0], ip_tile = 0;  // its record, and its first tile in the chunk
  struct Tile {
    uint32_t page[2];
    int key;
  };
  auto fetch = [&](int t) __attribute__((always_inline)) {
    while (t >= ip_tile + ip.tiles()) {
      ip_tile += ip.tiles();
      ip = load_piece(pieces + 8 * ++ip_index);
    }
    Tile x;
    x.key = ip.kv0 + kTile * (t - ip_tile);
    const int32_t *pt = page_table + ip.seq * pt_stride;
    // held unsigned: page ids are non-negative, and widen without a sign
    x.page[0] = static_cast<uint32_t>(pt[x.key >> page_shift]);
    x.page[1] = static_cast<uint32_t>(pt[min(x.key + 32, ip.kv1 - 1) >> page_shift]);
    return x;
  };
  // The layouts of the prefill kernel, conflict-free for the reads below; in
  // units of 8 dims: K unit(row, chunk) = (row / 16) * 256 + (chunk / 4) * 64 +
  // (row % 16) * 4 + (chunk % 4 ^ row / 4 % 4), V unit(row, chunk) = (row / 4) *
  // 64 + (chunk / 4) * 16 + (row % 4) * 4 + chunk % 4. K instruction i loads 16
  // rows (16 (i / 4) ..) of four chunks, V instruction i four whole rows.
  const uint32_t k_off = 256 * (lane >> 2) + 16 * ((lane & 3) ^ ((lane >> 4) & 3));
  const uint32_t v_off = 256 * ((lane >> 2) & 3) + 64 * (lane >> 4) + 16 * (lane & 3);
  auto issue = [&](const Tile &x, int t) __attribute__((always_inline)) {
    uint16_t *dst = ring + (t % kStages) * kStage;
#pragma unroll
    for (int j = 0; j < kLoads / 2; ++j) {
      const int i = wave * (kLoads / 2) + j;
      const int half = i >> 3;
      const int64_t row = (static_cast<int64_t>(half ? x.page[1] : x.page[0]) << page_shift) +
                          ((x.key + 32 * half) & page_mask);
      load_to_lds(kh + row * kHeadDim + 2048 * ((i >> 2) & 1) + 32 * (i & 3), k_off, dst + 512 * i);
      load_to_lds(vh + row * kHeadDim + 512 * (i & 7), v_off, dst + kTile * kHeadDim + 512 * i);
    }
  };

  // ---- this wave's rows of the piece being computed ----------------------
  Piece cp = ip;
  int cp_index = ip_index, cp_tile = 0;
  const int r = 32 * wave + c;
  bool wave_live = false, live = false;
  bf16x8 qop[8];  // row c of Q^T
  f32x16 acc[4];  // O^T[32 db + 8 (i / 4) + 4 h + i % 4][row c]
  float base, shift, l_run;
  uint32_t *row_line = line + r * kMaskStride;
  auto start = [&]() __attribute__((always_inline)) {
    const int rows = (cp.q1 - cp.q0) << group_shift;
    wave_live = 32 * wave < rows;
    live = r < rows;
    base = -INFINITY;
    shift = 0.f;
    l_run = 0.f;
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[db][i] = 0.f;
    if (!wave_live) return;
    const int64_t tok = cp.q_row + cp.q0 + (live ? r >> group_shift : 0);
    const uint16_t *src = q + cp.seq * q_ss + tok * q_st + (h0 + (r & group_mask)) * q_sh + 8 * h;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      u32x4 w = load16(src + 16 * kk);
      if (!live) w = u32x4{0u, 0u, 0u, 0u};
      qop[kk] = __builtin_bit_cast(bf16x8, w);
    }
    if (h == 0)
#pragma unroll
      for (int j = 0; j < kMaskStride; ++j)
        row_line[j] = live && j < line_words ? lines[tok * line_words + j] : 0u;
  };
  // Closes the piece: its output rows, or this wave's partial: fp32, in the
  // accumulator's own order (16 groups of 64 lanes x 16 bytes), live rows only.
  auto finish = [&]() __attribute__((always_inline)) {
    if (!wave_live) return;
    const float l = halves_sum(l_run);
    if (cp.slot < 0) {
      const float inv = 1.0f / l;
      const int64_t tok = cp.q_row + cp.q0 + (r >> group_shift);
      uint16_t *dst = out + cp.seq * o_ss + tok * o_st + (h0 + (r & group_mask)) * o_sh + 4 * h;
      if (live)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int db = j >> 2, i = 4 * (j & 3);
          *reinterpret_cast<uint2 *>(dst + 8 * j) =
              make_uint2(pack_bf16x2_rne(acc[db][i] * inv, acc[db][i + 1] * inv),
                         pack_bf16x2_rne(acc[db][i + 2] * inv, acc[db][i + 3] * inv));
        }
      return;
    }
    const int64_t block = static_cast<int64_t>(kvh) * n_slots + cp.slot + wave;
    float *dst = ws_acc + block * 32 * kHeadDim + 4 * lane;
    if (live) {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int db = j >> 2, i = 4 * (j & 3);
        *reinterpret_cast<f32x4 *>(dst + 256 * j) =
            f32x4{acc[db][i], acc[db][i + 1], acc[db][i + 2], acc[db][i + 3]};
      }
      if (h == 0) *reinterpret_cast<float2 *>(ws_ml + (block * 32 + c) * 2) = make_float2(base, l);
    }
  };

  // LDS read bases (u16 units), as in the prefill kernel.
  const int r16 = lane & 15;
  const int q16 = lane >> 4;
  int k_base[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    k_base[i] = (c >> 4) * 2048 + (c & 15) * 32 + 8 * ((2 * i + h) ^ ((c >> 2) & 3));
  const int v_base = kTile * kHeadDim + 512 * (q16 >> 1) + 32 * (r16 >> 2) + 16 * (q16 & 1) +
                     4 * (r16 & 3);

  // The line bits of the 32 slots from key kb0 on (bit j: slot kb0 + j is seen);
  // slots before the drafted ones are all seen.
  auto line_bits = [&](int kb0) __attribute__((always_inline)) -> uint32_t {
    const int d = kb0 - cp.cache;  // > -32
    if (d < 0) return row_line[0] << -d | ((1u << -d) - 1);
    const uint32_t lo = row_line[d >> 5], hi = row_line[(d >> 5) + 1];
    return static_cast<uint32_t>((static_cast<uint64_t>(hi) << 32 | lo) >> (d & 31));
  };

  // One block of 32 keys from kb0 on, in half b of the stage.
  auto block = [&](const uint16_t *stage, int b, int kb0) __attribute__((always_inline)) {
    const uint16_t *kb = stage + 4096 * b;
    f32x16 s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      const bf16x8 kop = *reinterpret_cast<const bf16x8 *>(kb + k_base[kk & 1] + 512 * (kk >> 1));
      s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kop, qop[kk], s, 0, 0, 0);
    }
    const bool masked = kb0 + 32 > cp.cache;
    uint32_t bits = 0xffffffffu;
    if (masked) {
      bits = live ? line_bits(kb0) : 0u;
      const uint32_t mine = bits >> (4 * h);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        s[i] = mine >> (8 * (i >> 2) + (i & 3)) & 1 ? s[i] : -INFINITY;
    }
    s16x8 vop[8];
    const uint16_t *vb = kb + v_base;
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int kh2 = 0; kh2 < 2; ++kh2) {
        const s16x4 lo = tr_read(vb + 2048 * kh2 + 128 * db);
        const s16x4 hi = tr_read(vb + 2048 * kh2 + 128 * db + 1024);
        vop[2 * db + kh2] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      }

    // Online softmax on raw scores: p = exp2(s scale log2(e) - shift), shift the row's
    // exponent base (0 while it has none). The base moves only when a score exceeds
    // it by 2^8; below that no lane's probabilities sum to more.
    float p[16], psum;
    auto probs = [&]() __attribute__((always_inline)) {
      psum = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], scale_log2, -shift));
        psum += p[i];
      }
    };
    probs();
    // !(psum <= ...) also catches an overflowed sum and NaN
    if (__builtin_expect(__any(base == -INFINITY || !(psum <= kLazyP)), 0)) {
      float m = s[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) m = fmaxf(m, s[i]);
      m = halves_max(m);
      const bool need = base == -INFINITY
                            ? m != -INFINITY
                            : __builtin_fmaf(m, scale_log2, -shift) > kLazy;
      if (__any(need)) {
        const float next = need ? m * scale_log2 : shift;
        const float alpha = base == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(shift - next);
        if (need) base = shift = next;
        l_run *= alpha;
#pragma unroll
        for (int db = 0; db < 4; ++db) acc[db] *= alpha;
        probs();
      }
    }
    l_run += psum;
    bf16x8 pop[2];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      pop[0][i] = static_cast<__bf16>(p[i]);
      pop[1][i] = static_cast<__bf16>(p[8 + i]);
    }
    bool odd = false;  // a drafted slot of the block holds an infinity or NaN in V
    if (masked) {
      // values of slots past the piece are zeroed (they may be any bits)
      if (kb0 + 32 > cp.kv1) {
#pragma unroll
        for (int kh2 = 0; kh2 < 2; ++kh2) {
          s16x8 keep;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            keep[j] = kb0 + 16 * kh2 + 8 * (j >> 2) + 4 * h + (j & 3) < cp.kv1 ? -1 : 0;
#pragma unroll
          for (int db = 0; db < 4; ++db) vop[2 * db + kh2] &= keep;
        }
      }
      u16x2 top = {0, 0};
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const u32x4 w = __builtin_bit_cast(u32x4, vop[x]) & 0x7fff7fffu;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t pair = w[j];  // a bit cast of the element itself would take the first
          top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, pair));
        }
      }
      odd = __any(top[0] >= 0x7f80 || top[1] >= 0x7f80);
    }
    if (__builtin_expect(odd, 0)) {
      // rare: such values leave the product (0 times them is NaN) and reach only
      // the rows that see their slot
#pragma unroll
      for (int x = 0; x < 8; ++x)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if ((vop[x][j] & 0x7f80) == 0x7f80) vop[x][j] = 0;
      for (int key = 0; key < 32 && kb0 + key < cp.kv1; ++key) {
        const uint16_t *row = kb + kTile * kHeadDim + 512 * (key >> 2) + 32 * (key & 3);
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int dim = 8 * (i >> 2) + 4 * h + (i & 3);  // of the 32-dim slice db
            const uint16_t v = row[128 * db + 8 * (dim >> 3) + (dim & 7)];
            if ((v & 0x7f80) == 0x7f80 && (bits >> key & 1))
              acc[db][i] += __uint_as_float(static_cast<uint32_t>(v) << 16);
          }
      }
    }
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int kh2 = 0; kh2 < 2; ++kh2)
        acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            __builtin_bit_cast(bf16x8, vop[2 * db + kh2]), pop[kh2], acc[db], 0, 0, 0);
  };

  // ---- the chunk ---------------------------------------------------------
  start();
  Tile next = fetch(0);
  issue(next, 0);
  if (n_tiles > 1) issue(next = fetch(1), 1);
  if (n_tiles > 2) issue(next = fetch(2), 2);
  if (n_tiles > 3) next = fetch(3);
  for (int t = 0; t < n_tiles; ++t) {
    // tile t has arrived in every wave, and every wave is done with tile t - 1,
    // whose stage tile t + 3 takes
    if (t + 2 < n_tiles)
      wait_loads<(2 * kLoads < 63 ? 2 * kLoads : 63)>();
    else if (t + 1 < n_tiles)
      wait_loads<kLoads>();
    else
      wait_loads<0>();
    __builtin_amdgcn_s_barrier();
    __asm__ volatile("" ::: "memory");
    if (t + 3 < n_tiles) {
      issue(next, t + 3);
      if (t + 4 < n_tiles) next = fetch(t + 4);
    }
    const uint16_t *stage = ring + (t % kStages) * kStage;
    const int key = cp.kv0 + kTile * (t - cp_tile);
    if (wave_live) {
      block(stage, 0, key);
      if (key + 32 < cp.kv1) block(stage, 1, key + 32);
    }
    if (key + kTile >= cp.kv1) {
      finish();
      if (cp_index + 1 < p_end) {
        cp_tile = t + 1;
        cp = load_piece(pieces + 8 * ++cp_index);
        start();
      }
    }
  }
}

// Joins the partials of a request's rows: grid (kv head, merge item, 32-row
// group), thread = row c of the group and dims 8 j8 .. 8 j8 + 7. Item = {seq, q0,
// q1, first_slot, splits, q_row, row blocks a split, 0}. Rows past the item's are neither
// read nor written.
__global__ __launch_bounds__(512) void tree_merge_kernel(
    uint16_t *__restrict__ out, int64_t o_ss, int64_t o_st, int64_t o_sh,
    const int32_t *__restrict__ items, const float *__restrict__ ws_acc,
    const float *__restrict__ ws_ml, int n_slots, int group_shift) {
  const int32_t *it = items + 8 * blockIdx.y;
  const int q0 = it[1];
  const int rows = (it[2] - q0) << group_shift;
  const int splits = it[4];
  const int c = threadIdx.x & 31;
  const int j8 = threadIdx.x >> 5;
  const int row = 32 * blockIdx.z + c;
  // an empty record pads a list to a fixed launch size
  if (row >= rows || splits <= 0) return;
  float mx = -INFINITY, lsum = 0.f;
  f32x4 a0 = {0.f, 0.f, 0.f, 0.f}, a1 = {0.f, 0.f, 0.f, 0.f};
  // rounds of independent loads: the index is clamped to a real split, and the
  // ones past the last are replaced by the empty partial
  constexpr int kRound = 4;
  for (int s0 = 0; s0 < splits; s0 += kRound) {
    float m[kRound], l[kRound];
    f32x4 x0[kRound], x1[kRound];
#pragma unroll
    for (int j = 0; j < kRound; ++j) {
      const int64_t block = static_cast<int64_t>(blockIdx.x) * n_slots + it[3] +
                            min(s0 + j, splits - 1) * it[6] + blockIdx.z;
      const float2 ml = *reinterpret_cast<const float2 *>(ws_ml + (block * 32 + c) * 2);
      m[j] = ml.x;
      l[j] = ml.y;
      const float *src = ws_acc + block * 32 * kHeadDim + 256 * j8 + 4 * c;
      x0[j] = *reinterpret_cast<const f32x4 *>(src);
      x1[j] = *reinterpret_cast<const f32x4 *>(src + 128);
    }
    float cmx = mx;
#pragma unroll
    for (int j = 0; j < kRound; ++j) {
      if (s0 + j >= splits) m[j] = -INFINITY;
      cmx = fmaxf(cmx, m[j]);
    }
    const float f_old = mx == -INFINITY ? 0.f : exp2f(mx - cmx);
    lsum *= f_old;
    a0 *= f_old;
    a1 *= f_old;
#pragma unroll
    for (int j = 0; j < kRound; ++j) {
      if (m[j] == -INFINITY) continue;  // nothing seen (or no such split)
      const float f = exp2f(m[j] - cmx);
      lsum += f * l[j];
      a0 += f * x0[j];
      a1 += f * x1[j];
    }
    mx = cmx;
  }
  const int64_t tok = it[5] + q0 + (row >> group_shift);
  const int head = (blockIdx.x << group_shift) + (row & ((1 << group_shift) - 1));
  store16(out + it[0] * o_ss + tok * o_st + head * o_sh + 8 * j8,
          u32x4{pack_bf16x2_rne(a0[0] / lsum, a0[1] / lsum), pack_bf16x2_rne(a0[2] / lsum, a0[3] / lsum),
                pack_bf16x2_rne(a1[0] / lsum, a1[1] / lsum),
                pack_bf16x2_rne(a1[2] / lsum, a1[3] / lsum)});
}

int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

}  // namespace
}  // namespace hy

using hy::kHeadDim;

extern "C" int64_t hy_tree_workspace_bytes(int32_t n_slots, int32_t num_kv_heads,
                                           int32_t head_dim) {
  if (n_slots <= 0 || num_kv_heads <= 0 || head_dim <= 0) return 0;
  const int64_t rows = static_cast<int64_t>(n_slots) * num_kv_heads * 32;
  return hy::align256(rows * head_dim * 4) + hy::align256(rows * 2 * 4);
}

extern "C" int hy_paged_tree(
    const void *q, int64_t q_stride_seq, int64_t q_stride_tok, int64_t q_stride_head, void *out,
    int64_t o_stride_seq, int64_t o_stride_tok, int64_t o_stride_head, const void *k_pool,
    const void *v_pool, int64_t pool_head_stride, const int32_t *page_table,
    int64_t page_table_stride, const uint32_t *lines, int32_t line_words, const int32_t *items,
    int32_t n_chunks, int32_t max_rows, const int32_t *merge_items, int32_t n_merge,
    int32_t n_slots, void *workspace, int64_t workspace_bytes, int32_t num_q_heads,
    int32_t num_kv_heads, int32_t head_dim, int32_t page_size, float scale, void *stream) {
  hy::clear_error();
  HY_REQUIRE(scale > 0.f, "softmax scale must be positive");
  HY_REQUIRE(num_kv_heads >= 1 && num_q_heads >= num_kv_heads && num_q_heads % num_kv_heads == 0,
             "num_q_heads (%d) must be a positive multiple of num_kv_heads (%d)", num_q_heads,
             num_kv_heads);
  HY_REQUIRE_SUPPORTED(head_dim == kHeadDim, "head_dim %d unsupported (need %d)", head_dim,
                       kHeadDim);
  HY_REQUIRE_SUPPORTED(page_size >= 32 && (page_size & (page_size - 1)) == 0,
                       "page_size %d unsupported (power of two >= 32 required)", page_size);
  const int G = num_q_heads / num_kv_heads;
  HY_REQUIRE_SUPPORTED(G <= 16 && (G & (G - 1)) == 0,
                       "GQA group size %d unsupported (1, 2, 4, 8, 16)", G);
  HY_REQUIRE(n_chunks >= 0 && n_merge >= 0 && n_slots >= 0, "item counts must be non-negative");
  if (n_chunks == 0) return HY_OK;
  HY_REQUIRE(n_chunks <= 65535 && n_merge <= 65535,
             "%d chunks and %d merge items: the grid takes 65535", n_chunks, n_merge);
  HY_REQUIRE(max_rows >= 1 && max_rows <= hy::kTreeRows, "max_rows %d is not within 1 .. %d",
             max_rows, hy::kTreeRows);
  HY_REQUIRE(line_words >= 1 && line_words <= hy::kMaskWords, "line_words %d is not within 1 .. %d",
             line_words, hy::kMaskWords);
  HY_REQUIRE(q && out && k_pool && v_pool && page_table && lines && items &&
                 (merge_items || n_merge == 0),
             "hy_paged_tree: null pointer argument");
  HY_REQUIRE(((q_stride_seq | q_stride_tok | q_stride_head | o_stride_seq | o_stride_tok |
               o_stride_head | pool_head_stride) &
              7) == 0 &&
                 ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) |
                   reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool)) &
                  15) == 0,
             "hy_paged_tree: rows must be 16-byte aligned");
  const int64_t need = hy_tree_workspace_bytes(n_slots, num_kv_heads, head_dim);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) {
    hy::set_error("workspace too small: need %lld bytes, got %lld", static_cast<long long>(need),
                  static_cast<long long>(workspace_bytes));
    return HY_ENOSPACE;
  }
  float *ws_acc = static_cast<float *>(workspace);
  float *ws_ml = nullptr;
  if (need > 0)
    ws_ml = reinterpret_cast<float *>(
        static_cast<char *>(workspace) +
        hy::align256(static_cast<int64_t>(n_slots) * num_kv_heads * 32 * head_dim * 4));
  const int group_shift = __builtin_ctz(static_cast<unsigned>(G));
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto launch = [&](auto kernel, int waves) {
    hipLaunchKernelGGL(kernel, dim3(num_kv_heads, n_chunks), dim3(64 * waves), 0, st,
                       static_cast<const uint16_t *>(q), q_stride_seq, q_stride_tok, q_stride_head,
                       static_cast<uint16_t *>(out), o_stride_seq, o_stride_tok, o_stride_head,
                       static_cast<const uint16_t *>(k_pool), static_cast<const uint16_t *>(v_pool),
                       pool_head_stride, page_table, page_table_stride, items, n_chunks, lines,
                       line_words, ws_acc, ws_ml, n_slots, group_shift,
                       __builtin_ctz(static_cast<unsigned>(page_size)), scale * hy::kLog2e);
  };
  if (max_rows <= 64)
    launch(hy::tree_kernel<2>, 2);
  else if (max_rows <= 128)
    launch(hy::tree_kernel<4>, 4);
  else
    launch(hy::tree_kernel<8>, 8);
  if (int rc = hy::launch_status("hy_paged_tree")) return rc;
  if (n_merge == 0) return HY_OK;
  hipLaunchKernelGGL(hy::tree_merge_kernel, dim3(num_kv_heads, n_merge, (max_rows + 31) / 32),
                     dim3(512), 0, st, static_cast<uint16_t *>(out), o_stride_seq, o_stride_tok,
                     o_stride_head, merge_items, ws_acc, ws_ml, n_slots, group_shift);
  return hy::launch_status("hy_paged_tree");
}
