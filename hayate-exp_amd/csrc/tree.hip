// Attention for trees of drafted tokens over a paged cache (gfx950).
//
// A request with c cached tokens and n drafted ones holds them in slots 0 ..
// c + n - 1. Node i's query sees every cached token, its ancestors and itself:
//   o_i = sum_j softmax_j(scale q_i k_j) v_j,  j < c  or  j - c in line(i).
// Slots of other branches may hold anything, infinities and NaN included.
//
// Work split: as in the decode kernel, the key steps (64 keys) of all requests, in
// order, form one stream per kv head that the planner cuts into one chunk per
// compute unit (fewer in small ticks); a chunk holds pieces (the part of one
// request inside it). All rows (node, head of the group) of a request read each
// K/V row once, up to 256 of them, 32 a wave; more go into further tiles. A piece
// that is not a tile's whole stream leaves fp32 partials that tree_merge_kernel joins.
//
// What bounds it: up to about 128 rows HBM (32 chains of 5 nodes, 233 MB: 42.3 us, 5.5 TB/s,
// and 4.6 for the merge); with 256 the matrix cores, in part by the clock that the power limit
// leaves and in part by what stands between the products (8 trees of 64 nodes on 32 k tokens:
// 290 us a call with the merge, 902 TFLOP/s, 305 and 9.4 traced kernel by kernel; MFMAs are busy
// in 51 % of the cycles at 1.63 GHz; with all keys in L2 1,000 TFLOP/s, a large library product
// 1,415 to 1,649 by the layout of its right operand); in small ticks the latency of the steps and
// the launch (8 nodes on 500 tokens: 13.0 us, 8 steps of 0.45). The variants keep 37 to 67
// scalars, strides and bases above all, in lanes of vector registers, most of them in those
// with waves that only load.
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
// over the slots, loaded to LDS with the rows of Q.

#include <type_traits>

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

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

__device__ __forceinline__ s16x4 tr_read(const uint16_t *p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(const_cast<uint16_t *>(p)));
}

// 16 rows of 256 bytes (4 KiB) from rows + off[i] + 1024 i (lane l's own off) straight to LDS at
// lds + 1024 i + 16 l, four instructions for one M0: the instruction's offset counts on both
// sides. lds is wave-uniform, through M0, with the wait state the ISA asks for between its write
// and the load. The caller waits (wait_loads) before it reads them. kStream: nontemporal, for
// lines that no other workgroup reads.
template <bool kStream>
__device__ __forceinline__ void load_rows_to_lds(const uint16_t *rows, const uint32_t (&off)[4],
                                                 const uint16_t *lds) {
  // wave-uniform, and held in scalar registers
  const uint64_t at = reinterpret_cast<uintptr_t>(rows);
  const uint64_t base =
      static_cast<uint64_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at >> 32))) << 32 |
      static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at)));
  const uint32_t m0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
      (const __attribute__((address_space(3))) uint16_t *)lds));
  if constexpr (kStream)
    __asm__ volatile(
        "s_mov_b32 m0, %5\n\ts_nop 0\n\t"
        "global_load_lds_dwordx4 %0, %4 nt\n\t"
        "global_load_lds_dwordx4 %1, %4 offset:1024 nt\n\t"
        "global_load_lds_dwordx4 %2, %4 offset:2048 nt\n\t"
        "global_load_lds_dwordx4 %3, %4 offset:3*1024 nt"
        :
        : "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(base),
          "s"(__builtin_amdgcn_readfirstlane(m0))
        : "memory");
  else
    __asm__ volatile(
        "s_mov_b32 m0, %5\n\ts_nop 0\n\t"
        "global_load_lds_dwordx4 %0, %4\n\t"
        "global_load_lds_dwordx4 %1, %4 offset:1024\n\t"
        "global_load_lds_dwordx4 %2, %4 offset:2048\n\t"
        "global_load_lds_dwordx4 %3, %4 offset:3*1024"
        :
        : "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(base),
          "s"(__builtin_amdgcn_readfirstlane(m0))
        : "memory");
}

// 16 bytes from each lane's own address to lds + 16 l.
__device__ __forceinline__ void load_to_lds(const uint16_t *g, const uint16_t *lds) {
  const uint32_t m0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
      (const __attribute__((address_space(3))) uint16_t *)lds));
  __asm__ volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
                   :
                   : "v"(g), "s"(__builtin_amdgcn_readfirstlane(m0))
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

// Every wave's LDS accesses before it are done (LDS only: loads in flight stay so).
__device__ __forceinline__ void barrier() {
  __asm__ volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  __asm__ volatile("" ::: "memory");
}

// x, opaquely: what is computed from it in a rare branch is not kept in registers across
// the loop around it.
__device__ __forceinline__ int here(int x) {
  __asm__ volatile("" : "+v"(x));
  return x;
}

struct Piece {
  int seq, q0, q1, kv0, kv1, slot, q_row, cache;
  __device__ __forceinline__ int tiles() const { return (kv1 - kv0 + kTile - 1) / kTile; }
};

__device__ __forceinline__ Piece load_piece(const int32_t *r) {
  return Piece{r[0], r[1], r[2], r[3], r[4], r[5], r[6], r[7]};
}

// RW waves side by side hold 32 rows each; KS of them hold the same rows and share the 32-key
// blocks of a tile (KS == 2: one block each). LW more waves do nothing but load; with LW == 0
// the others load as well.
template <int RW, int KS, int LW>
__global__ __launch_bounds__(64 * (RW * KS + LW)) __attribute__((amdgpu_waves_per_eu(2, 2)))
void tree_kernel(const uint16_t *__restrict__ q, int64_t q_ss, int64_t q_st, int64_t q_sh,
                 uint16_t *__restrict__ out, int64_t o_ss, int64_t o_st, int64_t o_sh,
                 const uint16_t *__restrict__ k_pool, const uint16_t *__restrict__ v_pool,
                 int64_t pool_hs, const int32_t *__restrict__ page_table, int64_t pt_stride,
                 const int32_t *__restrict__ items, int n_chunks,
                 const uint32_t *__restrict__ lines, int line_words, float *__restrict__ ws_acc,
                 float *__restrict__ ws_ml, int n_slots, int group_shift, int page_shift,
                 float scale_log2) {
  constexpr int W = RW * KS + LW;
  constexpr int kLoaders = LW > 0 ? LW : W;
  constexpr int kLoads = 32 / kLoaders;       // load instructions of a loading wave per stage
  constexpr int kRows = 32 * RW;
  constexpr int kQStages = (kRows + 127) / 128;
  // load instructions of a loading wave for the rows' lines
  constexpr int kLineLoads = (kRows * kMaskWords + kLoaders * 256 - 1) / (kLoaders * 256);
  constexpr int kLineWords = kLineLoads * kLoaders * 256;
  static_assert(KS == 1 || RW <= 2, "finish() joins two waves' rows in one stage");
  __shared__ __attribute__((aligned(1024))) uint16_t ring[kStages * kStage];
  // A piece has two stages at least, so the one issued three stages ahead belongs at most to
  // the piece after the next.
  __shared__ __attribute__((aligned(1024))) uint32_t line[3][kLineWords];
  __shared__ float2 other_ml[kRows];
  __shared__ uint32_t sick[kMaskWords];  // drafted slots with an infinity or NaN in V

  const int32_t *ch = items + kTreeChunkInts * blockIdx.y;
  const int32_t *pieces = items + kTreeChunkInts * n_chunks;
  const int kvh = blockIdx.x;
  const int p_end = ch[1];
  // an empty chunk record pads a list to a fixed launch size
  if (ch[2] <= 0) return;
  const int n_stages = ch[2] + kQStages * (p_end - ch[0]);

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int c = lane & 31;
  const int h = lane >> 5;
  const int h0 = kvh << group_shift;
  const int group_mask = (1 << group_shift) - 1;
  const int page_mask = (1 << page_shift) - 1;
  const uint16_t *kh = k_pool + kvh * pool_hs;
  const uint16_t *vh = v_pool + kvh * pool_hs;

  // ---- stage loads ------------------------------------------------------
  // Issue cursor: the piece of the next stage to load, and the stage's step in it:
  // -kQStages .. -1 its rows of Q (and, with the first, their lines), then its tiles.
  // A tile's two 32-key halves each lie in one page (pages hold at least 32 keys, pieces
  // start at multiples of 64). Keys past the piece are read from its last page: in
  // bounds, and masked.
  Piece ip = load_piece(ch + 8);
  int ip_index = ch[0], ip_step = -kQStages;
  uint32_t page0 = 0, page1 = 0;
  auto fetch = [&]() __attribute__((always_inline)) {
    if (ip_step < 0) return;
    const int32_t *pt = page_table + ip.seq * pt_stride;
    const int key = ip.kv0 + kTile * ip_step;
    // held unsigned: page ids are non-negative, and widen without a sign
    page0 = static_cast<uint32_t>(pt[key >> page_shift]);
    page1 = static_cast<uint32_t>(pt[min(key + 32, ip.kv1 - 1) >> page_shift]);
  };
  auto advance = [&]() __attribute__((always_inline)) {
    if (++ip_step == ip.tiles()) {
      ip = load_piece(pieces + 8 * ++ip_index);
      ip_step = -kQStages;
    }
    fetch();
  };
  // Both tiles keep the rows' order, four to a KiB, so that one load instruction takes four whole
  // rows and its offset serves both sides; within, in units of 8 dims, unit(row, chunk) =
  // (row / 4) * 64 + (chunk / 4) * 16 + (row % 4) * 4 + x with x = chunk % 4 in a V tile and
  // chunk % 4 ^ row / 4 % 4 in a K tile (and for Q): the operand reads below are then
  // free of bank conflicts, and four neighbouring lanes load 64 bytes of a row.
  const int loader = LW > 0 ? wave - RW * KS : wave;
  // whether no other chunk reads this chunk's keys for other rows
  const bool alone = ch[3] != 0;
  auto issue_tile = [&](auto stream, uint16_t *dst, int lane_) __attribute__((always_inline)) {
    constexpr bool kStream = decltype(stream)::value;
    const int key = ip.kv0 + kTile * ip_step;
    const uint32_t row_off = 256 * ((lane_ >> 2) & 3) + 64 * (lane_ >> 4);
    const uint32_t v_off[4] = {row_off + 16 * (lane_ & 3), row_off + 16 * (lane_ & 3),
                               row_off + 16 * (lane_ & 3), row_off + 16 * (lane_ & 3)};
    const uint32_t k_off[4] = {v_off[0], row_off + 16 * ((lane_ & 3) ^ 1),
                               row_off + 16 * ((lane_ & 3) ^ 2), row_off + 16 * ((lane_ & 3) ^ 3)};
    // groups of 16 rows: four of K, then four of V
#pragma unroll
    for (int j = 0; j < 8 / kLoaders; ++j) {
      const int g = loader + kLoaders * j;
      // its rows' page; picked by bits, as a choice by address would put both in memory, and a
      // read from there waits for every load in flight
      const uint32_t page = page0 ^ ((page0 ^ page1) & (0u - ((g >> 1) & 1u)));
      const int64_t row = (static_cast<int64_t>(page) << page_shift) +
                          ((key + 16 * (g & 3)) & page_mask);
      if (g < 4)
        load_rows_to_lds<kStream>(kh + row * kHeadDim, k_off, dst + 2048 * g);
      else
        load_rows_to_lds<kStream>(vh + row * kHeadDim, v_off, dst + 2048 * g);
    }
  };
  auto issue = [&](int stage) __attribute__((always_inline)) {
    if (LW > 0 && loader < 0) return;
    uint16_t *dst = ring + (stage % kStages) * kStage;
    const int lane_ = here(lane);
    if (ip_step < 0) {
      // rows past the piece's are read from its first node, and zeroed on use
      const int row0 = 128 * (ip_step + kQStages);
      const uint16_t *base = q + ip.seq * q_ss + static_cast<int64_t>(ip.q_row) * q_st;
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int i = loader * kLoads + j;
        const int row = row0 + 4 * i + ((lane_ >> 2) & 3);
        const int tok = ip.q0 + (row >> group_shift);
        load_to_lds(base + (tok < ip.q1 ? tok : ip.q0) * q_st + (h0 + (row & group_mask)) * q_sh +
                        32 * (lane_ >> 4) + 8 * ((lane_ & 3) ^ (i & 3)),
                    dst + 512 * i);
      }
      if (ip_step == -kQStages) {
        const int last = (ip.q1 - ip.q0) * line_words - 4;
#pragma unroll
        for (int j = 0; j < kLineLoads; ++j) {
          const int at = 256 * (loader * kLineLoads + j);
          load_to_lds(reinterpret_cast<const uint16_t *>(
                          lines + static_cast<int64_t>(ip.q_row + ip.q0) * line_words +
                          min(at + 4 * lane_, last)),
                      reinterpret_cast<uint16_t *>(line[ip_index % 3] + at));
        }
      }
      return;
    }
    if (alone)
      issue_tile(std::true_type{}, dst, lane_);
    else
      issue_tile(std::false_type{}, dst, lane_);
  };

  // ---- this wave's rows of the piece being computed ----------------------
  Piece cp = ip;
  const uint32_t *own_line = line[0];
  const int rw = wave % RW;
  const int ks = wave / RW;
  bool wave_live = false;
  const int r = 32 * rw + c;  // this lane's row
  bool live = false;
  bf16x8 qop[2][4];  // the row of Q^T
  f32x16 acc[4];     // O^T[32 db + 8 (i / 4) + 4 h + i % 4][row]
  float base, shift, l_run;

  // LDS read bases (u16 units).
  const int r16 = lane & 15;
  const int q16 = lane >> 4;
  int k_base[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    k_base[i] = (c >> 2) * 512 + (c & 3) * 32 + 8 * ((2 * i + h) ^ ((c >> 2) & 3));
  const int v_base = kTile * kHeadDim + 512 * (q16 >> 1) + 32 * (r16 >> 2) + 16 * (q16 & 1) +
                     4 * (r16 & 3);
  // Dims 64 half .. 64 half + 63 of 32 rows of K or Q, as the first product's operands.
  auto read_rows = [&](bf16x8(&x)[4], const uint16_t *rows, int half) __attribute__((always_inline)) {
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
      x[kk] = *reinterpret_cast<const bf16x8 *>(rows + k_base[kk & 1] + 128 * (2 * half + (kk >> 1)));
  };
  auto scores = [&](f32x16 &s, const bf16x8(&kop)[4], int half) __attribute__((always_inline)) {
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
      s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kop[kk], qop[half][kk], s, 0, 0, 0);
  };
  auto start = [&]() __attribute__((always_inline)) {
    const int rows = (cp.q1 - cp.q0) << group_shift;
    wave_live = wave < RW * KS && 32 * rw < rows;
    live = r < rows;
    base = -INFINITY;
    shift = 0.f;
    l_run = 0.f;
#pragma unroll
    for (int db = 0; db < 4; ++db) acc[db] = f32x16{};
  };

  // Drafted slots among the 32 keys from kb0 on: the rows' lines mask their scores. A line's
  // bits for them (bit j: slot of key kb0 + j is seen); slots before the drafted ones are
  // all seen.
  auto mask = [&](f32x16 &s, int kb0) __attribute__((always_inline)) {
    const int d = kb0 - cp.cache;
    if (d <= -32) return;
    uint32_t bits = 0u;
    if (live) {
      const int lane_ = here(lane);
      const uint32_t *words =
          own_line + ((32 * rw + (lane_ & 31)) >> group_shift) * line_words;
      if (d < 0) {
        bits = words[0] << -d | ((1u << -d) - 1);
      } else {
        const int w = d >> 5;  // the slot lies in the tree: below line_words
        const uint32_t hi = w + 1 < line_words ? words[w + 1] : 0u;
        bits = static_cast<uint32_t>((static_cast<uint64_t>(hi) << 32 | words[w]) >> (d & 31));
      }
      bits >>= 4 * (lane_ >> 5);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = bits >> (8 * (i >> 2) + (i & 3)) & 1 ? s[i] : -INFINITY;
  };
  // Online softmax on raw scores: p = exp2(s scale log2(e) - shift), shift the row's
  // exponent base (0 while it has none).
  auto probs = [&](const f32x16 &s, bf16x8(&pop)[2]) __attribute__((always_inline)) {
    float a[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      a[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], scale_log2, -shift));
      pop[i >> 3][i & 7] = static_cast<__bf16>(a[i]);
    }
#pragma unroll
    for (int n = 8; n > 0; n >>= 1)  // pairwise: four dependent sums
#pragma unroll
      for (int i = 0; i < n; ++i) a[i] = a[2 * i] + a[2 * i + 1];
    return a[0];
  };
  // The base moves only when a score exceeds it by 2^8 (or the row sees its first key);
  // below that no lane's probabilities sum to more. Rare, and then they are redone.
  auto rebase = [&](const f32x16 &s, bf16x8(&pop)[2], float psum) __attribute__((always_inline)) {
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
        psum = probs(s, pop);
      }
    }
    l_run += psum;
  };
  // V^T operands of a block, dims 64 half .. 64 half + 63, and their product.
  auto read_v = [&](s16x8(&vop)[4], const uint16_t *kb, int half) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint16_t *vb = kb + v_base + 128 * (2 * half + (i >> 1)) + 2048 * (i & 1);
      vop[i] = __builtin_shufflevector(tr_read(vb), tr_read(vb + 1024), 0, 1, 2, 3, 4, 5, 6, 7);
    }
  };
  auto pv = [&](const s16x8(&vop)[4], const bf16x8(&pop)[2], int half) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f32x16 &a = acc[2 * half + (i >> 1)];
      a = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, vop[i]), pop[i & 1], a,
                                                  0, 0, 0);
    }
  };

  // One block of 32 keys from kb0 on at kb (K rows; V behind). The scores of a wave's next block
  // are not computed beside this one's softmax: with 256 rows (two waves a SIMD, which cover
  // each other) that gave 315 against 317 us on 8 x 64 nodes over 32k keys, two row blocks a
  // wave to pair 314, and with fewer rows the loads take longer than the blocks.
  auto block = [&](const uint16_t *kb, int kb0) __attribute__((always_inline)) {
    bf16x8 kop[4], pop[2];
    s16x8 v0[4], v1[4];
    f32x16 s = f32x16{};
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      read_rows(kop, kb, half);
      scores(s, kop, half);
    }
    read_v(v0, kb, 0);
    read_v(v1, kb, 1);
    mask(s, kb0);
    rebase(s, pop, probs(s, pop));
    pv(v0, pop, 0);
    pv(v1, pop, 1);
  };

  // V rows of drafted slots in the stage `cur`, keys from `key` on, before they meet the
  // probabilities (0 times an infinity or NaN is NaN): rows past the piece, which may hold
  // any bits, become 0, and so do infinities and NaN, whose slots are marked; finish()
  // gives them to the rows that see them. Every thread of the workgroup takes part, and
  // a barrier follows.
  auto clean = [&](uint16_t *cur, int key) __attribute__((always_inline)) {
    for (int u = 64 * wave + here(lane); u < kTile * kHeadDim / 8; u += 64 * W) {
      const int slot_key = key + 4 * (u >> 6) + ((u >> 2) & 3);
      if (slot_key < cp.cache) continue;
      uint16_t *at = cur + kTile * kHeadDim + 8 * u;
      u32x4 x = *reinterpret_cast<const u32x4 *>(at);
      bool found = slot_key >= cp.kv1;
      if (found) {
        x = u32x4{0u, 0u, 0u, 0u};
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool lo = (x[j] & 0x7f80u) == 0x7f80u, hi = (x[j] & 0x7f800000u) == 0x7f800000u;
          found = found || lo || hi;
          x[j] &= (lo ? 0xffff0000u : 0xffffffffu) & (hi ? 0x0000ffffu : 0xffffffffu);
        }
        const int slot = slot_key - cp.cache;
        if (found) atomicOr(&sick[slot >> 5], 1u << (slot & 31));
      }
      if (found) *reinterpret_cast<u32x4 *>(at) = x;
    }
    barrier();
  };

  // Closes the piece: its output rows, or a partial: fp32, in the accumulator's own
  // order (16 groups of 64 lanes x 16 bytes), live rows only. With KS == 2 the second
  // wave's rows are joined first, through the stage of the tile just used: it is
  // free once every wave has left it, until the loads that follow the next barrier.
  auto finish = [&](uint16_t *stage) __attribute__((always_inline)) {
    const int lane_ = here(lane), c_ = lane_ & 31, h_ = lane_ >> 5, r_ = 32 * rw + c_;
    float l = halves_sum(l_run);
    if constexpr (KS == 2) {
      float *box = reinterpret_cast<float *>(stage) + 4096 * rw + 4 * lane_;
      barrier();
      if (ks == 1 && wave_live) {
        if (h_ == 0) other_ml[r_] = make_float2(base, l);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const f32x16 &a = acc[j >> 2];
          const int i = 4 * (j & 3);
          *reinterpret_cast<f32x4 *>(box + 256 * j) = f32x4{a[i], a[i + 1], a[i + 2], a[i + 3]};
        }
      }
      barrier();
      if (ks == 0 && wave_live) {
        const float2 o = other_ml[r_];
        const float top = fmaxf(base, o.x);
        // a wave that saw nothing adds nothing (its sums are 0)
        const float mine = base == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(base - top);
        const float theirs = o.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(o.x - top);
        l = l * mine + o.y * theirs;
        base = top;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          f32x16 &a = acc[j >> 2];
          const int i = 4 * (j & 3);
          const f32x4 x = *reinterpret_cast<const f32x4 *>(box + 256 * j);
#pragma unroll
          for (int e = 0; e < 4; ++e) a[i + e] = a[i + e] * mine + x[e] * theirs;
        }
      }
    }
    if (ks != 0 || !wave_live) return;
    // infinities and NaN of marked slots (none, as a rule), from the pool
    for (int w = 0; w < line_words; ++w) {
      uint32_t marks = __builtin_amdgcn_readfirstlane(sick[w]);
      while (marks != 0) {
        const int bit = __builtin_ctz(marks), key = cp.cache + 32 * w + bit;
        marks &= marks - 1;
        const bool sees = live && own_line[(r_ >> group_shift) * line_words + w] >> bit & 1;
        const int64_t row =
            (static_cast<int64_t>(page_table[cp.seq * pt_stride + (key >> page_shift)]) << page_shift) +
            (key & page_mask);
        const uint16_t *v = vh + row * kHeadDim + 4 * h_;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const uint2 x = *reinterpret_cast<const uint2 *>(v + 8 * j);
          const float value[4] = {bf16_lo(x.x), bf16_hi(x.x), bf16_lo(x.y), bf16_hi(x.y)};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (sees && (__float_as_uint(value[e]) & 0x7f800000u) == 0x7f800000u)
              acc[j >> 2][4 * (j & 3) + e] += value[e];
        }
      }
    }
    if (!live) return;
    if (cp.slot < 0) {
      const float inv = 1.0f / l;
      const int64_t tok = cp.q_row + cp.q0 + (r_ >> group_shift);
      uint16_t *dst = out + cp.seq * o_ss + tok * o_st + (h0 + (r_ & group_mask)) * o_sh + 4 * h_;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const f32x16 &a = acc[j >> 2];
        const int i = 4 * (j & 3);
        *reinterpret_cast<uint2 *>(dst + 8 * j) =
            make_uint2(pack_bf16x2_rne(a[i] * inv, a[i + 1] * inv),
                       pack_bf16x2_rne(a[i + 2] * inv, a[i + 3] * inv));
      }
      return;
    }
    // a sum that is NaN counts as seen (the merge drops rows that saw nothing)
    if (base == -INFINITY && l != l) base = 0.f;
    const int64_t at = static_cast<int64_t>(kvh) * n_slots + cp.slot + rw;
    float *dst = ws_acc + at * 32 * kHeadDim + 4 * lane_;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const f32x16 &a = acc[j >> 2];
      const int i = 4 * (j & 3);
      *reinterpret_cast<f32x4 *>(dst + 256 * j) = f32x4{a[i], a[i + 1], a[i + 2], a[i + 3]};
    }
    if (h_ == 0) *reinterpret_cast<float2 *>(ws_ml + (at * 32 + c_) * 2) = make_float2(base, l);
  };

  // ---- the chunk ---------------------------------------------------------
  // Two waves a SIMD that compute: one of them goes first, which keeps the two apart (309 against
  // 321 us on 8 x 64 nodes over 32k keys; a priority by region, or a delay, gave less).
  if (RW * KS == 8 && wave >= 4) __builtin_amdgcn_s_setprio(1);
  issue(0);
  for (int i = 1; i < 3 && i < n_stages; ++i) {
    advance();
    issue(i);
  }
  if (n_stages > 3) advance();
  int t = 0;  // stages computed
  uint16_t *cur;
  auto next_stage = [&]() __attribute__((always_inline)) {
    // The page ids of the next loads are read here and waited for with the stage: a scalar
    // load outstanding would make every wait for an LDS read in a block wait for it too.
    if ((LW == 0 || loader >= 0) && t > 0 && t + 3 < n_stages) advance();
    // stage t has arrived in every wave, and every wave is done with stage t - 1, which
    // stage t + 3 takes
    if (LW > 0 && loader < 0) {
      // (nothing of its own in flight)
    } else if (t + 2 < n_stages) {
      wait_loads<2 * kLoads>();
    } else if (t + 1 < n_stages) {
      wait_loads<kLoads>();
    } else {
      wait_loads<0>();
    }
    barrier();
    if (t + 3 < n_stages) issue(t + 3);
    cur = ring + (t % kStages) * kStage;
    ++t;
  };
  for (int cp_index = ch[0]; cp_index < p_end; ++cp_index) {
    cp = load_piece(pieces + 8 * cp_index);
    own_line = line[cp_index % 3];
    start();
    for (int part = 0; part < kQStages; ++part) {
      next_stage();
      if (part == 0 && wave == 0 && lane < kMaskWords) sick[lane] = 0;
      if (part != rw >> 2) continue;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        read_rows(qop[half], cur + 4096 * (rw & 3), half);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          if (!live) qop[half][kk] = bf16x8{};
      }
    }
    for (int key = cp.kv0; key < cp.kv1; key += kTile) {
      next_stage();
      if (key + kTile > cp.cache) clean(cur, key);
      if (!wave_live) continue;
      if constexpr (KS == 2) {
        if (key + 32 * ks < cp.kv1) block(cur + 4096 * ks, key + 32 * ks);
      } else {
        block(cur, key);
        if (key + 32 < cp.kv1) block(cur + 4096, key + 32);
      }
    }
    finish(cur);
  }
}

// Joins the partials of a request's rows: grid (kv head, merge item, 32-row group and part of
// the dims), thread = row c of the group and dims 8 j8 .. 8 j8 + 7. Item = {seq, q0,
// q1, first_slot, splits, q_row, row blocks a split, 0}. Rows past the item's are neither
// read nor written. One wave a workgroup, for the few items of a small tick: 8 nodes on
// 8,000 tokens (32 splits) 16.1 us with the attention, 16.6 with two waves, 17.7 with four, 19.6
// with eight.
constexpr int kMergeThreads = 64;
constexpr int kMergeParts = 512 / kMergeThreads;

__global__ __launch_bounds__(kMergeThreads) void tree_merge_kernel(
    uint16_t *__restrict__ out, int64_t o_ss, int64_t o_st, int64_t o_sh,
    const int32_t *__restrict__ items, const float *__restrict__ ws_acc,
    const float *__restrict__ ws_ml, int n_slots, int group_shift) {
  const int32_t *it = items + 8 * blockIdx.y;
  const int q0 = it[1];
  const int rows = (it[2] - q0) << group_shift;
  const int splits = it[4], blocks = it[6];
  const int c = threadIdx.x & 31;
  const int j8 = (kMergeThreads / 32) * (blockIdx.z % kMergeParts) + (threadIdx.x >> 5);
  const int row_block = blockIdx.z / kMergeParts;
  const int row = 32 * row_block + c;
  // an empty record pads a list to a fixed launch size
  if (row >= rows || splits <= 0) return;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * n_slots + it[3] + row_block;
  const float *ml_row = ws_ml + (first * 32 + c) * 2;
  const float *acc_row = ws_acc + first * 32 * kHeadDim + 256 * j8 + 4 * c;
  float mx = -INFINITY, lsum = 0.f;
  f32x4 a0 = {0.f, 0.f, 0.f, 0.f}, a1 = {0.f, 0.f, 0.f, 0.f};
  // A round of independent loads: the index is clamped to a real split, and the ones past
  // the last are replaced by the empty partial. Rounds of 8, the last of 4 or 2: with 8
  // only, items of two or three splits read too much (4 trees of 200 nodes 63.0 us against
  // 61.6), with 4 only, 8 nodes on 8,000 tokens take 17.1.
  auto round = [&](auto n, int s0) __attribute__((always_inline)) {
    constexpr int kRound = decltype(n)::value;
    float m[kRound], l[kRound];
    f32x4 x0[kRound], x1[kRound];
#pragma unroll
    for (int j = 0; j < kRound; ++j) {
      const int64_t block = static_cast<int64_t>(min(s0 + j, splits - 1)) * blocks;
      const float2 ml = *reinterpret_cast<const float2 *>(ml_row + block * 64);
      m[j] = ml.x;
      l[j] = ml.y;
      const float *src = acc_row + block * 32 * kHeadDim;
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
  };
  int s0 = 0;
  for (; splits - s0 > 4; s0 += 8) round(std::integral_constant<int, 8>{}, s0);
  if (splits - s0 > 2)
    round(std::integral_constant<int, 4>{}, s0);
  else if (splits > s0)
    round(std::integral_constant<int, 2>{}, s0);
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
  HY_REQUIRE(n_merge == 0 || n_slots > 0, "%d merge items without partials", n_merge);
  HY_REQUIRE(line_words == 4 || line_words == 8, "line_words is %d, not 4 or 8", line_words);
  HY_REQUIRE(q && out && k_pool && v_pool && page_table && lines && items &&
                 (merge_items || n_merge == 0),
             "hy_paged_tree: null pointer argument");
  HY_REQUIRE(((q_stride_seq | q_stride_tok | q_stride_head | o_stride_seq | o_stride_tok |
               o_stride_head | pool_head_stride) &
              7) == 0 &&
                 ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) |
                   reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool) |
                   reinterpret_cast<uintptr_t>(lines)) &
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
  // The narrowest variant that holds the largest tile. Up to 128 rows, four waves only load: one
  // wave issues such a load every 130 cycles or so, and the others' would wait behind products
  // (32 chains: 54 us without them, 42 with); up to 64 rows two waves share a row block's keys.
  // With 256 rows the eight waves are needed for the products. Geometric means over 16
  // batches in the next wider variant: 8 nodes (32 rows) 27.9 us against 27.2, 16 nodes 23.4
  // against 22.2, 32 nodes 35.4 against 32.5.
  if (max_rows <= 32)
    launch(hy::tree_kernel<1, 2, 4>, 6);
  else if (max_rows <= 64)
    launch(hy::tree_kernel<2, 2, 4>, 8);
  else if (max_rows <= 128)
    launch(hy::tree_kernel<4, 1, 4>, 8);
  else
    launch(hy::tree_kernel<8, 1, 0>, 8);
  if (int rc = hy::launch_status("hy_paged_tree")) return rc;
  if (n_merge == 0) return HY_OK;
  hipLaunchKernelGGL(hy::tree_merge_kernel, dim3(num_kv_heads, n_merge, (max_rows + 31) / 32 * hy::kMergeParts),
                     dim3(hy::kMergeThreads), 0, st, static_cast<uint16_t *>(out), o_stride_seq, o_stride_tok,
                     o_stride_head, merge_items, ws_acc, ws_ml, n_slots, group_shift);
  return hy::launch_status("hy_paged_tree");
}
