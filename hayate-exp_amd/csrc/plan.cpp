// Tick planner: turns per-sequence (q_len, kv_len) into the work lists the
// decode and prefill kernels consume. Host-only code, no device access.
//
// Decode sequences (q_len == 1): their K/V rows, concatenated in sequence
// order, are cut into one chunk per CU and kv head, equal in cost (tokens
// plus a fixed charge for every piece after a chunk's first; cuts inside a
// sequence on multiples of 32 tokens); each piece of a sequence in
// a chunk gets W workspace slots (one per wave of the decode workgroup) and
// every decode sequence one merge item over its pieces' slots.
// Prefill sequences (q_len > 1) are cut into query tiles of kPrefillRows / G
// tokens (prefill_shape.h);
// the longest tiles are split along their key range when the simulated
// dispatch says so, and work is ordered longest first so the short items
// fill in behind the long ones.

#include <math.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include <algorithm>
#include <array>
#include <functional>
#include <new>
#include <queue>
#include <vector>

#include "../../include/hayate_attn.h"
#include "decode_shape.h"
#include "prefill_shape.h"
#include "tree_shape.h"
#include "weigh_shape.h"
#include "window.h"

namespace hy {
void set_error(const char *fmt, ...);
void clear_error();
}  // namespace hy

namespace {

constexpr int kSlice = 32;        // decode kernel's token slice
using hy::kPrefillRows;                          // rows of a prefill workgroup
constexpr int kPrefillKeys = hy::kPrefillTileKeys;  // keys per prefill step
// Prefill cost model, in units of one step (64 keys) of one workgroup,
// measured on MI355X from per-workgroup start/end stamps (s_memrealtime) on
// the 4 x 512 chunked prefill and the mixed tick: a workgroup takes 5.35 us
// + 1.86 us per step, so its fixed cost (Q load, first tiles, epilogue) is
// about 2.9 steps; a workgroup that follows another on the same CU starts
// 6.4 us (3.4 steps) after the previous one's last step; the merge launch
// costs about two steps and one split partial (write + read of its rows of
// fp32 O) a fortieth of a step.
// The prologue and epilogue have since lost about 2 us; settings of 1.4-2.9
// fixed, 1.9-3.4 gap and 1.2-2.0 for the merge stay within 1 % of each other on
// eleven prompt and mixed ticks, so these were kept.
constexpr double kPrefillFixed = 2.9;
constexpr double kPrefillGap = 3.4;
constexpr double kMergeLaunch = 2.0;
constexpr double kPartialCost = 0.025;
constexpr int kDecodeWgPerCu = 1;     // decode workgroups (chunks) per CU
using hy::kDecodeWaves;                // waves per decode workgroup: partials per piece
constexpr int64_t kMinChunk = 64;     // smallest decode chunk, in tokens (two slices)
// Cost of a decode piece after a chunk's first, in tokens: per-wave stamps
// (s_memrealtime) of the batch-32 decode on MI355X put a chunk at 43.4 /
// 45.0 / 45.7 / 46.5 us with 1 / 2 / 3 / 4 pieces for the same tokens
// (~1.1 us per piece: a partial flush, the next query rows and a partial
// last slice) at ~0.0192 us per token.
constexpr int64_t kDecodePieceCost = 64;

// How a prefill tile of `steps` key steps is cut into key ranges (parts).
// Even: the fewest parts of at most `len` steps, of equal length (+-1).
// Capped: parts of exactly `len` steps from the start and the remainder as a
// last, shorter part when it has at least `min_rest` steps (a short part
// fills the second slot of a CU whose first workgroup was short); a smaller
// remainder is spread over the full parts instead.
struct SplitRule {
  bool capped;
  int64_t len, min_rest;
};

void split_tile(int64_t steps, const SplitRule &r, std::vector<int64_t> &parts) {
  parts.clear();
  if (steps <= r.len) {
    parts.push_back(steps);
    return;
  }
  int64_t n = (steps + r.len - 1) / r.len;
  if (r.capped) {
    const int64_t full = steps / r.len;
    const int64_t rest = steps - full * r.len;
    if (rest == 0 || rest >= r.min_rest) {
      for (int64_t i = 0; i < full; ++i) parts.push_back(r.len);
      if (rest) parts.push_back(rest);
      return;
    }
    n = full;
  }
  for (int64_t i = 0; i < n; ++i) parts.push_back(steps / n + (i < steps % n ? 1 : 0));
}

// Makespan (in steps) of prefill tiles cut by `rule`, dispatched longest
// first onto `slots` workgroup slots (each kv head a separate workgroup),
// plus the merge launch and the merge traffic of the partials they create.
// With the slots a multiple of the kv heads, the copies of an item for the
// kv heads go to equally loaded slots, so one head on slots / heads slots
// gives the same makespan. The buffers are kept between calls, and a run
// stops as soon as it cannot end below `bound` (its value is then >= bound).
struct PrefillSim {
  std::vector<double> costs, free_at;
  std::vector<int64_t> parts;

  double cost(const std::vector<int64_t> &tile_steps, const SplitRule &rule, int num_kv_heads,
              int64_t slots, double bound) {
    costs.clear();
    int64_t partials = 0;
    double longest = 0.0, total = 0.0;
    for (int64_t st : tile_steps) {
      split_tile(st, rule, parts);
      for (int64_t p : parts) {
        costs.push_back(static_cast<double>(p) + kPrefillFixed);
        longest = std::max(longest, costs.back());
        total += costs.back();
      }
      if (parts.size() > 1) partials += static_cast<int64_t>(parts.size());
    }
    const double extra =
        (partials ? kMergeLaunch : 0.0) + kPartialCost * static_cast<double>(partials * num_kv_heads);
    int copies = num_kv_heads;
    if (slots % num_kv_heads == 0) {
      slots /= num_kv_heads;
      copies = 1;
    }
    // Lower bounds first: the longest part, and all the work spread evenly.
    const double lower = std::max(longest, total * copies / static_cast<double>(slots)) + extra;
    if (costs.empty() || lower >= bound) return lower;
    std::sort(costs.begin(), costs.end(), std::greater<double>());
    free_at.assign(static_cast<size_t>(slots), 0.0);  // a min-heap (all equal)
    double makespan = 0.0;
    for (double c : costs)
      for (int h = 0; h < copies; ++h) {
        std::pop_heap(free_at.begin(), free_at.end(), std::greater<double>());
        double &slot = free_at.back();
        slot += c + (slot > 0.0 ? kPrefillGap : 0.0);
        makespan = std::max(makespan, slot);
        std::push_heap(free_at.begin(), free_at.end(), std::greater<double>());
        if (makespan + extra >= bound) return makespan + extra;
      }
    return makespan + extra;
  }
};

// window 0: none. Otherwise decode pieces and prefill ranges are cut from the numbers of the
// keys in sight (window.h), for the sequence's token and for a tile's first one.
int plan_tick(const int32_t *q_lens, const int32_t *kv_lens, int32_t num_seqs,
              int32_t num_q_heads, int32_t num_kv_heads, int32_t page_size, int32_t num_cus,
              int32_t target_tokens_per_split, int32_t window, int32_t sinks,
              int32_t *decode_items, int32_t decode_capacity, int32_t *merge_items,
              int32_t merge_capacity, int32_t *prefill_items, int32_t prefill_capacity,
              int32_t *prefill_merge_items, int32_t prefill_merge_capacity,
              int32_t *counts_out) {
  if (num_seqs < 0 || (num_seqs > 0 && (q_lens == nullptr || kv_lens == nullptr)) ||
      counts_out == nullptr) {
    hy::set_error("hy_plan_tick: invalid sequence arrays");
    return HY_EINVAL;
  }
  if (num_kv_heads < 1 || num_q_heads < num_kv_heads || num_q_heads % num_kv_heads) {
    hy::set_error("hy_plan_tick: num_q_heads (%d) must be a multiple of num_kv_heads (%d)",
                  num_q_heads, num_kv_heads);
    return HY_EINVAL;
  }
  if (page_size < kSlice || (page_size & (page_size - 1))) {
    hy::set_error("hy_plan_tick: page_size %d must be a power of two >= %d", page_size, kSlice);
    return HY_EUNSUPPORTED;
  }
  const int G = num_q_heads / num_kv_heads;
  if (kPrefillRows % G) {
    hy::set_error("hy_plan_tick: GQA group size %d unsupported", G);
    return HY_EUNSUPPORTED;
  }
  // Keys of a decode sequence's stream, and those a tile from token q0 on leaves out.
  auto decode_keys = [&](int b) {
    return window > 0 ? kv_lens[b] - hy::window_keys(kv_lens[b] - 1, window, sinks).gap
                      : kv_lens[b];
  };
  auto tile_gap = [&](int32_t first_pos) {
    return window > 0 ? hy::window_keys(first_pos, window, sinks).gap : 0;
  };
  int64_t decode_tokens = 0;
  for (int b = 0; b < num_seqs; ++b) {
    if (q_lens[b] < 0 || kv_lens[b] < q_lens[b]) {
      hy::set_error("hy_plan_tick: sequence %d has q_len %d, kv_len %d", b, q_lens[b],
                    kv_lens[b]);
      return HY_EINVAL;
    }
    if (q_lens[b] == 1) decode_tokens += decode_keys(b);
  }

  // Decode: the K/V rows of all decode sequences, concatenated in sequence
  // order, form one token stream per kv head that is cut into n_chunks
  // chunks of equal cost, one workgroup each. A cut inside a sequence
  // falls on a multiple of 32 tokens of that sequence. A chunk holds one or
  // more pieces (the part of one sequence inside the chunk); each wave of a
  // chunk's workgroup leaves one partial per piece, and the merge pass
  // combines all partials of a sequence.
  std::vector<int32_t> q_begin(static_cast<size_t>(num_seqs) + 1, 0);
  for (int b = 0; b < num_seqs; ++b) q_begin[b + 1] = q_begin[b] + q_lens[b];
  int64_t n_chunks = 0;
  if (decode_tokens > 0) {
    if (target_tokens_per_split > 0) {
      n_chunks = (decode_tokens + target_tokens_per_split - 1) / target_tokens_per_split;
    } else {
      const int64_t cus = num_cus > 0 ? num_cus : 256;
      n_chunks = std::max<int64_t>(1, (cus * kDecodeWgPerCu + num_kv_heads - 1) / num_kv_heads);
      n_chunks = std::min<int64_t>(n_chunks, std::max<int64_t>(1, decode_tokens / kMinChunk));
    }
  }
  struct PieceRec {
    int32_t seq, t0, t1, slice_begin;
  };
  struct ChunkRec {
    int32_t piece_begin, piece_end, n_slices;
  };
  struct DecodeCut {
    std::vector<PieceRec> pieces;
    std::vector<ChunkRec> chunks;
  };
  const int32_t max_pieces = hy::decode_max_pieces(G);
  // Cuts the decode stream into n_chunks chunks of equal cost, where a
  // chunk's cost is its tokens plus `piece_cost` for every piece after its
  // first, and `total` is the whole stream's cost.
  auto cut_stream = [&](int64_t total, int64_t piece_cost, DecodeCut &d) {
    d.pieces.clear();
    d.chunks.clear();
    int64_t pos = 0;          // stream cost before the next piece
    int64_t chunk = 0;        // index of the chunk being filled
    int64_t chunk_start = 0;  // stream cost where it began
    int32_t first = 0;        // its first piece
    int32_t slices = 0;       // its slices so far
    auto close_chunk = [&]() {
      if (static_cast<int32_t>(d.pieces.size()) > first)
        d.chunks.push_back({first, static_cast<int32_t>(d.pieces.size()), slices});
      first = static_cast<int32_t>(d.pieces.size());
      slices = 0;
      ++chunk;
      chunk_start = pos;
    };
    // Where the chunk being filled should end: the rest of the stream shared
    // evenly by the chunks still to fill. A chunk that the piece limit closed
    // early thus leaves its unfilled share to all later chunks instead of
    // moving every later cut one chunk ahead of the stream.
    auto chunk_target = [&]() -> int64_t {
      return chunk_start + (total - chunk_start) / (n_chunks - chunk);
    };
    for (int b = 0; b < num_seqs; ++b) {
      if (q_lens[b] != 1) continue;
      const int64_t kv = decode_keys(b);
      int64_t t = 0;
      while (t < kv) {
        // stream cost at token t once the piece's own cost is paid
        const int64_t at =
            pos + (static_cast<int32_t>(d.pieces.size()) > first ? piece_cost : 0);
        int64_t end = kv;
        bool cut = false;
        if (chunk < n_chunks - 1) {
          const int64_t chunk_end = chunk_target();
          if (chunk_end - at < kv - t) {
            end = std::min<int64_t>(
                kv, std::max<int64_t>(t, t + (chunk_end - at + kSlice / 2) / kSlice * kSlice));
            cut = true;
          }
        }
        if (end > t) {
          d.pieces.push_back({b, static_cast<int32_t>(t), static_cast<int32_t>(end), slices});
          slices += static_cast<int32_t>((end - t + kSlice - 1) / kSlice);
          pos = at + (end - t);
          t = end;
        }
        // A chunk also ends at the size of the kernel's query table.
        if (cut || static_cast<int32_t>(d.pieces.size()) - first >= max_pieces) close_chunk();
      }
    }
    if (static_cast<int32_t>(d.pieces.size()) > first)
      d.chunks.push_back({first, static_cast<int32_t>(d.pieces.size()), slices});
  };
  // The costliest chunk: its slices' tokens plus kDecodePieceCost for every
  // piece after its first.
  auto max_chunk_cost = [&](const DecodeCut &d) {
    int64_t worst = 0;
    for (const ChunkRec &c : d.chunks)
      worst = std::max<int64_t>(worst, static_cast<int64_t>(c.n_slices) * kSlice +
                                           kDecodePieceCost * (c.piece_end - c.piece_begin - 1));
    return worst;
  };
  // Equal tokens per chunk first; then cuts that price each extra piece,
  // the stream's total cost taken from the previous cut's piece count; the
  // cut with the cheapest costliest chunk is kept.
  DecodeCut best, trial;
  cut_stream(decode_tokens, 0, best);
  int64_t best_cost = max_chunk_cost(best);
  int64_t total = decode_tokens;
  for (int pass = 0; pass < 3 && n_chunks > 1; ++pass) {
    cut_stream(total, kDecodePieceCost, trial);
    const int64_t c = max_chunk_cost(trial);
    total = decode_tokens + kDecodePieceCost * static_cast<int64_t>(trial.pieces.size() -
                                                                    trial.chunks.size());
    if (c < best_cost) {
      best_cost = c;
      std::swap(best, trial);
    }
  }
  const std::vector<PieceRec> &pieces = best.pieces;
  const std::vector<ChunkRec> &chunks = best.chunks;
  // One merge item per decode sequence over its pieces' slots (its pieces
  // are consecutive).
  int32_t n_merge = 0, n_pre = 0;
  for (size_t i = 0; i < pieces.size();) {
    size_t j = i;
    while (j < pieces.size() && pieces[j].seq == pieces[i].seq) ++j;
    if (n_merge >= merge_capacity) {
      hy::set_error("hy_plan_tick: merge capacity %d too small", merge_capacity);
      return HY_ENOSPACE;
    }
    int32_t *mt = merge_items + 4 * n_merge++;
    mt[0] = pieces[i].seq;
    mt[1] = kDecodeWaves * static_cast<int32_t>(i);
    mt[2] = kDecodeWaves * static_cast<int32_t>(j - i);
    mt[3] = q_begin[pieces[i].seq];
    i = j;
  }
  const int32_t n_dec = static_cast<int32_t>(chunks.size());
  const int32_t n_pieces = static_cast<int32_t>(pieces.size());
  const int32_t n_slots = kDecodeWaves * n_pieces;
  if (static_cast<int64_t>(n_dec) + n_pieces > decode_capacity) {
    hy::set_error("hy_plan_tick: decode capacity %d too small (need %d)", decode_capacity,
                  n_dec + n_pieces);
    return HY_ENOSPACE;
  }
  // Chunk records carry their first piece so that a workgroup can issue its
  // first loads after one dependent read.
  for (int32_t i = 0; i < n_dec; ++i) {
    int32_t *it = decode_items + 8 * i;
    const PieceRec &f = pieces[chunks[i].piece_begin];
    it[0] = chunks[i].piece_begin;
    it[1] = chunks[i].piece_end;
    it[2] = chunks[i].n_slices;
    it[3] = f.seq;
    it[4] = f.t0;
    it[5] = f.t1;
    it[6] = kDecodeWaves * chunks[i].piece_begin;
    it[7] = q_begin[f.seq];
  }
  for (int32_t i = 0; i < n_pieces; ++i) {
    int32_t *it = decode_items + 8 * (n_dec + i);
    it[0] = pieces[i].seq;
    it[1] = pieces[i].t0;
    it[2] = pieces[i].t1;
    it[3] = kDecodeWaves * i;
    it[4] = pieces[i].slice_begin;
    it[5] = q_begin[pieces[i].seq];
    it[6] = kv_lens[pieces[i].seq] - 1;  // position of the sequence's query token
    it[7] = pieces[i].t1 == decode_keys(pieces[i].seq);  // the piece holds that token
  }

  // Prefill: query tiles of kPrefillRows / G tokens; the key range of a tile is
  // [0, cache_len + q_end). The longest tiles are split into key ranges by
  // the split rule whose simulated run is shortest.
  struct Tile {
    int32_t seq, q0, q1, kv_end;
    int64_t steps;
  };
  std::vector<Tile> tiles;
  const int tile = kPrefillRows / G;
  int64_t max_tile_steps = 0;
  for (int b = 0; b < num_seqs; ++b) {
    const int ql = q_lens[b];
    if (ql <= 1) continue;
    const int cache = kv_lens[b] - ql;
    for (int q0 = 0; q0 < ql; q0 += tile) {
      const int q1 = std::min(ql, q0 + tile);
      const int32_t end = cache + q1 - tile_gap(cache + q0);
      const int64_t st = (end + kPrefillKeys - 1) / kPrefillKeys;
      tiles.push_back({b, q0, q1, end, st});
      max_tile_steps = std::max(max_tile_steps, st);
    }
  }
  SplitRule rule{false, std::max<int64_t>(max_tile_steps, 1), 0};
  if (!tiles.empty()) {
    std::vector<int64_t> tile_steps;
    for (const Tile &t : tiles) tile_steps.push_back(t.steps);
    const int64_t slots = static_cast<int64_t>(num_cus > 0 ? num_cus : 256) * hy::kPrefillWgPerCu;
    PrefillSim sim;
    double best = sim.cost(tile_steps, rule, num_kv_heads, slots, HUGE_VAL);
    // Candidates: every length down to 2 steps for short ranges, at most 32
    // evenly spaced ones for long ranges (the simulation is cheap), each cut
    // evenly and capped with a few remainder thresholds.
    const int64_t top = rule.len;
    const int64_t step = std::max<int64_t>(1, (top - 2) / 32);
    for (int64_t len = top - step; len >= 2; len -= step) {
      const SplitRule cands[] = {{false, len, 0}, {true, len, 1}, {true, len, 2},
                                 {true, len, 4}, {true, len, 8}, {true, len, len / 2}};
      for (const SplitRule &c : cands) {
        const double t = sim.cost(tile_steps, c, num_kv_heads, slots, best);
        if (t < best) {
          best = t;
          rule = c;
        }
      }
    }
  }
  struct PItem {
    int32_t seq, q0, q1, kv0, kv1, slot;
  };
  std::vector<PItem> pitems;
  int32_t n_pmerge = 0, n_pslots = 0;
  std::vector<int64_t> lens;
  for (const Tile &t : tiles) {
    split_tile(t.steps, rule, lens);
    const int64_t n = static_cast<int64_t>(lens.size());
    int64_t parts = 0, a = 0;
    for (int64_t len : lens) {
      const int32_t kv0 = static_cast<int32_t>(a * kPrefillKeys);
      const int32_t kv1 = static_cast<int32_t>(std::min<int64_t>(t.kv_end, (a + len) * kPrefillKeys));
      pitems.push_back({t.seq, t.q0, t.q1, kv0, kv1, n > 1 ? n_pslots + static_cast<int32_t>(parts) : -1});
      ++parts;
      a += len;
    }
    if (n > 1) {
      if (n_pmerge >= prefill_merge_capacity) {
        hy::set_error("hy_plan_tick: prefill merge capacity %d too small", prefill_merge_capacity);
        return HY_ENOSPACE;
      }
      int32_t *mt = prefill_merge_items + 8 * n_pmerge++;
      mt[0] = t.seq;
      mt[1] = t.q0;
      mt[2] = t.q1;
      mt[3] = n_pslots;
      mt[4] = static_cast<int32_t>(parts);
      mt[5] = q_begin[t.seq];
      mt[6] = mt[7] = 0;
      n_pslots += static_cast<int32_t>(parts);
    }
  }
  std::stable_sort(pitems.begin(), pitems.end(), [](const PItem &a, const PItem &b) {
    return a.kv1 - a.kv0 > b.kv1 - b.kv0;
  });
  if (static_cast<int64_t>(pitems.size()) > prefill_capacity) {
    hy::set_error("hy_plan_tick: prefill capacity %d too small (need %zu)", prefill_capacity,
                  pitems.size());
    return HY_ENOSPACE;
  }
  for (const PItem &p : pitems) {
    int32_t *pt = prefill_items + 8 * n_pre++;
    pt[0] = p.seq;
    pt[1] = p.q0;
    pt[2] = p.q1;
    pt[3] = p.kv0;
    pt[4] = p.kv1;
    pt[5] = p.slot;
    pt[6] = q_begin[p.seq];
    pt[7] = kv_lens[p.seq] - q_lens[p.seq];  // cached keys before the chunk
  }
  counts_out[0] = n_dec;
  counts_out[1] = n_merge;
  counts_out[2] = n_slots;
  counts_out[3] = n_pre;
  counts_out[4] = n_pmerge;
  counts_out[5] = n_pslots;
  counts_out[6] = n_pieces;
  return HY_OK;
}

}  // namespace

extern "C" int hy_plan_tick(const int32_t *q_lens, const int32_t *kv_lens,
                            int32_t num_seqs, int32_t num_q_heads,
                            int32_t num_kv_heads, int32_t page_size,
                            int32_t num_cus, int32_t target_tokens_per_split,
                            int32_t *decode_items, int32_t decode_capacity,
                            int32_t *merge_items, int32_t merge_capacity,
                            int32_t *prefill_items, int32_t prefill_capacity,
                            int32_t *prefill_merge_items, int32_t prefill_merge_capacity,
                            int32_t *counts_out) {
  hy::clear_error();
  return plan_tick(q_lens, kv_lens, num_seqs, num_q_heads, num_kv_heads, page_size, num_cus,
                   target_tokens_per_split, 0, 0, decode_items, decode_capacity, merge_items,
                   merge_capacity, prefill_items, prefill_capacity, prefill_merge_items,
                   prefill_merge_capacity, counts_out);
}

extern "C" int hy_plan_tick_window(
    const int32_t *q_lens, const int32_t *kv_lens, int32_t num_seqs, int32_t num_q_heads,
    int32_t num_kv_heads, int32_t page_size, int32_t num_cus, int32_t target_tokens_per_split,
    int32_t window, int32_t sinks, int32_t *decode_items, int32_t decode_capacity,
    int32_t *merge_items, int32_t merge_capacity, int32_t *prefill_items,
    int32_t prefill_capacity, int32_t *prefill_merge_items, int32_t prefill_merge_capacity,
    int32_t *counts_out) {
  hy::clear_error();
  if (window < 1 || sinks < 0 || sinks > hy::kMaxSinks) {
    hy::set_error("hy_plan_tick_window: window %d (at least 1), sinks %d (0 to %d)", window, sinks,
                  hy::kMaxSinks);
    return HY_EINVAL;
  }
  try {
    return plan_tick(q_lens, kv_lens, num_seqs, num_q_heads, num_kv_heads, page_size, num_cus,
                     target_tokens_per_split, window, sinks, decode_items, decode_capacity,
                     merge_items, merge_capacity, prefill_items, prefill_capacity,
                     prefill_merge_items, prefill_merge_capacity, counts_out);
  } catch (const std::bad_alloc &) {
    hy::set_error("hy_plan_tick_window: out of host memory");
    return HY_ENOSPACE;
  }
}

namespace {

// Costs of drafted-tree attention, in sixteenths of a key step.
constexpr int64_t kTreeStep = 16;
// A step of a tile of at most 128 rows in a launch of more: one wave a SIMD computes instead of
// two. Geometric means over 14 batches each: 4 trees of 200 nodes (three full tiles and one of
// 32 rows each) on 1.5 to 4 k tokens 66.2 us at 16, 64.8 at 14, 64.6 at 13, 65.3 at 12, 66.3 at
// 11; 2 to 32 trees of 5 to 100 nodes 66.2, 65.3, 64.6, 65.3 and 66.7. (With equal tiles, all at
// 16: 67.0 and 66.2.)
constexpr int64_t kTreeFewRowsStep = 13;
// Tiles of 128 rows instead of 256 read keys twice but leave more of the work to units that
// would idle, often without a merge: 5 to 100 nodes on up to 1,500 tokens 30 -> 22 us, 26 -> 20;
// on long caches, where every unit is busy, 390 -> 440. A step of theirs is taken as 11 (9:
// 67.0 us over the 14 mixed batches, 10: 62.9, 11: 62.6, 12: 62.8, only full tiles 65.4), the
// merge as 8 full steps.
constexpr int64_t kTreeHalfStep = 11;
constexpr int64_t kTreeSplitCost = 128;
// A piece after a chunk's first, in launches of at most 128 rows and of more: the rows of Q come
// and the partials go between its steps and the others'. Geometric means over 16 batches each: 2
// to 40 chains of 3 to 8 nodes 22.4 us at 16, 21.2 at 32, 20.7 at 64, 21.1 at 112; trees of 20
// to 32 nodes 41.0, 40.0, 39.3 and 39.9; 4 of 200 nodes 63.7 at 16, 61.7 at 48, 61.8 at 64, 62.9
// at 80.
constexpr int64_t kTreeFewRowsPiece = 64;
constexpr int64_t kTreePiece = 48;
// The merge launch, in launches of at most 32 rows (a step takes 0.45 us there while few units
// run) and of more (1.1 us): 8 nodes on 500 tokens 12.6 us in one piece, 11.8 in two and a merge,
// but then the host takes 13.2; 26 nodes 17.6 and 12.4. Where all units run a merge reads
// more: 9 large trees 31 us whole, 35 at 40 and 32 at 72.
constexpr int64_t kTreeMergeCost = 128;
constexpr int64_t kTreeMergeCostRows = 72;
// Key steps of a chunk at least, on average: more chunks add partials. 8 nodes on 2,000 tokens in
// one launch take 16.0 us at 1, 13.7 at 2, 13.6 at 3 and 13.4 at 4, 64 nodes 24.1, 18.3, 17.4
// and 17.1, on 800 tokens 15.0, 15.0, 14.7 and 14.9; 8 nodes there 12.6, 12.0, 12.0 and 15.7.
constexpr int64_t kTreeChunkSteps = 3;

struct TreePieceRec {
  int32_t tile, step0, step1;  // query tile, and its key steps
};
// Chunk i holds pieces [ends[i - 1], ends[i]).
struct TreeCut {
  std::vector<TreePieceRec> pieces;
  std::vector<int32_t> ends;
  int64_t worst = 0;  // the costliest chunk
  bool split = false;
};

// Cuts the key steps of the query tiles, in order, into at most n_chunks chunks of
// equal cost; `total` is what the whole stream is taken to cost, a step of tile t cost[t] and a
// piece after a chunk's first piece_cost.
void cut_tree(const std::vector<int32_t> &steps, const std::vector<int32_t> &cost, int64_t n_chunks,
              int64_t total, int64_t piece_cost, TreeCut &cut) {
  cut = TreeCut();
  int64_t spent = 0, in_chunk = 0;
  int32_t first = 0;
  auto size = [&]() { return static_cast<int32_t>(cut.pieces.size()); };
  auto close = [&]() {
    cut.worst = std::max(cut.worst, in_chunk);
    spent += in_chunk;
    in_chunk = 0;
    first = size();
    cut.ends.push_back(first);
  };
  for (size_t t = 0; t < steps.size(); ++t) {
    int32_t at = 0;
    while (at < steps[t]) {
      const int64_t left = n_chunks - static_cast<int64_t>(cut.ends.size());  // this one included
      const int64_t share =
          left > 1 ? (std::max<int64_t>(total - spent, 1) + left - 1) / left : INT64_MAX;
      const int64_t extra = size() > first ? piece_cost : 0;
      const int64_t room = share - in_chunk - extra;
      if (room <= 0 && size() > first) {
        close();
        continue;
      }
      const int64_t fit = (std::max<int64_t>(room, 1) - 1) / cost[t] + 1;
      const int32_t n = static_cast<int32_t>(std::min<int64_t>(steps[t] - at, fit));
      cut.pieces.push_back({static_cast<int32_t>(t), at, at + n});
      cut.split = cut.split || n < steps[t];
      in_chunk += n * static_cast<int64_t>(cost[t]) + extra;
      at += n;
    }
  }
  if (size() > first) close();
}

// The query tiles whole, in order, in at most n_chunks chunks of at most `most`; false if they
// do not fit.
bool whole_tree(const std::vector<int32_t> &steps, const std::vector<int32_t> &cost,
                int64_t n_chunks, int64_t most, int64_t piece_cost, TreeCut &cut) {
  cut = TreeCut();
  int64_t in_chunk = 0;
  for (size_t t = 0; t < steps.size(); ++t) {
    const int64_t all = steps[t] * static_cast<int64_t>(cost[t]);
    if (all > most) return false;
    if (in_chunk > 0 && in_chunk + piece_cost + all > most) {
      cut.ends.push_back(static_cast<int32_t>(t));
      in_chunk = 0;
    }
    in_chunk += all + (in_chunk > 0 ? piece_cost : 0);
    cut.pieces.push_back({static_cast<int32_t>(t), 0, steps[t]});
    cut.worst = std::max(cut.worst, in_chunk);
  }
  if (!steps.empty()) cut.ends.push_back(static_cast<int32_t>(steps.size()));
  return static_cast<int64_t>(cut.ends.size()) <= n_chunks;
}

struct TreeTile {
  int32_t seq, q0, q1, kv_end;
};
struct TreeTiling {
  std::vector<TreeTile> tiles;
  std::vector<int32_t> steps;  // a tile's key steps
  int32_t max_rows = 0;
  TreeCut cut;
};

// The requests' rows in tiles of at most tile_rows, and the chunks of their key steps.
void tile_tree(const int32_t *q_lens, const int32_t *kv_lens, int32_t num_seqs, int32_t G,
               int64_t n_units, int32_t tile_rows, TreeTiling &out) {
  std::vector<int32_t> &steps = out.steps, cost;
  int64_t all = 0, all_cost = 0;
  for (int b = 0; b < num_seqs; ++b) {
    // nodes beyond one workgroup's rows: full tiles, and the rest
    const int32_t per = tile_rows / G;
    for (int32_t q0 = 0; q0 < q_lens[b]; q0 += per) {
      const int32_t q1 = std::min(q_lens[b], q0 + per);
      const int32_t end = kv_lens[b] - q_lens[b] + q1;
      out.tiles.push_back({b, q0, q1, end});
      steps.push_back((end + hy::kTreeTileKeys - 1) / hy::kTreeTileKeys);
      all += steps.back();
      out.max_rows = std::max(out.max_rows, (q1 - q0) * G);
    }
  }
  for (size_t t = 0; t < steps.size(); ++t) {
    const bool few = out.max_rows > 128 && (out.tiles[t].q1 - out.tiles[t].q0) * G <= 128;
    cost.push_back(static_cast<int32_t>(few ? kTreeFewRowsStep : kTreeStep));
    all_cost += steps[t] * static_cast<int64_t>(cost[t]);
  }
  const int64_t n_chunks = std::max<int64_t>(1, std::min<int64_t>(n_units, all / kTreeChunkSteps));
  const int64_t piece = out.max_rows > 128 ? kTreePiece : kTreeFewRowsPiece;
  TreeCut trial, &best = out.cut;
  cut_tree(steps, cost, n_chunks, all_cost, piece, best);
  for (int pass = 0; pass < 3; ++pass) {
    const TreeCut &last = pass ? trial : best;
    const int64_t total =
        all_cost + piece * static_cast<int64_t>(last.pieces.size() - last.ends.size());
    cut_tree(steps, cost, n_chunks, total, piece, trial);
    if (trial.worst < best.worst) best = trial;
  }
  // Tiles that need no merge are worth a longer chunk; the shortest such chunk by bisection.
  if (best.split) {
    int64_t fits = best.worst + (out.max_rows > 32 ? kTreeMergeCostRows : kTreeMergeCost), low = 0;
    while (low < fits && whole_tree(steps, cost, n_chunks, fits, piece, trial)) {
      best = trial;
      const int64_t mid = low + (fits - low) / 2;
      if (whole_tree(steps, cost, n_chunks, mid, piece, trial))
        fits = mid;
      else
        low = mid + 1;
    }
  }
}

int plan_tree(const int32_t *q_lens, const int32_t *kv_lens, int32_t num_seqs, int32_t G,
              int32_t num_kv_heads, int32_t num_cus, int32_t *items, int32_t item_capacity,
              int32_t *merge_items, int32_t merge_capacity, int32_t *counts_out) {
  std::vector<int32_t> q_begin(static_cast<size_t>(num_seqs) + 1, 0);
  for (int b = 0; b < num_seqs; ++b) q_begin[b + 1] = q_begin[b] + q_lens[b];
  const int64_t cus = num_cus > 0 ? num_cus : 256, n_units = (cus + num_kv_heads - 1) / num_kv_heads;
  // the tiling whose costliest chunk, and merge, take the shorter time
  TreeTiling full, half;
  tile_tree(q_lens, kv_lens, num_seqs, G, n_units, hy::kTreeRows, full);
  const TreeTiling *tiling = &full;
  if (full.max_rows > 128) {
    tile_tree(q_lens, kv_lens, num_seqs, G, n_units, 128, half);
    auto time = [](const TreeTiling &t, int64_t step) {
      return t.cut.worst * step / kTreeStep + (t.cut.split ? kTreeSplitCost : 0);
    };
    if (time(half, kTreeHalfStep) < time(full, kTreeStep)) tiling = &half;
  }
  const std::vector<TreeTile> &tiles = tiling->tiles;
  const std::vector<int32_t> &steps = tiling->steps;
  const TreeCut &best = tiling->cut;
  const int32_t max_rows = tiling->max_rows;
  const std::vector<TreePieceRec> &pieces = best.pieces;
  const std::vector<int32_t> &ends = best.ends;
  const int64_t need = 2 * static_cast<int64_t>(ends.size()) + static_cast<int64_t>(pieces.size());
  if (need > item_capacity) {
    hy::set_error("hy_plan_tree: item capacity %d too small (need %lld)", item_capacity,
                  static_cast<long long>(need));
    return HY_ENOSPACE;
  }
  int32_t n_merge = 0;
  int64_t n_slots = 0;
  int32_t *rec = items + hy::kTreeChunkInts * static_cast<int64_t>(ends.size());
  for (size_t i = 0; i < pieces.size(); ++i) {
    const TreeTile &t = tiles[pieces[i].tile];
    const int32_t blocks = ((t.q1 - t.q0) * G + 31) / 32;
    const bool whole = pieces[i].step0 == 0 && pieces[i].step1 == steps[pieces[i].tile];
    if (!whole) {
      if (pieces[i].step0 == 0) {
        if (n_merge >= merge_capacity) {
          hy::set_error("hy_plan_tree: merge capacity %d too small", merge_capacity);
          return HY_ENOSPACE;
        }
        int32_t *m = merge_items + 8 * n_merge++;
        m[0] = t.seq;
        m[1] = t.q0;
        m[2] = t.q1;
        m[3] = static_cast<int32_t>(n_slots);
        m[4] = 0;
        m[5] = q_begin[t.seq];
        m[6] = blocks;
        m[7] = 0;
      }
      ++merge_items[8 * (n_merge - 1) + 4];  // a tile's pieces are consecutive
    }
    int32_t *r = rec + 8 * i;
    r[0] = t.seq;
    r[1] = t.q0;
    r[2] = t.q1;
    r[3] = pieces[i].step0 * hy::kTreeTileKeys;
    r[4] = std::min(t.kv_end, pieces[i].step1 * hy::kTreeTileKeys);
    r[5] = whole ? -1 : static_cast<int32_t>(n_slots);
    r[6] = q_begin[t.seq];
    r[7] = kv_lens[t.seq] - q_lens[t.seq];
    if (!whole) n_slots += blocks;
    if (n_slots > INT32_MAX) {
      hy::set_error("hy_plan_tree: too many partials");
      return HY_EINVAL;
    }
  }
  for (size_t i = 0; i < ends.size(); ++i) {
    const int32_t first = i ? ends[i - 1] : 0;
    int32_t *ch = items + hy::kTreeChunkInts * i;
    int32_t n = 0;
    for (int32_t p = first; p < ends[i]; ++p) n += pieces[p].step1 - pieces[p].step0;
    ch[0] = first;
    ch[1] = ends[i];
    ch[2] = n;
    ch[3] = 1;
    for (int32_t p = first; p < ends[i]; ++p) {
      const TreeTile &t = tiles[pieces[p].tile];
      if (t.q1 - t.q0 < q_lens[t.seq]) ch[3] = 0;
    }
    for (int j = 4; j < 8; ++j) ch[j] = 0;
    for (int j = 0; j < 8; ++j) ch[8 + j] = rec[8 * first + j];
  }
  counts_out[0] = static_cast<int32_t>(ends.size());
  counts_out[1] = static_cast<int32_t>(pieces.size());
  counts_out[2] = n_merge;
  counts_out[3] = static_cast<int32_t>(n_slots);
  counts_out[4] = max_rows;
  return HY_OK;
}

}  // namespace

extern "C" int hy_tree_lines(const int32_t *parents, const int32_t *q_lens, int32_t num_seqs,
                             int32_t line_words, uint32_t *lines, int32_t *depths) {
  hy::clear_error();
  if (num_seqs < 0 || (num_seqs > 0 && (!parents || !q_lens || !lines || !depths)) ||
      (line_words != 4 && line_words != 8)) {
    hy::set_error("hy_tree_lines: invalid arrays");
    return HY_EINVAL;
  }
  int64_t row = 0;
  for (int32_t b = 0; b < num_seqs; ++b) {
    if (q_lens[b] < 1 || q_lens[b] > 32 * line_words) {
      hy::set_error("hy_tree_lines: tree %d has %d nodes, not 1 to %d", b, q_lens[b],
                    32 * line_words);
      return HY_EINVAL;
    }
    const int64_t first = row;
    for (int32_t i = 0; i < q_lens[b]; ++i, ++row) {
      const int32_t p = parents[row];
      if (p < -1 || p >= i) {
        hy::set_error("hy_tree_lines: tree %d: the parent of node %d is %d, not an earlier node or -1",
                      b, i, p);
        return HY_EINVAL;
      }
      for (int32_t w = 0; w < line_words; ++w)
        lines[row * line_words + w] = p < 0 ? 0u : lines[(first + p) * line_words + w];
      lines[row * line_words + (i >> 5)] |= 1u << (i & 31);
      depths[row] = p < 0 ? 0 : depths[first + p] + 1;
    }
  }
  return HY_OK;
}

extern "C" int32_t hy_tree_max_nodes(void) { return hy::kTreeMaxNodes; }

extern "C" int hy_plan_tree(const int32_t *q_lens, const int32_t *kv_lens, int32_t num_seqs,
                            int32_t num_q_heads, int32_t num_kv_heads, int32_t num_cus,
                            int32_t *items, int32_t item_capacity, int32_t *merge_items,
                            int32_t merge_capacity, int32_t *counts_out) {
  hy::clear_error();
  if (num_seqs < 0 || (num_seqs > 0 && (q_lens == nullptr || kv_lens == nullptr)) ||
      counts_out == nullptr || (item_capacity > 0 && items == nullptr) ||
      (merge_capacity > 0 && merge_items == nullptr)) {
    hy::set_error("hy_plan_tree: invalid arrays");
    return HY_EINVAL;
  }
  if (num_kv_heads < 1 || num_q_heads < num_kv_heads || num_q_heads % num_kv_heads) {
    hy::set_error("hy_plan_tree: num_q_heads (%d) must be a multiple of num_kv_heads (%d)",
                  num_q_heads, num_kv_heads);
    return HY_EINVAL;
  }
  const int32_t G = num_q_heads / num_kv_heads;
  if (G > 16 || (G & (G - 1))) {
    hy::set_error("hy_plan_tree: GQA group size %d unsupported (1, 2, 4, 8, 16)", G);
    return HY_EUNSUPPORTED;
  }
  int64_t rows = 0;
  for (int b = 0; b < num_seqs; ++b) {
    if (q_lens[b] < 1 || kv_lens[b] < q_lens[b]) {
      hy::set_error("hy_plan_tree: sequence %d has q_len %d, kv_len %d", b, q_lens[b], kv_lens[b]);
      return HY_EINVAL;
    }
    if (q_lens[b] > hy::kTreeMaxNodes) {
      hy::set_error("hy_plan_tree: sequence %d has %d nodes, at most %d are supported", b,
                    q_lens[b], hy::kTreeMaxNodes);
      return HY_EUNSUPPORTED;
    }
    // the kernel counts keys to the end of the next tile in 32 bits
    if (kv_lens[b] > INT32_MAX - 2 * hy::kTreeTileKeys) {
      hy::set_error("hy_plan_tree: sequence %d has kv_len %d, too long", b, kv_lens[b]);
      return HY_EUNSUPPORTED;
    }
    rows += q_lens[b];
  }
  if (rows > INT32_MAX) {
    hy::set_error("hy_plan_tree: too many rows");
    return HY_EINVAL;
  }
  try {
    return plan_tree(q_lens, kv_lens, num_seqs, G, num_kv_heads, num_cus, items, item_capacity,
                     merge_items, merge_capacity, counts_out);
  } catch (const std::bad_alloc &) {
    hy::set_error("hy_plan_tree: out of host memory");
    return HY_ENOSPACE;
  }
}

namespace {

// Weigh workgroups a compute unit holds, and what an item costs besides its row stages, in stages
// (measured on MI355X, two a unit: 2.6 us a stage, about 5 us for the keys, the first rows and the
// sums).
constexpr int64_t kWeighPerCu = 2;
constexpr double kWeighFixed = 2.0;
// Items a slot beyond which no cut evens out more than it costs.
constexpr int64_t kWeighItems = 6;

// One sequence's chunk in row ranges ("parts") of equal length.
struct WeighParts {
  int64_t count, tokens;
  WeighParts(int64_t ql, int64_t range) {
    count = (ql + range - 1) / range;
    tokens = (ql + count - 1) / count;
    count = (ql + tokens - 1) / tokens;
  }
};

// The range of tokens whose items, longest first, are done soonest.
int64_t weigh_range(const int32_t *q_lens, const int32_t *kv_lens, int32_t num_seqs, int64_t G,
                    int64_t slots) {
  constexpr int64_t keys = hy::kWeighKeys;
  int64_t longest = 1;
  for (int b = 0; b < num_seqs; ++b) longest = std::max<int64_t>(longest, q_lens[b]);
  int64_t best_range = longest;
  double best = HUGE_VAL;
  std::vector<double> costs, free_at;
  const int64_t least = std::max<int64_t>(1, hy::kWeighRows / G);  // one stage
  for (int64_t n = 1; n <= 32; ++n) {
    const int64_t range = (longest + n - 1) / n;
    if (n > 1 && range < least) break;
    costs.clear();
    for (int b = 0; b < num_seqs; ++b) {
      const int64_t ql = q_lens[b], cache = kv_lens[b] - ql;
      if (ql <= 1) continue;
      const WeighParts parts(ql, range);
      for (int64_t t0 = 0; t0 < kv_lens[b]; t0 += keys)
        for (int64_t p = t0 <= cache ? 0 : (t0 - cache) / parts.tokens; p < parts.count; ++p) {
          const int64_t from = std::max(p * parts.tokens, t0 - cache);
          const int64_t rows = (std::min(ql, (p + 1) * parts.tokens) - from) * G;
          costs.push_back(kWeighFixed + static_cast<double>((rows + hy::kWeighRows - 1) / hy::kWeighRows));
        }
      if (n > 1 && static_cast<int64_t>(costs.size()) > kWeighItems * slots) return best_range;
    }
    std::sort(costs.begin(), costs.end(), std::greater<double>());
    free_at.assign(static_cast<size_t>(slots), 0.0);
    double end = 0;
    for (double c : costs) {
      std::pop_heap(free_at.begin(), free_at.end(), std::greater<double>());
      end = std::max(end, free_at.back() += c);
      std::push_heap(free_at.begin(), free_at.end(), std::greater<double>());
    }
    if (end < best) {
      best = end;
      best_range = range;
    }
  }
  return best_range;
}

int plan_weigh(const int32_t *q_lens, const int32_t *kv_lens, const int32_t *rows,
               int32_t num_seqs, int32_t num_q_heads, int32_t num_kv_heads, int32_t num_cus,
               const int32_t *merge_items, int32_t n_merge, int32_t *score_start, int32_t *items,
               int32_t item_capacity, int32_t *adds, int32_t add_capacity, int64_t *counts_out) {
  constexpr int64_t keys = hy::kWeighKeys;
  const int64_t G = num_q_heads / num_kv_heads;
  const int64_t cus = num_cus > 0 ? num_cus : 256;
  const int64_t slots = std::max<int64_t>(1, cus * kWeighPerCu / num_kv_heads);
  const int64_t range = weigh_range(q_lens, kv_lens, num_seqs, G, slots);
  int64_t scores = 0, partials = 0, q_row = 0, n_items = 0, n_adds = 0, parts_max = 0;
  // the partial slots of every decode token
  std::vector<const int32_t *> slots_of(static_cast<size_t>(num_seqs), nullptr);
  for (int i = 0; i < n_merge; ++i) slots_of[merge_items[4 * i]] = merge_items + 4 * i;
  for (int b = 0; b < num_seqs; ++b) {
    if (q_lens[b] == 1 && slots_of[b] == nullptr) {
      hy::set_error("hy_plan_weigh: sequence %d has no merge item", b);
      return HY_EINVAL;
    }
    const int64_t kv = kv_lens[b], ql = q_lens[b], cache = kv - ql;
    const bool chunk = ql > 1;
    const WeighParts parts(ql, range);
    const int64_t per = parts.tokens, n_parts = parts.count;
    score_start[b] = chunk ? 0 : static_cast<int32_t>(scores);
    for (int64_t t0 = 0; t0 < kv; t0 += keys) {
      // parts whose last token sees the first key
      const int64_t first = !chunk || t0 <= cache ? 0 : (t0 - cache) / per;
      if (n_adds >= add_capacity) {
        hy::set_error("hy_plan_weigh: addition capacity %d too small", add_capacity);
        return HY_ENOSPACE;
      }
      int32_t *a = adds + 8 * n_adds++;
      a[0] = rows[b];
      a[1] = static_cast<int32_t>(t0);
      a[2] = static_cast<int32_t>(std::min(kv, t0 + keys));
      a[3] = chunk ? static_cast<int32_t>((n_parts - first) * num_kv_heads) : slots_of[b][2];
      a[4] = chunk ? static_cast<int32_t>(first * num_kv_heads) : slots_of[b][1];
      a[5] = !chunk;
      a[6] = static_cast<int32_t>(chunk ? partials : scores);
      a[7] = 0;
      for (int64_t p = first; chunk && p < n_parts; ++p) {
        if (n_items >= item_capacity) {
          hy::set_error("hy_plan_weigh: item capacity %d too small", item_capacity);
          return HY_ENOSPACE;
        }
        int32_t *it = items + 8 * n_items++;
        it[0] = b;
        it[1] = static_cast<int32_t>(t0);
        it[2] = static_cast<int32_t>(p * per);
        it[3] = static_cast<int32_t>(std::min(ql, (p + 1) * per));
        it[4] = static_cast<int32_t>(p);
        it[5] = static_cast<int32_t>(q_row);
        it[6] = static_cast<int32_t>(cache);
        it[7] = static_cast<int32_t>(partials);
      }
    }
    if (chunk) {
      partials += (kv + keys - 1) / keys * keys;
      parts_max = std::max(parts_max, n_parts);
    } else {
      scores += (kv + hy::kWeighPad - 1) / hy::kWeighPad * hy::kWeighPad;
    }
    q_row += ql;
    if (scores > INT32_MAX - 2 * keys || partials > INT32_MAX - 2 * keys ||
        q_row * num_q_heads > INT32_MAX) {
      hy::set_error("hy_plan_weigh: too many keys or rows in one batch");
      return HY_EUNSUPPORTED;
    }
  }
  // the longest first, as weigh_range() has them
  std::vector<std::array<int32_t, 8>> order(static_cast<size_t>(n_items));
  if (n_items > 0) std::copy_n(items, 8 * n_items, order[0].data());
  auto tokens = [](const std::array<int32_t, 8> &x) { return x[3] - std::max(x[2], x[1] - x[6]); };
  std::stable_sort(order.begin(), order.end(),
                   [&](const auto &x, const auto &y) { return tokens(x) > tokens(y); });
  for (size_t i = 0; i < order.size(); ++i) std::copy(order[i].begin(), order[i].end(), items + 8 * i);
  counts_out[0] = n_items;
  counts_out[1] = n_adds;
  counts_out[2] = scores;
  counts_out[3] = partials;
  counts_out[4] = parts_max;
  return HY_OK;
}

}  // namespace

extern "C" int hy_plan_weigh(const int32_t *q_lens, const int32_t *kv_lens, const int32_t *rows,
                             int32_t num_seqs, int32_t num_q_heads, int32_t num_kv_heads,
                             int32_t num_cus, const int32_t *merge_items, int32_t n_merge,
                             int32_t *score_start, int32_t *items, int32_t item_capacity,
                             int32_t *adds, int32_t add_capacity, int64_t *counts_out) {
  hy::clear_error();
  if (num_seqs < 0 || counts_out == nullptr ||
      (num_seqs > 0 && (!q_lens || !kv_lens || !rows || !score_start)) ||
      (item_capacity > 0 && items == nullptr) || (add_capacity > 0 && adds == nullptr) ||
      n_merge < 0 || (n_merge > 0 && merge_items == nullptr)) {
    hy::set_error("hy_plan_weigh: invalid arrays");
    return HY_EINVAL;
  }
  for (int i = 0; i < n_merge; ++i) {
    if (merge_items[4 * i] < 0 || merge_items[4 * i] >= num_seqs) {
      hy::set_error("hy_plan_weigh: merge item %d is of sequence %d", i, merge_items[4 * i]);
      return HY_EINVAL;
    }
  }
  if (num_kv_heads < 1 || num_q_heads < num_kv_heads || num_q_heads % num_kv_heads) {
    hy::set_error("hy_plan_weigh: num_q_heads (%d) must be a multiple of num_kv_heads (%d)",
                  num_q_heads, num_kv_heads);
    return HY_EINVAL;
  }
  const int32_t G = num_q_heads / num_kv_heads;
  if (G > 16 || (G & (G - 1))) {
    hy::set_error("hy_plan_weigh: GQA group size %d unsupported (1, 2, 4, 8, 16)", G);
    return HY_EUNSUPPORTED;
  }
  for (int b = 0; b < num_seqs; ++b) {
    if (q_lens[b] < 1 || kv_lens[b] < q_lens[b] || rows[b] < 0) {
      hy::set_error("hy_plan_weigh: sequence %d has q_len %d, kv_len %d, row %d", b, q_lens[b],
                    kv_lens[b], rows[b]);
      return HY_EINVAL;
    }
  }
  try {
    return plan_weigh(q_lens, kv_lens, rows, num_seqs, num_q_heads, num_kv_heads, num_cus,
                      merge_items, n_merge, score_start, items, item_capacity, adds, add_capacity,
                      counts_out);
  } catch (const std::bad_alloc &) {
    hy::set_error("hy_plan_weigh: out of host memory");
    return HY_ENOSPACE;
  }
}
