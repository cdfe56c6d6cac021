// Launches that the combined attention calls are made of; the functions behind the C entries of
// the same kind, with what a window or the weights of tokens add to them.
#pragma once

#include <stdint.h>

namespace hy {

// Packed rows: element strides of a sequence, a token and a head.
struct Rows {
  void *at;
  int64_t seq, tok, head;
};
struct Pools {
  void *k, *v;
  int64_t head_stride;
  const int32_t *page_table;
  int64_t page_table_stride;
};
struct Shape {
  int32_t num_seqs, num_q_heads, num_kv_heads, head_dim, page_size;
  float scale;
};
struct Workspace {
  void *at;
  int64_t bytes;
};
// A list of work and the partial slots that it leaves or joins.
struct Items {
  const int32_t *at;
  int32_t count, slots;
};
struct Window {
  int32_t window, sinks;  // window 0: none
};
// Raw scores of decode tokens (null: not kept).
struct Scores {
  float *at;
  const int32_t *start;
  int64_t stride;
};
struct AppendArgs;

int decode(const char *name, const Rows &q, const Rows &out, const Pools &pools,
           const int32_t *q_start, const Items &items, const Workspace &ws, const Shape &shape,
           const Window &window, const Scores &scores, const AppendArgs *append, void *stream);
int decode_merge(const char *name, const Rows &out, const int32_t *q_start, const Items &items,
                 const Workspace &ws, const Shape &shape, void *stream);
int prefill(const char *name, const Rows &q, const Rows &out, const Pools &pools,
            const int32_t *q_start, const int32_t *kv_lens, const Items &items,
            const Workspace &ws, const Shape &shape, const Window &window, float *row_ml,
            void *stream);
int prefill_merge(const char *name, const Rows &out, const int32_t *q_start, const Items &items,
                  const Workspace &ws, const Shape &shape, float *row_ml, void *stream);
// The weights of a tick's tokens: what its chunks' products (computed again) and its decode tokens'
// scores say. finish_weights() joins the decode tokens' partials, as decode_merge() does, and adds
// to the table.
struct Weigh {
  const int32_t *items;
  int32_t n_items;
  const int32_t *adds;
  int32_t n_adds;
  Scores scores;
  float *partials;
  int64_t partial_stride;
  float *row_ml;
  float *weights;
  int64_t weights_stride;
};
int check_weigh(const char *name, const Rows &q, const Shape &shape, const Weigh &weigh);
int weigh_chunks(const char *name, const Rows &q, const Pools &pools, const Shape &shape,
                 const Weigh &weigh, void *stream);
int finish_weights(const char *name, const Rows &out, const Items &merge, const Workspace &ws,
                   const Shape &shape, const Weigh &weigh, void *stream);

int check_window(const char *name, const Window &window);

}  // namespace hy
