// Attention of a whole tick in one call: the launches of its decode and prefill lists and their
// merges, with a window, or with the weights of the cached tokens.

#include "attend.h"

#include "../../include/hayate_attn.h"

namespace hy {
void set_error(const char *fmt, ...);
void clear_error();
}  // namespace hy

namespace {

struct Tick {
  hy::Rows q, out;
  hy::Pools pools;
  const int32_t *q_start, *kv_lens;
  hy::Items decode, decode_merge, prefill, prefill_merge;
  hy::Workspace decode_ws, prefill_ws;
  hy::Shape shape;
};

int check(const char *name, const Tick &t) {
  if (t.decode.count < 0 || t.decode_merge.count < 0 || t.prefill.count < 0 ||
      t.prefill_merge.count < 0) {
    hy::set_error("%s: item counts must be non-negative", name);
    return HY_EINVAL;
  }
  if ((t.decode.count == 0) != (t.decode_merge.count == 0) ||
      (t.prefill.count == 0 && t.prefill_merge.count > 0)) {
    hy::set_error("%s: a merge list without the work before it, or the reverse", name);
    return HY_EINVAL;
  }
  return HY_OK;
}

int attend_chunks(const char *name, const Tick &t, const hy::Window &window, float *row_ml,
                  void *stream) {
  if (int rc = hy::prefill(name, t.q, t.out, t.pools, t.q_start, t.kv_lens, t.prefill, t.prefill_ws,
                           t.shape, window, row_ml, stream))
    return rc;
  return hy::prefill_merge(name, t.out, t.q_start, t.prefill_merge, t.prefill_ws, t.shape, row_ml,
                           stream);
}

}  // namespace

#define HY_TICK                                                                                   \
  Tick {                                                                                          \
    {const_cast<void *>(q), q_stride_seq, q_stride_tok, q_stride_head},                           \
        {out, o_stride_seq, o_stride_tok, o_stride_head},                                         \
        {const_cast<void *>(k_pool), const_cast<void *>(v_pool), pool_head_stride, page_table,    \
         page_table_stride},                                                                      \
        q_start, kv_lens, {decode_items, n_decode, n_slots}, {merge_items, n_merge, n_slots},     \
        {prefill_items, n_prefill, n_prefill_slots},                                              \
        {prefill_merge_items, n_prefill_merge, n_prefill_slots}, {workspace, workspace_bytes},    \
        {prefill_workspace, prefill_workspace_bytes}, {                                           \
      num_seqs, num_q_heads, num_kv_heads, head_dim, page_size, scale                             \
    }                                                                                             \
  }

extern "C" int hy_paged_window(
    const void *q, int64_t q_stride_seq, int64_t q_stride_tok, int64_t q_stride_head, void *out,
    int64_t o_stride_seq, int64_t o_stride_tok, int64_t o_stride_head, const void *k_pool,
    const void *v_pool, int64_t pool_head_stride, const int32_t *page_table,
    int64_t page_table_stride, const int32_t *q_start, const int32_t *kv_lens,
    const int32_t *decode_items, int32_t n_decode, const int32_t *merge_items, int32_t n_merge,
    int32_t n_slots, void *workspace, int64_t workspace_bytes, const int32_t *prefill_items,
    int32_t n_prefill, const int32_t *prefill_merge_items, int32_t n_prefill_merge,
    int32_t n_prefill_slots, void *prefill_workspace, int64_t prefill_workspace_bytes,
    int32_t num_seqs, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    int32_t page_size, int32_t window, int32_t sinks, float scale, void *stream) {
  const char *name = "hy_paged_window";
  hy::clear_error();
  const hy::Window w{window, sinks};
  if (int rc = hy::check_window(name, w)) return rc;
  const Tick t = HY_TICK;
  if (int rc = check(name, t)) return rc;
  if (int rc = hy::decode(name, t.q, t.out, t.pools, t.q_start, t.decode, t.decode_ws, t.shape, w, {},
                          nullptr, stream))
    return rc;
  if (int rc = hy::decode_merge(name, t.out, t.q_start, t.decode_merge, t.decode_ws, t.shape, stream))
    return rc;
  return attend_chunks(name, t, w, nullptr, stream);
}

extern "C" int hy_paged_weigh(
    const void *q, int64_t q_stride_seq, int64_t q_stride_tok, int64_t q_stride_head, void *out,
    int64_t o_stride_seq, int64_t o_stride_tok, int64_t o_stride_head, const void *k_pool,
    const void *v_pool, int64_t pool_head_stride, const int32_t *page_table,
    int64_t page_table_stride, const int32_t *q_start, const int32_t *kv_lens,
    const int32_t *decode_items, int32_t n_decode, const int32_t *merge_items, int32_t n_merge,
    int32_t n_slots, void *workspace, int64_t workspace_bytes, const int32_t *prefill_items,
    int32_t n_prefill, const int32_t *prefill_merge_items, int32_t n_prefill_merge,
    int32_t n_prefill_slots, void *prefill_workspace, int64_t prefill_workspace_bytes,
    int32_t num_seqs, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    int32_t page_size, const int32_t *weigh_items, int32_t n_weigh, const int32_t *add_items,
    int32_t n_add, const int32_t *score_start, float *scores, int64_t score_stride,
    float *partials, int64_t partial_stride, float *row_ml, float *weights,
    int64_t weights_stride, float scale, void *stream) {
  const char *name = "hy_paged_weigh";
  hy::clear_error();
  const Tick t = HY_TICK;
  if (int rc = check(name, t)) return rc;
  if ((n_decode > 0 && !(scores && score_start)) || (n_prefill > 0 && !(partials && row_ml))) {
    hy::set_error("%s: null pointer argument", name);
    return HY_EINVAL;
  }
  const hy::Weigh w{weigh_items, n_weigh,        add_items, n_add,
                    {n_decode > 0 ? scores : nullptr, score_start, score_stride},
                    partials,    partial_stride, row_ml,    weights, weights_stride};
  if (int rc = hy::check_weigh(name, t.q, t.shape, w)) return rc;
  if (int rc = hy::decode(name, t.q, t.out, t.pools, t.q_start, t.decode, t.decode_ws, t.shape, {},
                          w.scores, nullptr, stream))
    return rc;
  if (int rc = attend_chunks(name, t, {}, row_ml, stream)) return rc;
  if (int rc = hy::weigh_chunks(name, t.q, t.pools, t.shape, w, stream)) return rc;
  return hy::finish_weights(name, t.out, t.decode_merge, t.decode_ws, t.shape, w, stream);
}
