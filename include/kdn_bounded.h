/* kdn_bounded.h -- C ABI of bounded contexts: what keeps an anchor layer's cache and its time from growing with a stream's
 * whole past, next to recurrent states of fixed size.  Attention that sees a sliding window and a few first tokens, and the
 * eviction of keys by the attention weight that they got.  Part of libkdn.so; the conventions and argument structs are those of
 * kdn_anchor.h.
 *
 * Reference interfaces (paths relative to jatin-yadav-acad/kernel-deltanet): the softmax anchor pages of HybridMemoryPool,
 * serving/hybrid_memory_pool.{h,cpp}, which the reference never bounds.
 */
#ifndef KDN_BOUNDED_H
#define KDN_BOUNDED_H

#include "kdn_anchor.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Version of this header's entry points: major << 16 | minor. */
int kdn_bounded_version(void);

/* ---- A sliding window and sinks -----------------------------------------------------------------------------------
 * A query at position p of its keys (the last query's position is the last key's) sees key j if j <= p and
 * (j > p - window or j < sinks): the last `window` keys, its own among them, and the first `sinks`.  window >= 1, sinks >= 0;
 * all else is kdn_attn_fwd's and kdn_attn_bwd's, y_low and lse included: the backward takes what the forward of the same
 * window and sinks wrote. */
int kdn_attn_window_fwd(const kdn_attn_args* a, int64_t window, int64_t sinks, void* stream);
size_t kdn_attn_window_bwd_workspace_bytes(const kdn_attn_bwd_args* a, int64_t window, int64_t sinks);   /* 0: invalid; reads sizes only */
int kdn_attn_window_bwd(const kdn_attn_bwd_args* a, int64_t window, int64_t sinks, void* stream);

/* ---- New tokens over pages: a window, and what each key got -------------------------------------------------------
 * kdn_tree_attn in which a token, at position context_lens[b] + its depth (the number of new tokens that it sees besides
 * itself), sees of the context and of the new tokens only those in the window or among the sinks, as above; window 0: all.
 *   weights: to the weight of each key of the context, weights[slot of b][key head][place], is added the sum of its softmax weights
 * over the stream's new tokens and the query heads that share its head; the new tokens' own places, behind the context, are
 * set to theirs.  Places past `places` are skipped, and streams whose slot is negative or past num_slots.  Slots are distinct.  Runs of
 * tokens alone (no parents: a refused draft would count), at most 32 rows to a key head (max_new * H / H_kv); summed in a fixed
 * order. */
typedef struct kdn_tree_bound_args {
  int64_t window, sinks;
  float* weights; int64_t weights_stride[2];  /* [slot][head], places next to one another; NULL: none */
  int64_t places, num_slots;
  const int32_t* slots;         /* device [num_seqs]: a stream's slot; NULL: its number */
} kdn_tree_bound_args;
size_t kdn_tree_attn_bounded_workspace_bytes(const kdn_tree_attn_args* a, const kdn_tree_bound_args* b);   /* 0: invalid; reads sizes only,
                                                                         and whether there are weights */
int kdn_tree_attn_bounded(const kdn_tree_attn_args* a, const kdn_tree_bound_args* b, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* KDN_BOUNDED_H */
