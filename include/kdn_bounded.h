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

/* ---- What each key of a prompt got -------------------------------------------------------------------------------
 * weights[slot of b][e][j] = the sum, over the query rows of sequence b that see its key j and the query heads of key head e, of
 * exp(scale q.k - lse): with kdn_attn_fwd's lse, the column sums of its softmax.  Rows and offsets as there (the rows may be the
 * last ones of a sequence alone), window as above, 0: none.  With `add` the keys before a sequence's first row (j < len_k - len_q),
 * whose earlier rows' weights are there already, are added to; all others are set.  Places past `places`, and slots out of range,
 * are skipped; slots are distinct.  Summed in a fixed order. */
typedef struct kdn_attn_weights_args {
  int64_t num_seqs, total_q, total_k;
  int64_t H, H_kv;
  int d, dtype, add;
  float scale;
  int64_t window, sinks;
  const int64_t* cu_q;          /* device [num_seqs + 1] */
  const int64_t* cu_k;          /* device [num_seqs + 1]; NULL: cu_q */
  const void* q; int64_t q_stride[2];   /* [token][head] */
  const void* k; int64_t k_stride[2];
  const float* lse;             /* [H][total_q] */
  float* weights; int64_t weights_stride[2];  /* [slot][head], places next to one another */
  int64_t places, num_slots;
  const int32_t* slots;         /* device [num_seqs]: a sequence's slot; NULL: its number */
  void* workspace; size_t workspace_bytes;
} kdn_attn_weights_args;
size_t kdn_attn_weights_workspace_bytes(const kdn_attn_weights_args* a);   /* 0: invalid; reads sizes only, and whether there are slots */
int kdn_attn_weights(const kdn_attn_weights_args* a, void* stream);

/* ---- Eviction ----------------------------------------------------------------------------------------------------
 * Cuts each stream's cache from L = lens[b] places to N = min(L, keep[b]), of each layer and key head on its own.  Place j of a
 * stream holds the token at position positions[slot][layer][head][j] if j < settled[b], else j + evicted[b] (what a stream's
 * tokens so far are more than its places).  Of the places stay: those of positions below `sinks`, then those of the last `recent` of
 * the L + evicted[b] positions, then those of largest weight (a weight that is no positive number counts as 0); of equals the
 * lowest (of the last `recent`, too, where they and the sinks are more than N: give at most N - sinks to have the latest).  The kept places from N on move, in order, to the given-up ones before it, in order: key, value, weight and position;
 * afterwards positions[0 .. N) are all there (settled is N, evicted L - N more).  What lies from N on is left as it is.
 * The pages of places below N are the stream's own: no other stream has them.  Slots out of range are skipped; slots and pages are
 * distinct, and no stride over several pages, layers, heads, tokens or slots is 0 (KDN_ERR_INVALID_ARGUMENT).  Needs max_len >= every lens[b] (longer ones are cut), `places` and the page table's room for it. */
typedef struct kdn_evict_args {
  int64_t num_seqs, layers, H_kv;
  int d, dtype;
  int64_t page_tokens, num_pages, table_width, table_stride;
  int64_t max_len, sinks, recent;
  const int32_t* page_table;    /* device [num_seqs][table_width], rows table_stride apart */
  const int32_t* lens;          /* device [num_seqs] */
  const int32_t* keep;          /* device [num_seqs] */
  const int32_t* settled;       /* device [num_seqs], or NULL: 0 */
  const int32_t* evicted;       /* device [num_seqs], or NULL: 0 */
  const int32_t* slots;         /* device [num_seqs]: a stream's slot; NULL: its number */
  void* k_pages; int64_t k_pages_stride[4];      /* [page][layer][head][token] */
  void* v_pages; int64_t v_pages_stride[4];
  float* weights; int64_t weights_stride[3];     /* [slot][layer][head], places next to one another */
  int32_t* positions; int64_t positions_stride[3];
  int64_t places, num_slots;
  void* workspace; size_t workspace_bytes;       /* 16-byte aligned */
} kdn_evict_args;
size_t kdn_evict_workspace_bytes(const kdn_evict_args* a);   /* 0: invalid; reads sizes only, and whether there are slots */
int kdn_evict(const kdn_evict_args* a, void* stream);

/* ---- The pages' bookkeeping for it (host only, as kdn_page_pool_*) -------------------------------------------------- */
/* The pages of the stream's first `tokens` tokens become its own: each that another stream has is replaced, and pairs[0 .. 2 n) are
 * the copies to make before anything is written; n is returned (KDN_ERR_CAPACITY, and nothing changed, if it is over room or the
 * free pages). */
int64_t kdn_page_pool_own(kdn_page_pool* pool, int stream, int64_t tokens, int32_t* pairs, int64_t room);
/* Takes the full pages first .. first + pages - 1 out of the stream: those behind them move up, and the stream is pages *
 * page_tokens shorter (what no window reaches any more). */
int kdn_page_pool_drop(kdn_page_pool* pool, int stream, int64_t first, int64_t pages);

#ifdef __cplusplus
}
#endif

#endif /* KDN_BOUNDED_H */
