/* kdn_anchor.h -- C ABI of the softmax anchor layers: the attention layers that a hybrid model keeps between its
 * recurrent ones, and the pages their keys and values live in.  Part of libkdn.so; the conventions are those of kdn.h
 * (caller-allocated device buffers, stream-ordered, a negative kdn_status on error, element strides with a contiguous
 * innermost dimension, no library state).  Head dimension d: 64 or 128.  dtype: KDN_DTYPE_BF16 or KDN_DTYPE_F32 for all
 * of a call's tensors; rows start on 16 bytes.
 *
 * Reference interfaces (paths relative to jatin-yadav-acad/kernel-deltanet): the softmax anchor pages of
 * HybridMemoryPool, serving/hybrid_memory_pool.{h,cpp} (16-token reference-counted pages, shared by fork_stream), whose
 * attention the reference leaves to its host framework.
 */
#ifndef KDN_ANCHOR_H
#define KDN_ANCHOR_H

#include "kdn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Version of this header's entry points: major << 16 | minor. */
int kdn_anchor_version(void);

/* ---- Causal attention over packed sequences -------------------------------------------------------------------
 * y_i = sum_j p_ij v_j, p_i. = softmax over the visible j of scale q_i . k_j.  Sequence b is the query rows
 * cu_q[b] .. cu_q[b+1]-1 and the key rows cu_k[b] .. cu_k[b+1]-1; its query i sees the keys j <= i + (len_k - len_q)
 * (the last query sees the last key).  A row that sees no key gets zeros, its lse -infinity and its gradient zero;
 * so do rows that no sequence has (before the first offset, from the last on), and such keys' gradients are zero.
 * Query head h uses key head h / (H / H_kv).  Offsets are read on the device; the grid follows from total_q and num_seqs.
 * A row has an infinity or NaN of a key or value only if it sees that key. */
typedef struct kdn_attn_args {
  int64_t num_seqs, total_q, total_k;
  int64_t H, H_kv;              /* H a multiple of H_kv */
  int d, dtype;
  float scale;                  /* finite, > 0 */
  const int64_t* cu_q;          /* device [num_seqs + 1], not decreasing, within [0, total_q] */
  const int64_t* cu_k;          /* device [num_seqs + 1]; NULL: cu_q (total_k = total_q) */
  const void* q; int64_t q_stride[2];   /* [token][head] */
  const void* k; int64_t k_stride[2];
  const void* v; int64_t v_stride[2];
  void* y;       int64_t y_stride[2];
  float* lse;                   /* [H][total_q]: log of the sum of exp(scale q.k), or NULL */
  void* y_low;   int64_t y_low_stride[2];   /* what rounding to bf16 took from y, for the backward, or NULL (unused with fp32) */
} kdn_attn_args;
int kdn_attn_fwd(const kdn_attn_args* a, void* stream);

/* Gradients of a loss through kdn_attn_fwd, given dy = dL/dy: `fwd` holds the forward's arguments with its y and lse
 * (both required) and y_low (if the forward wrote it: dy . y is formed from both; without it from the rounded y).  dq, dk,
 * dv in the inputs' dtype, each rounded once from fp32 sums, summed in a fixed order (the same bits every time); every row is
 * written.  An infinity or NaN in a sequence's q, k, v or dy stays in that sequence's gradients, but may reach
 * those of rows that do not see it.  workspace: kdn_attn_bwd_workspace_bytes, 16-byte aligned. */
typedef struct kdn_attn_bwd_args {
  const kdn_attn_args* fwd;
  const void* dy; int64_t dy_stride[2];
  void* dq;       int64_t dq_stride[2];
  void* dk;       int64_t dk_stride[2];
  void* dv;       int64_t dv_stride[2];
  void* workspace; size_t workspace_bytes;
} kdn_attn_bwd_args;
size_t kdn_attn_bwd_workspace_bytes(const kdn_attn_bwd_args* a);   /* 0: invalid; reads sizes only */
int kdn_attn_bwd(const kdn_attn_bwd_args* a, void* stream);

/* ---- Rotary positions ------------------------------------------------------------------------------------------
 * Of each head's first `rotary_dim` values, pair j (j < rotary_dim / 2) at elements (2j, 2j + 1) (interleaved) or
 * (j, j + rotary_dim / 2) turns by the angle t = positions[token] * inv_freq[j]:
 * (a, b) -> magnitude (a cos t - b sin t, b cos t + a sin t); inverse turns by -t (the gradient).  The other values are
 * copied.  t is formed in 64 bits.  q and k in one launch; k NULL (H_kv 0): q alone.  The outputs may be the inputs. */
typedef struct kdn_rotary_args {
  int64_t tokens, H, H_kv;
  int d, rotary_dim, dtype, interleaved, inverse;
  float magnitude;
  const int64_t* positions;     /* device [tokens], |position| < 2^52 */
  const double* inv_freq;       /* device [rotary_dim / 2], radians a position */
  const void* q; int64_t q_stride[2];
  const void* k; int64_t k_stride[2];
  void* q_out;   int64_t q_out_stride[2];
  void* k_out;   int64_t k_out_stride[2];
} kdn_rotary_args;
int kdn_rotary(const kdn_rotary_args* a, void* stream);

/* ---- Pages ------------------------------------------------------------------------------------------------------
 * A cache is a slab of num_pages equal pages of page_tokens tokens (a power of two from 16 on).  Inside a page the caller
 * lays out what it likes (layers, keys and values); an operator takes base pointers and the strides [page][head][token]. */

/* Copies whole pages inside a slab: page pairs[2i] to page pairs[2i + 1] (host array, read before the call returns; no
 * device copy of it is made).  No page may be the target of two pairs, or the target of one and the source of another.
 * page_bytes a multiple of 16. */
int kdn_page_copy(void* slab, int64_t num_pages, int64_t page_bytes, const int32_t* pairs, int64_t n, void* stream);

/* Puts the keys and values of new tokens into their places: token i to row rows[i] % page_tokens of page
 * rows[i] / page_tokens.  A token whose row lies outside the slab (a negative one: padding) is skipped.  Rows distinct. */
typedef struct kdn_page_append_args {
  int64_t tokens, H_kv;
  int d, dtype;
  int64_t page_tokens, num_pages;
  const int64_t* rows;          /* device [tokens] */
  const void* k; int64_t k_stride[2];         /* [token][head] */
  const void* v; int64_t v_stride[2];
  void* k_pages; int64_t k_pages_stride[3];   /* [page][head][token] */
  void* v_pages; int64_t v_pages_stride[3];
} kdn_page_append_args;
int kdn_page_append(const kdn_page_append_args* a, void* stream);

/* Bookkeeping of the pages on the host, single-threaded per pool: which pages a stream's tokens lie on, shared by forks
 * and counted (hybrid_memory_pool.cpp:20-22, 86-135).  Nothing here touches the device: what has to be copied comes back
 * as pairs for kdn_page_copy.  Negative returns are kdn_status; a call that fails changes nothing. */
typedef struct kdn_page_pool kdn_page_pool;
int kdn_page_pool_create(int64_t num_pages, int64_t page_tokens, int64_t max_streams, kdn_page_pool** out);
void kdn_page_pool_destroy(kdn_page_pool* pool);
int kdn_page_pool_open(kdn_page_pool* pool);                      /* a new empty stream's number */
int kdn_page_pool_fork(kdn_page_pool* pool, int stream);          /* a new stream that shares all of `stream`'s pages */
int kdn_page_pool_close(kdn_page_pool* pool, int stream);         /* its pages are free once no stream has them */
/* Room for `tokens` more tokens of `stream`.  A partly filled last page that another stream shares is replaced by a page of
 * its own: then 1 is returned and pair[0..1] is the copy to make before anything is written; otherwise 0. */
int kdn_page_pool_extend(kdn_page_pool* pool, int stream, int64_t tokens, int32_t pair[2]);
int kdn_page_pool_truncate(kdn_page_pool* pool, int stream, int64_t tokens);   /* keeps the first `tokens` tokens */
int64_t kdn_page_pool_length(const kdn_page_pool* pool, int stream);           /* tokens */
/* The stream's page numbers into table[0 .. width): their count (KDN_ERR_CAPACITY if it is over width). */
int64_t kdn_page_pool_table(const kdn_page_pool* pool, int stream, int32_t* table, int64_t width);
/* rows[i] = where token first + i lies (page * page_tokens + place), for kdn_page_append. */
int kdn_page_pool_rows(const kdn_page_pool* pool, int stream, int64_t first, int64_t n, int64_t* rows);
/* Moves the pages in use to the lowest numbers: the moves as (from, to) into pairs[0 .. 2 * room), their count returned
 * (KDN_ERR_CAPACITY, and nothing moved, if they are more than room).  The caller makes the copies before anything else. */
int64_t kdn_page_pool_compact(kdn_page_pool* pool, int32_t* pairs, int64_t room);
int64_t kdn_page_pool_used(const kdn_page_pool* pool);            /* pages in use */
int64_t kdn_page_pool_free(const kdn_page_pool* pool);

/* ---- Attention of new tokens over the pages ---------------------------------------------------------------------
 * Sequence b has the new tokens cu_new[b] .. cu_new[b+1]-1 (at most max_new <= 64) behind a context of context_lens[b]
 * tokens, token j of which lies on page page_table[b][j / page_tokens].  New token t sees the whole context, itself, and
 * along its parents the new tokens it hangs on: parents[cu_new[b] + t] is a number below t, or negative for one that hangs
 * on the context (parents NULL: each hangs on the one before it).  k and v hold the new tokens' own keys and values, which
 * need not be in the pages.  Softmax and heads as kdn_attn_fwd.  max_context bounds the context lengths (longer ones are
 * cut) and sizes the grid; nothing is read back to the host.  Rows of y that no such token has are zeros: those before
 * cu_new[0], from cu_new[num_seqs] on (a step padded to a fixed size), and past max_new of a sequence.  At 16 bytes: every
 * row; workspace. */
typedef struct kdn_tree_attn_args {
  int64_t num_seqs, total_new, max_new, max_context;
  int64_t H, H_kv;
  int d, dtype;
  float scale;
  int64_t page_tokens, num_pages, table_width, table_stride;
  const int64_t* cu_new;        /* device [num_seqs + 1] */
  const int32_t* context_lens;  /* device [num_seqs] */
  const int32_t* page_table;    /* device [num_seqs][table_width], rows table_stride apart */
  const int32_t* parents;       /* device [total_new] or NULL */
  const void* q; int64_t q_stride[2];         /* [token][head] */
  const void* k; int64_t k_stride[2];
  const void* v; int64_t v_stride[2];
  const void* k_pages; int64_t k_pages_stride[3];
  const void* v_pages; int64_t v_pages_stride[3];
  void* y; int64_t y_stride[2];
  void* workspace; size_t workspace_bytes;
} kdn_tree_attn_args;
size_t kdn_tree_attn_workspace_bytes(const kdn_tree_attn_args* a);   /* 0: invalid; reads sizes only */
int kdn_tree_attn(const kdn_tree_attn_args* a, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* KDN_ANCHOR_H */
