/*
 * fa2_b200_lm — C ABI of the operators for language models that stand beside fa2_fwd / fa2_bwd:
 * attention with changed scores (tanh cap, distance bias) under document and prefix masks, forward
 * and backward, and attention over a paged key/value cache with the calls that feed it.
 *
 * The conventions are those of fa2_b200.h: device pointers owned by the caller, element strides, a
 * stream, a negative fa2_status and a message in fa2_last_error on failure, nothing allocated, nothing
 * synchronised. None of these calls has a counterpart in the reference.
 */
#ifndef FA2_B200_LM_H_
#define FA2_B200_LM_H_

#include "fa2_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Version of this header (major * 1000 + minor), apart from that of fa2_b200.h. */
#define FA2_LM_ABI_VERSION 1001
int fa2_lm_version(void);

/* ---------------------------------------------------------------------------------------------
 * Attention with changed scores
 *   s = softmax_scale * q.k ;  s <- softcap * tanh(s / softcap) ;  s <- s - slope_h * |i + Sk - Sq - j|
 * Query i sees key j iff all that is given holds:
 *   causal   : j <= i + Sk - Sq, or j < prefix_lens[b]
 *   documents: i and j belong to the same document. A document is a run of equal ids; tokens with a
 *              negative id are padding, they see nothing and are seen by nothing.
 * A query that sees nothing gets zeros (lse -inf) and no gradient. Values of q, k, v and d_o must be
 * finite, in masked places and padding too: a masked weight is an exact 0, and 0 * inf is NaN.
 * ------------------------------------------------------------------------------------------- */
typedef struct {
  float softcap;               /* 0: none; else in [2^-10, 1024]                                 */
  const float* alibi_slopes;   /* float32 [heads_q] on the device, or NULL; takes no gradient    */
  const int32_t* prefix_lens;  /* int32 [batch] on the device, or NULL; needs causal             */
  const int32_t* document_layout;   /* what fa2_document_layout wrote, or NULL; needs Sq == Sk   */
  /* [batch, seqlen_q, heads_q, head_dim] in the q dtype, or NULL: the forward writes there what rounding o
   * to 16 bits dropped, the backward adds it to o where it forms rowsum(o * d_o). In bf16 that rounding is
   * the largest part of the gradients' error where single keys dominate; fp16 does not need it.         */
  void* o_rest;
  fa2_strides o_rest_strides;
} fa2_score_mod;

/* Bytes of the layout of `batch` rows of `seqlen` document ids. */
size_t fa2_document_layout_bytes(int32_t batch, int32_t seqlen);

/* Reads document ids (int32, rows `stride_b` elements apart) and writes the layout that the two calls
 * below take: for every token the first and one past the last token of its document, the same over
 * every 128 tokens, and an order of work. `layout`: 16-byte aligned, fa2_document_layout_bytes. One layout serves the forward
 * and backward calls of every layer that works on these rows. */
int fa2_document_layout(const int32_t* document_ids, int64_t stride_b, int32_t batch, int32_t seqlen,
                        int32_t* layout, size_t layout_bytes, void* cuda_stream);

/* fa2_fwd / fa2_bwd with changed scores. The parameter blocks are those of fa2_b200.h without bias,
 * mask, dropout, seqlens, dbias and dropout_bits (refused); softmax_scale must be positive;
 * fa2_fwd_workspace_bytes sizes the scratch of the forward. The backward needs fa2_bwd_workspace_bytes; with
 * fa2_scored_bwd_workspace_bytes it may deal the query heads of a key/value head to several SMs where there are few tiles
 * (dk and dv are the same from call to call either way, but not between the two). Both depend on the current device's
 * number of SMs. */
int fa2_scored_fwd(const fa2_fwd_params* params, const fa2_score_mod* mod, void* cuda_stream);
size_t fa2_scored_bwd_workspace_bytes(const fa2_problem* problem);
int fa2_scored_bwd(const fa2_bwd_params* params, const fa2_score_mod* mod, void* cuda_stream);

/* ---------------------------------------------------------------------------------------------
 * Serving with a paged key/value cache
 *   k_cache, v_cache: [pages][page_size][heads_kv][head_dim], any strides in multiples of 8 elements;
 *   page_size a power of two from 8 to 2^20. A slot is page * page_size + place in the page. A request's
 *   row of the block table holds its pages in order. The new tokens of all requests lie one behind the
 *   other in packed tensors of num_tokens rows; rows behind the last request are left alone.
 * ------------------------------------------------------------------------------------------- */
typedef struct {
  const int32_t* context_lens;  /* [requests] tokens in the cache; below 0 counts as 0             */
  const int32_t* new_lens;      /* [requests] new tokens, 0 allowed; those beyond num_tokens are cut */
  int32_t requests;             /* 1 .. 8192                                                       */
  int32_t* block_table;         /* [requests][table_width], updated: new pages are entered         */
  int64_t table_stride;         /* elements between its rows                                       */
  int32_t table_width;
  const int32_t* free_pages;    /* [n_free] pages to take from, in this order                      */
  int32_t n_free;
  const int32_t* free_start;    /* one int32 on the device, or NULL (0): entries already taken     */
  int32_t page_size, num_tokens;
  int32_t heads_q, heads_kv;    /* of the attention that will use the work list                    */
  int32_t* cu_seqlens;          /* out [requests + 1]: first row of every request                  */
  int32_t* seqlens_k;           /* out [requests]: tokens in the cache with the new ones           */
  int64_t* slot_map;            /* out [num_tokens]: slot of every new token; -1 behind the last request
                                   and where no page was left                                      */
  int32_t* positions;           /* out [num_tokens]; 0 behind the last request                     */
  int32_t* pages_taken;         /* out [1]: entries of free_pages that this step needs; more than there
                                   are: the pages that were missing are -1 in the table            */
  int32_t* work;                /* out: work list of fa2_paged_attention, 16-byte aligned          */
  size_t work_bytes;            /* at least fa2_paged_work_bytes                                   */
} fa2_paged_plan_params;

/* Depends, like the plan itself, on the current device's number of SMs. */
size_t fa2_paged_work_bytes(int32_t requests, int32_t num_tokens, int32_t heads_q, int32_t heads_kv);
int fa2_paged_plan(const fa2_paged_plan_params* params, void* cuda_stream);

typedef struct {
  const void* ptr;
  int64_t stride_page, stride_slot, stride_head;
} fa2_paged_cache;

/* Writes the keys and values of new tokens, [tokens][heads][head_dim] with 16-bit elements of any type, to
 * their slots. Slots outside the cache (-1) are skipped; slots must not occur twice (the slot then holds
 * pieces of either row). Pointers 16-byte aligned, strides and head_dim multiples of 8. */
typedef struct {
  const void* k; int64_t k_stride_t, k_stride_h;
  const void* v; int64_t v_stride_t, v_stride_h;
  fa2_paged_cache k_cache, v_cache;
  const int64_t* slot_map;
  int32_t tokens, heads, head_dim, pages, page_size;
} fa2_paged_write_params;

int fa2_paged_cache_write(const fa2_paged_write_params* params, void* cuda_stream);

/* Attention of the packed new tokens over the cache that holds their keys and values already: token i of
 * request b, at position p = context + i, sees the keys 0 .. p. head_dim up to 128, heads_q / heads_kv up
 * to 128. `work` comes from fa2_paged_plan with the same requests, tokens, heads, page size and table.
 * Entries of the table outside the pool read as zeros; what lies in the pages behind a request's last key
 * is ignored, NaN included. */
typedef struct {
  const void* q; int64_t q_stride_t, q_stride_h;      /* [tokens][heads_q][head_dim]              */
  void* o; int64_t o_stride_t, o_stride_h;
  float* lse;                                          /* [tokens][heads_q] natural log, or NULL   */
  fa2_paged_cache k_cache, v_cache;
  int32_t tokens, heads_q, heads_kv, head_dim, dtype, pages, page_size;
  const int32_t* block_table; int64_t table_stride; int32_t table_width, requests;
  const int32_t* work;
  float softmax_scale;                                 /* positive                                 */
  float softcap;                                       /* as in fa2_score_mod                      */
  const float* alibi_slopes;
  void* workspace; size_t workspace_bytes;             /* fa2_paged_workspace_bytes, 128-byte aligned */
} fa2_paged_attention_params;

/* Depends on the current device's number of SMs. */
size_t fa2_paged_workspace_bytes(int32_t head_dim);
int fa2_paged_attention(const fa2_paged_attention_params* params, void* cuda_stream);

#ifdef __cplusplus
}
#endif
#endif /* FA2_B200_LM_H_ */
