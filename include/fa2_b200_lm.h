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
#define FA2_LM_ABI_VERSION 1000
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
} fa2_score_mod;

/* Bytes of the layout of `batch` rows of `seqlen` document ids. */
size_t fa2_document_layout_bytes(int32_t batch, int32_t seqlen);

/* Reads document ids (int32, rows `stride_b` elements apart) and writes the layout that the two calls
 * below take: for every token the first and one past the last token of its document, and the same over
 * every 128 tokens. `layout`: 16-byte aligned, fa2_document_layout_bytes. One layout serves the forward
 * and backward calls of every layer that works on these rows. */
int fa2_document_layout(const int32_t* document_ids, int64_t stride_b, int32_t batch, int32_t seqlen,
                        int32_t* layout, size_t layout_bytes, void* cuda_stream);

/* fa2_fwd / fa2_bwd with changed scores. The parameter blocks are those of fa2_b200.h without bias,
 * mask, dropout, seqlens, dbias and dropout_bits (refused); softmax_scale must be positive;
 * fa2_fwd_workspace_bytes / fa2_bwd_workspace_bytes size the scratch. */
int fa2_scored_fwd(const fa2_fwd_params* params, const fa2_score_mod* mod, void* cuda_stream);
int fa2_scored_bwd(const fa2_bwd_params* params, const fa2_score_mod* mod, void* cuda_stream);

#ifdef __cplusplus
}
#endif
#endif /* FA2_B200_LM_H_ */
