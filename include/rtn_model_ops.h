/*
 * C ABI of the MI355X (gfx950) operators of whole language models (librtn_model_ops.so): the gated delta rule, an embedding
 * table, and a step of beam search.
 *
 * As in rtn_sequence_ops.h: plain pointers and sizes; all data pointers are DEVICE pointers on the current HIP device (but for
 * the lists of rtn_reorder_rows), aligned to their element type; `hip_stream` is a hipStream_t (NULL = the default stream).
 * Every entry only enqueues work on that stream: no device synchronisation, no allocation (scratch comes in through
 * `workspace`, 16-byte aligned, whose contents are neither expected nor kept), inputs are never written, outputs are
 * caller-allocated, overlap nothing and are fully overwritten.  All entries can be recorded into a HIP graph.  Nothing is
 * enqueued where a status other than RTN_OK is returned for a reason that the host can see.
 */
#ifndef RTN_MODEL_OPS_H
#define RTN_MODEL_OPS_H

#include <stddef.h>
#include <stdint.h>

#include "rtn_native_lstm2.h" /* status codes and element types */

#ifdef __cplusplus
extern "C" {
#endif

/* ABI version of this header: 1. */
int rtn_model_ops_abi_version(void);

/* Text of the last error of the calling thread ("" if its last call succeeded). */
const char* rtn_model_ops_last_error(void);

/*
 * Gated delta rule.  Each head has a state S [dk,dv]; with a_t = exp(g_t)
 *
 *   S_t = a_t S_{t-1} + k_t u_t^T,   u_t = beta_t (v_t - a_t S_{t-1}^T k_t),   y_t = scale S_t^T q_t
 *
 * q, k   [T,B,key_heads,dk], v [T,B,heads,dv]; row (t,b) starts at element (t*B+b)*ld (0: contiguous).  heads is a multiple of key_heads,
 *        heads / key_heads neighbouring heads share queries and keys.  1 <= dk <= 128, 1 <= dv <= 65536, T up to 2^30.  Beyond 16 frames, and with a
 *        gradient, a frame of all sequences (B*ld elements) is at most 64 MiB (RTN_ERR_SHAPE).
 * g, beta [T,B,heads] float32; g is at most 0 (log of the decay; minus infinity forgets everything before)
 * s0     [B,heads,dk,dv] float32 state before the first frame; NULL: zeros
 * lens   [B] frames per sequence (clamped to 0..T); NULL: T each.  Frames past them are not read: y is 0 there and the state stays.
 *        direction -1: from each sequence's last frame to its first.
 * y      [T,B,heads,dv] in the type of q, k and v; sN [B,heads,dk,dv] float32, the state behind the last frame visited
 * saved  what the gradient wants to know (rtn_delta_rule_saved_bytes), or NULL
 * A number that is not finite (or of float32 and above 3.38e38, the largest of bfloat16) in a frame that there is spoils the outputs of its head from its chunk of 64 frames (float32: 32) on,
 *        not from its own frame on.  (Up to 16 frames without `saved` go frame by frame, where it does so from its own on.)
 */
size_t rtn_delta_rule_fwd_workspace_bytes(int64_t T, int32_t B, int32_t key_heads, int32_t heads, int32_t dk, int32_t dv, int32_t dtype, int32_t keep);
size_t rtn_delta_rule_saved_bytes(int64_t T, int32_t B, int32_t key_heads, int32_t heads, int32_t dk, int32_t dv, int32_t dtype);
int rtn_delta_rule_fwd(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, const float* g, const float* beta, const float* s0,
                       const int64_t* lens, void* y, float* sN, void* saved, int64_t T, int32_t B, int32_t key_heads, int32_t heads, int32_t dk, int32_t dv,
                       int32_t dtype, float scale, int32_t direction, void* workspace, size_t workspace_bytes, void* hip_stream);

/*
 * Its gradient.  dy [T,B,heads,dv] (rows lddy elements apart, 0: contiguous), not read past a sequence's length; dsN [B,heads,dk,dv] float32 or NULL (zero).
 * dq, dk_out [T,B,key_heads,dk], dv_out [T,B,heads,dv] contiguous, in the type of q, k and v; dg, dbeta [T,B,heads], ds0 [B,heads,dk,dv] float32; all but ds0 are 0 past a
 * sequence's length.  `saved` is what the forward call with the same q, k, v, g, beta, s0, lens and direction left.  Heads that share queries and keys are
 * added in their order; without any (heads = 0) the gradients of queries and keys are 0.
 */
size_t rtn_delta_rule_bwd_workspace_bytes(int64_t T, int32_t B, int32_t key_heads, int32_t heads, int32_t dk, int32_t dv, int32_t dtype);
int rtn_delta_rule_bwd(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, const float* g, const float* beta, const int64_t* lens,
                       const void* saved, const void* dy, int64_t lddy, const float* dsN, void* dq, void* dk_out, void* dv_out, float* dg, float* dbeta, float* ds0,
                       int64_t T, int32_t B, int32_t key_heads, int32_t heads, int32_t dk, int32_t dv, int32_t dtype, float scale, int32_t direction, void* workspace,
                       size_t workspace_bytes, void* hip_stream);

/*
 * Rows of a table: y[r] = scale table[tokens[r]].
 *
 * tokens [rows]; a negative one marks a row without a token: y is 0 there.  One of V or more makes its row NaN.
 * table  [V,D], row v at element v*ld (0: D); y [rows,D] contiguous.  rows below 2^31, V below 2^31.
 */
int rtn_embedding_fwd(const int64_t* tokens, const void* table, int64_t ld, void* y, int64_t rows, int64_t V, int64_t D, int32_t dtype, float scale, void* hip_stream);

/*
 * Its gradient: Dtable[v] = scale * the sum of dy[r] over the rows of token v, in float32: these rows are added in the order of r in blocks of 8, 16 or 32 (by rows and D), and
 * the blocks' sums in order.  So the rows of other tokens have no part in how they are added.
 * dy [rows,D] (rows ld elements apart, 0: D), not read where there is no token of the table; Dtable [V,D] contiguous.
 */
size_t rtn_embedding_bwd_workspace_bytes(int64_t rows, int64_t V, int64_t D, int32_t dtype);
int rtn_embedding_bwd(const int64_t* tokens, const void* dy, int64_t ld, void* Dtable, int64_t rows, int64_t V, int64_t D, int32_t dtype, float scale, void* workspace,
                      size_t workspace_bytes, void* hip_stream);

/*
 * The best continuations of a batch of searches.
 *
 *   joint[b,k,v] = totals[b,k] + scores[b,k,v]   (one addition, rounded to float32)
 *
 * scores [B,K,V], row (b,k) at element (b*K+k)*ld (0: V); totals [B,K] float32
 * ended  [B,K] (0 or not), or NULL: the scores of a hypothesis that has ended are taken as 0 for v = end_token and -inf for all others, and not
 *        read.  end_token in 0..V-1 where `ended` is not NULL.
 * out_totals, sources, tokens [B,beam]: joint, k and v of the `beam` largest of a search in descending order, among equal ones the lowest k first and
 *        among those the lowest v; a NaN before everything.  1 <= beam <= min(64, K V), V up to 2^26, K V below 2^31, and B K pieces of a hypothesis'
 *        scores (of 8192 at least) below 2^22 (else RTN_ERR_SHAPE).
 */
size_t rtn_beam_select_workspace_bytes(int32_t B, int32_t K, int64_t V, int32_t dtype, int32_t beam);
int rtn_beam_select(const void* scores, int64_t ld, const float* totals, const uint8_t* ended, int64_t end_token, float* out_totals, int64_t* sources, int64_t* tokens,
                    int32_t B, int32_t K, int64_t V, int32_t dtype, int32_t beam, void* workspace, size_t workspace_bytes, void* hip_stream);

/*
 * Rows of several tensors by their source: out[n][b,j] = in[n][b,sources[b,j]], rows of row_bytes[n] bytes.
 *
 * in, out, row_bytes: lists of `count` on the HOST, read before the call returns; in[n] [B,K] rows, out[n] [B,beam] rows, at any address.
 * A source that is not in 0..K-1 gives a row of zero bytes.
 */
int rtn_reorder_rows(int32_t count, const void* const* in, void* const* out, const int64_t* row_bytes, const int64_t* sources, int32_t B, int32_t K, int32_t beam,
                     void* hip_stream);

#ifdef __cplusplus
}
#endif
#endif /* RTN_MODEL_OPS_H */
