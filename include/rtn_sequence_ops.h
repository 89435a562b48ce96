/*
 * C ABI of the MI355X (gfx950) operators around the recurrent layers (librtn_sequence_ops.so): a gated linear
 * recurrence, dropout from a counter, and log probabilities of tokens.
 *
 * As in rtn_native_lstm2.h: plain pointers and sizes; all data pointers are DEVICE pointers on the current HIP device,
 * aligned to their element type; `hip_stream` is a hipStream_t (NULL = the default stream).  Every entry only enqueues
 * work on that stream: no device synchronisation, no allocation (scratch comes in through `workspace`, 16-byte aligned,
 * whose contents are neither expected nor kept), inputs are never written, outputs are caller-allocated and fully
 * overwritten.  All entries can be recorded into a HIP graph.  Nothing is enqueued where a status other than RTN_OK is
 * returned for a reason that the host can see; sizes whose launch would have 2^32 threads or more are such a reason (RTN_ERR_SHAPE).
 */
#ifndef RTN_SEQUENCE_OPS_H
#define RTN_SEQUENCE_OPS_H

#include <stddef.h>
#include <stdint.h>

#include "rtn_native_lstm2.h" /* status codes and element types */

#ifdef __cplusplus
extern "C" {
#endif

/* ABI version of this header: 1. */
int rtn_sequence_ops_abi_version(void);

/* Text of the last error of the calling thread ("" if its last call succeeded). */
const char* rtn_sequence_last_error(void);

/*
 * Gated linear recurrence: NativeLstm2's gates without its recurrent product.
 *
 *   c_t = sigmoid(f_t) c_{t-1} + sigmoid(i_t) tanh(z_t),   y_t = sigmoid(o_t) c_t
 *
 * X     [T,B,4n] gates before their activation, along the last axis z (cell-in), i (input), f (forget), o (output);
 *       row (t,b) starts at element (t*B+b)*ldX (0: 4n)
 * c0    [B,n] float32 state before the first frame; NULL: zeros
 * lens  [B] frames per sequence (clamped to 0..T); NULL: T each.  Frames past them are not read: Y is 0 there and the
 *       state stays.  direction -1: from each sequence's last frame to its first.
 * Y     [T,B,n] in X's type; cN [B,n] float32, the state after the last frame visited
 * saved what the gradient wants to know (rtn_gated_recurrence_saved_bytes), or NULL
 * The state is float32 throughout, whatever the type.  T up to 2^30, n up to 2^26.
 */
size_t rtn_gated_recurrence_saved_bytes(int64_t T, int32_t B, int32_t n, int32_t dtype);
size_t rtn_gated_recurrence_fwd_workspace_bytes(int64_t T, int32_t B, int32_t n, int32_t dtype);
int rtn_gated_recurrence_fwd(const void* X, int64_t ldX, const float* c0, const int64_t* lens, void* Y, float* cN, void* saved, int64_t T, int32_t B, int32_t n,
                             int32_t dtype, int32_t direction, void* workspace, size_t workspace_bytes, void* hip_stream);

/*
 * Its gradient.  DY [T,B,n] (rows ldDY elements apart, 0: n) in X's type, not read past a sequence's length; DcN [B,n]
 * float32 or NULL (zero).  DX [T,B,4n] contiguous, 0 past a sequence's length; Dc0 [B,n] float32.
 * `saved` is what the forward call with the same X, lens, direction left, in which its c0 is held: c0 is not read here and may be NULL.
 */
size_t rtn_gated_recurrence_bwd_workspace_bytes(int64_t T, int32_t B, int32_t n, int32_t dtype);
int rtn_gated_recurrence_bwd(const void* X, int64_t ldX, const float* c0, const int64_t* lens, const void* saved, const void* DY, int64_t ldDY, const float* DcN,
                             void* DX, float* Dc0, int64_t T, int32_t B, int32_t n, int32_t dtype, int32_t direction, void* workspace, size_t workspace_bytes,
                             void* hip_stream);

/*
 * Dropout whose mask is a function of (seed, offset, index), never stored:
 *
 *   y = keep(e) ? x * 65536 / (65536 - threshold) : 0,   plus the residual where there is one
 *
 * keep(e): the 16-bit draw of element e is at least `threshold` (0..65536: the drop probability times 65536).  The draws
 * of the elements 8g..8g+7 are the 16-bit halves, the lower one first, of the four words of Philox4x32-10 (Salmon,
 * Moraes, Dror, Shaw 2011) with key (seed low, seed high) and counter (g low, g high, offset low, offset high).
 * x     [times,rows,width], row r of time t at element (t*rows+r)*ldx (0: width); y contiguous; `residual` [times,rows,width]
 *       with ldr, or NULL
 * e     (t*rows + r)*width + column, or, where `same_over_time` is not 0, r*width + column
 * offset_ptr: one int64 on the device that is added to `offset`, or NULL.  (A recorded call draws anew at each replay.)
 * The gradient with respect to x is this call on the error of y without a residual; that of the residual is the error itself.
 */
int rtn_dropout(const void* x, int64_t ldx, const void* residual, int64_t ldr, void* y, int64_t times, int64_t rows, int64_t width, int32_t dtype, int32_t threshold,
                uint64_t seed, uint64_t offset, const int64_t* offset_ptr, int32_t same_over_time, void* hip_stream);

/*
 * Log probabilities under softmax over the last axis.
 *
 * logits  [rows,V], row r at element r*ld (0: V); V up to 2^26
 * targets [rows] token per row, or NULL (no log_prob; every row counts).  A negative target marks a row without a token:
 *         it is not read, log_prob and entropy are 0, the alternatives -inf with index -1, its gradient 0.
 *         A target of V or more gives a log_prob of NaN and a row of NaN as gradient.
 * log_prob [rows] = logits[target] - lse, entropy [rows] = -sum p log p
 * norm    [rows,2] the two parts of lse = log sum exp: a reference m, which is the largest logit or at most 22 below it, and log sum exp(logits - m).
 *         (One number would round away what the gradient needs where logits are large.)
 * top_log_prob, top_ids [rows,top_k]: the top_k largest logits of a row in descending order, among equal ones the lower index
 *         first, a NaN before everything; as log probabilities and indices.  0 <= top_k <= min(64, V).
 * All in float32, indices int64.  entropy, log_prob, norm: NULL if not wanted.  A logit of -inf has probability 0 and adds nothing;
 * a row of nothing else has every log probability -inf, entropy 0 and gradient 0.
 */
size_t rtn_token_log_probs_workspace_bytes(int64_t rows, int64_t V, int32_t dtype, int32_t top_k);
int rtn_token_log_probs_fwd(const void* logits, int64_t ld, const int64_t* targets, int64_t rows, int64_t V, int32_t dtype, int32_t top_k, float* log_prob, float* norm,
                            float* entropy, float* top_log_prob, int64_t* top_ids, void* workspace, size_t workspace_bytes, void* hip_stream);

/*
 * Gradient of sum_r d_log_prob[r] log_prob[r] + d_entropy[r] entropy[r] with respect to the logits:
 *
 *   D[r,v] = d_log_prob[r] (1[v = target] - p_v) - d_entropy[r] p_v (log p_v + entropy[r])
 *
 * norm and entropy as the forward call wrote them; d_log_prob (needs targets), d_entropy (needs entropy): NULL for zero.
 * D [rows,V], contiguous, in the type of the logits.
 */
int rtn_token_log_probs_bwd(const void* logits, int64_t ld, const int64_t* targets, const float* norm, const float* entropy, const float* d_log_prob, const float* d_entropy,
                            void* D, int64_t rows, int64_t V, int32_t dtype, void* hip_stream);

#ifdef __cplusplus
}
#endif
#endif /* RTN_SEQUENCE_OPS_H */
