/* MI355X token sampler: the steps between ids and logits (libd3sampler.so).
 *
 * What a caller needs around the draws (d3s_sampler.h) and the layers
 * (d3s_train.h): the verification of tokens that a smaller model drafted, the
 * rows that ids stand for and their gradient, the norm in front of a head or
 * a layer and its gradient, and dropout.
 * The conventions are those of d3s_train.h: plain pointers and sizes, every
 * array in device memory unless said otherwise, strides in elements between two
 * rows, `stream` a hipStream_t, calls that enqueue work and return a status
 * code (D3S_OK or D3S_ERR_*) before anything is launched, the *_ws forms for a
 * workspace that the caller sizes (*_workspace_bytes), clears once
 * (d3s_workspace_init) and passes to every call on one stream, the calls
 * without _ws for the block that the library keeps for the stream (while the
 * stream is being captured, calls without _ws that need a workspace return
 * D3S_ERR_WORKSPACE).  The same inputs give the same bits at every call.
 * Outputs may overlap inputs only where it is said. */
#ifndef D3S_STEP_H
#define D3S_STEP_H

#include "d3s_train.h"

#ifdef __cplusplus
extern "C" {
#endif

/* 8 bits: 4 of exponent, 3 of mantissa, greatest value 448, no infinity (outputs
 * of d3s_rms_norm only) */
#define D3S_DTYPE_E4M3 2

/* the most drafted tokens of a sequence, candidates of a row, ids of a row */
#define D3S_MAX_DRAFT 64
#define D3S_MAX_RANKED 1024
#define D3S_MAX_IDS 64

/* Verification of drafted tokens (speculative sampling), for each sequence b
 * with L = lengths[b] drafts x_0 .. x_{L-1} (lengths NULL: n_draft; clamped
 * to 0 .. n_draft) and
 *   p_i = softmax(target row b (n_draft + 1) + i / T),  i = 0 .. L,
 *   q_i = softmax(draft row b n_draft + i / Td),        i = 0 .. L - 1,
 * T = max(temperature, 1e-5), Td likewise, -inf logits masked.  draft NULL: the
 * drafts were certain, q_i is 1 at x_i and 0 elsewhere.
 *   Draft i is accepted if u_accept[b, i] q_i(x_i) < p_i(x_i) and all before it
 * were.  At the first that is not, a token is drawn from max(p_i - q_i, 0) (from
 * p_i where that is 0 everywhere); behind the last accepted one, from p_L.  So
 * the tokens are distributed as draws from the target alone.
 *   The draw from weights r_j is the least j with r_0 + .. + r_j > u_draw[b] Z, Z
 * their sum, all in 64 bits (the last j with r_j > 0 where rounding leaves none).
 * tokens [n_seqs, n_draft + 1]: the accepted drafts, the drawn token, then -1.
 * n_accepted [n_seqs].  accept [n_seqs, n_draft] (may be NULL): min(1,
 * p_i(x_i) / q_i(x_i)) for i < L, of all drafts and not the accepted only (q = 0:
 * 1 if p > 0, else 0), then 0.
 * A draft outside [0, vocab) has p = 0 and is never accepted.
 * Rows count only up to the token that is drawn: where one of them has a NaN or
 * +inf logit, or its sequence's temperature is not finite, the sequence ends there:
 * n_accepted as far, -1 in place of the token (accept is NaN for such a row wherever it
 * is).  A target row that is masked everywhere has p = 0, and 0 is drawn
 * from it.  counters: as d3s_sample's, the first two slots, one count a sequence. */
typedef struct {
  const void *target; /* [n_seqs (n_draft + 1), vocab] */
  int target_dtype;
  int64_t target_stride;
  const void *draft; /* [n_seqs n_draft, vocab], or NULL */
  int draft_dtype;
  int64_t draft_stride;
  int64_t n_seqs;
  int n_draft; /* 0 .. D3S_MAX_DRAFT */
  int64_t vocab;
  const int32_t *drafted;         /* [n_seqs, n_draft] */
  const int32_t *lengths;         /* [n_seqs], or NULL */
  const float *temperature;       /* [n_seqs], or NULL: the scalar */
  float temperature_scalar;
  const float *draft_temperature; /* the same of the draft model */
  float draft_temperature_scalar;
  const float *u_accept; /* [n_seqs, n_draft] in [0, 1) */
  const float *u_draw;   /* [n_seqs] in [0, 1) */
  int32_t *tokens;
  int32_t *n_accepted;
  float *accept;
  uint32_t *counters;
} d3s_verify_params;

int d3s_verify(const d3s_verify_params *params, void *stream);

/* Bytes of workspace d3s_verify_ws needs (0: none), or a negative status (the
 * pointers of params are not looked at). */
int64_t d3s_verify_workspace_bytes(const d3s_verify_params *params);

/* d3s_verify with the workspace given: never allocates, may be captured. */
int d3s_verify_ws(const d3s_verify_params *params, void *workspace, int64_t workspace_bytes, void *stream);

/* The same from ranked candidates, for models that draw with top_k and top_p:
 * target_cand and target_probs [n_seqs (n_draft + 1), target_k], draft_cand and
 * draft_probs [n_seqs n_draft, draft_k] are what d3s_sample writes to cand and
 * probs (a rank past the cut has probability 0; a candidate stands once in a row).
 * draft_cand and draft_probs both NULL: the drafts were certain.  The draw is
 * the sampler's race with u_draw [n_seqs, target_k]: the first greatest r_j /
 * -log(1 - u_j) over the ranks with r_j > 0, so that without drafts it is
 * d3s_sample's own (as there, -log(1 - 0) is -0: a rank with u_j = 0 is drawn only
 * where no other has r_j > 0).  Outputs and the rest as above; a row of d3s_sample's with
 * candidates -1 was refused, and one whose probabilities are NaN was masked. */
int d3s_verify_ranked(const int32_t *target_cand, const float *target_probs, int target_k, const int32_t *draft_cand,
                      const float *draft_probs, int draft_k, int64_t n_seqs, int n_draft, const int32_t *drafted,
                      const int32_t *lengths, const float *u_accept, const float *u_draw, int32_t *tokens,
                      int32_t *n_accepted, float *accept, uint32_t *counters, void *stream);

/* The rows that ids stand for: y[r] = scale * sum_t table[t slot_rows + ids[r, t]],
 * summed in fp32 in the order of t, rounded once.
 * ids [n_rows, n_ids], n_ids 1 .. D3S_MAX_IDS; an id outside [0, vocab) is none
 * and adds nothing.  slot_rows 0: one table of vocab rows for all; vocab or
 * more (less is D3S_ERR_ARG): the t-th id has a part of the table of its own.  table [.., width] and
 * y [n_rows, width] fp32 or bf16 each. */
int d3s_embed(const int32_t *ids, int64_t n_rows, int n_ids, const void *table, int dtype, int64_t table_stride,
              int64_t vocab, int64_t slot_rows, int64_t width, float scale, void *y, int y_dtype, int64_t y_stride,
              void *stream);

/* Its gradient in the table: grad[t slot_rows + v] = scale * the sum of dy[r] over
 * the ids[r, t] that are v, in fp32 in a fixed order, rounded once; with
 * accumulate not 0, added to what is there before the rounding, else rows that no id
 * names are zeros (those between two slots' parts too).  dy [n_rows, width], grad
 * [vocab (+ (n_ids - 1) slot_rows), width]; fp32 or bf16 each.  slot_rows is 0
 * or at least vocab; n_rows * n_ids at most 2^31 - 65536. */
int d3s_embed_backward(const int32_t *ids, int64_t n_rows, int n_ids, const void *dy, int dtype, int64_t dy_stride,
                       int64_t vocab, int64_t slot_rows, int64_t width, float scale, int accumulate, void *grad,
                       int grad_dtype, int64_t grad_stride, void *stream);
int64_t d3s_embed_backward_workspace_bytes(int64_t n_rows, int n_ids, int64_t vocab, int64_t slot_rows, int64_t width);
int d3s_embed_backward_ws(const int32_t *ids, int64_t n_rows, int n_ids, const void *dy, int dtype, int64_t dy_stride,
                          int64_t vocab, int64_t slot_rows, int64_t width, float scale, int accumulate, void *grad,
                          int grad_dtype, int64_t grad_stride, void *workspace, int64_t workspace_bytes, void *stream);

/* Root-mean-square norm: with h = x + residual (residual may be NULL: h = x),
 *   rstd[r] = 1 / sqrt(mean_j h[r, j]^2 + eps),  y = h rstd gain,
 * in fp32 (h is not rounded before), each output rounded once.  x, residual,
 * sum and gain [width] are of `dtype` (fp32 or bf16); gain may be NULL: 1.
 * sum [n_rows, width] receives h, for the residual path and the backward (it may
 * be NULL, or be x or residual themselves, with the same stride).
 * rstd [n_rows] fp32, may be NULL.
 * y_dtype D3S_DTYPE_F32 or _BF16 (y may be x or residual itself where types and
 * strides agree and sum is elsewhere), or D3S_DTYPE_E4M3: each `group`
 * elements of a row (32, 64, 128 or 256; 0: the whole row; the last group may be
 * shorter) share scales[r, g] = greatest |y| / 448, and y holds the fp32 quotient y / scale rounded to
 * the nearest 8 bits, so that q times scale stands for y.  A group of zeros has scale
 * 0 and zeros; one that holds a NaN or an infinity has scale NaN and NaNs. scales
 * [n_rows, ceil(width / group)] fp32 is needed then, and else not looked at.
 * eps >= 0; a row of zeros with eps 0 gives rstd +inf and NaN, as the formula does. */
int d3s_rms_norm(const void *x, int dtype, int64_t x_stride, const void *residual, int64_t residual_stride, void *sum,
                 int64_t sum_stride, const void *gain, float eps, int64_t n_rows, int64_t width, void *y, int y_dtype,
                 int64_t y_stride, int group, float *scales, float *rstd, void *stream);

/* Its gradient: with xhat = h rstd and a = dy gain,
 *   dx = rstd (a - xhat mean_j(a xhat)) + dsum   (x's and the residual's alike),
 *   dgain[j] = sum_r dy xhat   (fp32, before any rounding),
 * h and rstd what the forward call wrote (h: sum, or x without a residual), dsum the
 * gradient that reaches sum by another way, or NULL.  dy, h, gain, dsum and dx
 * are of `dtype`; gain NULL: 1.  dx may be dy, h or dsum itself, with the same stride,
 * or NULL; dgain may be NULL. */
int d3s_rms_norm_backward(const void *dy, int dtype, int64_t dy_stride, const void *h, int64_t h_stride,
                          const void *gain, const float *rstd, const void *dsum, int64_t dsum_stride, int64_t n_rows,
                          int64_t width, void *dx, int64_t dx_stride, float *dgain, void *stream);
int64_t d3s_rms_norm_backward_workspace_bytes(int64_t n_rows, int64_t width, int has_dgain);
int d3s_rms_norm_backward_ws(const void *dy, int dtype, int64_t dy_stride, const void *h, int64_t h_stride,
                             const void *gain, const float *rstd, const void *dsum, int64_t dsum_stride, int64_t n_rows,
                             int64_t width, void *dx, int64_t dx_stride, float *dgain, void *workspace,
                             int64_t workspace_bytes, void *stream);

/* Dropout: y[r, j] = residual[r, j] + (u >= p ? x[r, j] / (1 - p) : 0), u the uniform
 * number r width + j of draw `draw` (plus *draw_add, a device counter, if it is
 * not NULL: so that a captured call drops other elements at every replay) under
 * `seed`, as d3s_uniform_fill writes it.  No mask is stored: the gradient is the
 * same call on dy, with the same p, seed and draw and no residual.  p in [0, 1];
 * p = 1 drops everything.  A dropped element is 0 whatever x holds.  x,
 * residual (may be NULL) and y are of `dtype`; computed in fp32, rounded once.  y may
 * be x or residual itself, with the same stride. */
int d3s_dropout(const void *x, int dtype, int64_t x_stride, const void *residual, int64_t residual_stride,
                int64_t n_rows, int64_t width, float p, uint64_t seed, uint64_t draw, const uint64_t *draw_add, void *y,
                int64_t y_stride, void *stream);

#ifdef __cplusplus
}
#endif

#endif
