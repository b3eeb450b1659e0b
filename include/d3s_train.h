/* MI355X token sampler: scoring and training operators (libd3sampler.so).
 *
 * What a caller needs next to a draw (d3s_sampler.h): the log probability of
 * the tokens that were drawn or given, the gradient of a loss on them, the
 * layers that make the logits at matrix-core rate with their gradients, and
 * the global norm of a set of gradients with clipping.
 * The conventions are those of d3s_sampler.h: plain pointers and sizes, every
 * array in device memory unless said otherwise, `stream` a hipStream_t, calls
 * that enqueue work and return a status code (D3S_OK or D3S_ERR_*) before
 * anything is launched, the *_ws forms for a workspace that the caller sizes
 * (*_workspace_bytes), clears once (d3s_workspace_init) and passes to every
 * call on one stream, the calls without _ws for the block that the library
 * keeps for the stream (while the stream is being captured, calls without _ws
 * that need a workspace return D3S_ERR_WORKSPACE).  The same inputs give the same bits at every call: no
 * result depends on the order in which workgroups end. */
#ifndef D3S_TRAIN_H
#define D3S_TRAIN_H

#include "d3s_sampler.h"

#ifdef __cplusplus
extern "C" {
#endif

/* the most given tokens and alternatives of a row */
#define D3S_MAX_TOKENS 64
#define D3S_MAX_TOP 64

/* Log probabilities of given tokens, entropy and the best alternatives, for
 * each row of logits [n_rows, vocab] (fp32 or bf16, row r at logits + r *
 * row_stride elements).  Per row, with T = max(temperature, 1e-5), the banned
 * index set to -inf and -inf logits masked:
 *   m = the greatest logit, S = sum_j exp((l_j - m) / T),
 *   logprobs[r, t] = (l_token - m) / T - log S,
 *   entropy[r] = -sum_j p_j log p_j,  p_j = exp((l_j - m) / T) / S,
 *   row_stats[r] = { m, log S }   (the row's log-sum-exp is m / T + log S),
 *   top_ids[r, i], top_logprobs[r, i]: the i-th greatest logit's index and log
 *   probability, ties to the lowest index, masked ones last.
 * Sums are held in fp32.
 * temperature: per-row array [n_rows], or NULL for temperature_scalar.  banned:
 * a per-row index (any value outside [0, vocab): none), or NULL.  tokens
 * [n_rows, n_tokens], n_tokens 0 .. D3S_MAX_TOKENS; a token outside [0, vocab)
 * is none: its log probability is 0.  A masked token's is -inf.  n_top 0 ..
 * min(D3S_MAX_TOP, vocab).  logprobs (with n_tokens), entropy, row_stats
 * [n_rows, 2] and top_ids / top_logprobs [n_rows, n_top] may each be NULL.
 * counters: as d3s_sample's, the first two slots.
 * A row with a NaN or +inf logit, or a temperature that is not finite (-infinity
 * too, which a draw takes as 1e-5), is refused: every number NaN (log
 * probabilities of no token too), top_ids -1.
 * A row whose logits are all masked has log probabilities -inf (0 for no
 * token), entropy 0, row_stats -inf and top_ids 0, 1, ... */
int d3s_logprob(const void *logits, int dtype, int64_t n_rows, int64_t vocab, int64_t row_stride,
                const float *temperature, float temperature_scalar, const int32_t *banned, const int32_t *tokens,
                int n_tokens, float *logprobs, float *entropy, float *row_stats, int n_top, int32_t *top_ids,
                float *top_logprobs, uint32_t *counters, void *stream);

/* Bytes of workspace d3s_logprob_ws needs (0: none), with n_top alternatives or
 * with top_ids and top_logprobs both NULL, or a negative status. */
int64_t d3s_logprob_workspace_bytes(int dtype, int64_t n_rows, int64_t vocab, int n_top);

/* d3s_logprob with the workspace given: never allocates, may be captured. */
int d3s_logprob_ws(const void *logits, int dtype, int64_t n_rows, int64_t vocab, int64_t row_stride,
                   const float *temperature, float temperature_scalar, const int32_t *banned, const int32_t *tokens,
                   int n_tokens, float *logprobs, float *entropy, float *row_stats, int n_top, int32_t *top_ids,
                   float *top_logprobs, uint32_t *counters, void *workspace, int64_t workspace_bytes, void *stream);

/* The gradient of sum_r ( sum_t grad_logprobs[r, t] logprobs[r, t] +
 * grad_entropy[r] entropy[r] ) in the logits:
 *   grad_logits[r, j] = (1 / T) [ sum_t g_t (1{j = token_t} - p_j)
 *                                 - g_H p_j (log p_j + entropy) ],
 * 0 at masked places, in the logits' type (rows grad_row_stride elements
 * apart; computed in fp32, rounded once).  row_stats and entropy are what
 * d3s_logprob wrote (entropy may be NULL with grad_entropy NULL).  Tokens that
 * are none have no gradient; a token given twice has both.  A row all of whose
 * gradients are 0 gets zeros whatever it holds; any other refused row gets
 * NaN (0 at masked places).  grad_logits may be logits itself (with the same row stride), else the
 * two must not overlap.  Needs no workspace. */
int d3s_logprob_backward(const void *logits, int dtype, int64_t n_rows, int64_t vocab, int64_t row_stride,
                         const float *temperature, float temperature_scalar, const int32_t *banned,
                         const int32_t *tokens, int n_tokens, const float *row_stats, const float *entropy,
                         const float *grad_logprobs, const float *grad_entropy, void *grad_logits,
                         int64_t grad_row_stride, void *stream);

/* activations of a dense layer */
#define D3S_ACT_NONE 0
#define D3S_ACT_RELU 1
#define D3S_ACT_SILU 2      /* z / (1 + exp(-z)) */
#define D3S_ACT_GELU 3      /* z (1 + erf(z / sqrt 2)) / 2 */
#define D3S_ACT_GELU_TANH 4 /* z (1 + tanh(sqrt(2 / pi) (z + 0.044715 z^3))) / 2 */

/* A dense layer's operands: y [m, n] = residual + act(x w^T + bias), x [m, k]
 * and w [n, k] bf16, sums in fp32, rounded once.
 * x_transposed: x is stored [k, m]; w_transposed: w is stored [k, n].  So the
 * gradients are the same call: dx [m, k'] = dz w (w_transposed, inner length
 * n), dw [n, k'] = dz^T x (both transposed, inner length m).
 * Strides are in elements between two stored rows.  bias [n] bf16, residual
 * [m, n] of y's type (it may be y itself, with y's stride: sums over
 * micro-batches) and z [m, n] bf16 (the pre-activation x w^T + bias, kept for the
 * backward) may be NULL.
 * No other output may overlap an input.  y_dtype D3S_DTYPE_F32 or
 * D3S_DTYPE_BF16.  m, n, k from 0 up to 2^31 - 1024; k = 0 sums nothing. */
typedef struct {
  const uint16_t *x;
  int64_t x_stride;
  int x_transposed;
  const uint16_t *w;
  int64_t w_stride;
  int w_transposed;
  int64_t m, n, k;
  const uint16_t *bias;
  int activation;
  const void *residual;
  int64_t residual_stride;
  uint16_t *z;
  int64_t z_stride;
  void *y;
  int64_t y_stride;
  int y_dtype;
} d3s_dense_params;

int d3s_dense_bf16(const d3s_dense_params *params, void *stream);

/* Bytes of workspace d3s_dense_bf16_ws needs (0: none), or a negative status
 * (the pointers of params are not looked at). */
int64_t d3s_dense_workspace_bytes(const d3s_dense_params *params);

/* d3s_dense_bf16 with the workspace given: never allocates, may be captured. */
int d3s_dense_bf16_ws(const d3s_dense_params *params, void *workspace, int64_t workspace_bytes, void *stream);

/* The gradient through a dense layer's epilogue: dz [m, n] = dy act'(z) (bf16,
 * rounded once; it may be dy itself, with dy's stride, or NULL) and dbias[n] =
 * the column sums of dy act'(z) in fp32, before the rounding (may be NULL).  z may
 * be NULL with D3S_ACT_NONE. */
int d3s_dense_activation_backward_bf16(const uint16_t *dy, int64_t dy_stride, const uint16_t *z, int64_t z_stride,
                                       int64_t m, int64_t n, int activation, uint16_t *dz, int64_t dz_stride,
                                       float *dbias, void *stream);
int64_t d3s_dense_activation_backward_workspace_bytes(int64_t m, int64_t n, int has_dbias);
int d3s_dense_activation_backward_bf16_ws(const uint16_t *dy, int64_t dy_stride, const uint16_t *z, int64_t z_stride,
                                          int64_t m, int64_t n, int activation, uint16_t *dz, int64_t dz_stride,
                                          float *dbias, void *workspace, int64_t workspace_bytes, void *stream);

/* The global L2 norm of n_tensors gradients, and the gradients clipped to it:
 *   norm = sqrt(sum over all elements g^2)   (summed in 64 bits),
 *   dst = g * (max_norm / norm) where norm > max_norm, else dst = g.
 * src, dst, numel and dtypes are host arrays of n_tensors device addresses,
 * lengths (0 allowed) and D3S_DTYPE_*; they are read before the call returns.
 * dst[i] may be src[i] (then nothing is written unless the norm passes
 * max_norm), any other overlap is not allowed; dst NULL: the norm alone.
 * norm: one fp32 in device memory.  A norm that is not finite clips nothing:
 * the gradients keep their bits, and the caller sees the norm.  max_norm > 0. */
int d3s_clip_grads(const void *const *src, void *const *dst, const int64_t *numel, const int32_t *dtypes,
                   int n_tensors, float max_norm, float *norm, void *stream);
int64_t d3s_clip_grads_workspace_bytes(int n_tensors);
int d3s_clip_grads_ws(const void *const *src, void *const *dst, const int64_t *numel, const int32_t *dtypes,
                      int n_tensors, float max_norm, float *norm, void *workspace, int64_t workspace_bytes,
                      void *stream);

#ifdef __cplusplus
}
#endif

#endif
