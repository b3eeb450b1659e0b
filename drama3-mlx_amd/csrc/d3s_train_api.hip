/* C-ABI of the scoring and training operators (include/d3s_train.h): argument
 * checks, workspaces, launches.  Nothing here throws: the checks come first,
 * and the only allocation is the stream's block. */
#include "d3s_room.h"

using namespace d3s;

namespace {

int check_rows(int dtype, int64_t n_rows, int64_t vocab) {
  if (!known(dtype)) return D3S_ERR_DTYPE;
  if (n_rows < 0 || n_rows > INT_MOST || vocab < 1) return D3S_ERR_ARG;
  return vocab > D3S_MAX_VOCAB ? D3S_ERR_UNSUPPORTED : D3S_OK;
}

int logprob_call(const void *logits, int dtype, int64_t n_rows, int64_t vocab, int64_t row_stride,
                 const float *temperature, float temperature_scalar, const int32_t *banned, const int32_t *tokens,
                 int n_tokens, float *logprobs, float *entropy, float *row_stats, int n_top, int32_t *top_ids,
                 float *top_logprobs, uint32_t *counters, Room room, void *stream) {
  if (const int rc = check_rows(dtype, n_rows, vocab)) return rc;
  if (row_stride < vocab || n_tokens < 0 || n_tokens > D3S_MAX_TOKENS || n_top < 0 || n_top > D3S_MAX_TOP ||
      n_top > vocab)
    return D3S_ERR_ARG;
  if (n_rows == 0) return D3S_OK;
  if (!logits || off(logits, size_of(dtype)) || (n_tokens > 0 && !tokens)) return D3S_ERR_ARG;
  if (!top_ids && !top_logprobs) n_top = 0;
  d3s::ScoreArgs a{};
  a.logits = logits;
  a.row_stride = row_stride;
  a.vocab = (int)vocab;
  a.n_rows = (int)n_rows;
  a.temperature = temperature;
  a.temperature_scalar = temperature_scalar;
  a.banned = banned;
  a.tokens = tokens;
  a.n_tokens = logprobs ? n_tokens : 0;
  a.logprobs = logprobs;
  a.entropy = entropy;
  a.row_stats = row_stats;
  a.n_top = n_top;
  a.top_ids = top_ids;
  a.top_logprobs = top_logprobs;
  a.counters = counters;
  const d3s::Dtype dt = type_of(dtype);
  hipStream_t s = (hipStream_t)stream;
  void *ws = nullptr;
  if (const int rc = take_room(room, d3s::score_workspace_bytes(dt, n_rows, a.vocab, n_top), s, &ws)) return rc;
  d3s::launch_score(a, dt, ws, s);
  return done();
}

/* (a tile or a stage past the end still counts in 32 bits) */
constexpr int64_t SIZE_MOST = INT_MOST - 1023;

bool product_shape(const d3s_dense_params *p) {
  if (p->m < 0 || p->n < 0 || p->k < 0 || p->m > SIZE_MOST || p->n > SIZE_MOST || p->k > SIZE_MOST) return false;
  return p->x_stride >= (p->x_transposed ? p->m : p->k) && p->w_stride >= (p->w_transposed ? p->n : p->k);
}

int check_dense(const d3s_dense_params *p) {
  if (!p) return D3S_ERR_ARG;
  if (!known(p->y_dtype)) return D3S_ERR_DTYPE;
  if (!product_shape(p) || p->activation < D3S_ACT_NONE || p->activation > D3S_ACT_GELU_TANH) return D3S_ERR_ARG;
  return D3S_OK;
}

int dense_call(const d3s_dense_params *p, Room room, void *stream) {
  if (const int rc = check_dense(p)) return rc;
  if (p->y_stride < p->n || (p->residual && p->residual_stride < p->n) || (p->z && p->z_stride < p->n))
    return D3S_ERR_ARG;
  if (p->m == 0 || p->n == 0) return D3S_OK;
  /* (at another stride one workgroup's outputs would be rows that another has yet to read) */
  if (p->residual == p->y && p->residual && p->residual_stride != p->y_stride && p->m > 1) return D3S_ERR_ARG;
  const size_t ys = size_of(p->y_dtype);
  if (!p->y || off(p->y, ys) || off(p->residual, ys) || off(p->bias, 2) || off(p->z, 2)) return D3S_ERR_ARG;
  if (p->k > 0 && (!p->x || !p->w || off(p->x, 2) || off(p->w, 2))) return D3S_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  void *ws = nullptr;
  if (const int rc = take_room(room, d3s::dense_workspace_bytes(*p), s, &ws)) return rc;
  d3s::launch_dense(*p, ws, s);
  return done();
}

int act_grad_call(const uint16_t *dy, int64_t dy_stride, const uint16_t *z, int64_t z_stride, int64_t m, int64_t n,
                  int activation, uint16_t *dz, int64_t dz_stride, float *dbias, Room room, void *stream) {
  if (m < 0 || n < 0 || m > INT_MOST || n > INT_MOST || activation < D3S_ACT_NONE || activation > D3S_ACT_GELU_TANH ||
      dy_stride < n || (z && z_stride < n) || (dz && dz_stride < n))
    return D3S_ERR_ARG;
  if (n == 0 || (!dz && !dbias)) return D3S_OK;
  if (dz && dz == dy && dz_stride != dy_stride && m > 1) return D3S_ERR_ARG; /* (as a residual in place, above) */
  if (off(dbias, 4)) return D3S_ERR_ARG;
  if (m > 0 && (!dy || (!z && activation != D3S_ACT_NONE) || off(dy, 2) || off(z, 2) || off(dz, 2)))
    return D3S_ERR_ARG;
  if (m == 0 && !dbias) return D3S_OK;
  hipStream_t s = (hipStream_t)stream;
  void *ws = nullptr;
  if (const int rc = take_room(room, d3s::act_grad_workspace_bytes(m, n, dbias != nullptr), s, &ws)) return rc;
  d3s::launch_act_grad({dy, activation == D3S_ACT_NONE ? nullptr : z, dy_stride, z_stride, (int)m, (int)n, activation,
                        dz, dz_stride, dbias},
                       ws, s);
  return done();
}

int clip_call(const void *const *src, void *const *dst, const int64_t *numel, const int32_t *dtypes, int n_tensors,
              float max_norm, float *norm, Room room, void *stream) {
  if (n_tensors < 0 || !(max_norm > 0.0f) || !norm || off(norm, 4)) return D3S_ERR_ARG;
  if (n_tensors > 0 && (!src || !numel || !dtypes)) return D3S_ERR_ARG;
  for (int i = 0; i < n_tensors; i++) {
    if (!known(dtypes[i])) return D3S_ERR_DTYPE;
    /* (element counts whose bytes and chunks stay far inside 64 bits) */
    if (numel[i] < 0 || numel[i] > ((int64_t)1 << 46)) return D3S_ERR_ARG;
    if (numel[i] > 0 && (!src[i] || off(src[i], size_of(dtypes[i])) ||
                         (dst && (!dst[i] || off(dst[i], size_of(dtypes[i]))))))
      return D3S_ERR_ARG;
  }
  hipStream_t s = (hipStream_t)stream;
  void *ws = nullptr;
  if (const int rc = take_room(room, d3s::clip_workspace_bytes(n_tensors), s, &ws)) return rc;
  d3s::launch_clip(src, dst, numel, dtypes, n_tensors, max_norm, norm, ws, s);
  return done();
}

}  // namespace

extern "C" {

int d3s_logprob(const void *logits, int dtype, int64_t n_rows, int64_t vocab, int64_t row_stride,
                const float *temperature, float temperature_scalar, const int32_t *banned, const int32_t *tokens,
                int n_tokens, float *logprobs, float *entropy, float *row_stats, int n_top, int32_t *top_ids,
                float *top_logprobs, uint32_t *counters, void *stream) {
  return locked(stream, [&] {
    return logprob_call(logits, dtype, n_rows, vocab, row_stride, temperature, temperature_scalar, banned, tokens,
                      n_tokens, logprobs, entropy, row_stats, n_top, top_ids, top_logprobs, counters,
                      Room{false, nullptr, 0}, stream);
  });
}

int64_t d3s_logprob_workspace_bytes(int dtype, int64_t n_rows, int64_t vocab, int n_top) {
  if (const int rc = check_rows(dtype, n_rows, vocab)) return rc;
  if (n_top < 0 || n_top > D3S_MAX_TOP || n_top > vocab) return D3S_ERR_ARG;
  /* (a call with neither array of alternatives has none: other segments) */
  const size_t with = d3s::score_workspace_bytes(type_of(dtype), n_rows, (int)vocab, n_top);
  const size_t without = d3s::score_workspace_bytes(type_of(dtype), n_rows, (int)vocab, 0);
  return (int64_t)(with > without ? with : without);
}

int d3s_logprob_ws(const void *logits, int dtype, int64_t n_rows, int64_t vocab, int64_t row_stride,
                   const float *temperature, float temperature_scalar, const int32_t *banned, const int32_t *tokens,
                   int n_tokens, float *logprobs, float *entropy, float *row_stats, int n_top, int32_t *top_ids,
                   float *top_logprobs, uint32_t *counters, void *workspace, int64_t workspace_bytes, void *stream) {
  return logprob_call(logits, dtype, n_rows, vocab, row_stride, temperature, temperature_scalar, banned, tokens,
                      n_tokens, logprobs, entropy, row_stats, n_top, top_ids, top_logprobs, counters,
                      Room{true, workspace, workspace_bytes}, stream);
}

int d3s_logprob_backward(const void *logits, int dtype, int64_t n_rows, int64_t vocab, int64_t row_stride,
                         const float *temperature, float temperature_scalar, const int32_t *banned,
                         const int32_t *tokens, int n_tokens, const float *row_stats, const float *entropy,
                         const float *grad_logprobs, const float *grad_entropy, void *grad_logits,
                         int64_t grad_row_stride, void *stream) {
  if (const int rc = check_rows(dtype, n_rows, vocab)) return rc;
  if (row_stride < vocab || grad_row_stride < vocab || n_tokens < 0 || n_tokens > D3S_MAX_TOKENS) return D3S_ERR_ARG;
  if (n_rows == 0) return D3S_OK;
  const size_t es = size_of(dtype);
  if (!logits || !grad_logits || !row_stats || off(logits, es) || off(grad_logits, es)) return D3S_ERR_ARG;
  if (n_tokens > 0 && (!tokens || !grad_logprobs)) return D3S_ERR_ARG;
  if (grad_entropy && !entropy) return D3S_ERR_ARG;
  if (grad_logits == logits && grad_row_stride != row_stride) return D3S_ERR_ARG;
  d3s::ScoreArgs a{};
  a.logits = logits;
  a.row_stride = row_stride;
  a.vocab = (int)vocab;
  a.n_rows = (int)n_rows;
  a.temperature = temperature;
  a.temperature_scalar = temperature_scalar;
  a.banned = banned;
  a.tokens = tokens;
  a.n_tokens = n_tokens;
  a.stats_in = row_stats;
  a.entropy_in = entropy;
  a.grad_logprobs = grad_logprobs;
  a.grad_entropy = grad_entropy;
  a.grad = grad_logits;
  a.grad_stride = grad_row_stride;
  d3s::launch_score_backward(a, type_of(dtype), (hipStream_t)stream);
  return done();
}

int d3s_dense_bf16(const d3s_dense_params *params, void *stream) {
  return locked(stream, [&] {
    return dense_call(params, Room{false, nullptr, 0}, stream);
  });
}

int64_t d3s_dense_workspace_bytes(const d3s_dense_params *params) {
  if (const int rc = check_dense(params)) return rc;
  return (int64_t)d3s::dense_workspace_bytes(*params);
}

int d3s_dense_bf16_ws(const d3s_dense_params *params, void *workspace, int64_t workspace_bytes, void *stream) {
  return dense_call(params, Room{true, workspace, workspace_bytes}, stream);
}

int d3s_dense_activation_backward_bf16(const uint16_t *dy, int64_t dy_stride, const uint16_t *z, int64_t z_stride,
                                       int64_t m, int64_t n, int activation, uint16_t *dz, int64_t dz_stride,
                                       float *dbias, void *stream) {
  return locked(stream, [&] {
    return act_grad_call(dy, dy_stride, z, z_stride, m, n, activation, dz, dz_stride, dbias, Room{false, nullptr, 0},
                       stream);
  });
}

int64_t d3s_dense_activation_backward_workspace_bytes(int64_t m, int64_t n, int has_dbias) {
  if (m < 0 || n < 0 || m > INT_MOST || n > INT_MOST) return D3S_ERR_ARG;
  return (int64_t)d3s::act_grad_workspace_bytes(m, n, has_dbias != 0);
}

int d3s_dense_activation_backward_bf16_ws(const uint16_t *dy, int64_t dy_stride, const uint16_t *z, int64_t z_stride,
                                          int64_t m, int64_t n, int activation, uint16_t *dz, int64_t dz_stride,
                                          float *dbias, void *workspace, int64_t workspace_bytes, void *stream) {
  return act_grad_call(dy, dy_stride, z, z_stride, m, n, activation, dz, dz_stride, dbias,
                       Room{true, workspace, workspace_bytes}, stream);
}

int d3s_clip_grads(const void *const *src, void *const *dst, const int64_t *numel, const int32_t *dtypes,
                   int n_tensors, float max_norm, float *norm, void *stream) {
  return locked(stream, [&] {
    return clip_call(src, dst, numel, dtypes, n_tensors, max_norm, norm, Room{false, nullptr, 0}, stream);
  });
}

int64_t d3s_clip_grads_workspace_bytes(int n_tensors) {
  return n_tensors < 0 ? D3S_ERR_ARG : (int64_t)d3s::clip_workspace_bytes(n_tensors);
}

int d3s_clip_grads_ws(const void *const *src, void *const *dst, const int64_t *numel, const int32_t *dtypes,
                      int n_tensors, float max_norm, float *norm, void *workspace, int64_t workspace_bytes,
                      void *stream) {
  return clip_call(src, dst, numel, dtypes, n_tensors, max_norm, norm, Room{true, workspace, workspace_bytes}, stream);
}

}  // extern "C"
