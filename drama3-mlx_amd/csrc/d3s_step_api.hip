/* C-ABI of the operators between ids and logits (include/d3s_step.h): argument
 * checks, workspaces, launches.  Nothing here throws: the checks come first,
 * and the only allocation is the stream's block. */
#include "d3s_room.h"
#include "d3s_step_internal.h"

using namespace d3s;

namespace {

/* rows by a stride stay inside 63 bits of bytes */
constexpr int64_t STRIDE_MOST = (int64_t)1 << 40;
/* ids of a gradient: their places, and those that lanes look ahead to, are counted in 32 bits */
constexpr int64_t IDS_MOST = ((int64_t)1 << 31) - 65536;
bool stride_ok(int64_t stride, int64_t width) { return stride >= width && stride <= STRIDE_MOST; }

int check_verify(const d3s_verify_params *p) {
  if (!p) return D3S_ERR_ARG;
  if (!known(p->target_dtype) || (p->draft && !known(p->draft_dtype))) return D3S_ERR_DTYPE;
  if (p->n_seqs < 0 || p->n_draft < 0 || p->n_draft > D3S_MAX_DRAFT || p->vocab < 1 ||
      p->n_seqs > INT_MOST / (2 * D3S_MAX_DRAFT + 1))
    return D3S_ERR_ARG;
  if (p->vocab > D3S_MAX_VOCAB) return D3S_ERR_UNSUPPORTED;
  if (!stride_ok(p->target_stride, p->vocab) || (p->draft && !stride_ok(p->draft_stride, p->vocab))) return D3S_ERR_ARG;
  return D3S_OK;
}

int verify_call(const d3s_verify_params *params, Room room, void *stream) {
  if (const int rc = check_verify(params)) return rc;
  const d3s_verify_params &p = *params;
  if (p.n_seqs == 0) return D3S_OK;
  if (!p.target || off(p.target, size_of(p.target_dtype)) || (p.draft && off(p.draft, size_of(p.draft_dtype))))
    return D3S_ERR_ARG;
  if (!p.u_draw || !p.tokens || !p.n_accepted || (p.n_draft > 0 && (!p.drafted || !p.u_accept))) return D3S_ERR_ARG;
  for (const void *q : {(const void *)p.drafted, (const void *)p.lengths, (const void *)p.temperature,
                        (const void *)p.draft_temperature, (const void *)p.u_accept, (const void *)p.u_draw,
                        (const void *)p.tokens, (const void *)p.n_accepted, (const void *)p.accept, (const void *)p.counters})
    if (off(q, 4)) return D3S_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  void *ws = nullptr;
  if (const int rc = take_room(room, verify_workspace_bytes(p), s, &ws)) return rc;
  launch_verify(p, ws, s);
  return done();
}

/* the rows of the table, parts and what lies between them (0: the arguments are out of range) */
int64_t table_rows(int64_t n_rows, int n_ids, int64_t vocab, int64_t slot_rows, int64_t width) {
  if (n_rows < 0 || n_rows > INT_MOST || n_ids < 1 || n_ids > D3S_MAX_IDS || vocab < 1 || vocab > INT_MOST || width < 0 ||
      width > INT_MOST || slot_rows < 0 || slot_rows > INT_MOST || (slot_rows != 0 && slot_rows < vocab))
    return 0;
  return vocab + (n_ids - 1) * slot_rows;
}

int embed_grad_check(const int32_t *ids, int64_t n_rows, int n_ids, const void *dy, int dtype, int64_t dy_stride,
                     int64_t vocab, int64_t slot_rows, int64_t width, void *grad, int grad_dtype, int64_t grad_stride) {
  if (!known(dtype) || !known(grad_dtype)) return D3S_ERR_DTYPE;
  if (!table_rows(n_rows, n_ids, vocab, slot_rows, width) || n_rows > IDS_MOST / n_ids || !stride_ok(dy_stride, width) || !stride_ok(grad_stride, width))
    return D3S_ERR_ARG;
  if (width == 0) return D3S_OK;
  if (!grad || off(grad, size_of(grad_dtype))) return D3S_ERR_ARG;
  if (n_rows > 0 && (!ids || !dy || off(dy, size_of(dtype)) || off(ids, 4))) return D3S_ERR_ARG;
  return D3S_OK;
}

int embed_grad_call(const int32_t *ids, int64_t n_rows, int n_ids, const void *dy, int dtype, int64_t dy_stride,
                    int64_t vocab, int64_t slot_rows, int64_t width, float scale, int accumulate, void *grad,
                    int grad_dtype, int64_t grad_stride, Room room, void *stream) {
  if (const int rc = embed_grad_check(ids, n_rows, n_ids, dy, dtype, dy_stride, vocab, slot_rows, width, grad, grad_dtype,
                                      grad_stride))
    return rc;
  if (width == 0 || (accumulate && n_rows == 0)) return D3S_OK;
  hipStream_t s = (hipStream_t)stream;
  void *ws = nullptr;
  if (const int rc = take_room(room, embed_grad_workspace_bytes(n_rows, n_ids, vocab, slot_rows, width), s, &ws)) return rc;
  launch_embed_grad({ids, n_rows, n_ids, vocab, slot_rows, width, scale, dy, dy_stride, grad, grad_stride, accumulate},
                    type_of(dtype), type_of(grad_dtype), ws, s);
  return done();
}

bool rows_ok(int64_t n_rows, int64_t width) { return n_rows >= 0 && n_rows <= INT_MOST && width >= 0 && width <= INT_MOST; }
/* an array that may be another one, at one stride */
bool apart(const void *a, int64_t a_stride, const void *b, int64_t b_stride, int64_t rows) {
  return !a || a != b || a_stride == b_stride || rows <= 1;
}

int norm_grad_call(const void *dy, int dtype, int64_t dy_stride, const void *h, int64_t h_stride, const void *gain,
                   const float *rstd, const void *dsum, int64_t dsum_stride, int64_t n_rows, int64_t width, void *dx,
                   int64_t dx_stride, float *dgain, Room room, void *stream) {
  if (!known(dtype)) return D3S_ERR_DTYPE;
  if (!rows_ok(n_rows, width) || !stride_ok(dy_stride, width) || !stride_ok(h_stride, width) ||
      (dsum && !stride_ok(dsum_stride, width)) || (dx && !stride_ok(dx_stride, width)))
    return D3S_ERR_ARG;
  if (width == 0 || (!dx && !dgain) || (n_rows == 0 && !dgain)) return D3S_OK;
  const size_t es = size_of(dtype);
  if (off(dgain, 4) || off(gain, es) || off(dx, es) || off(dsum, es)) return D3S_ERR_ARG;
  if (n_rows > 0 && (!dy || !h || !rstd || off(dy, es) || off(h, es) || off(rstd, 4))) return D3S_ERR_ARG;
  if (!apart(dx, dx_stride, dy, dy_stride, n_rows) || !apart(dx, dx_stride, h, h_stride, n_rows) ||
      !apart(dx, dx_stride, dsum, dsum_stride, n_rows))
    return D3S_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  void *ws = nullptr;
  if (const int rc = take_room(room, norm_grad_workspace_bytes(n_rows, width, dgain != nullptr), s, &ws)) return rc;
  launch_norm_grad({dy, h, gain, dsum, dy_stride, h_stride, dsum_stride, rstd, n_rows, width, dx, dx_stride, dgain},
                   type_of(dtype), ws, s);
  return done();
}

}  // namespace

extern "C" {

int d3s_verify(const d3s_verify_params *params, void *stream) {
  return locked(stream, [&] { return verify_call(params, Room{false, nullptr, 0}, stream); });
}

int64_t d3s_verify_workspace_bytes(const d3s_verify_params *params) {
  if (const int rc = check_verify(params)) return rc;
  return params->n_seqs == 0 ? 0 : (int64_t)verify_workspace_bytes(*params);
}

int d3s_verify_ws(const d3s_verify_params *params, void *workspace, int64_t workspace_bytes, void *stream) {
  return verify_call(params, Room{true, workspace, workspace_bytes}, stream);
}

int d3s_verify_ranked(const int32_t *target_cand, const float *target_probs, int target_k, const int32_t *draft_cand,
                      const float *draft_probs, int draft_k, int64_t n_seqs, int n_draft, const int32_t *drafted,
                      const int32_t *lengths, const float *u_accept, const float *u_draw, int32_t *tokens,
                      int32_t *n_accepted, float *accept, uint32_t *counters, void *stream) {
  const bool drafts = draft_cand || draft_probs;
  if (n_seqs < 0 || n_seqs > INT_MOST / (2 * D3S_MAX_DRAFT + 1) || n_draft < 0 || n_draft > D3S_MAX_DRAFT || target_k < 1 ||
      (drafts && draft_k < 1))
    return D3S_ERR_ARG;
  if (target_k > D3S_MAX_RANKED || (drafts && draft_k > D3S_MAX_RANKED)) return D3S_ERR_UNSUPPORTED;
  if (n_seqs == 0) return D3S_OK;
  if (!target_cand || !target_probs || (drafts && (!draft_cand || !draft_probs)) || !u_draw || !tokens || !n_accepted ||
      (n_draft > 0 && (!drafted || !u_accept)))
    return D3S_ERR_ARG;
  for (const void *q : {(const void *)target_cand, (const void *)target_probs, (const void *)draft_cand,
                        (const void *)draft_probs, (const void *)drafted, (const void *)lengths, (const void *)u_accept,
                        (const void *)u_draw, (const void *)tokens, (const void *)n_accepted, (const void *)accept,
                        (const void *)counters})
    if (off(q, 4)) return D3S_ERR_ARG;
  launch_verify_ranked({target_cand, target_probs, target_k, draft_cand, draft_probs, drafts ? draft_k : 0, (int)n_seqs,
                        n_draft, drafted, lengths, u_accept, u_draw, tokens, n_accepted, accept, counters},
                       (hipStream_t)stream);
  return done();
}

int d3s_embed(const int32_t *ids, int64_t n_rows, int n_ids, const void *table, int dtype, int64_t table_stride,
              int64_t vocab, int64_t slot_rows, int64_t width, float scale, void *y, int y_dtype, int64_t y_stride,
              void *stream) {
  if (!known(dtype) || !known(y_dtype)) return D3S_ERR_DTYPE;
  if (!table_rows(n_rows, n_ids, vocab, slot_rows, width) || !stride_ok(table_stride, width) || !stride_ok(y_stride, width))
    return D3S_ERR_ARG;
  if (n_rows == 0 || width == 0) return D3S_OK;
  if (!ids || !table || !y || off(ids, 4) || off(table, size_of(dtype)) || off(y, size_of(y_dtype))) return D3S_ERR_ARG;
  launch_embed({ids, n_rows, n_ids, vocab, slot_rows, width, scale, table, table_stride, y, y_stride, 0}, type_of(dtype),
               type_of(y_dtype), (hipStream_t)stream);
  return done();
}

int d3s_embed_backward(const int32_t *ids, int64_t n_rows, int n_ids, const void *dy, int dtype, int64_t dy_stride,
                       int64_t vocab, int64_t slot_rows, int64_t width, float scale, int accumulate, void *grad,
                       int grad_dtype, int64_t grad_stride, void *stream) {
  return locked(stream, [&] {
    return embed_grad_call(ids, n_rows, n_ids, dy, dtype, dy_stride, vocab, slot_rows, width, scale, accumulate, grad,
                           grad_dtype, grad_stride, Room{false, nullptr, 0}, stream);
  });
}

int64_t d3s_embed_backward_workspace_bytes(int64_t n_rows, int n_ids, int64_t vocab, int64_t slot_rows, int64_t width) {
  if (!table_rows(n_rows, n_ids, vocab, slot_rows, width) || n_rows > IDS_MOST / n_ids) return D3S_ERR_ARG;
  return (int64_t)embed_grad_workspace_bytes(n_rows, n_ids, vocab, slot_rows, width);
}

int d3s_embed_backward_ws(const int32_t *ids, int64_t n_rows, int n_ids, const void *dy, int dtype, int64_t dy_stride,
                          int64_t vocab, int64_t slot_rows, int64_t width, float scale, int accumulate, void *grad,
                          int grad_dtype, int64_t grad_stride, void *workspace, int64_t workspace_bytes, void *stream) {
  return embed_grad_call(ids, n_rows, n_ids, dy, dtype, dy_stride, vocab, slot_rows, width, scale, accumulate, grad,
                         grad_dtype, grad_stride, Room{true, workspace, workspace_bytes}, stream);
}

int d3s_rms_norm(const void *x, int dtype, int64_t x_stride, const void *residual, int64_t residual_stride, void *sum,
                 int64_t sum_stride, const void *gain, float eps, int64_t n_rows, int64_t width, void *y, int y_dtype,
                 int64_t y_stride, int group, float *scales, float *rstd, void *stream) {
  const bool e4m3 = y_dtype == D3S_DTYPE_E4M3;
  if (!known(dtype) || (!known(y_dtype) && !e4m3)) return D3S_ERR_DTYPE;
  if (!rows_ok(n_rows, width) || !(eps >= 0.0f) || !stride_ok(x_stride, width) || !stride_ok(y_stride, width) ||
      (residual && !stride_ok(residual_stride, width)) || (sum && !stride_ok(sum_stride, width)))
    return D3S_ERR_ARG;
  if (e4m3 && group != 0 && group != 32 && group != 64 && group != 128 && group != 256) return D3S_ERR_ARG;
  if (n_rows == 0 || width == 0) return D3S_OK;
  const size_t es = size_of(dtype), ys = e4m3 ? 1 : size_of(y_dtype);
  if (!x || !y || off(x, es) || off(residual, es) || off(sum, es) || off(gain, es) || off(y, ys) || off(rstd, 4))
    return D3S_ERR_ARG;
  if (e4m3 && (!scales || off(scales, 4))) return D3S_ERR_ARG;
  /* in place: the same elements by the same thread, at one stride and type; y and sum are two outputs */
  if (y == sum || ((y == x || y == residual) && y_dtype != dtype)) return D3S_ERR_ARG;
  if (!apart(sum, sum_stride, x, x_stride, n_rows) || !apart(sum, sum_stride, residual, residual_stride, n_rows) ||
      !apart(y, y_stride, x, x_stride, n_rows) || !apart(y, y_stride, residual, residual_stride, n_rows))
    return D3S_ERR_ARG;
  launch_norm({x, residual, x_stride, residual_stride, sum, sum_stride, gain, eps, n_rows, width, y, y_dtype, y_stride,
               e4m3 ? group : 0, scales, rstd},
              type_of(dtype), (hipStream_t)stream);
  return done();
}

int d3s_rms_norm_backward(const void *dy, int dtype, int64_t dy_stride, const void *h, int64_t h_stride,
                          const void *gain, const float *rstd, const void *dsum, int64_t dsum_stride, int64_t n_rows,
                          int64_t width, void *dx, int64_t dx_stride, float *dgain, void *stream) {
  return locked(stream, [&] {
    return norm_grad_call(dy, dtype, dy_stride, h, h_stride, gain, rstd, dsum, dsum_stride, n_rows, width, dx, dx_stride,
                          dgain, Room{false, nullptr, 0}, stream);
  });
}

int64_t d3s_rms_norm_backward_workspace_bytes(int64_t n_rows, int64_t width, int has_dgain) {
  if (!rows_ok(n_rows, width)) return D3S_ERR_ARG;
  return (int64_t)norm_grad_workspace_bytes(n_rows, width, has_dgain != 0);
}

int d3s_rms_norm_backward_ws(const void *dy, int dtype, int64_t dy_stride, const void *h, int64_t h_stride,
                             const void *gain, const float *rstd, const void *dsum, int64_t dsum_stride, int64_t n_rows,
                             int64_t width, void *dx, int64_t dx_stride, float *dgain, void *workspace,
                             int64_t workspace_bytes, void *stream) {
  return norm_grad_call(dy, dtype, dy_stride, h, h_stride, gain, rstd, dsum, dsum_stride, n_rows, width, dx, dx_stride,
                        dgain, Room{true, workspace, workspace_bytes}, stream);
}

int d3s_dropout(const void *x, int dtype, int64_t x_stride, const void *residual, int64_t residual_stride,
                int64_t n_rows, int64_t width, float p, uint64_t seed, uint64_t draw, const uint64_t *draw_add, void *y,
                int64_t y_stride, void *stream) {
  if (!known(dtype)) return D3S_ERR_DTYPE;
  if (!rows_ok(n_rows, width) || !(p >= 0.0f && p <= 1.0f) || !stride_ok(x_stride, width) || !stride_ok(y_stride, width) ||
      (residual && !stride_ok(residual_stride, width)))
    return D3S_ERR_ARG;
  if (n_rows == 0 || width == 0) return D3S_OK;
  const size_t es = size_of(dtype);
  if (!x || !y || off(x, es) || off(y, es) || off(residual, es) || off(draw_add, 8)) return D3S_ERR_ARG;
  if (!apart(y, y_stride, x, x_stride, n_rows) || !apart(y, y_stride, residual, residual_stride, n_rows)) return D3S_ERR_ARG;
  /* u = w 2^-24 >= p iff the whole number w >= p 2^24 (exact in fp32: a power of two) */
  const float bar = p * 16777216.0f;
  const uint32_t least = (uint32_t)bar + ((float)(uint32_t)bar < bar ? 1u : 0u);
  const float scale = p < 1.0f ? (float)(1.0 / (1.0 - (double)p)) : 0.0f;
  launch_dropout({x, residual, x_stride, residual_stride, n_rows, width, least, scale, seed, draw, draw_add, y, y_stride},
                 type_of(dtype), (hipStream_t)stream);
  return done();
}

}  // extern "C"
