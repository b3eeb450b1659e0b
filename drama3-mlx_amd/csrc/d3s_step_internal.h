/* Internal launch interface of the operators between ids and logits
 * (include/d3s_step.h): d3s_step_api.hip checks and sizes, the kernels are in
 * d3s_verify.hip, d3s_embed.hip, d3s_norm.hip and d3s_dropout.hip. */
#ifndef D3S_STEP_INTERNAL_H
#define D3S_STEP_INTERNAL_H

#include "../../include/d3s_step.h"
#include "d3s_internal.h"

namespace d3s {

/* workgroups a launch at most: their threads are counted in 32 bits (kernels of
 * more work loop over it) */
constexpr int STEP_GRID = 1 << 20;

size_t verify_workspace_bytes(const d3s_verify_params &p);
void launch_verify(const d3s_verify_params &p, void *ws, hipStream_t s);

struct RankedArgs {
  const int32_t *target_cand;
  const float *target_probs;
  int target_k;
  const int32_t *draft_cand;
  const float *draft_probs;
  int draft_k;
  int n_seqs, n_draft;
  const int32_t *drafted, *lengths;
  const float *u_accept, *u_draw;
  int32_t *tokens, *n_accepted;
  float *accept;
  uint32_t *counters;
};
void launch_verify_ranked(const RankedArgs &a, hipStream_t s);

struct EmbedArgs {
  const int32_t *ids;
  int64_t n_rows;
  int n_ids;
  int64_t vocab, slot_rows, width;
  float scale;
  const void *in; /* the table, or dy */
  int64_t in_stride;
  void *out; /* y, or the gradient */
  int64_t out_stride;
  int accumulate;
};
void launch_embed(const EmbedArgs &a, Dtype in, Dtype out, hipStream_t s);
size_t embed_grad_workspace_bytes(int64_t n_rows, int n_ids, int64_t vocab, int64_t slot_rows, int64_t width);
void launch_embed_grad(const EmbedArgs &a, Dtype in, Dtype out, void *ws, hipStream_t s);

struct NormArgs {
  const void *x, *residual;
  int64_t x_stride, residual_stride;
  void *sum;
  int64_t sum_stride;
  const void *gain;
  float eps;
  int64_t n_rows, width;
  void *y;
  int y_dtype;
  int64_t y_stride;
  int group; /* of E4M3, 0 for whole rows */
  float *scales, *rstd;
};
void launch_norm(const NormArgs &a, Dtype dt, hipStream_t s);

struct NormGradArgs {
  const void *dy, *h, *gain, *dsum;
  int64_t dy_stride, h_stride, dsum_stride;
  const float *rstd;
  int64_t n_rows, width;
  void *dx;
  int64_t dx_stride;
  float *dgain;
};
size_t norm_grad_workspace_bytes(int64_t n_rows, int64_t width, bool dgain);
void launch_norm_grad(const NormGradArgs &a, Dtype dt, void *ws, hipStream_t s);

struct DropoutArgs {
  const void *x, *residual;
  int64_t x_stride, residual_stride, n_rows, width;
  uint32_t least; /* kept iff the word's upper 24 bits are at least this */
  float scale;
  uint64_t seed, draw;
  const uint64_t *draw_add;
  void *y;
  int64_t y_stride;
};
void launch_dropout(const DropoutArgs &a, Dtype dt, hipStream_t s);

}  // namespace d3s

#endif
