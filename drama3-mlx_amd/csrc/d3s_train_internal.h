/* Internal launch interface of the scoring and training operators
 * (include/d3s_train.h): d3s_train_api.hip checks and sizes, the kernels are
 * in d3s_score.hip, d3s_dense.hip and d3s_clip.hip. */
#ifndef D3S_TRAIN_INTERNAL_H
#define D3S_TRAIN_INTERNAL_H

#include <mutex>

#include "../../include/d3s_train.h"
#include "d3s_internal.h"

namespace d3s {

/* held while a call that uses the stream's block enqueues its launches */
std::unique_lock<std::recursive_mutex> stream_call_lock(hipStream_t s);

struct ScoreArgs {
  const void *logits;
  int64_t row_stride;
  int vocab, n_rows;
  const float *temperature;
  float temperature_scalar;
  const int32_t *banned;
  const int32_t *tokens;
  int n_tokens;
  /* forward */
  float *logprobs, *entropy, *row_stats;
  int n_top;
  int32_t *top_ids;
  float *top_logprobs;
  uint32_t *counters;
  /* backward */
  const float *stats_in, *entropy_in, *grad_logprobs, *grad_entropy;
  void *grad;
  int64_t grad_stride;
};

/* segments a row is cut into, and the workspace that takes (0: one segment);
 * the records lie after the counters' block */
int score_segments(Dtype dt, int64_t n_rows, int vocab, int n_top);
size_t score_workspace_bytes(Dtype dt, int64_t n_rows, int vocab, int n_top);
void launch_score(const ScoreArgs &a, Dtype dt, void *ws, hipStream_t s);
void launch_score_backward(const ScoreArgs &a, Dtype dt, hipStream_t s);

size_t dense_workspace_bytes(const d3s_dense_params &p);
void launch_dense(const d3s_dense_params &p, void *ws, hipStream_t s);

struct ActGradArgs {
  const uint16_t *dy, *z;
  int64_t dy_stride, z_stride;
  int m, n, act;
  uint16_t *dz;
  int64_t dz_stride;
  float *dbias;
};
size_t act_grad_workspace_bytes(int64_t m, int64_t n, bool dbias);
void launch_act_grad(const ActGradArgs &a, void *ws, hipStream_t s);

size_t clip_workspace_bytes(int n_tensors);
void launch_clip(const void *const *src, void *const *dst, const int64_t *numel, const int32_t *dtypes, int n_tensors,
                 float max_norm, float *norm, void *ws, hipStream_t s);

}  // namespace d3s

#endif
