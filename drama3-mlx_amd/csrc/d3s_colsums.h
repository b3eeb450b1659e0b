/* The second launch of column sums: the first leaves a row of partial sums for each
 * of its runs of rows. */
#ifndef D3S_COLSUMS_H
#define D3S_COLSUMS_H

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace d3s {
namespace {

/* 16 columns a workgroup, 16 threads a column, each a sixteenth of the runs */
__global__ __launch_bounds__(256) void k_column_sums(const float *parts, int runs, int n, int group0, float *dbias) {
  __shared__ float sum[16][17];
  const int c = (int)threadIdx.x % 16, q = (int)threadIdx.x / 16;
  const int64_t col = ((int64_t)group0 + blockIdx.x) * 16 + c;
  const int per = (runs + 15) / 16, r1 = min(runs, (q + 1) * per);
  float v = 0.0f;
  if (col < n) {
#pragma unroll 16
    for (int r = q * per; r < r1; r++) v += parts[(int64_t)r * n + col];
  }
  sum[q][c] = v;
  __syncthreads();
  if (q == 0 && col < n) {
    v = 0.0f;
    for (int i = 0; i < 16; i++) v += sum[i][c];
    dbias[col] = v;
  }
}

void launch_column_sums(const float *parts, int runs, int n, float *out, hipStream_t s) {
  constexpr int MOST = 1 << 22; /* workgroups a launch */
  const int64_t groups = ((int64_t)n + 15) / 16;
  /* (up to 2^27 workgroups: 2^35 threads would pass the launch's count) */
  for (int64_t g = 0; g < groups; g += MOST)
    k_column_sums<<<dim3((unsigned)min((int64_t)MOST, groups - g)), 256, 0, s>>>(parts, runs, n, (int)g, out);
}

}  // namespace
}  // namespace d3s

#endif
