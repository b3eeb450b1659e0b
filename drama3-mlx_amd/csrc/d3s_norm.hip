/* k_norm_rows, k_norm_grad_rows: root-mean-square norm with the residual's addition
 * and an output in 8 bits, and its gradient (gfx950, wave64; include/d3s_step.h). */
#include "d3s_step_internal.h"
#include "d3s_vec.h"

namespace d3s {
namespace {

constexpr int NT = 256;
constexpr int NW = NT / WAVE;
constexpr float E4M3_MOST = 448.0f;

/* the sum (or greatest) over the workgroup, in every thread, added in one order */
__device__ __forceinline__ float block_sum(float v, float *part) {
  v = readlane_f(wave_scan_add_f32(v), 63);
  __syncthreads();
  if (lane_id() == 0) part[threadIdx.x / WAVE] = v;
  __syncthreads();
  float t = 0.0f;
#pragma unroll
  for (int w = 0; w < NW; w++) t += part[w];
  return t;
}
__device__ __forceinline__ float block_max(float v, float *part) {
  v = wave_max_f(v);
  __syncthreads();
  if (lane_id() == 0) part[threadIdx.x / WAVE] = v;
  __syncthreads();
  float t = part[0];
#pragma unroll
  for (int w = 1; w < NW; w++) t = __builtin_elementwise_maximum(t, part[w]);
  return t;
}

/* eight values over their group's greatest, as 8 bits (saturating: a quotient is
 * at most 448 and a rounding) */
__device__ __forceinline__ uint64_t pack_e4m3(const float *v, float scale) {
  uint32_t w[2] = {0u, 0u};
  float q[8];
#pragma unroll
  for (int e = 0; e < 8; e++) {
    q[e] = scale > 0.0f ? v[e] / scale : scale == 0.0f ? 0.0f : __builtin_nanf("");
    if (scale > 0.0f) q[e] = fminf(fmaxf(q[e], -E4M3_MOST), E4M3_MOST);
  }
#pragma unroll
  for (int i = 0; i < 2; i++) {
    w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i], q[4 * i + 1], 0, false);
    w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i + 2], q[4 * i + 3], (int)w[i], true);
  }
  return (uint64_t)w[1] << 32 | w[0];
}

/* the scale of a group whose greatest |y| is `most` (NaN in, NaN out; an infinity
 * is one too) */
__device__ __forceinline__ float e4m3_scale(float most) {
  return most < __builtin_inff() ? most / E4M3_MOST : __builtin_nanf("");
}

template <bool BF16>
__global__ __launch_bounds__(NT) void k_norm_rows(NormArgs a) {
  constexpr int ES = BF16 ? 2 : 4;
  __shared__ float part[NW];
  const int tid = (int)threadIdx.x;
  for (int64_t row = blockIdx.x; row < a.n_rows; row += gridDim.x) {
    const char *x = (const char *)a.x + row * a.x_stride * ES;
    const char *res = a.residual ? (const char *)a.residual + row * a.residual_stride * ES : nullptr;
    auto get = [&](int64_t j, int left, float *h) {
      load8<BF16>(x, j, left, h);
      if (res) {
        float r[8];
        load8<BF16>(res, j, left, r);
#pragma unroll
        for (int e = 0; e < 8; e++) h[e] += r[e];
      }
    };
    auto left_at = [&](int64_t j) { return j < a.width ? (int)min((int64_t)8, a.width - j) : 0; };
    float s = 0.0f;
    for (int64_t j = tid * 8; j < a.width; j += NT * 8) {
      float h[8];
      get(j, left_at(j), h);
#pragma unroll
      for (int e = 0; e < 8; e++) s = fmaf(h[e], h[e], s);
    }
    s = block_sum(s, part);
    const float rstd = 1.0f / sqrtf(s / (float)a.width + a.eps);
    if (tid == 0 && a.rstd) a.rstd[row] = rstd;
    auto scaled = [&](int64_t j, int left, float *h) {
      float g[8] = {1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f};
      if (a.gain) load8<BF16>(a.gain, j, left, g);
#pragma unroll
      for (int e = 0; e < 8; e++) h[e] = h[e] * rstd * g[e];
    };
    auto greatest = [&](const float *y, int left) {
      float most = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; e++) most = __builtin_elementwise_maximum(most, e < left ? fabsf(y[e]) : 0.0f);
      return most;
    };
    float row_scale = 0.0f;
    const bool whole = a.y_dtype == D3S_DTYPE_E4M3 && a.group == 0;
    if (whole) {
      float most = 0.0f;
      for (int64_t j = tid * 8; j < a.width; j += NT * 8) {
        float h[8];
        get(j, left_at(j), h);
        scaled(j, left_at(j), h);
        most = __builtin_elementwise_maximum(most, greatest(h, left_at(j)));
      }
      row_scale = e4m3_scale(block_max(most, part));
      if (tid == 0) a.scales[row] = row_scale;
    }
    for (int64_t base = 0; base < a.width; base += NT * 8) {
      const int64_t j = base + tid * 8;
      const int left = left_at(j);
      float h[8];
      get(j, left, h);
      if (a.sum && left > 0) store8<BF16>((char *)a.sum + row * a.sum_stride * ES, j, left, h);
      scaled(j, left, h);
      if (a.y_dtype == D3S_DTYPE_BF16) {
        if (left > 0) store8<true>((char *)a.y + row * a.y_stride * 2, j, left, h);
      } else if (a.y_dtype == D3S_DTYPE_F32) {
        if (left > 0) store8<false>((char *)a.y + row * a.y_stride * 4, j, left, h);
      } else {
        float scale = row_scale;
        if (!whole) {
          float most = left > 0 ? greatest(h, left) : 0.0f;
          for (int d = 1; d < a.group / 8; d *= 2) most = __builtin_elementwise_maximum(most, __shfl_xor(most, d));
          scale = e4m3_scale(most);
          if (left > 0 && j % a.group == 0)
            a.scales[row * ((a.width + a.group - 1) / a.group) + j / a.group] = scale;
        }
        const uint64_t q = pack_e4m3(h, scale);
        uint8_t *y = (uint8_t *)a.y + row * a.y_stride + j;
        if (left == 8)
          __builtin_memcpy(y, &q, 8);
        else
          for (int e = 0; e < left; e++) y[e] = (uint8_t)(q >> 8 * e);
      }
    }
  }
}

template <bool BF16>
__global__ __launch_bounds__(NT) void k_norm_grad_rows(NormGradArgs a) {
  constexpr int ES = BF16 ? 2 : 4;
  __shared__ float part[NW];
  const int tid = (int)threadIdx.x;
  for (int64_t row = blockIdx.x; row < a.n_rows; row += gridDim.x) {
    const char *dy = (const char *)a.dy + row * a.dy_stride * ES, *h = (const char *)a.h + row * a.h_stride * ES;
    const float rstd = a.rstd[row];
    auto get = [&](int64_t j, int left, float *p, float *xhat) {
      float g[8] = {1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f};
      load8<BF16>(dy, j, left, p);
      load8<BF16>(h, j, left, xhat);
      if (a.gain) load8<BF16>(a.gain, j, left, g);
#pragma unroll
      for (int e = 0; e < 8; e++) p[e] *= g[e], xhat[e] *= rstd;
    };
    float s = 0.0f;
    for (int64_t j = tid * 8; j < a.width; j += NT * 8) {
      float p[8], xhat[8];
      get(j, (int)min((int64_t)8, a.width - j), p, xhat);
#pragma unroll
      for (int e = 0; e < 8; e++) s = fmaf(p[e], xhat[e], s);
    }
    const float mean = block_sum(s, part) / (float)a.width;
    for (int64_t j = tid * 8; j < a.width; j += NT * 8) {
      const int left = (int)min((int64_t)8, a.width - j);
      float p[8], xhat[8], d[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
      get(j, left, p, xhat);
      if (a.dsum) load8<BF16>((const char *)a.dsum + row * a.dsum_stride * ES, j, left, d);
#pragma unroll
      for (int e = 0; e < 8; e++) p[e] = rstd * (p[e] - xhat[e] * mean) + d[e];
      store8<BF16>((char *)a.dx + row * a.dx_stride * ES, j, left, p);
    }
  }
}

/* dgain: a thread a column, the rows in order */
template <bool BF16>
__global__ __launch_bounds__(NT) void k_norm_dgain(NormGradArgs a) {
  for (int64_t j = (int64_t)blockIdx.x * NT + threadIdx.x; j < a.width; j += (int64_t)gridDim.x * NT) {
    float s = 0.0f;
    for (int64_t r = 0; r < a.n_rows; r++)
      s = fmaf(load_at<BF16>(a.dy, r * a.dy_stride + j), load_at<BF16>(a.h, r * a.h_stride + j) * a.rstd[r], s);
    a.dgain[j] = s;
  }
}

}  // namespace

void launch_norm(const NormArgs &args, Dtype dt, hipStream_t s) {
  const NormArgs a = args;
  const dim3 grid((unsigned)(a.n_rows < STEP_GRID ? a.n_rows : STEP_GRID));
  if (dt == DT_BF16)
    k_norm_rows<true><<<grid, NT, 0, s>>>(a);
  else
    k_norm_rows<false><<<grid, NT, 0, s>>>(a);
}

size_t norm_grad_workspace_bytes(int64_t, int64_t, bool) { return 0; }

void launch_norm_grad(const NormGradArgs &args, Dtype dt, void *, hipStream_t s) {
  const NormGradArgs a = args;
  /* (dgain first: dx may be dy or h) */
  const int64_t cols = (a.width + NT - 1) / NT;
  const dim3 strips((unsigned)(cols < STEP_GRID ? cols : STEP_GRID));
  const dim3 grid((unsigned)(a.n_rows < STEP_GRID ? a.n_rows : STEP_GRID));
  if (a.dgain) dt == DT_BF16 ? k_norm_dgain<true><<<strips, NT, 0, s>>>(a) : k_norm_dgain<false><<<strips, NT, 0, s>>>(a);
  if (!a.dx || a.n_rows == 0) return;
  dt == DT_BF16 ? k_norm_grad_rows<true><<<grid, NT, 0, s>>>(a) : k_norm_grad_rows<false><<<grid, NT, 0, s>>>(a);
}

}  // namespace d3s
