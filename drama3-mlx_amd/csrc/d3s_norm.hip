/* k_norm, k_norm_grad: root-mean-square norm with the residual's addition and an
 * output in 8 bits, and its gradient (gfx950, wave64; include/d3s_step.h).
 *
 * A row's inputs are read once, all in flight together, and stay in registers: up to 256
 * columns a part of a wave a row, up to 2048 (the gradient's three rows: 1024) a wave, up to 16384 a workgroup of 256 to
 * 1024 threads; longer rows are read once for each pass (k_norm_rows, k_norm_grad_rows, k_norm_dgain).  Squares are summed in fp32,
 * a lane's in order and then by a tree.  h stays in fp32 from the addition to y; rstd is
 * a correctly rounded root and quotient.  8 bits: a group's greatest |y| by exchanges among the lanes
 * that hold it, its scale an fp32 quotient, each y rounded once.
 * The gradient's column sums (dgain) stay in registers over the rows that a workgroup takes, one row of sums
 * for each workgroup goes to the workspace, and a second launch adds them in order: no atomics.
 *
 * Bound: HBM.  bf16 8192 x 2048 with residual and kept sum, e4m3 by groups of 128: 25.7 us (4.6 TB/s);
 * its gradient with dsum and dgain 28 us (4.8 TB/s) and 4.4 of the second launch; 100000 x 64
 * 9.7 us (5.3 TB/s).  One row of 2048: 3.5 us, a launch and two dependent loads' latency. */
#include "d3s_colsums.h"
#include "d3s_step_internal.h"
#include "d3s_vec.h"

namespace d3s {
namespace {

constexpr int NT = 256;
constexpr int NW = NT / WAVE;
constexpr float E4M3_MOST = 448.0f;

/* the sum (or greatest) over a workgroup of T threads, in every thread, added in one order */
template <int T>
__device__ __forceinline__ float block_sum(float v, float *part) {
  v = readlane_f(wave_scan_add_f32(v), 63);
  __syncthreads();
  if (lane_id() == 0) part[threadIdx.x / WAVE] = v;
  __syncthreads();
  float t = 0.0f;
#pragma unroll
  for (int w = 0; w < T / WAVE; w++) t += part[w];
  return t;
}
template <int T>
__device__ __forceinline__ float block_max(float v, float *part) {
  v = wave_max_f(v);
  __syncthreads();
  if (lane_id() == 0) part[threadIdx.x / WAVE] = v;
  __syncthreads();
  float t = part[0];
#pragma unroll
  for (int w = 1; w < T / WAVE; w++) t = __builtin_elementwise_maximum(t, part[w]);
  return t;
}

/* eight values over their group's scale, as 8 bits; saturating: the greatest quotient is
 * 448 and a rounding.  The quotient is the correctly rounded one of fp32, by the scale's reciprocal in 64 bits: the
 * product is within 2^-52 of it, and no quotient of two 24-bit numbers is nearer than 2^-49 (both relative) to
 * the middle of two fp32 numbers, which has 25. */
__device__ __forceinline__ uint64_t pack_e4m3(const float *v, float scale) {
  uint32_t w[2] = {0u, 0u};
  float q[8];
  const double inv = scale == 0.0f ? 0.0 : 1.0 / (double)scale;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    q[e] = (float)((double)v[e] * inv);
    q[e] = __builtin_elementwise_minimum(__builtin_elementwise_maximum(q[e], -E4M3_MOST), E4M3_MOST); /* (NaN stays) */
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

/* the sum (or greatest) over the G threads of a row, in each of them, added in one order */
template <int G>
__device__ __forceinline__ float row_sum(float v, float *part) {
  if constexpr (G >= NT) return block_sum<G>(v, part);
  if constexpr (G == WAVE) return readlane_f(wave_scan_add_f32(v), 63);
#pragma unroll
  for (int d = 1; d < G; d *= 2) v += __shfl_xor(v, d);
  return v;
}
template <int G>
__device__ __forceinline__ float row_max(float v, float *part) {
  if constexpr (G >= NT) return block_max<G>(v, part);
  if constexpr (G == WAVE) return wave_max_f(v);
#pragma unroll
  for (int d = 1; d < G; d *= 2) v = __builtin_elementwise_maximum(v, __shfl_xor(v, d));
  return v;
}

/* threads of a workgroup whose rows are held by G each */
constexpr int row_threads(int G) { return G > NT ? G : NT; }

/* G threads hold a row, U chunks of eight elements each, in registers: one read of
 * everything, all of it in flight together. */
/* elements that follow each other in a lane: as many as make a store of 16 bytes; eight for 8 bits */
template <bool BF16, int OUT>
constexpr int norm_elements() { return OUT != D3S_DTYPE_E4M3 && (!BF16 || OUT == D3S_DTYPE_F32) ? 4 : 8; }

template <bool BF16, int OUT, int G, int U>
__global__ __launch_bounds__(row_threads(G)) void k_norm(NormArgs a) {
  constexpr int ES = BF16 ? 2 : 4, ROWS = row_threads(G) / G, E = norm_elements<BF16, OUT>();
  __shared__ float part[row_threads(G) / WAVE];
  const int g = (int)threadIdx.x % G;
  for (int64_t row0 = (int64_t)blockIdx.x * ROWS; row0 < a.n_rows; row0 += (int64_t)gridDim.x * ROWS) {
    const int64_t row = min(row0 + threadIdx.x / G, a.n_rows - 1);
    const bool mine = row0 + threadIdx.x / G < a.n_rows; /* (the others shadow the last row and store nothing) */
    const int width = (int)a.width;
    const char *x = (const char *)a.x + row * a.x_stride * ES;
    Vec<BF16, E> q[U], r[U], w[U];
#pragma unroll
    for (int u = 0; u < U; u++) q[u].load_some(x, (u * G + g) * E, width - (u * G + g) * E);
    if (a.residual) {
      const char *res = (const char *)a.residual + row * a.residual_stride * ES;
#pragma unroll
      for (int u = 0; u < U; u++) r[u].load_some(res, (u * G + g) * E, width - (u * G + g) * E);
    }
    if (a.gain) {
#pragma unroll
      for (int u = 0; u < U; u++) w[u].load_some(a.gain, (u * G + g) * E, width - (u * G + g) * E);
    }
    float h[U][E], s = 0.0f;
#pragma unroll
    for (int u = 0; u < U; u++) {
      q[u].values(h[u]);
      if (a.residual) {
        float t[E];
        r[u].values(t);
#pragma unroll
        for (int e = 0; e < E; e++) h[u][e] += t[e];
      }
#pragma unroll
      for (int e = 0; e < E; e++) s = fmaf(h[u][e], h[u][e], s);
    }
    if (a.sum && mine) {
#pragma unroll
      for (int u = 0; u < U; u++)
        store_row<BF16, E, BF16 || E == 4>((char *)a.sum + row * a.sum_stride * ES, (u * G + g) * E, width - (u * G + g) * E, h[u]);
    }
    s = row_sum<G>(s, part);
    const float rstd = 1.0f / sqrtf(s / (float)width + a.eps);
    if (g == 0 && a.rstd && mine) a.rstd[row] = rstd;
#pragma unroll
    for (int u = 0; u < U; u++) {
      float t[E];
      if (a.gain) w[u].values(t);
#pragma unroll
      for (int e = 0; e < E; e++) {
        h[u][e] *= rstd;
        if (a.gain) h[u][e] *= t[e];
      }
    }
    if constexpr (OUT != D3S_DTYPE_E4M3) {
      constexpr int YS = OUT == D3S_DTYPE_BF16 ? 2 : 4;
      if (mine) {
#pragma unroll
        for (int u = 0; u < U; u++)
          store_row<OUT == D3S_DTYPE_BF16, E>((char *)a.y + row * a.y_stride * YS, (u * G + g) * E, width - (u * G + g) * E, h[u]);
      }
    } else {
      /* (places past the row hold x = 0 and, where rstd is infinite, 0 times it: not looked at) */
      float most[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        most[u] = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++)
          most[u] = __builtin_elementwise_maximum(most[u], (u * G + g) * E + e < width ? fabsf(h[u][e]) : 0.0f);
      }
      if (a.group == 0) {
#pragma unroll
        for (int u = 1; u < U; u++) most[0] = __builtin_elementwise_maximum(most[0], most[u]);
        most[0] = row_max<G>(most[0], part);
#pragma unroll
        for (int u = 1; u < U; u++) most[u] = most[0];
      } else {
        for (int d = 1; d < min(a.group / 8, G); d *= 2)
#pragma unroll
          for (int u = 0; u < U; u++) most[u] = __builtin_elementwise_maximum(most[u], __shfl_xor(most[u], d));
      }
      const int size = a.group ? a.group : width;
      const int64_t groups = (width + size - 1) / size;
      uint8_t *y = (uint8_t *)a.y + row * a.y_stride;
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int j = (u * G + g) * E, left = width - j;
        const float scale = e4m3_scale(most[u]);
        if (left <= 0 || !mine) continue;
        if (a.group ? j % a.group == 0 : j == 0) a.scales[row * groups + (a.group ? j / a.group : 0)] = scale;
        const uint64_t p = pack_e4m3(h[u], scale);
        if (left >= 8)
          __builtin_memcpy(y + j, &p, 8);
        else
          for (int e = 0; e < left; e++) y[j + e] = (uint8_t)(p >> 8 * e);
      }
    }
  }
}

/* The gradient, rows held the same way; a workgroup takes every gridDim.x-th set of
 * rows and keeps their columns' sums of dy xhat in registers. */
template <bool BF16, int G, int U, bool SUM>
__global__ __launch_bounds__(row_threads(G)) void k_norm_grad(NormGradArgs a, float *parts) {
  constexpr int ES = BF16 ? 2 : 4, ROWS = row_threads(G) / G, E = BF16 ? 8 : 4;
  __shared__ float part[row_threads(G) / WAVE];
  __shared__ float sums[SUM && ROWS > 1 ? NT * U * E : 1];
  const int g = (int)threadIdx.x % G, width = (int)a.width;
  Vec<BF16, E> w[U];
  if (a.gain) {
#pragma unroll
    for (int u = 0; u < U; u++) w[u].load_some(a.gain, (u * G + g) * E, width - (u * G + g) * E);
  }
  float acc[U][E];
#pragma unroll
  for (int u = 0; u < U; u++)
#pragma unroll
    for (int e = 0; e < E; e++) acc[u][e] = 0.0f;
  /* a row's inputs; the next row's are loaded while this one is worked on, where registers allow */
  constexpr bool AHEAD = U * E <= 8 || (G <= WAVE && U * E <= 16);
  struct In {
    Vec<BF16, E> d[U], h[U], r[U];
    float rstd;
  };
  auto get = [&](int64_t row0, In &in) {
    const int64_t row = min(row0 + threadIdx.x / G, a.n_rows - 1);
#pragma unroll
    for (int u = 0; u < U; u++) {
      in.d[u].load_some((const char *)a.dy + row * a.dy_stride * ES, (u * G + g) * E, width - (u * G + g) * E);
      in.h[u].load_some((const char *)a.h + row * a.h_stride * ES, (u * G + g) * E, width - (u * G + g) * E);
    }
    if (a.dsum && a.dx) {
#pragma unroll
      for (int u = 0; u < U; u++)
        in.r[u].load_some((const char *)a.dsum + row * a.dsum_stride * ES, (u * G + g) * E, width - (u * G + g) * E);
    }
    in.rstd = a.rstd[row];
  };
  In in, next;
  const int64_t step = (int64_t)gridDim.x * ROWS;
  if (AHEAD) get((int64_t)blockIdx.x * ROWS, in); /* (there is no workgroup without a row) */
  for (int64_t row0 = (int64_t)blockIdx.x * ROWS; row0 < a.n_rows; row0 += step) {
    const int64_t row = min(row0 + threadIdx.x / G, a.n_rows - 1);
    const bool mine = row0 + threadIdx.x / G < a.n_rows;
    if (!AHEAD) {
      get(row0, in);
    } else {
      if (row0 > (int64_t)blockIdx.x * ROWS) in = next;
      if (row0 + step < a.n_rows) get(row0 + step, next);
    }
    const auto &d = in.d, &h = in.h, &r = in.r;
    const float rstd = in.rstd;
    float s = 0.0f;
#pragma unroll
    for (int u = 0; u < U; u++) {
      float p[E], t[E], k[E];
      d[u].values(p);
      h[u].values(t);
      if (a.gain) w[u].values(k);
#pragma unroll
      for (int e = 0; e < E; e++) {
        const float xhat = t[e] * rstd;
        if (SUM && mine && (u * G + g) * E + e < width) acc[u][e] = fmaf(p[e], xhat, acc[u][e]);
        s = fmaf(a.gain ? p[e] * k[e] : p[e], (u * G + g) * E + e < width ? xhat : 0.0f, s);
      }
    }
    if (!a.dx) continue; /* (uniform) */
    const float mean = row_sum<G>(s, part) / (float)width;
    if (!mine) continue; /* (G == NT: always its own) */
#pragma unroll
    for (int u = 0; u < U; u++) {
      float p[E], t[E], k[E], o[E];
      d[u].values(p);
      h[u].values(t);
      if (a.gain) w[u].values(k);
      if (a.dsum) r[u].values(o);
#pragma unroll
      for (int e = 0; e < E; e++) {
        const float v = rstd * ((a.gain ? p[e] * k[e] : p[e]) - t[e] * rstd * mean);
        o[e] = a.dsum ? v + o[e] : v;
      }
      store_row<BF16, E>((char *)a.dx + row * a.dx_stride * ES, (u * G + g) * E, width - (u * G + g) * E, o);
    }
  }
  if constexpr (SUM) {
    float *out = parts + (int64_t)blockIdx.x * a.width;
    if constexpr (ROWS == 1) {
#pragma unroll
      for (int u = 0; u < U; u++)
        store_row<false, E, false>(out, (u * G + g) * E, width - (u * G + g) * E, acc[u]);
    } else {
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < E; e++) sums[(threadIdx.x / G) * (G * U * E) + (u * G + g) * E + e] = acc[u][e];
      __syncthreads();
      for (int j = (int)threadIdx.x; j < width; j += NT) {
        float v = 0.0f;
#pragma unroll 4
        for (int i = 0; i < ROWS; i++) v += sums[i * (G * U * E) + j];
        out[j] = v;
      }
    }
  }
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
      load_row<BF16, 8>(x, j, left, h);
      if (res) {
        float r[8];
        load_row<BF16, 8>(res, j, left, r);
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
    s = block_sum<NT>(s, part);
    const float rstd = 1.0f / sqrtf(s / (float)a.width + a.eps);
    if (tid == 0 && a.rstd) a.rstd[row] = rstd;
    auto scaled = [&](int64_t j, int left, float *h) {
      float g[8] = {1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f};
      if (a.gain) load_row<BF16, 8>(a.gain, j, left, g);
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
      row_scale = e4m3_scale(block_max<NT>(most, part));
      if (tid == 0) a.scales[row] = row_scale;
    }
    for (int64_t base = 0; base < a.width; base += NT * 8) {
      const int64_t j = base + tid * 8;
      const int left = left_at(j);
      float h[8];
      get(j, left, h);
      if (a.sum && left > 0) store_row<BF16, 8, BF16>((char *)a.sum + row * a.sum_stride * ES, j, left, h);
      scaled(j, left, h);
      if (a.y_dtype == D3S_DTYPE_BF16) {
        if (left > 0) store_row<true, 8>((char *)a.y + row * a.y_stride * 2, j, left, h);
      } else if (a.y_dtype == D3S_DTYPE_F32) {
        if (left > 0) store_row<false, 8, false>((char *)a.y + row * a.y_stride * 4, j, left, h);
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
      load_row<BF16, 8>(dy, j, left, p);
      load_row<BF16, 8>(h, j, left, xhat);
      if (a.gain) load_row<BF16, 8>(a.gain, j, left, g);
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
    const float mean = block_sum<NT>(s, part) / (float)a.width;
    for (int64_t j = tid * 8; j < a.width; j += NT * 8) {
      const int left = (int)min((int64_t)8, a.width - j);
      float p[8], xhat[8], d[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
      get(j, left, p, xhat);
      if (a.dsum) load_row<BF16, 8>((const char *)a.dsum + row * a.dsum_stride * ES, j, left, d);
#pragma unroll
      for (int e = 0; e < 8; e++) p[e] = rstd * (p[e] - xhat[e] * mean) + d[e];
      store_row<BF16, 8, BF16>((char *)a.dx + row * a.dx_stride * ES, j, left, p);
    }
  }
}

/* dgain of rows too long for registers: a thread a column, a run of rows each */
template <bool BF16>
__global__ __launch_bounds__(NT) void k_norm_dgain(NormGradArgs a, int64_t strips, int rows, float *parts) {
  const int64_t j = (int64_t)blockIdx.x % strips * NT + threadIdx.x, run = blockIdx.x / strips;
  if (j >= a.width) return;
  float s = 0.0f;
#pragma unroll 4
  for (int64_t r = run * rows; r < min(a.n_rows, (run + 1) * rows); r++)
    s = fmaf(load_at<BF16>(a.dy, r * a.dy_stride + j), load_at<BF16>(a.h, r * a.h_stride + j) * a.rstd[r], s);
  parts[run * a.width + j] = s;
}

/* f(T) for a workgroup of T threads, as few as hold `chunks` of a row, or false */
template <int... T, class F>
bool of_threads(int64_t chunks, F f) {
  return ((chunks <= T && (f(std::integral_constant<int, T>{}), true)) || ...);
}

/* The threads and chunks of E elements that hold a row: f(G, U), or false for one that is streamed.
 * Beyond 2048 columns a workgroup of about as many threads as have eight elements each, or 16 (bf16 6553 x 2560
 * 21 us, fp32 1524 x 11008 56; 256 threads that hold up to 64, 23.5 and 111); of 8 bits, whose groups' lanes wait for
 * each other, 16 where they can (4096 x 4096 23 us, 8 elements 26.6). */
template <int E, bool U1, class F>
bool in_registers(int64_t width, F f) { /* (U1: eight may do) */
  constexpr int M = 8 / E;
  using std::integral_constant;
  auto go = [&](auto g, auto u) { return f(g, u), true; };
  if (width <= 64) return go(integral_constant<int, 8>{}, integral_constant<int, M>{});
  if (width <= 128) return go(integral_constant<int, 16>{}, integral_constant<int, M>{});
  if (width <= 256) return go(integral_constant<int, 32>{}, integral_constant<int, M>{});
  if (width <= 512) return go(integral_constant<int, 64>{}, integral_constant<int, M>{});
  if (width <= 1024) return go(integral_constant<int, 64>{}, integral_constant<int, 2 * M>{});
  if (width <= 2048) return go(integral_constant<int, 64>{}, integral_constant<int, 4 * M>{});
  const int64_t chunks = (width + 7) / 8;
  return (U1 && of_threads<320, 384, 512, 640, 768, 1024>(chunks, [&](auto t) { go(t, integral_constant<int, M>{}); })) ||
         of_threads<256, 320, 384, 512, 640, 768, 1024>((chunks + 1) / 2, [&](auto t) { go(t, integral_constant<int, 2 * M>{}); });
}

/* The same for the gradient, whose inputs are three rows and whose sums stay: beyond 1024 columns a
 * workgroup a row, of as many threads as leave 8 elements each, so that the next row's loads fit beside them
 * (8192 x 2048 bf16: 32 us; a wave a row, without loads ahead, 43.  4096 x 5000 fp32: 80 us; 256 threads
 * 114).  32 beyond 8192 (1024 x 16384 fp32: 68 us; 1024 threads, whose registers spill, 77). */
template <int E, class F>
bool grad_in_registers(int64_t width, F f) {
  constexpr int M = 8 / E;
  auto go = [&](auto g, auto u) { return f(g, u), true; };
  using std::integral_constant;
  if (width <= 1024) return in_registers<E, false>(width, f);
  const int64_t chunks = (width + 7) / 8;
  return of_threads<256, 512, 1024>(chunks, [&](auto t) { go(t, integral_constant<int, M>{}); }) ||
         of_threads<512>((chunks + 3) / 4, [&](auto t) { go(t, integral_constant<int, 4 * M>{}); });
}

/* Workgroups of the gradient: the runs of its column sums.  As many as are resident (512: 36 us for
 * 8192 x 2048, 768 and 1024: 32, 1280 and 2048: 38); of wide rows fewer, since each leaves a row of
 * sums (4096 x 4096 bf16 with 512, 768 and 1024: 31, 37 and 37; 2048 x 8192 with 256, 384 and 512: 33, 41 and
 * 38). */
int64_t grad_runs(int64_t width) { return width <= 2048 ? 1024 : width <= 4096 ? 512 : 256; }
struct GradSplit {
  int64_t strips;
  int rows, runs;
};
GradSplit grad_split(int64_t n_rows, int64_t width) {
  GradSplit p{1, 0, 0};
  const bool held = grad_in_registers<8>(width, [&](auto g, auto) { p.rows = row_threads(decltype(g)::value) / decltype(g)::value; });
  if (held) {
    const int64_t sets = (n_rows + p.rows - 1) / p.rows;
    p.runs = (int)(sets < grad_runs(width) ? sets : grad_runs(width));
  } else {
    p.strips = (width + NT - 1) / NT;
    int64_t runs = 1024 / p.strips;
    if (runs < 1) runs = 1;
    p.rows = (int)((n_rows + runs - 1) / runs);
    p.runs = p.rows ? (int)((n_rows + p.rows - 1) / p.rows) : 0;
  }
  return p;
}

}  // namespace

void launch_norm(const NormArgs &args, Dtype dt, hipStream_t s) {
  const NormArgs a = args;
  auto grid = [&](int rows) {
    const int64_t n = (a.n_rows + rows - 1) / rows;
    return dim3((unsigned)(n < STEP_GRID ? n : STEP_GRID));
  };
  auto held = [&](auto bf16, auto type) {
    constexpr bool B = decltype(bf16)::value;
    constexpr int OUT = decltype(type)::value;
    return in_registers<norm_elements<B, OUT>(), OUT != D3S_DTYPE_E4M3>(a.width, [&](auto g, auto u) {
      constexpr int G = decltype(g)::value, T = row_threads(G);
      k_norm<B, OUT, G, decltype(u)::value><<<grid(T / G), T, 0, s>>>(a);
    });
  };
  auto of_type = [&](auto bf16) {
    return a.y_dtype == D3S_DTYPE_BF16  ? held(bf16, std::integral_constant<int, D3S_DTYPE_BF16>{})
           : a.y_dtype == D3S_DTYPE_F32 ? held(bf16, std::integral_constant<int, D3S_DTYPE_F32>{})
                                        : held(bf16, std::integral_constant<int, D3S_DTYPE_E4M3>{});
  };
  if (dt == DT_BF16 ? of_type(std::true_type{}) : of_type(std::false_type{})) return;
  if (dt == DT_BF16)
    k_norm_rows<true><<<grid(1), NT, 0, s>>>(a);
  else
    k_norm_rows<false><<<grid(1), NT, 0, s>>>(a);
}

size_t norm_grad_workspace_bytes(int64_t n_rows, int64_t width, bool dgain) {
  if (!dgain || n_rows == 0 || width == 0) return 0;
  const int runs = grad_split(n_rows, width).runs;
  return runs == 1 ? 0 : split_counter_bytes() + (size_t)runs * (size_t)width * sizeof(float);
}

void launch_norm_grad(const NormGradArgs &args, Dtype dt, void *ws, hipStream_t s) {
  const NormGradArgs a = args;
  const GradSplit p = grad_split(a.n_rows, a.width);
  /* (one run's sums are dgain) */
  float *parts = p.runs == 1 ? a.dgain : ws ? (float *)((char *)ws + split_counter_bytes()) : nullptr;
  auto rows_held = [&](auto bf16) {
    constexpr bool B = decltype(bf16)::value;
    return grad_in_registers<B ? 8 : 4>(a.width, [&](auto g, auto u) {
      constexpr int G = decltype(g)::value, U = decltype(u)::value;
      constexpr int T = row_threads(G);
      if (a.dgain)
        k_norm_grad<B, G, U, true><<<dim3((unsigned)p.runs), T, 0, s>>>(a, parts);
      else
        k_norm_grad<B, G, U, false><<<dim3((unsigned)p.runs), T, 0, s>>>(a, parts);
    });
  };
  const bool held = p.runs && (dt == DT_BF16 ? rows_held(std::true_type{}) : rows_held(std::false_type{}));
  if (!held && p.runs) { /* (dgain first: dx may be dy or h) */
    const dim3 strips((unsigned)(p.strips * p.runs)), rows((unsigned)(a.n_rows < STEP_GRID ? a.n_rows : STEP_GRID));
    if (a.dgain) {
      if (dt == DT_BF16)
        k_norm_dgain<true><<<strips, NT, 0, s>>>(a, p.strips, p.rows, parts);
      else
        k_norm_dgain<false><<<strips, NT, 0, s>>>(a, p.strips, p.rows, parts);
    }
    if (a.dx) dt == DT_BF16 ? k_norm_grad_rows<true><<<rows, NT, 0, s>>>(a) : k_norm_grad_rows<false><<<rows, NT, 0, s>>>(a);
  }
  if (a.dgain && p.runs != 1) launch_column_sums(parts, p.runs, (int)a.width, a.dgain, s);
}

}  // namespace d3s
