/* k_dense: y = residual + act(x w^T + bias) on the matrix cores, bf16 operands
 * in either order, fp32 sums (gfx950, wave64; include/d3s_train.h). */
#include "d3s_epilogue.h"

namespace d3s {
namespace {

constexpr int GRID_MOST = 1 << 22; /* workgroups a launch: their threads are counted in 32 bits */

struct Operands {
  const uint16_t *x, *w;
  int64_t x_stride, w_stride;
  int k;
};

/* ---- any stride, any size ----
 * A 128 x 128 tile a workgroup of four waves (64 x 64 each, 4 x 4 tiles of
 * 16 x 16 x 32), stages of 32 of the inner length through registers into LDS,
 * every 8-element piece loaded whole where it lies inside and element by
 * element at the edges.  The weights are the first operand, so that a lane
 * holds four neighbouring outputs of one row. */
constexpr int DT_M = 128, DT_K = 32, DT_PAD = 8, DT_ROW = DT_K + DT_PAD;
constexpr int DT_OUT = 64 + 4; /* a row of outputs in LDS */

/* 8 elements of a stored row from `at`, zeros past `left` */
__device__ __forceinline__ uint4 piece(const uint16_t *p, int left) {
  uint4 q = make_uint4(0u, 0u, 0u, 0u);
  if (left >= 8) {
    __builtin_memcpy(&q, p, 16);
  } else if (left > 0) {
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (e < left) w[e / 2] |= (uint32_t)p[e] << (16 * (e & 1));
    q = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return q;
}

/* a stage of one operand: rows r0 .., inner k0 .. of [rows, k] (T: stored [k, rows]) */
template <bool T>
struct Stage {
  uint4 q[2];
  __device__ __forceinline__ void load(const uint16_t *p, int64_t stride, int rows, int k, int r0, int k0) {
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int i = (int)threadIdx.x + u * 256;
      if constexpr (T) { /* 32 stored rows of 128 */
        const int kk = k0 + i / 16, r = r0 + i % 16 * 8;
        q[u] = kk < k ? piece(p + (int64_t)kk * stride + r, rows - r) : make_uint4(0u, 0u, 0u, 0u);
      } else { /* 128 stored rows of 32 */
        const int r = r0 + i / 4, kk = k0 + i % 4 * 8;
        q[u] = r < rows ? piece(p + (int64_t)r * stride + kk, k - kk) : make_uint4(0u, 0u, 0u, 0u);
      }
    }
  }
  __device__ __forceinline__ void store(uint16_t *lds) const {
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int i = (int)threadIdx.x + u * 256;
      if constexpr (T) {
        const uint32_t w[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
#pragma unroll
        for (int e = 0; e < 8; e++) lds[(i % 16 * 8 + e) * DT_ROW + i / 16] = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
      } else {
        *(uint4 *)(lds + i / 4 * DT_ROW + i % 4 * 8) = q[u];
      }
    }
  }
};

template <bool XT, bool WT>
__global__ __launch_bounds__(256) void k_dense_any(Operands a, Out o, int n_tiles, int64_t tile0) {
  __shared__ __attribute__((aligned(16))) uint16_t lx[DT_M * DT_ROW], lw[DT_M * DT_ROW];
  const int64_t tile = tile0 + blockIdx.x;
  const int i0 = (int)(tile / n_tiles) * DT_M, j0 = (int)(tile % n_tiles) * DT_M;
  const int lane = lane_id(), wid = threadIdx.x / WAVE;
  const int wi = wid / 2 * 64, wj = wid % 2 * 64; /* the wave's rows and outputs */
  f32x4 acc[4][4];
#pragma unroll
  for (int p = 0; p < 4; p++)
#pragma unroll
    for (int q = 0; q < 4; q++) acc[p][q] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  Stage<XT> sx;
  Stage<WT> sw;
  if (a.k > 0) {
    sx.load(a.x, a.x_stride, o.m, a.k, i0, 0);
    sw.load(a.w, a.w_stride, o.n, a.k, j0, 0);
  }
  for (int k0 = 0; k0 < a.k; k0 += DT_K) {
    __syncthreads();
    sx.store(lx);
    sw.store(lw);
    __syncthreads();
    if (a.k - k0 > DT_K) {
      sx.load(a.x, a.x_stride, o.m, a.k, i0, k0 + DT_K);
      sw.load(a.w, a.w_stride, o.n, a.k, j0, k0 + DT_K);
    }
    bf16x8 fx[4], fw[4];
#pragma unroll
    for (int p = 0; p < 4; p++) {
      fx[p] = *(const bf16x8 *)(lx + (wi + p * 16 + (lane & 15)) * DT_ROW + (lane >> 4) * 8);
      fw[p] = *(const bf16x8 *)(lw + (wj + p * 16 + (lane & 15)) * DT_ROW + (lane >> 4) * 8);
    }
#pragma unroll
    for (int p = 0; p < 4; p++)
#pragma unroll
      for (int q = 0; q < 4; q++) acc[p][q] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw[q], fx[p], acc[p][q], 0, 0, 0);
  }
  /* 16 rows of the wave's 64 outputs at a time through its part of LDS, so that
   * a row's outputs leave in whole lines */
  __syncthreads();
  float *mine = (float *)(wid < 2 ? lx : lw) + (wid & 1) * 16 * DT_OUT;
#pragma unroll
  for (int p = 0; p < 4; p++) {
    wave_lds_sync();
#pragma unroll
    for (int q = 0; q < 4; q++) *(f32x4 *)(mine + (lane & 15) * DT_OUT + q * 16 + (lane >> 4) * 4) = acc[p][q];
    wave_lds_sync();
#pragma nounroll
    for (int r = lane >> 4; r < 16; r += 4)
      put_edge(o, i0 + wi + p * 16 + r, j0 + wj + (lane & 15) * 4, *(const f32x4 *)(mine + r * DT_OUT + (lane & 15) * 4));
  }
}

template <bool XT, bool WT>
void launch_any(const Operands &a, const Out &o, hipStream_t s) {
  const int n_tiles = (int)(((int64_t)o.n + DT_M - 1) / DT_M);
  const int64_t tiles = ((int64_t)o.m + DT_M - 1) / DT_M * n_tiles;
  for (int64_t t0 = 0; t0 < tiles; t0 += GRID_MOST)
    k_dense_any<XT, WT><<<dim3((unsigned)min((int64_t)GRID_MOST, tiles - t0)), 256, 0, s>>>(a, o, n_tiles, t0);
}

}  // namespace

size_t dense_workspace_bytes(const d3s_dense_params &p) { return 0; }

void launch_dense(const d3s_dense_params &p, void *ws, hipStream_t s) {
  const Operands a{p.x, p.w, p.x_stride, p.w_stride, (int)p.k};
  const Out o{p.bias,     p.residual, p.z,        p.y,        p.residual_stride, p.z_stride,
              p.y_stride, (int)p.m,   (int)p.n,   p.activation, p.y_dtype == D3S_DTYPE_F32};
  if (p.x_transposed)
    p.w_transposed ? launch_any<true, true>(a, o, s) : launch_any<true, false>(a, o, s);
  else
    p.w_transposed ? launch_any<false, true>(a, o, s) : launch_any<false, false>(a, o, s);
}

}  // namespace d3s
