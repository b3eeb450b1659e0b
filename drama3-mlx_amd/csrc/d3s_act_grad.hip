/* k_act_grad: dz = dy act'(z) and its column sums (gfx950, wave64;
 * include/d3s_train.h).
 *
 * A workgroup takes a strip of columns (8 a lane) and a run of rows, its
 * threads `lanes` across and 256 / lanes rows at a time; each keeps its
 * columns' sums in fp32, the workgroup adds its threads' in order, and
 * k_column_sums adds the workgroups' in order.  No atomics: the sums do not
 * depend on which workgroup ends first.  Bound: HBM (two reads, one
 * write): 8192 x 2048 with silu and the sums 18 to 20 us (5.3 TB/s) and 3.9 of the second
 * launch; dz goes past the caches (through them 22.5 in all, so 21). */
#include "d3s_epilogue.h"

namespace d3s {
namespace {

constexpr int AT = 256;
constexpr int GRID_MOST = 1 << 22;

struct Split {
  int lanes, strips; /* lanes across, strips of 8 * lanes columns */
  int rows, runs;    /* rows a workgroup, runs of them */
};

Split split_of(int64_t m, int64_t n) {
  Split s;
  s.lanes = 1;
  while (s.lanes < WAVE && (int64_t)s.lanes * 8 < n) s.lanes *= 2;
  s.strips = (int)((n + s.lanes * 8 - 1) / (s.lanes * 8));
  const int at_once = AT / s.lanes;
  /* about 2048 workgroups (1024: 24.7 us for 8192 x 2048 with gelu, 2048: 22.5), each
   * of at least four rounds of rows */
  int64_t runs = 2048 / s.strips;
  if (runs < 1) runs = 1;
  int64_t rows = (m + runs - 1) / runs;
  rows = (rows + 4 * at_once - 1) / (4 * at_once) * (4 * at_once);
  if (rows > 0x7fffffff) rows = 0x7fffffff;
  s.rows = (int)rows;
  s.runs = rows ? (int)((m + rows - 1) / rows) : 0;
  return s;
}

template <bool SUM, int ACT>
__global__ __launch_bounds__(AT) void k_act_grad(ActGradArgs a, Split s, float *parts) {
  __shared__ float sum[SUM ? AT * 8 : 1];
  const int strip = (int)blockIdx.x % s.strips, run = (int)blockIdx.x / s.strips;
  const int across = (int)threadIdx.x % s.lanes, down = (int)threadIdx.x / s.lanes, at_once = AT / s.lanes;
  const int64_t j = ((int64_t)strip * s.lanes + across) * 8;
  const int64_t end = min((int64_t)a.m, (int64_t)(run + 1) * s.rows);
  float acc[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  const int left = j < a.n ? (int)min((int64_t)8, a.n - j) : 0;
  auto one = [&](float dy, float z) { return ACT == D3S_ACT_NONE ? dy : dy * slope<ACT>(z); };
  if (left == 8) {
#pragma unroll 2
    for (int64_t i = (int64_t)run * s.rows + down; i < end; i += at_once) {
      uint32_t d[4], z[4] = {0u, 0u, 0u, 0u}, w[4];
      __builtin_memcpy(d, a.dy + i * a.dy_stride + j, 16);
      if (ACT != D3S_ACT_NONE) __builtin_memcpy(z, a.z + i * a.z_stride + j, 16);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float x = one(d3s_u2f(d[e] << 16), d3s_u2f(z[e] << 16));
        const float y = one(d3s_u2f(d[e] & 0xffff0000u), d3s_u2f(z[e] & 0xffff0000u));
        acc[2 * e] += x;
        acc[2 * e + 1] += y;
        w[e] = pack2(x, y);
      }
      if (a.dz) stream16(a.dz + i * a.dz_stride + j, make_uint4(w[0], w[1], w[2], w[3]));
    }
  } else if (left > 0) {
    for (int64_t i = (int64_t)run * s.rows + down; i < end; i += at_once)
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (e < left) {
          const float v = one(bf(a.dy[i * a.dy_stride + j + e]), ACT != D3S_ACT_NONE ? bf(a.z[i * a.z_stride + j + e]) : 0.0f);
          acc[e] += v;
          if (a.dz) a.dz[i * a.dz_stride + j + e] = pack1(v);
        }
  }
  if constexpr (SUM) {
#pragma unroll
    for (int e = 0; e < 8; e++) sum[threadIdx.x * 8 + e] = acc[e];
    __syncthreads();
    const int cols = s.lanes * 8; /* up to 512 */
    for (int c = (int)threadIdx.x; c < cols; c += AT) {
      float v = 0.0f;
      for (int d = 0; d < at_once; d++) v += sum[d * cols + c];
      const int64_t col = (int64_t)strip * cols + c;
      if (col < a.n) parts[(int64_t)run * a.n + col] = v;
    }
  }
}

/* 16 columns a workgroup, 16 threads a column, each a sixteenth of the runs */
__global__ __launch_bounds__(AT) void k_column_sums(const float *parts, int runs, int n, int group0, float *dbias) {
  __shared__ float sum[16][17];
  const int c = (int)threadIdx.x % 16, q = (int)threadIdx.x / 16;
  const int64_t col = ((int64_t)group0 + blockIdx.x) * 16 + c;
  const int per = (runs + 15) / 16, r1 = min(runs, (q + 1) * per);
  float v = 0.0f;
  if (col < n) {
#pragma unroll 8
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

}  // namespace

size_t act_grad_workspace_bytes(int64_t m, int64_t n, bool dbias) {
  if (!dbias || m == 0 || n == 0) return 0;
  return split_counter_bytes() + (size_t)split_of(m, n).runs * (size_t)n * sizeof(float);
}

void launch_act_grad(const ActGradArgs &a, void *ws, hipStream_t s) {
  const Split sp = split_of(a.m, a.n);
  float *parts = ws ? (float *)((char *)ws + split_counter_bytes()) : nullptr;
  /* at most 2048 workgroups, or a strip of 512 columns each: 2^22 */
  const unsigned blocks = (unsigned)sp.strips * (unsigned)sp.runs;
  auto go = [&](auto kernel) { kernel<<<dim3(blocks), AT, 0, s>>>(a, sp, parts); };
  auto pick = [&](auto act) {
    constexpr int ACT = decltype(act)::value;
    a.dbias ? go(k_act_grad<true, ACT>) : go(k_act_grad<false, ACT>);
  };
  if (blocks) {
    switch (a.act) {
      case D3S_ACT_RELU: pick(std::integral_constant<int, D3S_ACT_RELU>{}); break;
      case D3S_ACT_SILU: pick(std::integral_constant<int, D3S_ACT_SILU>{}); break;
      case D3S_ACT_GELU: pick(std::integral_constant<int, D3S_ACT_GELU>{}); break;
      case D3S_ACT_GELU_TANH: pick(std::integral_constant<int, D3S_ACT_GELU_TANH>{}); break;
      default: pick(std::integral_constant<int, D3S_ACT_NONE>{});
    }
  }
  if (!a.dbias) return;
  const int64_t groups = ((int64_t)a.n + 15) / 16;
  /* (up to 2^27 workgroups: 2^35 threads would pass the launch's count) */
  for (int64_t g = 0; g < groups; g += GRID_MOST)
    k_column_sums<<<dim3((unsigned)min((int64_t)GRID_MOST, groups - g)), AT, 0, s>>>(
        parts, sp.runs, a.n, (int)g, a.dbias);
}

}  // namespace d3s
