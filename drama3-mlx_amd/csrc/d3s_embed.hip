/* k_embed, k_embed_grad: the rows that ids stand for, and their gradient in the
 * table (gfx950, wave64; include/d3s_step.h). */
#include "d3s_step_internal.h"
#include "d3s_vec.h"

namespace d3s {
namespace {

constexpr int ET = 256;

template <bool TB, bool YB>
__global__ __launch_bounds__(ET) void k_embed(EmbedArgs a, int lanes, int64_t strips, int64_t blocks) {
  const int across = (int)threadIdx.x % lanes, down = (int)threadIdx.x / lanes;
  for (int64_t blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
    const int64_t row = blk / strips * (ET / lanes) + down;
    const int64_t j = (blk % strips * lanes + across) * 8;
    if (row >= a.n_rows || j >= a.width) continue;
    const int left = (int)min((int64_t)8, a.width - j);
    float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    for (int t = 0; t < a.n_ids; t++) {
      const int id = a.ids[row * a.n_ids + t];
      if ((uint32_t)id >= (uint64_t)a.vocab) continue;
      float w[8];
      load8<TB>((const char *)a.in + (t * a.slot_rows + id) * a.in_stride * (TB ? 2 : 4), j, left, w);
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] += w[e];
    }
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] *= a.scale;
    store8<YB>((char *)a.out + row * a.out_stride * (YB ? 2 : 4), j, left, v);
  }
}

constexpr int GR = 8;         /* rows of the table that a workgroup sums */
constexpr int GC = ET * 8;    /* by columns */
constexpr int LOOK = ET * 4;  /* ids looked at together */

/* GR rows of one slot's part by GC columns, summed in LDS: the ids are looked
 * through in order, and those of these rows gathered in that order. */
template <bool DB, bool GB>
__global__ __launch_bounds__(ET) void k_embed_grad(EmbedArgs a, int64_t slots, int64_t part, int64_t blocks_part,
                                                   int64_t strips, int64_t blocks) {
  __shared__ float sum[GR][GC];
  __shared__ int64_t found[LOOK];
  __shared__ int which[LOOK];
  __shared__ int counts[ET / WAVE];
  const int tid = (int)threadIdx.x;
  const int64_t n = slots > 1 ? a.n_rows : a.n_rows * a.n_ids; /* ids to look through */
  for (int64_t blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
    const int64_t strip = blk % strips, slot = blk / strips / blocks_part;
    const int64_t v0 = blk / strips % blocks_part * GR;
    const int64_t j = strip * GC + tid * 8;
    const int left = j < a.width ? (int)min((int64_t)8, a.width - j) : 0;
    for (int r = 0; r < GR; r++)
      for (int e = 0; e < 8; e++) sum[r][e * ET + tid] = 0.0f;
    for (int64_t base = 0; base < n; base += LOOK) {
      /* a thread's four ids follow each other */
      int hit[4], mine = 0;
      for (int u = 0; u < 4; u++) {
        const int64_t i = base + tid * 4 + u;
        hit[u] = -1;
        if (i < n) {
          const int id = a.ids[slots > 1 ? i * a.n_ids + slot : i];
          if (id >= v0 && id < v0 + GR && id < a.vocab) hit[u] = (int)(id - v0), mine++;
        }
      }
      const uint32_t incl = wave_scan_add_u32((uint32_t)mine);
      __syncthreads();
      if (lane_id() == WAVE - 1) counts[tid / WAVE] = (int)incl;
      __syncthreads();
      int at = (int)incl - mine, total = 0;
      for (int w = 0; w < ET / WAVE; w++) {
        if (w < tid / WAVE) at += counts[w];
        total += counts[w];
      }
      for (int u = 0; u < 4; u++)
        if (hit[u] >= 0) {
          const int64_t i = base + tid * 4 + u;
          found[at] = slots > 1 ? i : i / a.n_ids;
          which[at++] = hit[u];
        }
      __syncthreads();
      for (int f = 0; f < total && left > 0; f++) {
        float d[8];
        load8<DB>((const char *)a.in + found[f] * a.in_stride * (DB ? 2 : 4), j, left, d);
#pragma unroll
        for (int e = 0; e < 8; e++) sum[which[f]][e * ET + tid] += d[e];
      }
    }
    for (int r = 0; r < GR && left > 0; r++) {
      if (v0 + r >= part) break;
      const int64_t row = slot * a.slot_rows + v0 + r;
      if (a.slot_rows && slot == slots - 1 && v0 + r >= a.vocab) break;
      if (a.accumulate && v0 + r >= a.vocab) break;
      char *out = (char *)a.out + row * a.out_stride * (GB ? 2 : 4);
      float v[8], o[8];
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = sum[r][e * ET + tid] * a.scale;
      if (a.accumulate) {
        load8<GB>(out, j, left, o);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] += o[e];
      }
      store8<GB>(out, j, left, v);
    }
    __syncthreads();
  }
}

}  // namespace

void launch_embed(const EmbedArgs &args, Dtype in, Dtype out, hipStream_t s) {
  const EmbedArgs a = args;
  int lanes = 1;
  while (lanes < ET && (int64_t)lanes * 8 < a.width) lanes *= 2;
  const int64_t strips = (a.width + lanes * 8 - 1) / (lanes * 8);
  const int64_t blocks = strips * ((a.n_rows + ET / lanes - 1) / (ET / lanes));
  const dim3 grid((unsigned)(blocks < STEP_GRID ? blocks : STEP_GRID));
  auto go = [&](auto kernel) { kernel<<<grid, ET, 0, s>>>(a, lanes, strips, blocks); };
  if (in == DT_BF16)
    out == DT_BF16 ? go(k_embed<true, true>) : go(k_embed<true, false>);
  else
    out == DT_BF16 ? go(k_embed<false, true>) : go(k_embed<false, false>);
}

size_t embed_grad_workspace_bytes(int64_t, int, int64_t, int64_t, int64_t) { return 0; }

void launch_embed_grad(const EmbedArgs &args, Dtype in, Dtype out, void *, hipStream_t s) {
  const EmbedArgs a = args;
  const int64_t slots = a.slot_rows ? a.n_ids : 1, part = a.slot_rows ? a.slot_rows : a.vocab;
  const int64_t blocks_part = (part + GR - 1) / GR, strips = (a.width + GC - 1) / GC;
  const int64_t blocks = slots * blocks_part * strips;
  const dim3 grid((unsigned)(blocks < STEP_GRID ? blocks : STEP_GRID));
  auto go = [&](auto kernel) { kernel<<<grid, ET, 0, s>>>(a, slots, part, blocks_part, strips, blocks); };
  if (in == DT_BF16)
    out == DT_BF16 ? go(k_embed_grad<true, true>) : go(k_embed_grad<true, false>);
  else
    out == DT_BF16 ? go(k_embed_grad<false, true>) : go(k_embed_grad<false, false>);
}

}  // namespace d3s
