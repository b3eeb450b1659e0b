/* k_dropout: y = residual + kept x / (1 - p), the mask drawn from Philox as it is
 * used (gfx950, wave64; include/d3s_step.h). */
#include "d3s_step_internal.h"
#include "d3s_vec.h"

namespace d3s {
namespace {

constexpr int DT_ = 256;

/* a workgroup takes DT_ / lanes rows by E * lanes columns */
struct DropSplit {
  int lanes;
  int64_t strips, blocks;
};

DropSplit drop_split(int64_t rows, int64_t width, int E) {
  DropSplit s;
  s.lanes = 1;
  while (s.lanes < DT_ && (int64_t)s.lanes * E < width) s.lanes *= 2;
  s.strips = (width + s.lanes * E - 1) / (s.lanes * E);
  s.blocks = s.strips * ((rows + DT_ / s.lanes - 1) / (DT_ / s.lanes));
  return s;
}

/* WHOLE: every lane's first element is a multiple of four in the generator's count, so that its
 * words are whole blocks of Philox; else it draws one block more and takes its words from
 * among them. */
template <bool BF16, bool WHOLE>
__global__ __launch_bounds__(DT_) void k_dropout(DropoutArgs a, DropSplit sp) {
  constexpr int E = BF16 ? 8 : 4, ES = BF16 ? 2 : 4, B = E / 4 + (WHOLE ? 0 : 1);
  const int across = (int)threadIdx.x % sp.lanes, down = (int)threadIdx.x / sp.lanes;
  const uint64_t draw = a.draw + (a.draw_add ? *a.draw_add : 0u);
  for (int64_t blk = blockIdx.x; blk < sp.blocks; blk += gridDim.x) {
    const int64_t row = blk / sp.strips * (DT_ / sp.lanes) + down;
    const int64_t j = (blk % sp.strips * sp.lanes + across) * E, left = a.width - j;
    if (row >= a.n_rows || left <= 0) continue;
    Vec<BF16, E> x, r;
    x.load_some((const char *)a.x + row * a.x_stride * ES, j, left);
    if (a.residual) r.load_some((const char *)a.residual + row * a.residual_stride * ES, j, left);
    const uint64_t at = (uint64_t)row * (uint64_t)a.width + (uint64_t)j;
    uint32_t w[4 * B];
#pragma unroll
    for (int b = 0; b < B; b++) {
      const uint64_t q = (at >> 2) + b;
      const d3s_u32x4 o = d3s_philox4x32_10({{(uint32_t)q, (uint32_t)(q >> 32), (uint32_t)draw, (uint32_t)(draw >> 32)}},
                                            (uint32_t)a.seed, (uint32_t)(a.seed >> 32));
#pragma unroll
      for (int i = 0; i < 4; i++) w[4 * b + i] = o.v[i];
    }
    if constexpr (!WHOLE) { /* the words from at & 3 on */
      const uint32_t s = (uint32_t)at & 3u;
#pragma unroll
      for (int e = 0; e < E + 2; e++) w[e] = s & 1u ? w[e + 1] : w[e];
#pragma unroll
      for (int e = 0; e < E; e++) w[e] = s & 2u ? w[e + 2] : w[e];
    }
    float v[E], o[E];
    x.values(v);
    if (a.residual) r.values(o);
#pragma unroll
    for (int e = 0; e < E; e++) {
      v[e] = (w[e] >> 8) >= a.least ? v[e] * a.scale : 0.0f;
      if (a.residual) v[e] += o[e];
    }
    store_row<BF16, E>((char *)a.y + row * a.y_stride * ES, j, left, v);
  }
}

}  // namespace

void launch_dropout(const DropoutArgs &args, Dtype dt, hipStream_t s) {
  DropoutArgs a = args;
  /* rows that follow each other are one */
  if (a.x_stride == a.width && a.y_stride == a.width && (!a.residual || a.residual_stride == a.width)) {
    a.width *= a.n_rows;
    a.n_rows = 1;
  }
  const DropSplit sp = drop_split(a.n_rows, a.width, dt == DT_BF16 ? 8 : 4);
  const dim3 grid((unsigned)(sp.blocks < STEP_GRID ? sp.blocks : STEP_GRID));
  auto go = [&](auto kernel) { kernel<<<grid, DT_, 0, s>>>(a, sp); };
  const bool whole = a.n_rows == 1 || a.width % 4 == 0;
  if (dt == DT_BF16)
    whole ? go(k_dropout<true, true>) : go(k_dropout<true, false>);
  else
    whole ? go(k_dropout<false, true>) : go(k_dropout<false, false>);
}

}  // namespace d3s
