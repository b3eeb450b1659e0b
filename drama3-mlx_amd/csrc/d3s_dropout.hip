/* k_dropout: y = residual + kept x / (1 - p), the mask drawn from Philox as it is
 * used (gfx950, wave64; include/d3s_step.h). */
#include "d3s_step_internal.h"
#include "d3s_vec.h"

namespace d3s {
namespace {

constexpr int DT_ = 256;

/* a workgroup takes DT_ / lanes rows by 8 * lanes columns */
struct DropSplit {
  int lanes;
  int64_t strips, blocks;
};

DropSplit drop_split(int64_t rows, int64_t width) {
  DropSplit s;
  s.lanes = 1;
  while (s.lanes < DT_ && (int64_t)s.lanes * 8 < width) s.lanes *= 2;
  s.strips = (width + s.lanes * 8 - 1) / (s.lanes * 8);
  s.blocks = s.strips * ((rows + DT_ / s.lanes - 1) / (DT_ / s.lanes));
  return s;
}

template <bool BF16>
__global__ __launch_bounds__(DT_) void k_dropout(DropoutArgs a, DropSplit sp) {
  const int across = (int)threadIdx.x % sp.lanes, down = (int)threadIdx.x / sp.lanes;
  const uint64_t draw = a.draw + (a.draw_add ? *a.draw_add : 0u);
  for (int64_t blk = blockIdx.x; blk < sp.blocks; blk += gridDim.x) {
    const int64_t row = blk / sp.strips * (DT_ / sp.lanes) + down;
    const int64_t j = (blk % sp.strips * sp.lanes + across) * 8;
    if (row >= a.n_rows || j >= a.width) continue;
    const int left = (int)min((int64_t)8, a.width - j);
    const char *x = (const char *)a.x + row * a.x_stride * (BF16 ? 2 : 4);
    char *y = (char *)a.y + row * a.y_stride * (BF16 ? 2 : 4);
    float v[8], r[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    load8<BF16>(x, j, left, v);
    if (a.residual) load8<BF16>((const char *)a.residual + row * a.residual_stride * (BF16 ? 2 : 4), j, left, r);
    const uint64_t at = (uint64_t)row * (uint64_t)a.width + (uint64_t)j;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      d3s_u32x4 c;
      const uint64_t q = (at + e) >> 2;
      c.v[0] = (uint32_t)q;
      c.v[1] = (uint32_t)(q >> 32);
      c.v[2] = (uint32_t)draw;
      c.v[3] = (uint32_t)(draw >> 32);
      const d3s_u32x4 o = d3s_philox4x32_10(c, (uint32_t)a.seed, (uint32_t)(a.seed >> 32));
      const uint32_t i = (uint32_t)(at + e) & 3u;
      const uint32_t w = i == 0 ? o.v[0] : i == 1 ? o.v[1] : i == 2 ? o.v[2] : o.v[3];
      v[e] = ((w >> 8) >= a.least ? v[e] * a.scale : 0.0f) + r[e];
    }
    store8<BF16>(y, j, left, v);
  }
}

}  // namespace

void launch_dropout(const DropoutArgs &args, Dtype dt, hipStream_t s) {
  const DropoutArgs a = args;
  const DropSplit sp = drop_split(a.n_rows, a.width);
  const dim3 grid((unsigned)(sp.blocks < STEP_GRID ? sp.blocks : STEP_GRID));
  if (dt == DT_BF16)
    k_dropout<true><<<grid, DT_, 0, s>>>(a, sp);
  else
    k_dropout<false><<<grid, DT_, 0, s>>>(a, sp);
}

}  // namespace d3s
