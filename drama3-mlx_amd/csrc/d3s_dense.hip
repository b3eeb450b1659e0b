/* Dense layers (include/d3s_train.h): which tiles a product is cut into
 * (gfx950; the kernel is in d3s_dense_tile.h). */
#include "d3s_dense.h"

namespace d3s {
namespace {

/* operands whose chunks go to LDS directly: rows at 16 bytes, a tile's 256 of
 * them within 32-bit offsets */
bool at_16(const uint16_t *p, int64_t stride) {
  return ((uintptr_t)p & 15u) == 0u && stride % 8 == 0 && stride < ((int64_t)1 << 22);
}

TilePlan plan(const d3s_dense_params &p, int tm, int tn) {
  TilePlan pl{};
  pl.tm = tm;
  pl.tn = tn;
  pl.m_tiles = (unsigned)((p.m + tm - 1) / tm);
  pl.n_tiles = (unsigned)((p.n + tn - 1) / tn);
  pl.tiles = pl.m_tiles * pl.n_tiles;
  pl.group = 8;
  pl.x_direct = at_16(p.x, p.x_stride);
  pl.w_direct = at_16(p.w, p.w_stride);
  pl.splits = 1;
  pl.stages = (int)(p.k / TILE_K);
  return pl;
}

}  // namespace

size_t dense_workspace_bytes(const d3s_dense_params &p) { return 0; }

void launch_dense(const d3s_dense_params &p, void *ws, hipStream_t s) {
  const Operands a{p.x, p.w, p.x_stride, p.w_stride, (int)p.k};
  const Out o{p.bias,     p.residual, p.z,        p.y,        p.residual_stride, p.z_stride,
              p.y_stride, (int)p.m,   (int)p.n,   p.activation, p.y_dtype == D3S_DTYPE_F32};
  const int t = p.m > 1024 && p.n > 1024 ? 256 : 128;
  const TilePlan pl = plan(p, t, t);
  if (p.x_transposed)
    p.w_transposed ? launch_tiles<true, true>(a, o, pl, s) : launch_tiles<true, false>(a, o, pl, s);
  else
    p.w_transposed ? launch_tiles<false, true>(a, o, pl, s) : launch_tiles<false, false>(a, o, pl, s);
}

}  // namespace d3s
