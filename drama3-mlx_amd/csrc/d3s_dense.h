/* What the products' kernels take (d3s_dense.hip plans, d3s_dense_tile.h computes). */
#ifndef D3S_DENSE_H
#define D3S_DENSE_H

#include "d3s_train_internal.h"

namespace d3s {

constexpr int TILE_K = 64; /* the inner length of a stage */

struct Operands {
  const uint16_t *x, *w;
  int64_t x_stride, w_stride;
  int k;
};

/* what a product's kernel needs to write its outputs */
struct Out {
  const uint16_t *bias;
  const void *residual;
  uint16_t *z;
  void *y;
  int64_t residual_stride, z_stride, y_stride;
  int m, n, act;
  bool f32;
};

/* m_tiles by n_tiles tiles of tm x tn from output (i0, j0), walked in columns
 * of `group`; each cut into `splits` of `stages` stages.  (An output takes two
 * bytes: the tiles of what fits the memory are counted in 32 bits.) */
struct TilePlan {
  unsigned tiles, first, m_tiles, n_tiles, group, splits;
  int i0, j0, stages;
  int tm, tn;
  bool x_direct, w_direct; /* operands by rows at 16 bytes: see Way */
};

template <bool XT, bool WT>
void launch_tiles(const Operands &a, const Out &o, const TilePlan &pl, hipStream_t s);

}  // namespace d3s

#endif
