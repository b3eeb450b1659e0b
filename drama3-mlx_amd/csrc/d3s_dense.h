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

/* m_tiles by n_tiles tiles of tm x tn, walked in columns of `group`; each cut into `splits` of `stages` stages.  (An output takes two
 * bytes: the tiles of what fits the memory are counted in 32 bits.) */
struct TilePlan {
  unsigned tiles, first, m_tiles, n_tiles, group, splits;
  int stages;
  int tm, tn;
  float *parts;       /* the splits' sums, and their arrivals (a 128-byte line a tile) */
  uint32_t *arrivals;
  bool x_direct, w_direct; /* operands by rows at 16 bytes: see Way */
};

/* k_few's: rows from i0 on (at most FEW_ROWS; or outputs, at most half as many:
 * the operands' roles exchanged), the inner length cut into `splits` of `batches` batches */
constexpr int FEW_ROWS = 64;
struct FewPlan {
  unsigned tiles, splits;
  int i0, batches;
  uint64_t *parts;
  uint32_t *arrivals;
};
int few_outputs(bool w_transposed); /* a workgroup's (exchanged: rows, by how x lies) */
int few_batch(bool w_transposed);
int few_waves(bool w_transposed); /* batches at a time */
size_t few_part_bytes(bool w_transposed, int rows); /* a split's sums of one workgroup */
void launch_few(const Operands &a, const Out &o, bool x_transposed, bool w_transposed, bool swap, const FewPlan &pl,
                hipStream_t s);

template <bool XT, bool WT>
void launch_tiles(const Operands &a, const Out &o, const TilePlan &pl, hipStream_t s);

}  // namespace d3s

#endif
