/* k_dropout: y = residual + kept x / (1 - p), the mask drawn from Philox as it is
 * used (gfx950, wave64; include/d3s_step.h).
 *
 * An element is kept iff the upper 24 bits of its word are at least p 2^24: the same as u >= p, since
 * u is those bits times 2^-24, without forming it.  1 / (1 - p) is rounded to fp32 once, the product and
 * the sum once each.  A lane takes one or two whole blocks of the generator (20 multiplies of 32 x 32 bits
 * each, about as long as its share of the memory traffic in bf16).
 *
 * Bound: HBM, the multiplies close behind.  bf16 8192 x 2048 with a residual 18 us (5.6 TB/s; a block
 * for each element 35); fp32 without 22 us (6.0 TB/s). */
#include "d3s_step_internal.h"
#include "d3s_vec.h"

namespace d3s {
namespace {

constexpr int DT_ = 256;

/* A lane's E elements begin at a multiple of four in the generator's count, so that its words are
 * whole blocks of Philox: in a row that does not (EVEN: none), the first lane's begin up to three
 * places before it.  (With lanes that begin with the row, a block more each and its words
 * picked, 8192 x 2049 bf16 with a residual at a stride of 2052 takes a third more.)  Rows' chunks are counted
 * through: these 22 us, a power of two of lanes for each row 36. */
template <bool BF16, bool EVEN>
__global__ __launch_bounds__(DT_) void k_dropout(DropoutArgs a, Spread c) {
  constexpr int E = BF16 ? 8 : 4, ES = BF16 ? 2 : 4;
  const uint64_t draw = a.draw + (a.draw_add ? *a.draw_add : 0u);
  for (int64_t blk = blockIdx.x; blk < c.blocks; blk += gridDim.x) {
    int64_t row, chunk;
    c.find<DT_>(blk, &row, &chunk);
    const uint64_t first = (uint64_t)row * (uint64_t)a.width;
    const int64_t j = chunk * E - (EVEN ? 0 : (int64_t)(first & 3u)), left = a.width - j;
    if (row >= a.n_rows || left <= 0) continue;
    const char *x = (const char *)a.x + row * a.x_stride * ES, *res = (const char *)a.residual + row * a.residual_stride * ES;
    char *y = (char *)a.y + row * a.y_stride * ES;
    Vec<BF16, E> q, r;
    const bool inside = EVEN || j >= 0;
    if (inside) {
      q.load_some(x, j, left);
      if (a.residual) r.load_some(res, j, left);
    }
    uint32_t w[E];
#pragma unroll
    for (int b = 0; b < E / 4; b++) {
      const uint64_t n = (first + (uint64_t)j) / 4u + b;
      const d3s_u32x4 o = d3s_philox4x32_10({{(uint32_t)n, (uint32_t)(n >> 32), (uint32_t)draw, (uint32_t)(draw >> 32)}},
                                            (uint32_t)a.seed, (uint32_t)(a.seed >> 32));
#pragma unroll
      for (int i = 0; i < 4; i++) w[4 * b + i] = o.v[i];
    }
    auto one = [&](int e, float v) { return (w[e] >> 8) >= a.least ? v * a.scale : 0.0f; };
    if (inside) {
      float v[E], o[E];
      q.values(v);
      if (a.residual) r.values(o);
#pragma unroll
      for (int e = 0; e < E; e++) {
        v[e] = one(e, v[e]);
        if (a.residual) v[e] += o[e];
      }
      store_row<BF16, E>(y, j, left, v);
    } else {
#pragma unroll
      for (int e = 0; e < E; e++)
        if (j + e >= 0 && e < left) {
          const float v = one(e, load_at<BF16>(x, j + e));
          store_at<BF16>(y, j + e, a.residual ? v + load_at<BF16>(res, j + e) : v);
        }
    }
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
  const bool even = a.n_rows == 1 || a.width % 4 == 0;
  const Spread c = Spread::of<DT_>(a.n_rows, a.width + (even ? 0 : 3), dt == DT_BF16 ? 8 : 4);
  const dim3 grid((unsigned)(c.blocks < STEP_GRID ? c.blocks : STEP_GRID));
  auto go = [&](auto kernel) { kernel<<<grid, DT_, 0, s>>>(a, c); };
  if (dt == DT_BF16)
    even ? go(k_dropout<true, true>) : go(k_dropout<true, false>);
  else
    even ? go(k_dropout<false, true>) : go(k_dropout<false, false>);
}

}  // namespace d3s
