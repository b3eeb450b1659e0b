/* Dense layers (include/d3s_train.h): which kernel takes a product, in which
 * tiles (gfx950; the kernels are in d3s_dense_tile.h and d3s_dense_few.hip). */
#include "d3s_dense.h"

namespace d3s {
namespace {

constexpr int CUS = 256;

/* operands whose chunks go to LDS directly: rows at 16 bytes, a tile's 256 of
 * them within 32-bit offsets */
bool direct_at(uintptr_t p, int64_t stride) { return p % 16 == 0 && stride % 8 == 0 && stride < ((int64_t)1 << 22); }

/* A product: its sizes, and how its operands lie. */
struct Product {
  int64_t m, n, k;
  bool x_turned, w_turned, x_direct, w_direct;
};

Product product_of(const d3s_dense_params &p, uintptr_t x, uintptr_t w) {
  Product r{p.m, p.n, p.k, p.x_transposed != 0, p.w_transposed != 0, false, false};
  r.x_direct = !r.x_turned && direct_at(x, p.x_stride);
  r.w_direct = !r.w_turned && direct_at(w, p.w_stride);
  return r;
}

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }

/* Microseconds of m rows and n outputs in tiles of tm x tn, one workgroup a CU: rounds of
 * workgroups, each its stages and what it spends before and after them.
 * Measured, by how many operands go to LDS directly: a stage of 256 x 256 1.45
 * (both), 1.65 (one) and 2.2, with an eighth of the CUs idle 1.1, 1.35 and 1.6; of
 * 128 x 256 0.93 and 1.2 (0.65 and 0.95); of 128 x 128 0.52 and 0.75 (with a
 * quarter idle 0.38 and 0.65).  Around them 14, 10 and 6, and for split sums 3 and 1 a split.
 * (8192 x 2048 x 2048, both direct: 63, 78 and 87 us in the three tiles;
 * 2048 x 2048 x 2048: 50, 29 and 22; 4096 x 2048 x 8192, both by the inner
 * index: 217, 160 and 210; 256 x 2048 x 8192: 128 x 128 with 1, 2, 4 and 8
 * splits 49, 31, 22 and 24.)  The middle tile is the wide one: few rows of tiles load
 * rows of x that are not at 4 bytes less often (heads of 4097 outputs, their weights'
 * gradient: 186 us, in tiles of 256 x 128 it was 205). */
double tile_us(const Product &p, int64_t m, int64_t n, int tm, int tn, int splits) {
  const int direct = p.x_direct + p.w_direct;
  const double wgs = (double)up(m, tm) * (double)up(n, tn) * splits;
  const double rounds = (double)(int64_t)((wgs + CUS - 1) / CUS), stages = (double)up(p.k, (int64_t)TILE_K * splits);
  const bool few = wgs <= (tn == 256 ? CUS * 7 / 8 : CUS * 3 / 4);
  if (tm == 256) {
    const double full = direct == 2 ? 1.45 : direct == 1 ? 1.65 : 2.2, some = direct == 2 ? 1.1 : direct == 1 ? 1.35 : 1.6;
    return rounds * (stages * (few ? some : full) + 14);
  }
  if (tn == 256) {
    const double full = direct == 2 ? 0.93 : 1.2, some = direct == 2 ? 0.65 : 0.95;
    return rounds * (stages * (few ? some : full) + 10);
  }
  const double stage = direct == 2 ? (few ? 0.38 : 0.52) : few ? 0.65 : 0.75;
  return rounds * (stages * stage + 6) + (splits > 1 ? 3 + splits : 0);
}

/* ... and of k_few, which reads `many` rows of the other operand at 4 TB/s */
double few_us(const Product &p, int64_t many) { return 6 + (double)many * (double)p.k * 2 / 4e6; }

struct Plan {
  TilePlan tile;         /* no tiles: no such launch */
  int64_t tile_m, tile_n;
  FewPlan few, few_outs; /* the rows after the tiles', and the outputs after theirs of the tiles' rows */
  double us;             /* what it should take */
};

size_t tile_bytes(const TilePlan &t) { return t.splits > 1 ? (size_t)t.tiles * t.splits * t.tm * t.tn * sizeof(float) : 0; }
size_t few_bytes(const FewPlan &f, bool turned, int64_t rows) {
  return f.splits > 1 ? (size_t)f.tiles * f.splits * few_part_bytes(turned, (int)rows) : 0;
}

/* `few` rows from i0 on against `many` of the other operand, turned or not */
FewPlan few_plan(int64_t i0, int64_t few, int64_t many, int64_t k, bool turned) {
  FewPlan f{};
  f.i0 = (int)i0;
  f.tiles = (unsigned)up(many, few_outputs(turned));
  /* the inner length over more workgroups while there are fewer than CUs, at
   * least two batches a wave (one with four fragments of rows) */
  const int64_t batches = up(k, few_batch(turned));
  int64_t most = batches / (few_waves(turned) * (few > 32 ? 1 : 2)), want = CUS / (int64_t)f.tiles;
  if (want < most) most = want;
  if (most > 16) most = 16; /* (32 splits of turned weights, 34 MB of them: 19.6 us, sixteen 15.4) */
  f.splits = most > 1 ? (unsigned)most : 1u;
  f.batches = (int)up(batches, f.splits);
  return f;
}

Plan plan(const Product &p) {
  Plan pl{};
  /* Few rows: k_few, which turns weights eight outputs at a time.  33 to 64 rows
   * (64 x 2048 x 2048: 9.3 us, in tiles 14.2; 64 x 4097 x 2048: 19.8, in tiles 15.8) while
   * its workgroups of 16 outputs, each of which reads all of x, run at once. */
  const bool rows_can = !p.w_turned || p.n >= 8;
  if (rows_can && (p.m <= 32 || (p.m <= FEW_ROWS && !p.w_turned && p.n <= 16 * CUS))) {
    pl.few = few_plan(0, p.m, p.n, p.k, p.w_turned);
    pl.us = few_us(p, p.n);
    return pl;
  }

  /* A last row or column of tiles that is nearly empty may cost a round of its
   * own: its rows, or outputs, are k_few's too. */
  double best = 1e300;
  TilePlan &t = pl.tile;
  for (int cut = 0; cut < 4; cut++) {
    const int64_t dm = cut & 1 ? p.m % 128 : 0, dn = cut & 2 ? p.n % 128 : 0, m = p.m - dm, n = p.n - dn;
    if ((cut & 1) && !(rows_can && dm > 0 && dm <= 32 && m >= 256)) continue;
    if ((cut & 2) && !(dn > 0 && dn <= 32 && n >= 256 && (!p.x_turned || m >= 8))) continue;
    const double also = (dm ? few_us(p, p.n) : 0) + (dn ? few_us(p, m) : 0);
    auto offer = [&](int tm, int tn, int splits) {
      const double us = tile_us(p, m, n, tm, tn, splits) + also;
      if (us >= best) return;
      best = us;
      pl.tile_m = m, pl.tile_n = n;
      t.tm = tm, t.tn = tn, t.splits = (unsigned)splits;
    };
    /* (256 x 256 turns eight rows at a time) */
    if (!(p.x_turned && m < 8) && !(p.w_turned && n < 8)) offer(256, 256, 1);
    offer(128, 256, 1);
    /* (Every split has its stages, and fewer workgroups than twice the CUs.  Eight at
     * most: the last to arrive reads every split's sums, so by the costs above more
     * only pay past an inner length of 8192; 256 x 256 x 16384, both by the inner
     * index, 32 us and with sixteen 29, 256 x 256 x 8192 23 either way.) */
    for (int s = 1; s <= 8; s++)
      if (s == 1 || (p.k >= (int64_t)4 * s * TILE_K && up(m, 128) * up(n, 128) * s <= 2 * CUS)) offer(128, 128, s);
  }
  pl.us = best;
  t.m_tiles = (unsigned)up(pl.tile_m, t.tm);
  t.n_tiles = (unsigned)up(pl.tile_n, t.tn);
  t.tiles = t.m_tiles * t.n_tiles;
  t.group = 8;
  t.stages = (int)up(p.k / TILE_K, t.splits);
  t.x_direct = p.x_direct;
  t.w_direct = p.w_direct;
  if (pl.tile_m < p.m) pl.few = few_plan(pl.tile_m, p.m - pl.tile_m, p.n, p.k, p.w_turned);
  if (pl.tile_n < p.n) pl.few_outs = few_plan(pl.tile_n, p.n - pl.tile_n, pl.tile_m, p.k, p.x_turned);
  return pl;
}

/* A product in two: the first part's rows and outputs, one of them the whole's.
 * Where the last round of tiles would be less than half full, what fills the rounds
 * before is a product of its own, and the rest another, in smaller tiles and
 * split sums (1500 x 11008 x 4096, w by the inner index, 258 tiles of 256 x 256: 205
 * us, so 135; 3000 x 11008 x 4096 by rows 271 and 216).  Whole rounds of whole tiles: both parts start where the
 * operands' alignment is the same. */
struct Cut {
  int64_t m, n;
};
Cut cut_of(const Product &p) {
  Cut best{p.m, p.n};
  const Plan whole = plan(p);
  if (!whole.tile.tiles) return best;
  double least = 0.92 * whole.us; /* (a launch more, and costs that are estimates) */
  const int tiles[3][2] = {{256, 256}, {128, 256}, {128, 128}};
  for (const auto &t : tiles) {
    const int64_t mt = up(p.m, t[0]), nt = up(p.n, t[1]), rounds = mt * nt / CUS;
    if (rounds < 1 || mt * nt % CUS == 0 || mt * nt % CUS >= CUS / 2) continue;
    const int64_t n = rounds * CUS / mt * t[1], m = rounds * CUS / nt * t[0];
    auto offer = [&](int64_t m1, int64_t n1, int64_t m2, int64_t n2) {
      Product a = p, b = p;
      a.m = m1, a.n = n1, b.m = m2, b.n = n2;
      const double us = plan(a).us + plan(b).us;
      if (us < least) least = us, best = {m1, n1};
    };
    if (n > 0 && n < p.n) offer(p.m, n, p.m, p.n - n);
    if (m > 0 && m < p.m) offer(m, p.n, p.m - m, p.n);
  }
  return best;
}

size_t bytes_of_part(const Product &p) {
  const Plan pl = plan(p);
  const size_t a = tile_bytes(pl.tile), b = few_bytes(pl.few, p.w_turned, p.m - pl.few.i0),
               c = few_bytes(pl.few_outs, p.x_turned, p.n - pl.few_outs.i0);
  const size_t ab = a > b ? a : b;
  return ab > c ? ab : c; /* (one launch after the other) */
}

size_t bytes_of(const Product &p) {
  const Cut c = cut_of(p);
  Product first = p, rest = p;
  first.m = c.m, first.n = c.n;
  const size_t a = bytes_of_part(first);
  if (c.m == p.m && c.n == p.n) return a;
  c.n < p.n ? rest.n -= c.n : rest.m -= c.m;
  const size_t b = bytes_of_part(rest);
  return a > b ? a : b;
}

}  // namespace

/* for whatever alignment the operands come at */
size_t dense_workspace_bytes(const d3s_dense_params &p) {
  size_t most = 0;
  for (int at = 0; at < 4; at++) {
    const size_t b = bytes_of(product_of(p, (uintptr_t)(at & 1) * 2, (uintptr_t)(at >> 1) * 2));
    most = b > most ? b : most;
  }
  return most ? split_counter_bytes() + most : 0;
}

static void launch_part(const d3s_dense_params &p, void *ws, hipStream_t s) {
  const Operands a{p.x, p.w, p.x_stride, p.w_stride, (int)p.k};
  Out o{p.bias,     p.residual, p.z,      p.y,          p.residual_stride,          p.z_stride,
        p.y_stride, (int)p.m,   (int)p.n, p.activation, p.y_dtype == D3S_DTYPE_F32};
  const Product pr = product_of(p, (uintptr_t)p.x, (uintptr_t)p.w);
  Plan pl = plan(pr);
  char *parts = ws ? (char *)ws + split_counter_bytes() : nullptr;
  if (pl.few.tiles) {
    pl.few.arrivals = (uint32_t *)ws;
    pl.few.parts = (uint64_t *)parts;
    launch_few(a, o, pr.x_turned, pr.w_turned, false, pl.few, s);
  }
  if (!pl.tile.tiles) return;
  o.m = (int)pl.tile_m;
  if (pl.few_outs.tiles) {
    pl.few_outs.arrivals = (uint32_t *)ws;
    pl.few_outs.parts = (uint64_t *)parts;
    launch_few(a, o, pr.x_turned, pr.w_turned, true, pl.few_outs, s);
  }
  o.n = (int)pl.tile_n;
  pl.tile.arrivals = (uint32_t *)ws;
  pl.tile.parts = (float *)parts;
  if (pr.x_turned)
    pr.w_turned ? launch_tiles<true, true>(a, o, pl.tile, s) : launch_tiles<true, false>(a, o, pl.tile, s);
  else
    pr.w_turned ? launch_tiles<false, true>(a, o, pl.tile, s) : launch_tiles<false, false>(a, o, pl.tile, s);
}

void launch_dense(const d3s_dense_params &p, void *ws, hipStream_t s) {
  const Cut c = cut_of(product_of(p, (uintptr_t)p.x, (uintptr_t)p.w));
  d3s_dense_params first = p, rest = p;
  first.m = c.m, first.n = c.n;
  launch_part(first, ws, s);
  const int64_t es = p.y_dtype == D3S_DTYPE_F32 ? 4 : 2;
  if (c.n < p.n) {
    rest.n -= c.n;
    rest.w += p.w_transposed ? c.n : c.n * p.w_stride;
    if (p.bias) rest.bias += c.n;
    if (p.z) rest.z += c.n;
    if (p.residual) rest.residual = (const char *)p.residual + c.n * es;
    rest.y = (char *)p.y + c.n * es;
    launch_part(rest, ws, s);
  } else if (c.m < p.m) {
    rest.m -= c.m;
    rest.x += p.x_transposed ? c.m : c.m * p.x_stride;
    if (p.z) rest.z += c.m * p.z_stride;
    if (p.residual) rest.residual = (const char *)p.residual + c.m * p.residual_stride * es;
    rest.y = (char *)p.y + c.m * p.y_stride * es;
    launch_part(rest, ws, s);
  }
}

}  // namespace d3s
