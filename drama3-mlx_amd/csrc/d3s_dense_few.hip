/* k_few: dense layers of up to 64 rows of x, or, with the operands' roles
 * exchanged, of up to 32 outputs (gfx950, wave64; include/d3s_train.h).
 *
 * Bound: the weights' bytes, which are read once, straight into the fragments
 * of 16 x 16 x 32 products (no LDS: nothing is shared between waves but x,
 * which the caches hold).  A workgroup's waves take the inner length in turns,
 * batches of 128 or 32, and join their sums in LDS; where the outputs alone do
 * not fill the chip the inner length is also cut over workgroups, whose sums
 * go through the workspace (the last to arrive adds them in order).
 * Weights by rows: a wave's 16 outputs, lane l row l % 16 and inner indices
 * 8 (l / 16) .. + 7 of a step.  Weights by the inner index: 128 outputs, lane l
 * eight of them (l % 16) at eight inner indices, turned in registers: fragment
 * e is outputs 8 r + e.
 * Rows that start between 4-byte words are loaded from the word below, with the word
 * behind, and moved down: a 16-byte load there takes far longer.
 *
 * Measured, repeated calls on the same weights: 1 x 2048 x
 * 2048 4.7 us (from HBM 6.5), 1 x 8192 x 8192 31 us (4.3 TB/s), 1 x 151936 x 2048
 * 138 us (4.5 TB/s), 64 x 2048 x 2048 9.4 us, 1 x 4097 x 4097 10.4 us. */
#include "d3s_dense_load.h"
#include "d3s_epilogue.h"
#include "d3s_rowcore.h"

namespace d3s {
namespace {

constexpr unsigned FEW_GRID = 1 << 20; /* workgroups a launch */

template <bool WT>
struct Shape {
  static constexpr int WAVES = WT ? 4 : 8;
  static constexpr int THREADS = WAVES * WAVE;
  static constexpr int OUTPUTS = WT ? 128 : 16; /* a workgroup */
  static constexpr int STEPS = WT ? 1 : 4;      /* of 32 a batch */
  static constexpr int FRAGMENTS = WT ? 8 : 1;  /* of 16 outputs */
};

/* eight elements at p, `odd` (0, 1) elements behind a 4-byte word */
__device__ __forceinline__ uint4 load_odd(const uint16_t *p, int odd) {
  const uint4 q = load16(p - odd);
  const uint32_t behind = *(const uint32_t *)(p - odd + 6 + 2 * odd);
  const int s = odd * 16;
  return make_uint4(__builtin_amdgcn_alignbit(q.y, q.x, s), __builtin_amdgcn_alignbit(q.z, q.y, s),
                    __builtin_amdgcn_alignbit(q.w, q.z, s), __builtin_amdgcn_alignbit(behind, q.w, s));
}

/* elements [at, at + 8) of row i of x, zeros past its end */
template <bool XT, bool ODD>
__device__ __forceinline__ bf16x8 x_fragment(const Operands &a, int i, int at, bool whole) {
  uint4 q = make_uint4(0u, 0u, 0u, 0u);
  if constexpr (XT) {
    uint32_t v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = whole || at + e < a.k ? a.x[(int64_t)(at + e) * a.x_stride + i] : 0u;
    q = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
  } else {
    const uint16_t *row = a.x + (int64_t)i * a.x_stride;
    if (whole)
      q = ODD ? load_odd(row + at, (int)((uintptr_t)row >> 1 & 1)) : load16(row + at);
    else if (at < a.k)
      q = row_chunk(row, at, a.k);
  }
  return __builtin_bit_cast(bf16x8, q);
}

template <int FR, bool XT, bool WT, bool ODD, bool SWAP>
__global__ __launch_bounds__(Shape<WT>::THREADS) void k_few(Operands a, Out o, FewPlan pl, unsigned first) {
  using S = Shape<WT>;
  constexpr int FG = S::FRAGMENTS, BATCH = S::STEPS * 32;
  __shared__ f32x4 sums[S::WAVES][FG][FR][WAVE];
  __shared__ unsigned last;
  const int lane = lane_id(), wid = (int)threadIdx.x / WAVE, g = lane >> 4, r = lane & 15;
  const int rows = SWAP ? o.n : o.m, outputs = SWAP ? o.m : o.n;
  const unsigned tile = (first + blockIdx.x) / pl.splits, split = (first + blockIdx.x) % pl.splits;
  const int j0 = (int)tile * S::OUTPUTS;
  const int batches = (int)(((int64_t)a.k + BATCH - 1) / BATCH);
  const int b1 = (int)min((int64_t)batches, (int64_t)(split + 1) * pl.batches);
  /* outputs past the end are the last again, and not written (turned: the last eight) */
  const int j = WT ? min(j0 + r * 8, outputs - 8) : min(j0 + r, outputs - 1);
  int xi[FR];
#pragma unroll
  for (int f = 0; f < FR; f++) xi[f] = min(pl.i0 + f * 16 + r, rows - 1);
  f32x4 acc[FG][FR];
#pragma unroll
  for (int e = 0; e < FG; e++)
#pragma unroll
    for (int f = 0; f < FR; f++) acc[e][f] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  auto batch = [&](int b, bool whole) {
    const int k0 = b * BATCH;
    bf16x8 fx[S::STEPS][FR];
    if constexpr (WT) {
      const int k = k0 + g * 8;
      uint4 q[8];
#pragma unroll
      for (int u = 0; u < 8; u++) q[u] = load16(a.w + (int64_t)(whole ? k + u : min(k + u, a.k - 1)) * a.w_stride + j);
#pragma unroll
      for (int f = 0; f < FR; f++) fx[0][f] = x_fragment<XT, ODD>(a, xi[f], k, whole);
      const int n = a.k - k;
      auto some = [&](int d) { return whole || n >= 2 * d + 2 ? ~0u : n == 2 * d + 1 ? 0xffffu : 0u; };
#pragma unroll
      for (int e = 0; e < 8; e++) {
        auto word = [&](int u) { return e < 2 ? q[u].x : e < 4 ? q[u].y : e < 6 ? q[u].z : q[u].w; };
        uint32_t v[4];
#pragma unroll
        for (int d = 0; d < 4; d++)
          v[d] = __builtin_amdgcn_perm(word(2 * d + 1), word(2 * d), e & 1 ? 0x07060302u : 0x05040100u) & some(d);
        const bf16x8 fw = __builtin_bit_cast(bf16x8, make_uint4(v[0], v[1], v[2], v[3]));
#pragma unroll
        for (int f = 0; f < FR; f++) acc[e][f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw, fx[0][f], acc[e][f], 0, 0, 0);
      }
    } else {
      bf16x8 fw[S::STEPS];
      const uint16_t *row = a.w + (int64_t)j * a.w_stride;
      const int odd = (int)((uintptr_t)row >> 1 & 1);
#pragma unroll
      for (int s = 0; s < S::STEPS; s++) {
        const int k = k0 + s * 32 + g * 8;
        fw[s] = __builtin_bit_cast(bf16x8, whole ? (ODD ? load_odd(row + k, odd) : load16(row + k)) : k < a.k ? row_chunk(row, k, a.k) : make_uint4(0u, 0u, 0u, 0u));
#pragma unroll
        for (int f = 0; f < FR; f++) fx[s][f] = x_fragment<XT, ODD>(a, xi[f], k, whole);
      }
#pragma unroll
      for (int s = 0; s < S::STEPS; s++)
#pragma unroll
        for (int f = 0; f < FR; f++) acc[0][f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw[s], fx[s][f], acc[0][f], 0, 0, 0);
    }
  };
  int b = (int)split * pl.batches + wid;
#pragma unroll 2
  for (; b < b1 && (int64_t)(b + 1) * BATCH <= a.k; b += S::WAVES) batch(b, true);
  if (b < b1) batch(b, false);

#pragma unroll
  for (int e = 0; e < FG; e++)
#pragma unroll
    for (int f = 0; f < FR; f++) sums[wid][e][f][lane] = acc[e][f];
  __syncthreads();

  /* Lane l of a fragment's sums holds row l % 16 of x and outputs 4 (l / 16) .. + 3
   * of it.  A thread takes EACH neighbouring outputs of one row: by rows the
   * lane's four, turned the eight of one of its outputs. */
  constexpr int EACH = WT ? 8 : 4, ITEMS = FR * 16 * S::OUTPUTS / EACH;
  constexpr int ROUNDS = (ITEMS + S::THREADS - 1) / S::THREADS;
  float v[ROUNDS][EACH];
  int at_i[ROUNDS], at_j[ROUNDS], skip[ROUNDS];
#pragma unroll
  for (int c = 0; c < ROUNDS; c++) {
    const int t = c * S::THREADS + (int)threadIdx.x;
    /* items in order of rows, then outputs */
    const int i = t / (S::OUTPUTS / EACH) % 16, f = t / (S::OUTPUTS / EACH) / 16 % FR, across = t % (S::OUTPUTS / EACH);
    at_i[c] = t < ITEMS ? pl.i0 + f * 16 + i : rows;
    at_j[c] = WT ? (int)min((int64_t)j0 + across * 8, (int64_t)outputs - 8) : j0 + across * 4;
    skip[c] = j0 + across * EACH - at_j[c]; /* (what the item before writes: a residual in place is added once) */
    const int from = WT ? (across >> 2) * 16 + i : across * 16 + i;
#pragma unroll
    for (int e = 0; e < EACH; e++) v[c][e] = 0.0f;
    for (int w = 0; w < S::WAVES; w++) {
      if constexpr (WT) {
#pragma unroll
        for (int e = 0; e < 8; e++) v[c][e] += ((const float *)&sums[w][e][f][from])[across & 3];
      } else {
        const f32x4 s = sums[w][0][f][from];
#pragma unroll
        for (int e = 0; e < 4; e++) v[c][e] += s[e];
      }
    }
  }
  if (pl.splits > 1) {
    constexpr int WORDS = EACH / 2; /* pairs of sums, 8 bytes */
    uint64_t *part = pl.parts + (size_t)tile * pl.splits * (ROUNDS * S::THREADS * WORDS);
    auto place = [&](unsigned s, int c, int w) {
      return part + (((size_t)s * ROUNDS + c) * WORDS + w) * S::THREADS + threadIdx.x;
    };
#pragma unroll
    for (int c = 0; c < ROUNDS; c++)
#pragma unroll
      for (int w = 0; w < WORDS; w++)
        st_agent(place(split, c, w), (uint64_t)d3s_f2u(v[c][2 * w]) | (uint64_t)d3s_f2u(v[c][2 * w + 1]) << 32);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
      uint32_t *count = pl.arrivals + (size_t)tile * 32;
      last = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == pl.splits - 1;
      if (last) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!last) return;
#pragma unroll
    for (int c = 0; c < ROUNDS; c++)
#pragma unroll
      for (int e = 0; e < EACH; e++) v[c][e] = 0.0f;
#pragma unroll 4
    for (unsigned s = 0; s < pl.splits; s++)
#pragma unroll
      for (int c = 0; c < ROUNDS; c++)
#pragma unroll
        for (int w = 0; w < WORDS; w++) {
          const uint64_t q = ld_agent(place(s, c, w));
          v[c][2 * w] += d3s_u2f((uint32_t)q);
          v[c][2 * w + 1] += d3s_u2f((uint32_t)(q >> 32));
        }
  }
#pragma unroll
  for (int c = 0; c < ROUNDS; c++) put_some<EACH, SWAP>(o, at_i[c], at_j[c], skip[c], v[c]);
}

template <int FR, bool XT, bool WT, bool SWAP>
void few_launch(const Operands &a, const Out &o, const FewPlan &pl, hipStream_t s) {
  const unsigned all = pl.tiles * pl.splits;
  /* (transposed loads are not moved: x's are single elements, the weights' eight rows each) */
  const bool odd = (!XT && ((uintptr_t)a.x % 4 != 0 || a.x_stride % 2 != 0)) || (!WT && ((uintptr_t)a.w % 4 != 0 || a.w_stride % 2 != 0));
  for (unsigned first = 0; first < all; first += FEW_GRID) {
    const dim3 grid(min(FEW_GRID, all - first));
    if constexpr (!(XT && WT)) {
      if (odd) {
        k_few<FR, XT, WT, true, SWAP><<<grid, Shape<WT>::THREADS, 0, s>>>(a, o, pl, first);
        continue;
      }
    }
    k_few<FR, XT, WT, false, SWAP><<<grid, Shape<WT>::THREADS, 0, s>>>(a, o, pl, first);
  }
}
template <bool XT, bool WT>
void few_rows(const Operands &a, const Out &o, bool swap, const FewPlan &pl, hipStream_t s) {
  const int rows = (swap ? o.n : o.m) - pl.i0;
  if (swap) return rows <= 16 ? few_launch<1, XT, WT, true>(a, o, pl, s) : few_launch<2, XT, WT, true>(a, o, pl, s);
  if (rows <= 16) return few_launch<1, XT, WT, false>(a, o, pl, s);
  if constexpr (!WT) { /* (33 rows and more: weights by rows only) */
    if (rows > 32) return few_launch<4, XT, WT, false>(a, o, pl, s);
  }
  few_launch<2, XT, WT, false>(a, o, pl, s);
}

}  // namespace

int few_outputs(bool w_transposed) { return w_transposed ? Shape<true>::OUTPUTS : Shape<false>::OUTPUTS; }
int few_batch(bool w_transposed) { return 32 * (w_transposed ? Shape<true>::STEPS : Shape<false>::STEPS); }
int few_waves(bool w_transposed) { return w_transposed ? Shape<true>::WAVES : Shape<false>::WAVES; }
size_t few_part_bytes(bool w_transposed, int rows) {
  const size_t fr = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  const size_t items = fr * 16 * (size_t)few_outputs(w_transposed), threads = (size_t)few_waves(w_transposed) * WAVE;
  const size_t each = w_transposed ? 8 : 4;
  return (items / each + threads - 1) / threads * threads * each * sizeof(float);
}

void launch_few(const Operands &a, const Out &o, bool x_transposed, bool w_transposed, bool swap, const FewPlan &pl,
                hipStream_t s) {
  const Operands b{a.w, a.x, a.w_stride, a.x_stride, a.k};
  const Operands &in = swap ? b : a;
  const bool xt = swap ? w_transposed : x_transposed, wt = swap ? x_transposed : w_transposed;
  if (xt)
    wt ? few_rows<true, true>(in, o, swap, pl, s) : few_rows<true, false>(in, o, swap, pl, s);
  else
    wt ? few_rows<false, true>(in, o, swap, pl, s) : few_rows<false, false>(in, o, swap, pl, s);
}

}  // namespace d3s
