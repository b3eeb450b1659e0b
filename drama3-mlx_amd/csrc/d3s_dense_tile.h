/* k_tile: a tile of y = residual + act(x w^T + bias) on the matrix cores, bf16
 * operands in either order, fp32 sums (gfx950, wave64; include/d3s_train.h).
 * Device code and its launch; each order of the operands is a translation unit.
 *
 * A workgroup of four waves owns TM x TN outputs; the inner length runs in
 * stages of 64, each operand's stage in LDS as [row][64]: rows of eight 16-byte
 * chunks, chunk c of row r at place c ^ (r ^ r / 8) % 8, so that a wave's reads
 * (one chunk of 32 rows) and its writes touch every bank alike.
 * Two stages lie in LDS (three or four of the small tiles' direct ones).
 * Fragments are read one step of 16 ahead of the matrix
 * instructions; the last step of a stage runs after the barrier that frees it,
 * so the next stage's first reads, and the filling of the freed one, hide
 * behind its products.
 * A stage reaches LDS directly (operands stored by rows, at 16 bytes), through
 * registers as it is (the same at any other element), through registers and
 * turned (operands stored by the inner index: a thread holds 8 rows of R / 32
 * inner indices and writes each row's together), or through registers as it
 * is stored by the inner index, [inner][row], to be read transposed.
 *
 * Bound: the matrix pipe, as far as LDS reads and the loads' issue leave it busy: 35 (both
 * operands by the inner index) to 51 % of a call.  On operands that are used again:
 * 8192 x 2048 x 2048 59 us (1160 TFLOP/s; from cold operands with every part of the
 * epilogue 77), 8192 x 8192 x 8192 805 us (1370 TFLOP/s), 8192 x 4097 x 2048 128 us (1070),
 * 4096 x 2048 x 8192 with both by the inner index 152 us (900 TFLOP/s). */
#ifndef D3S_DENSE_TILE_H
#define D3S_DENSE_TILE_H

#include <type_traits>

#include "d3s_dense_load.h"
#include "d3s_epilogue.h"

namespace d3s {
namespace {

constexpr int TT = 256;        /* threads of a workgroup */
constexpr int TK = TILE_K;     /* the inner length of a stage */
constexpr int STEP = 16;       /* ... of a matrix instruction */
constexpr unsigned TILE_GRID = 1 << 22; /* workgroups a launch: their threads are counted in 32 bits */

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

#define D3S_LDS __attribute__((address_space(3)))

/* how an operand's stages reach LDS, and how they lie there (above) */
enum Way { DIRECT, ROWS, TURNED, INNER };

/* One operand's part of a tile: R rows from r0 of [rows, k] (TURNED, INNER: stored [k, rows];
 * TURNED: eight rows at least). */
template <int R, Way WAY, int SETS>
struct Part {
  static constexpr int BYTES = R * TK * 2;
  static constexpr int PER = R * TK / 8 / TT;                      /* 16-byte loads a thread */
  static constexpr int DIRECTS = WAY == DIRECT ? PER : 0;          /* of them into LDS */
  static constexpr int LOADS = WAY == DIRECT ? 0 : PER;            /* ... into registers */
  static constexpr int WRITES = WAY == DIRECT ? 0 : WAY == TURNED ? 8 : PER; /* and from them */
  const uint16_t *p;
  int64_t stride;
  int rows, r0;
  uint32_t off[WAY == DIRECT ? PER : 1]; /* bytes from the tile's first row, and where that is */
  __amdgpu_buffer_rsrc_t from;
  const uint16_t *mine;                  /* TURNED, INNER: the thread's first chunk of stage 0 */
  int to;                                /* TURNED: its first row in LDS (below 0: not the tile's) */
  uint4 q[SETS][PER];

  static __device__ __forceinline__ int tid() { return (int)threadIdx.x; }
  static __device__ __forceinline__ int turn(int r) { return (r ^ r >> 3) & 7; }
  /* DIRECT, ROWS: the u-th place's row and chunk (eight places a row, in order) */
  static __device__ __forceinline__ int row(int u) { return (u * TT + tid()) / 8; }
  static __device__ __forceinline__ int chunk(int u) { return tid() % 8 ^ turn(row(u)); }
  /* TURNED: the thread's inner indices inside a stage, PER of them from here */
  static __device__ __forceinline__ int inner() { return tid() / (R / 8) * PER; }
  /* INNER: the u-th place's inner index, and its chunk: ACROSS places an index, in
   * order (the same chunk for every u) */
  static constexpr int ACROSS = R / 8;
  static __device__ __forceinline__ int spin(int k) { return (k & 3) << 2 & (ACROSS - 1); }
  static __device__ __forceinline__ int inner(int u) { return u * (TT / ACROSS) + tid() / ACROSS; }
  static __device__ __forceinline__ int across() { return tid() % ACROSS ^ spin(inner(0)); }

  __device__ __forceinline__ Part(const uint16_t *base, int64_t st, int n, int first)
      : p(base), stride(st), rows(n), r0(first) {
    /* rows past the end are the last one again: their outputs are not written */
    if constexpr (WAY == DIRECT) {
      from = __builtin_amdgcn_make_buffer_rsrc((void *)(p + (int64_t)r0 * stride), 0, -1, 0x00020000);
#pragma unroll
      for (int u = 0; u < PER; u++) off[u] = (uint32_t)(min(row(u), rows - 1 - r0) * stride + chunk(u) * 8) * 2u;
    } else if constexpr (WAY == TURNED) {
      /* eight rows that end with the last (written twice, the same) */
      to = min(tid() % (R / 8) * 8, rows - 8 - r0);
      mine = p + (int64_t)inner() * stride + (r0 + to);
    } else if constexpr (WAY == INNER) {
      /* (chunks past the rows are the last one again; one that is cut reads on into
       * the next inner index: see whole()) */
      to = min(across() * 8, (rows - 1 - r0) / 8 * 8);
      mine = p + (int64_t)inner(0) * stride + (r0 + to);
    }
  }
  /* the u-th 16 bytes of stage k0, straight into LDS (a buffer load: one 32-bit
   * register of address a lane; the sum of its offsets stays below 2^32) */
  __device__ __forceinline__ void direct(int u, int k0, char *lds) const {
    const int wid = __builtin_amdgcn_readfirstlane(tid() / WAVE);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (D3S_LDS void *)(lds + (u * TT + wid * WAVE) * 16), 16, (int)off[u],
                                             k0 * 2, 0, 0);
  }
  /* inner indices of which whole stages may be loaded: not the last, or of short
   * rows the last eight, where an INNER chunk is cut: it would read past the operand's end */
  __device__ __forceinline__ int whole(int k) const {
    const bool cut = WAY == INNER && r0 + R > rows && rows % 8 != 0;
    return cut ? max(k - (stride >= 8 ? 1 : 8), 0) : k;
  }
  /* the same into registers, from start(k0): a whole stage */
  __device__ __forceinline__ const uint16_t *start(int k0) const {
    return WAY == TURNED || WAY == INNER ? mine + (int64_t)k0 * stride : p + k0;
  }
  __device__ __forceinline__ void load(int set, int u, const uint16_t *at) {
    if constexpr (WAY == ROWS)
      q[set][u] = load16(at + ((int64_t)min(r0 + row(u), rows - 1) * stride + chunk(u) * 8));
    else
      q[set][u] = load16(at + u * (WAY == INNER ? TT / ACROSS * stride : stride));
  }
  /* the same of any stage: something finite or not from k1 on */
  __device__ __forceinline__ void load_some(int k0, int k1) {
#pragma unroll
    for (int u = 0; u < PER; u++) {
      if constexpr (WAY == TURNED) {
        q[0][u] = load16(p + (int64_t)min(k0 + inner() + u, k1 - 1) * stride + (r0 + to));
      } else if constexpr (WAY == INNER) {
        q[0][u] = row_chunk(p + (int64_t)min(k0 + inner(u), k1 - 1) * stride, r0 + to, rows);
      } else {
        const int k = k0 + chunk(u) * 8;
        const uint16_t *at = p + (int64_t)min(r0 + row(u), rows - 1) * stride;
        q[0][u] = k >= k1 ? make_uint4(0u, 0u, 0u, 0u) : WAY == DIRECT ? load16(at + k) : row_chunk(at, k, k1);
      }
    }
  }
  /* the v-th write of the registers into a stage (rows that are not the tile's: to `spare`) */
  __device__ __forceinline__ void write(int set, int v, char *lds, char *spare) const {
    if constexpr (WAY != TURNED) {
      *(uint4 *)(lds + (v * TT + tid()) * 16) = q[set][v];
    } else {
      static_assert(PER == 8, "a row's eight inner indices are one chunk");
      uint32_t w[4];
      auto word = [&](int u) { return v < 2 ? q[set][u].x : v < 4 ? q[set][u].y : v < 6 ? q[set][u].z : q[set][u].w; };
#pragma unroll
      for (int u = 0; u < 8; u += 2)
        w[u / 2] = __builtin_amdgcn_perm(word(u + 1), word(u), v & 1 ? 0x07060302u : 0x05040100u);
      const int r = to + v, k = inner();
      char *at = r < 0 ? spare : lds + (r * (TK * 2) + (k / 8 ^ turn(r)) * 16);
      *(uint4 *)at = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  __device__ __forceinline__ void write_all(char *lds, char *spare) const {
#pragma unroll
    for (int v = 0; v < (WAY == TURNED ? 8 : PER); v++) write(0, v, lds, spare);
  }
  /* the fragment of rows r .. r + 31 (r a multiple of 32), inner indices 16 step .. + 15 */
  static __device__ __forceinline__ bf16x8 fragment(const char *lds, int r, int step) {
    if constexpr (WAY == INNER) { /* two transposing reads: four inner indices of 16 rows a lane group */
      const int g = lane_id() >> 4, i = lane_id() & 15, k = step * STEP + (g >> 1) * 8 + (i >> 2);
      const int c = (r / 8 + (g & 1) * 2 + (i >> 1 & 1)) ^ spin(i >> 2);
      const char *at = lds + k * (R * 2) + c * 16 + (i & 1) * 8;
      const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((D3S_LDS bf16x4 *)at);
      const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((D3S_LDS bf16x4 *)(at + 4 * R * 2));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    const int at = r + (lane_id() & 31), c = (step * 2 + (lane_id() >> 5)) ^ turn(at);
    return *(const bf16x8 *)(lds + at * (TK * 2) + c * 16);
  }
};

/* all but the last N loads of the wave are there, and its reads of LDS; then every wave's */
template <int N>
__device__ __forceinline__ void stage_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | 7 << 4 | (N >> 4) << 14); /* vmcnt N, lgkmcnt 0 */
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

/* 16 bytes past the caches of one XCD */
constexpr int DEVICE_SCOPE = 16;

/* BUFS: stages in LDS.  AHEAD: stages through registers are loaded that many
 * before the one that is written next. */
template <int TM, int TN, int WAVES_M, int BUFS, int AHEAD, bool SPLIT, Way WX, Way WW>
__global__ __launch_bounds__(TT, 1) void k_tile(Operands a, Out o, TilePlan pl) {
  constexpr int WAVES_N = 4 / WAVES_M;
  constexpr int WM = TM / WAVES_M, WN = TN / WAVES_N, FM = WM / 32, FN = WN / 32;
  constexpr int STEPS = TK / STEP, SETS = AHEAD + 1;
  using PX = Part<TM, WX, SETS>;
  using PW = Part<TN, WW, SETS>;
  constexpr int STAGE = PX::BYTES + PW::BYTES;
  constexpr int OUT_ROW = WN + 4; /* a row of outputs in LDS, fp32 */
  constexpr int OUT_BYTES = 4 * 32 * OUT_ROW * 4;
  constexpr int ROOM = BUFS * STAGE > OUT_BYTES ? BUFS * STAGE : OUT_BYTES;
  __shared__ __attribute__((aligned(1024))) char lds[ROOM + 16];
  char *spare = lds + ROOM;
  static_assert(WX == DIRECT && WW == DIRECT ? AHEAD == 0 : BUFS == 2, "what the waits below count");
  static_assert(SETS <= 2, "the loop over stages takes two at a time");

  /* workgroups go to the eight XCDs in turn: each takes a run of neighbouring
   * tiles, in columns of eight, whose operands its L2 then holds */
  const unsigned turn = blockIdx.x % 8, each = gridDim.x / 8;
  const unsigned t = pl.first + turn * each + min(turn, gridDim.x % 8) + blockIdx.x / 8;
  const unsigned split = SPLIT ? t / pl.tiles : 0u, tile = SPLIT ? t % pl.tiles : t;
  const unsigned wide = pl.group * pl.n_tiles, band = tile / wide, in = tile % wide;
  const unsigned high = min(pl.group, pl.m_tiles - band * pl.group); /* tiles in a column of the band */
  const int i0 = (int)(band * pl.group + in % high) * TM, j0 = (int)(in / high) * TN;

  const int lane = lane_id(), wid = __builtin_amdgcn_readfirstlane((int)threadIdx.x / WAVE);
  const int wi = wid / WAVES_N * WM, wj = wid % WAVES_N * WN; /* the wave's rows and outputs */
  PX px(a.x, a.x_stride, o.m, i0);
  PW pw(a.w, a.w_stride, o.n, j0);

  f32x16 acc[FM][FN];
#pragma unroll
  for (int p = 0; p < FM; p++)
#pragma unroll
    for (int q = 0; q < FN; q++)
#pragma unroll
      for (int i = 0; i < 16; i++) acc[p][q][i] = 0.0f;

  const int whole = min(px.whole(a.k), pw.whole(a.k)) / TK;
  const int s0 = min(whole, (int)split * pl.stages);
  const int s1 = split == pl.splits - 1 ? whole : min(whole, s0 + pl.stages);
  bf16x8 fx[2][FM], fw[2][FN];
  auto read = [&](int to, const char *stage, int step, int f) {
    if (f < FM)
      fx[to][f] = PX::fragment(stage, wi + f * 32, step);
    else
      fw[to][f - FM] = PW::fragment(stage + PX::BYTES, wj + (f - FM) * 32, step);
  };
  auto read_all = [&](int to, const char *stage, int step) {
#pragma unroll
    for (int f = 0; f < FM + FN; f++) read(to, stage, step, f);
  };
  constexpr int DIRECTS = PX::DIRECTS + PW::DIRECTS, LOADS = PX::LOADS + PW::LOADS, WRITES = PX::WRITES + PW::WRITES;
  auto direct = [&](int u, int k0, char *to) {
    if (u < PX::DIRECTS)
      px.direct(u, k0, to);
    else
      pw.direct(u - PX::DIRECTS, k0, to + PX::BYTES);
  };
  struct Start {
    const uint16_t *x, *w;
  };
  auto start = [&](int k0) { return Start{px.start(k0), pw.start(k0)}; };
  auto load = [&](int set, int u, const Start &at) {
    if (u < PX::LOADS)
      px.load(set, u, at.x);
    else
      pw.load(set, u - PX::LOADS, at.w);
  };
  auto write = [&](int set, int v, char *to) {
    if (v < PX::WRITES)
      px.write(set, v, to, spare);
    else
      pw.write(set, v - PX::WRITES, to + PX::BYTES, spare);
  };
  /* the products of fragments `from`; after the n-th of them, and pinned there,
   * beside(n): its share of what goes on meanwhile */
  constexpr int PRODUCTS = FM * FN;
  auto multiply = [&](int from, auto beside) {
#pragma unroll
    for (int n = 0; n < PRODUCTS; n++) {
      const int p = n / FN, q = n % FN;
      acc[p][q] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fw[from][q], fx[from][p], acc[p][q], 0, 0, 0);
      beside(n);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  /* product n's share of `of` things spread over the products from `from` to `to` */
  auto share = [](int n, int from, int to, int of, auto each) {
    const int size = (of + to - from - 1) / (to - from), i0 = (n - from) * size;
#pragma unroll
    for (int i = i0; i < i0 + size; i++)
      if (n >= from && n < to && i < of) each(i);
  };
  /* Direct loads: the issue of one takes longer than a product hides beside an
   * LDS read, so they follow the reads, half of them in the next stage's first two
   * steps (8192 x 2048 x 8192: all in the last step 232 us, so 211).  With operands through registers they come last (an LDS write behind
   * them would wait for them), all at once. */
  constexpr int LATE = LOADS == 0 ? DIRECTS / 2 : 0, SOON = DIRECTS - LATE, HALF = PRODUCTS / 2;
  static_assert(LATE % 2 == 0, "two steps' shares");
  constexpr int WRITTEN = DIRECTS > 0 && HALF > 0 ? HALF : PRODUCTS;

  if (s0 < s1) {
    auto k_of = [&](int s) { return min(s, s1 - 1) * TK; }; /* (loads past the end: the last stage's, not read) */
#pragma unroll
    for (int b = 0; b < BUFS; b++) {
      const Start at = start(k_of(s0 + b));
#pragma unroll
      for (int u = 0; u < LOADS; u++) load(b % SETS, u, at);
#pragma unroll
      for (int u = 0; u < (b < BUFS - 1 ? DIRECTS : SOON); u++) direct(u, k_of(s0 + b), lds + b * STAGE);
#pragma unroll
      for (int v = 0; v < WRITES; v++) write(b % SETS, v, lds + b * STAGE);
    }
#pragma unroll
    for (int b = 2; b < 2 + AHEAD; b++) {
      const Start at = start(k_of(s0 + b));
#pragma unroll
      for (int u = 0; u < LOADS; u++) load(b % SETS, u, at);
    }
    stage_barrier<(BUFS - 2) * DIRECTS + SOON + AHEAD * LOADS>(); /* (registers' loads have been waited for) */
    read_all(0, lds, 0);
    char *here = lds;
    /* stage s, `turn` stages after a multiple of SETS */
    auto stage = [&](int s, auto turn) {
      constexpr int V = decltype(turn)::value;
      char *next = here == lds + (BUFS - 1) * STAGE ? lds : here + STAGE;
      char *back = here == lds ? lds + (BUFS - 1) * STAGE : here - STAGE;
      const int near = k_of(s + BUFS - 1), far = k_of(s + BUFS);
      const Start at = start(k_of(s + 2 + AHEAD));
#pragma unroll
      for (int j = 0; j < STEPS - 1; j++)
        multiply(j & 1, [&](int n) {
          share(n, 0, PRODUCTS, FM + FN, [&](int f) { read((j + 1) & 1, here, j + 1, f); });
          if (j < 2) share(n, HALF, PRODUCTS, LATE / 2, [&](int u) { direct(SOON + u + j * (LATE / 2), near, back); });
          if (j == 0) share(n, 0, PRODUCTS, LOADS, [&](int u) { load((V + 1) % SETS, u, at); });
        });
      /* the next stage is there: loads after its own may still be on their way */
      stage_barrier<(BUFS - 2) * DIRECTS + (AHEAD + 1) * LOADS>();
      multiply(1, [&](int n) {
        share(n, 0, PRODUCTS, FM + FN, [&](int f) { read(0, next, 0, f); });
        share(n, 0, WRITTEN, WRITES, [&](int v) { write((V + 2) % SETS, v, here); });
        share(n, HALF, PRODUCTS, SOON, [&](int u) { direct(u, far, here); });
      });
      here = next;
    };
    for (int s = s0; s < s1; s += SETS) {
      stage(s, std::integral_constant<int, 0>{});
      if constexpr (SETS > 1)
        if (s + 1 < s1) stage(s + 1, std::integral_constant<int, 1 % SETS>{});
    }
  }
  /* the rest of the inner length, what whole loads do not reach: zeros from its end on */
  const int end = split == pl.splits - 1 ? a.k : s1 * TK;
  for (int k0 = s1 * TK; k0 < end; k0 += TK) {
    px.load_some(k0, end);
    pw.load_some(k0, end);
    stage_barrier<0>();
    px.write_all(lds, spare);
    pw.write_all(lds + PX::BYTES, spare);
    stage_barrier<0>();
#pragma nounroll
    for (int j = 0; j < STEPS && k0 + j * STEP < end; j++) {
      read_all(0, lds, j);
      const int n = end - (k0 + j * STEP + (lane >> 5) * 8); /* of the lane's eight */
      uint4 mask;
      auto some = [&](int d) { return n >= 2 * d + 2 ? ~0u : n == 2 * d + 1 ? 0xffffu : 0u; };
      mask = make_uint4(some(0), some(1), some(2), some(3));
      auto cut = [&](bf16x8 &f) {
        uint4 v = __builtin_bit_cast(uint4, f);
        f = __builtin_bit_cast(bf16x8, make_uint4(v.x & mask.x, v.y & mask.y, v.z & mask.z, v.w & mask.w));
      };
#pragma unroll
      for (int p = 0; p < FM; p++) cut(fx[0][p]);
#pragma unroll
      for (int q = 0; q < FN; q++) cut(fw[0][q]);
      multiply(0, [](int) {});
    }
  }

  /* A split's sums go to the workspace, complete before its arrival is counted;
   * the last to arrive adds them below, in the order of the splits, so the bits
   * do not depend on who that is. */
  const int at = (int)threadIdx.x * 16;
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  auto block = [&](unsigned s) {
    float *parts = pl.parts + ((size_t)tile * pl.splits + s) * (TM * TN);
    return __builtin_amdgcn_make_buffer_rsrc(parts, 0, TM * TN * 4, 0x00020000);
  };
  if constexpr (SPLIT) {
    const __amdgpu_buffer_rsrc_t own = block(split);
#pragma unroll
    for (int c = 0; c < FM * FN * 4; c++) {
      const f32x16 &v = acc[c / 4 / FN][c / 4 % FN];
      const f32x4 s = {v[c % 4 * 4], v[c % 4 * 4 + 1], v[c % 4 * 4 + 2], v[c % 4 * 4 + 3]};
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, s), own, at, c * (TT * 16), DEVICE_SCOPE);
    }
    stage_barrier<0>();
    unsigned *last = (unsigned *)spare;
    if (threadIdx.x == 0) {
      uint32_t *count = pl.arrivals + (size_t)tile * 32;
      const bool is = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == pl.splits - 1;
      if (is) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      *last = is;
    }
    __syncthreads();
    if (!*last) return;
  }

  /* Each wave's outputs, 32 rows at a time, through its part of LDS, so that
   * a row leaves in whole lines.  Lane l holds row l % 32, and four neighbouring
   * outputs from 8 i + 4 (l / 32) in registers 4 i .. 4 i + 3.  One copy of the
   * code that writes rows (unrolled four times it does not fit the instruction
   * cache); the residual's rows are loaded 32 ahead. */
  stage_barrier<0>();
  constexpr int ACROSS = WN / 8, DOWN = WAVE / ACROSS, ROUNDS = 32 / DOWN;
  float *mine = (float *)lds + wid * 32 * OUT_ROW;
  float *row = mine + lane / ACROSS * OUT_ROW + lane % ACROSS * 8;
  const Eights<ROUNDS, DOWN, OUT_ROW> out(o, i0 + wi + lane / ACROSS, j0 + wj + lane % ACROSS * 8);
  const bool works = o.bias || o.z || o.act != D3S_ACT_NONE;
  typename Eights<ROUNDS, DOWN, OUT_ROW>::Residual now, ahead;
  out.get(ahead, 0);
#pragma nounroll
  for (int p = 0; p < FM; p++) {
    wave_lds_sync();
    auto stage_out = [&](int q, int i, f32x4 v) {
      *(f32x4 *)(mine + (lane & 31) * OUT_ROW + q * 32 + i * 8 + (lane >> 5) * 4) = v;
    };
    if constexpr (SPLIT) {
      f32x4 sum[FN * 4];
#pragma unroll
      for (int c = 0; c < FN * 4; c++) sum[c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 2
      for (unsigned s = 0; s < pl.splits; s++) {
        const __amdgpu_buffer_rsrc_t from = block(s);
#pragma unroll
        for (int c = 0; c < FN * 4; c++)
          sum[c] += __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(from, at, (p * FN * 4 + c) * (TT * 16), DEVICE_SCOPE));
      }
#pragma unroll
      for (int c = 0; c < FN * 4; c++) stage_out(c / 4, c % 4, sum[c]);
    } else {
#pragma unroll
      for (int c = 0; c < FM; c++)
        if (c == p) {
#pragma unroll
          for (int q = 0; q < FN; q++)
#pragma unroll
            for (int i = 0; i < 4; i++)
              stage_out(q, i, f32x4{acc[c][q][4 * i], acc[c][q][4 * i + 1], acc[c][q][4 * i + 2], acc[c][q][4 * i + 3]});
        }
    }
    wave_lds_sync();
    now = ahead;
    if (p + 1 < FM) out.get(ahead, (p + 1) * 32);
    if (works) out.activate(row, p * 32);
    out.put(row, p * 32, now);
    out.put_rest(row, p * 32);
  }
}

template <int TM, int TN, int WAVES_M, int BUFS, int AHEAD, Way WX, Way WW>
void launch_ways(const Operands &a, const Out &o, TilePlan pl, hipStream_t s) {
  const unsigned all = pl.tiles * pl.splits;
  for (pl.first = 0; pl.first < all; pl.first += TILE_GRID) {
    const dim3 grid(min(TILE_GRID, all - pl.first));
    bool split = false;
    if constexpr (TM == 128 && TN == 128) {
      split = pl.splits > 1;
      if (split) k_tile<TM, TN, WAVES_M, BUFS, AHEAD, true, WX, WW><<<grid, TT, 0, s>>>(a, o, pl);
    }
    if (!split) k_tile<TM, TN, WAVES_M, BUFS, AHEAD, false, WX, WW><<<grid, TT, 0, s>>>(a, o, pl);
  }
}

/* Small tiles: both operands directly, or both through registers (a write
 * behind a direct load waits for it, and small tiles' loads are many stages ahead). */
template <int TM, int TN, int WAVES_M, int BUFS, int AHEAD, bool XT, bool WT>
void launch_small(const Operands &a, const Out &o, const TilePlan &pl, hipStream_t s) {
  if constexpr (!XT && !WT) {
    if (pl.x_direct && pl.w_direct) return launch_ways<TM, TN, WAVES_M, BUFS, 0, DIRECT, DIRECT>(a, o, pl, s);
  }
  launch_ways<TM, TN, WAVES_M, 2, AHEAD, XT ? INNER : ROWS, WT ? INNER : ROWS>(a, o, pl, s);
}

/* The large tile turns (8192 x 2048 x 8192, both by the inner index: 305 us, as they
 * are 335; one beside direct rows, k 4096: 121, as it is beside rows through
 * registers 134), the small ones read transposed (4096 x 2048 x 8192 in 128 x 256:
 * 160, turned 173; their writes have fewer products to hide behind). */
template <bool XT, bool WT>
void launch_large(const Operands &a, const Out &o, const TilePlan &pl, hipStream_t s) {
  if constexpr (XT && WT) {
    launch_ways<256, 256, 2, 2, 0, TURNED, TURNED>(a, o, pl, s);
  } else if constexpr (XT) {
    pl.w_direct ? launch_ways<256, 256, 2, 2, 0, TURNED, DIRECT>(a, o, pl, s) : launch_ways<256, 256, 2, 2, 0, TURNED, ROWS>(a, o, pl, s);
  } else if constexpr (WT) {
    pl.x_direct ? launch_ways<256, 256, 2, 2, 0, DIRECT, TURNED>(a, o, pl, s) : launch_ways<256, 256, 2, 2, 0, ROWS, TURNED>(a, o, pl, s);
  } else {
    if (pl.x_direct)
      pl.w_direct ? launch_ways<256, 256, 2, 2, 0, DIRECT, DIRECT>(a, o, pl, s) : launch_ways<256, 256, 2, 2, 0, DIRECT, ROWS>(a, o, pl, s);
    else
      pl.w_direct ? launch_ways<256, 256, 2, 2, 0, ROWS, DIRECT>(a, o, pl, s) : launch_ways<256, 256, 2, 2, 0, ROWS, ROWS>(a, o, pl, s);
  }
}

}  // namespace

template <bool XT, bool WT>
void launch_tiles(const Operands &a, const Out &o, const TilePlan &pl, hipStream_t s) {
  if (pl.tm == 256 && pl.tn == 256)
    launch_large<XT, WT>(a, o, pl, s);
  else if (pl.tn == 256)
    launch_small<128, 256, 2, 3, 1, XT, WT>(a, o, pl, s);
  else
    launch_small<128, 128, 2, 4, 1, XT, WT>(a, o, pl, s);
}

}  // namespace d3s

#endif
