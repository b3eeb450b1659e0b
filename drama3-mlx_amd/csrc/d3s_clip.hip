/* k_norm, k_clip: the global L2 norm of many gradients, and the gradients
 * scaled to it (gfx950, wave64; include/d3s_train.h).
 *
 * The tensors' addresses and lengths travel as kernel arguments (as many a
 * launch as 4 KiB hold: a launch costs more than a short tensor's work), those of
 * many tensors on to k_clip in the workspace, so the call keeps nothing and may be
 * captured; a tensor of more than 2^30 elements
 * travels in pieces.  A launch's elements are cut into chunks of one size.
 * k_norm: workgroups take chunks in turn, square in 64 bits (a bf16's square is
 * exact and an fp32's keeps its range: nothing overflows, and the order costs no
 * accuracy; the conversions hide behind the loads) and leave one partial sum
 * each (a later launch of the same call adds to them).  k_clip: every workgroup
 * adds all partial sums in one order (they are 8 KiB of L2; a launch of its own for
 * it would cost more), and scales its chunks, from the last to the first: the end
 * of the norm's pass is what the cache still holds, and the stores leave it there.
 * Bound: HBM; the second pass over the gradients is the operation's own.  Ten
 * tensors of 8.4 million fp32: the norm 59 us (5.7 TB/s), the scaling 103 (6.5 TB/s;
 * with stores through the caches 200 in all, so 162); 150 ragged tensors of 2
 * million elements in all: 14 us, two launches. */
#include <type_traits>

#include "d3s_device.h"
#include "d3s_stream.h"
#include "d3s_train_internal.h"

namespace d3s {
namespace {

constexpr int CT = 256;
constexpr int CW = CT / WAVE;
constexpr int NORM_PIECES = 248;  /* a launch of k_norm */
constexpr int CLIP_PIECES = 164;  /* a launch of k_clip */
constexpr int64_t PIECE = (int64_t)1 << 30; /* elements, at most */
constexpr int CLIP_GROUPS = 1024;  /* workgroups a launch of k_norm: its partial sums */
constexpr int CU = 4;              /* 16-byte loads a lane has in flight */

template <int MOST>
struct Pieces {
  const void *src[MOST];
  uint32_t first[MOST]; /* the piece's first chunk */
  uint32_t numel[MOST]; /* elements << 1 | bf16 */
  int n;
  uint32_t chunks;
  uint32_t chunk; /* 16-byte units a chunk */
};
struct ClipOut {
  void *dst[CLIP_PIECES];
};

/* the pieces of many tensors, in the workspace */
struct Table {
  const void **src;
  void **dst;
  uint32_t *first, *numel;
  int n;
  uint32_t chunks, chunk;
};

/* what a launch of k_norm files there: its pieces from `at` on, chunks from `chunk0` */
struct Filed {
  void *dst[CLIP_PIECES];
  Table to;
  int at;
  uint32_t chunk0;
};
struct Nothing {};

/* a chunk of a piece: elements [j0, j1) from an aligned start, or cut by the piece's ends */
struct Chunk {
  int t;
  bool bf16;
  int64_t j0, j1;
};

/* chunk i of a piece that starts with chunk `first` */
__device__ __forceinline__ Chunk chunk_of(const void *src, uint32_t numel, uint32_t first, uint32_t chunk, uint32_t i) {
  Chunk c;
  c.bf16 = (numel & 1u) != 0u;
  const int64_t n = (int64_t)(numel >> 1), per = (int64_t)chunk * (c.bf16 ? 8 : 4);
  const int64_t lead = (int64_t)((uintptr_t)src & 15u) / (c.bf16 ? 2 : 4);
  c.j0 = (int64_t)(i - first) * per - lead;
  c.j1 = c.j0 + per < n ? c.j0 + per : n;
  return c;
}

/* chunk i's piece: the last of those that start at or before it, all starts loaded
 * at once (they ascend; a search would wait for one load after the other) */
template <int MOST>
__device__ __forceinline__ Chunk find_chunk(const Pieces<MOST> &a, uint32_t i) {
  int lo = -1;
#pragma unroll
  for (int w = 0; w < MOST; w += WAVE) {
    const int at = w + lane_id();
    lo += (int)__popcll(__ballot(at < a.n && a.first[min(at, MOST - 1)] <= i));
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  Chunk c = chunk_of(a.src[lo], a.numel[lo], a.first[lo], a.chunk, i);
  c.t = lo;
  return c;
}

/* the same in a table: the last 64th piece that starts at or before it, then the last of the 64 from there */
__device__ __forceinline__ Chunk find_chunk(const Table &a, uint32_t i) {
  int lo = -1;
  for (int w = 0; w < a.n; w += WAVE * WAVE) {
    const int at = w + lane_id() * WAVE;
    lo += (int)__popcll(__ballot(at < a.n && a.first[min(at, a.n - 1)] <= i));
  }
  const int at = lo * WAVE + lane_id();
  lo = lo * WAVE - 1 + (int)__popcll(__ballot(at < a.n && a.first[min(at, a.n - 1)] <= i));
  lo = __builtin_amdgcn_readfirstlane(lo);
  Chunk c = chunk_of(a.src[lo], a.numel[lo], a.first[lo], a.chunk, i);
  c.t = lo;
  return c;
}

__device__ __forceinline__ double square(float g) { return (double)g * (double)g; }

template <bool BF16>
__device__ __forceinline__ double squares(uint4 q) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (BF16) {
      const double x = d3s_u2f(w[i] << 16), y = d3s_u2f(w[i] & 0xffff0000u);
      s = fma(y, y, fma(x, x, s));
    } else {
      const double x = d3s_u2f(w[i]);
      s = fma(x, x, s);
    }
  }
  return s;
}

template <bool BF16>
__device__ __forceinline__ float element(const void *p, int64_t j) {
  if constexpr (BF16) return d3s_u2f((uint32_t)((const uint16_t *)p)[j] << 16);
  return ((const float *)p)[j];
}

/* the whole 16-byte units of [j0, j1) (j0 at an aligned address, or before the
 * tensor's start), and the elements before and after them */
template <bool BF16>
struct Span {
  static constexpr int EPC = BF16 ? 8 : 4;
  int64_t head0, head1, tail0, tail1; /* single elements */
  int64_t body;                       /* the first whole unit's element */
  int units;
  __device__ __forceinline__ Span(const Chunk &c) {
    body = c.j0 < 0 ? c.j0 + EPC : c.j0;
    if (body > c.j1) body = c.j1;
    head0 = c.j0 < 0 ? 0 : c.j0;
    head1 = body;
    units = (int)((c.j1 - body) / EPC);
    tail0 = body + (int64_t)units * EPC;
    tail1 = c.j1;
  }
};

template <bool BF16>
__device__ __forceinline__ double chunk_squares(const void *p, const Chunk &c) {
  const Span<BF16> s(c);
  const uint4 *b = (const uint4 *)((const char *)p + s.body * (BF16 ? 2 : 4));
  double sum[2] = {0.0, 0.0};
  int i = (int)threadIdx.x;
  for (; i + (CU - 1) * CT < s.units; i += CU * CT) {
    uint4 q[CU];
#pragma unroll
    for (int u = 0; u < CU; u++) q[u] = b[i + u * CT];
#pragma unroll
    for (int u = 0; u < CU; u++) sum[u & 1] += squares<BF16>(q[u]);
  }
  for (; i < s.units; i += CT) sum[0] += squares<BF16>(b[i]);
  const int64_t h = s.head0 + threadIdx.x, e = s.tail0 + threadIdx.x;
  if (h < s.head1) sum[1] += square(element<BF16>(p, h));
  if (e < s.tail1) sum[1] += square(element<BF16>(p, e));
  return sum[0] + sum[1];
}

/* the workgroup's sum, in thread order by a fixed tree, in every thread */
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[CW];
#pragma unroll
  for (int o = WAVE / 2; o > 0; o /= 2) v += __shfl_xor(v, o);
  __syncthreads();
  if (lane_id() == 0) part[threadIdx.x / WAVE] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int w = 1; w < CW; w++) v += part[w];
  return v;
}

template <int MOST, class F>
__global__ __launch_bounds__(CT) void k_norm(Pieces<MOST> a, F filed, double *parts, int have) {
  double sum = 0.0;
  if constexpr (!std::is_same_v<F, Nothing>) {
    if (blockIdx.x == 0 && (int)threadIdx.x < a.n) {
      static_assert(MOST <= CT, "a thread a piece");
      const int i = (int)threadIdx.x;
      filed.to.src[filed.at + i] = a.src[i];
      filed.to.dst[filed.at + i] = filed.dst[i];
      filed.to.first[filed.at + i] = filed.chunk0 + a.first[i];
      filed.to.numel[filed.at + i] = a.numel[i];
    }
  }
  for (uint32_t i = blockIdx.x; i < a.chunks; i += gridDim.x) {
    const Chunk c = find_chunk(a, i);
    sum += c.bf16 ? chunk_squares<true>(a.src[c.t], c) : chunk_squares<false>(a.src[c.t], c);
  }
  sum = block_sum(sum);
  if (threadIdx.x == 0) parts[blockIdx.x] = (int)blockIdx.x < have ? parts[blockIdx.x] + sum : sum;
}

/* the norm from its partial sums, in every thread */
__device__ __forceinline__ float norm_of(const double *parts, int n_parts) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n_parts; i += CT) s += parts[i];
  return (float)sqrt(block_sum(s));
}

__global__ __launch_bounds__(CT) void k_norm_write(const double *parts, int n_parts, float *norm) {
  const float v = norm_of(parts, n_parts);
  if (threadIdx.x == 0) *norm = v;
}

template <bool BF16>
__device__ __forceinline__ uint4 scaled(uint4 q, float scale) {
  uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (BF16) {
      const float x = d3s_u2f(w[i] << 16) * scale, y = d3s_u2f(w[i] & 0xffff0000u) * scale;
      w[i] = (uint32_t)d3s_f32_to_bf16_rn(x) | (uint32_t)d3s_f32_to_bf16_rn(y) << 16;
    } else {
      w[i] = d3s_f2u(d3s_u2f(w[i]) * scale);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <bool BF16>
__device__ __forceinline__ void scale_one(const void *p, void *d, int64_t j, float scale, bool keep) {
  if constexpr (BF16) {
    const uint16_t g = ((const uint16_t *)p)[j];
    ((uint16_t *)d)[j] = keep ? g : d3s_f32_to_bf16_rn(d3s_u2f((uint32_t)g << 16) * scale);
  } else {
    const float g = ((const float *)p)[j];
    ((float *)d)[j] = keep ? g : g * scale;
  }
}

/* keep: the bits as they are (no clipping) */
template <bool BF16>
__device__ __forceinline__ void chunk_scale(const void *p, void *d, const Chunk &c, float scale, bool keep) {
  const Span<BF16> s(c);
  constexpr int ES = BF16 ? 2 : 4;
  const uint4 *b = (const uint4 *)((const char *)p + s.body * ES);
  char *o = (char *)d + s.body * ES; /* (at any element: the stores may be unaligned) */
  int i = (int)threadIdx.x;
  for (; i + (CU - 1) * CT < s.units; i += CU * CT) {
    uint4 q[CU];
#pragma unroll
    for (int u = 0; u < CU; u++) q[u] = last16(b + i + u * CT);
#pragma unroll
    for (int u = 0; u < CU; u++) {
      if (!keep) q[u] = scaled<BF16>(q[u], scale);
      stream16(o + (int64_t)(i + u * CT) * 16, q[u]);
    }
  }
  for (; i < s.units; i += CT) {
    uint4 q = b[i];
    if (!keep) q = scaled<BF16>(q, scale);
    stream16(o + (int64_t)i * 16, q);
  }
  const int64_t h = s.head0 + threadIdx.x, e = s.tail0 + threadIdx.x;
  if (h < s.head1) scale_one<BF16>(p, d, h, scale, keep);
  if (e < s.tail1) scale_one<BF16>(p, d, e, scale, keep);
}

template <class P, class O>
__global__ __launch_bounds__(CT) void k_clip(P a, O out, const double *parts, int n_parts, float max_norm, float *norm) {
  const float v = norm_of(parts, n_parts);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = v;
  const bool keep = !(v > max_norm && v < __builtin_inff());
  const float scale = max_norm / v;
  for (uint32_t i = blockIdx.x; i < a.chunks; i += gridDim.x) {
    const Chunk c = find_chunk(a, a.chunks - 1 - i);
    if (keep && out.dst[c.t] == a.src[c.t]) continue;
    if (c.bf16)
      chunk_scale<true>(a.src[c.t], out.dst[c.t], c, scale, keep);
    else
      chunk_scale<false>(a.src[c.t], out.dst[c.t], c, scale, keep);
  }
}

/* chunks of 4 KiB (a 16-byte unit a lane) up to 64 KiB, by what fills the workgroups of some launches */
uint32_t chunk_for(int64_t units, int64_t launches) {
  uint32_t chunk = CT;
  while (chunk < 16 * CT && units > (int64_t)chunk * CLIP_GROUPS * launches) chunk *= 2;
  return chunk;
}

/* walks the tensors' pieces, MOST at a time */
struct Walk {
  const void *const *src;
  void *const *dst;
  const int64_t *numel;
  const int32_t *dtypes;
  int n_tensors, t;
  int64_t at; /* elements of tensor t that are behind */

  /* the next pieces and their chunks, of `chunk` units (0: by the pieces' lengths); false: there are none left */
  template <int MOST>
  bool fill(Pieces<MOST> &a, void **out, uint32_t chunk = 0) {
    int64_t total = 0;
    a.n = 0;
    uint32_t units[MOST];
    while (t < n_tensors && a.n < MOST) {
      const int size = dtypes[t] == D3S_DTYPE_BF16 ? 2 : 4;
      const int64_t left = numel[t] - at, n = left < PIECE ? left : PIECE;
      if (n > 0) {
        a.src[a.n] = (const char *)src[t] + at * size;
        if (out) out[a.n] = (char *)dst[t] + at * size;
        a.numel[a.n] = (uint32_t)n << 1 | (size == 2 ? 1u : 0u);
        units[a.n] = (uint32_t)((n * size + (int64_t)((uintptr_t)a.src[a.n] & 15u) + 15) / 16);
        total += units[a.n];
        a.n++;
      }
      at += n;
      if (at >= numel[t]) t++, at = 0;
    }
    if (chunk == 0) chunk = chunk_for(total, 1);
    uint32_t first = 0; /* (at most 248 pieces of 2^18 chunks) */
    for (int i = 0; i < a.n; i++) {
      a.first[i] = first;
      first += (units[i] + chunk - 1) / chunk;
    }
    a.chunks = first;
    a.chunk = chunk;
    return a.n > 0;
  }
};

}  // namespace

/* More tensors than a launch of k_clip holds: the launches of k_norm file their
 * pieces in a table, and one launch of k_clip takes them from there (700000 fp32
 * elements in 260 tensors 14.3 us, 18.6 with a launch for every 164 of them, in 1000
 * 39 and 53, in 170 12.7 and 13.5; 8 million bf16 in 214: 20.7 and 21.9).  A tensor of several pieces:
 * launch by launch (the table's room is by the tensors' number). */
static bool tabled(const int64_t *numel, const int32_t *dtypes, int n_tensors, int64_t *units) {
  int n = 0;
  *units = 0;
  for (int t = 0; t < n_tensors; t++) {
    if (numel[t] > PIECE) return false;
    n += numel[t] > 0;
    *units += (numel[t] * (dtypes[t] == D3S_DTYPE_BF16 ? 2 : 4) + 15) / 16;
  }
  return n > CLIP_PIECES;
}

size_t clip_workspace_bytes(int n_tensors) {
  const size_t table = n_tensors > CLIP_PIECES ? (size_t)n_tensors * (2 * sizeof(void *) + 2 * sizeof(uint32_t)) : 0;
  return split_counter_bytes() + CLIP_GROUPS * sizeof(double) + table;
}

void launch_clip(const void *const *src, void *const *dst, const int64_t *numel, const int32_t *dtypes, int n_tensors,
                 float max_norm, float *norm, void *ws, hipStream_t s) {
  double *parts = (double *)((char *)ws + split_counter_bytes());
  int n_parts = 0;
  int64_t units;
  if (dst && tabled(numel, dtypes, n_tensors, &units)) {
    Table to;
    to.src = (const void **)(parts + CLIP_GROUPS);
    to.dst = (void **)(to.src + n_tensors);
    to.first = (uint32_t *)(to.dst + n_tensors);
    to.numel = to.first + n_tensors;
    to.n = 0, to.chunks = 0;
    to.chunk = chunk_for(units, (n_tensors + CLIP_PIECES - 1) / CLIP_PIECES);
    Pieces<CLIP_PIECES> a;
    Filed f;
    Walk w{src, dst, numel, dtypes, n_tensors, 0, 0};
    while (w.fill(a, f.dst, to.chunk)) {
      f.to = to, f.at = to.n, f.chunk0 = to.chunks;
      const int groups = a.chunks < CLIP_GROUPS ? (int)a.chunks : CLIP_GROUPS;
      k_norm<<<groups, CT, 0, s>>>(a, f, parts, n_parts);
      if (groups > n_parts) n_parts = groups;
      to.n += a.n, to.chunks += a.chunks;
    }
    const int groups = to.chunks < 2 * CLIP_GROUPS ? (int)to.chunks : 2 * CLIP_GROUPS;
    k_clip<<<groups, CT, 0, s>>>(to, to, parts, n_parts, max_norm, norm);
    return;
  }
  {
    Pieces<NORM_PIECES> a;
    Walk w{src, dst, numel, dtypes, n_tensors, 0, 0};
    while (w.fill(a, nullptr)) {
      const int groups = a.chunks < CLIP_GROUPS ? (int)a.chunks : CLIP_GROUPS;
      k_norm<<<groups, CT, 0, s>>>(a, Nothing{}, parts, n_parts);
      if (groups > n_parts) n_parts = groups;
    }
  }
  bool written = false;
  if (dst) {
    Pieces<CLIP_PIECES> a;
    ClipOut o;
    Walk w{src, dst, numel, dtypes, n_tensors, 0, 0};
    while (w.fill(a, o.dst)) {
      const int groups = a.chunks < 2 * CLIP_GROUPS ? (int)a.chunks : 2 * CLIP_GROUPS;
      k_clip<<<groups, CT, 0, s>>>(a, o, parts, n_parts, max_norm, written ? nullptr : norm);
      written = true;
    }
  }
  if (!written) k_norm_write<<<1, CT, 0, s>>>(parts, n_parts, norm);
}

}  // namespace d3s
