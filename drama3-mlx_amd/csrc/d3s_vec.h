/* A lane's elements of a row, fp32 or bf16, at any element.  Device code only.
 *
 * A lane takes E elements that follow each other, so that a store of 16 bytes a lane writes
 * whole lines: 8 where the output is bf16, 4 where it is fp32.  (8 fp32 elements are two
 * stores of half lines each: past the caches 40970 x 2048 of them took 110 us, so 74.) */
#ifndef D3S_VEC_H
#define D3S_VEC_H

#include "d3s_device.h"
#include "d3s_stream.h"

namespace d3s {
namespace {

/* rounded to the nearest even, a NaN to a quiet one (v_cvt_pk_bf16_f32) */
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
}

template <bool BF16>
__device__ __forceinline__ float load_at(const void *row, int64_t j) {
  if constexpr (BF16) return d3s_u2f((uint32_t)((const uint16_t *)row)[j] << 16);
  return ((const float *)row)[j];
}
template <bool BF16>
__device__ __forceinline__ void store_at(void *row, int64_t j, float v) {
  if constexpr (BF16)
    ((uint16_t *)row)[j] = (uint16_t)pack_bf16(v, 0.0f);
  else
    ((float *)row)[j] = v;
}

/* E elements as they are stored */
template <bool BF16, int E>
struct Vec {
  static constexpr int W = E * (BF16 ? 2 : 4) / 4;
  uint32_t w[W];

  __device__ __forceinline__ void load(const void *row, int64_t j) { __builtin_memcpy(w, (const char *)row + j * (BF16 ? 2 : 4), 4 * W); }
  /* elements j .. j + E - 1 of which `left` (any number) are inside, the rest +0 */
  __device__ __forceinline__ void load_some(const void *row, int64_t j, int64_t left) {
    if (left >= E) {
      load(row, j);
      return;
    }
#pragma unroll
    for (int i = 0; i < W; i++) w[i] = 0u;
    if (left <= 0) return;
    /* (put together behind the loads, so that none waits for the one before: the norm's gradient of bf16 4092 x 4100
     * 47 us, so 60, of 3276 x 5120 31 and 41) */
    uint32_t t[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
      t[e] = 0u;
      if (e >= left) continue;
      if constexpr (BF16)
        t[e] = ((const uint16_t *)row)[j + e];
      else
        t[e] = ((const uint32_t *)row)[j + e];
    }
#pragma unroll
    for (int e = 0; e < E; e++) {
      if constexpr (BF16)
        w[e / 2] |= t[e] << 16 * (e % 2);
      else
        w[e] = t[e];
    }
  }
  __device__ __forceinline__ void values(float *v) const {
#pragma unroll
    for (int i = 0; i < W; i++) {
      if constexpr (BF16) {
        v[2 * i] = d3s_u2f(w[i] << 16);
        v[2 * i + 1] = d3s_u2f(w[i] & 0xffff0000u);
      } else {
        v[i] = d3s_u2f(w[i]);
      }
    }
  }
};

/* elements j .. j + E - 1 of a row, of which `left` are inside (the rest: 0) */
template <bool BF16, int E>
__device__ __forceinline__ void load_row(const void *row, int64_t j, int64_t left, float *v) {
  Vec<BF16, E> q;
  q.load_some(row, j, left);
  q.values(v);
}

/* the first `left` of E elements, to j .. of a row.  PAST: past the caches, for what is not
 * read again soon */
template <bool BF16, int E, bool PAST = true>
__device__ __forceinline__ void store_row(void *row, int64_t j, int64_t left, const float *v) {
  if (left >= E) {
    char *p = (char *)row + j * (BF16 ? 2 : 4);
    constexpr int W = Vec<BF16, E>::W;
    uint32_t w[W];
#pragma unroll
    for (int i = 0; i < W; i++) w[i] = BF16 ? pack_bf16(v[2 * i], v[2 * i + 1]) : d3s_f2u(v[i]);
    if constexpr (PAST && W >= 4) { /* (a loop over the stores would lose their being non-temporal) */
      stream16(p, make_uint4(w[0], w[1], w[2], w[3]));
      if constexpr (W > 4) stream16(p + 16, make_uint4(w[W - 4], w[W - 3], w[W - 2], w[W - 1]));
    } else {
      __builtin_memcpy(p, w, 4 * W);
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; e++)
      if (e < left) store_at<BF16>(row, j + e, v[e]);
  }
}

/* Rows of chunks, the chunks of all rows counted through, so that no lane is idle behind a row's
 * end.  A thread finds its row from its workgroup's first chunk: one division for the workgroup, and
 * a comparison (or, in short rows, a product by `over`, 2^20 / chunks rounded up: exact below
 * 512) for the thread. */
struct Spread {
  int64_t chunks; /* of a row */
  uint32_t over;
  int64_t blocks; /* of T threads */

  template <int T>
  static Spread of(int64_t rows, int64_t width, int elements) {
    static_assert(T <= 256, "");
    Spread c;
    c.chunks = (width + elements - 1) / elements;
    c.over = c.chunks < T ? (uint32_t)(((1 << 20) + c.chunks - 1) / c.chunks) : 0u;
    c.blocks = (rows * c.chunks + T - 1) / T;
    return c;
  }
  template <int T>
  __device__ __forceinline__ void find(int64_t blk, int64_t *row, int64_t *chunk) const {
    const int64_t first = blk * T, r0 = first / chunks, c0 = first - r0 * chunks;
    if (chunks < T) { /* c0 + threadIdx.x < 2 T */
      const uint32_t t = (uint32_t)c0 + threadIdx.x, r = t * over >> 20;
      *row = r0 + r, *chunk = t - r * (uint32_t)chunks;
    } else {
      const int64_t t = c0 + threadIdx.x;
      const bool next = t >= chunks;
      *row = r0 + next, *chunk = next ? t - chunks : t;
    }
  }
};

}  // namespace
}  // namespace d3s

#endif
