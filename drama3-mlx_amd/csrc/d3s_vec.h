/* Eight elements of a row, fp32 or bf16, at any element.  Device code only. */
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
struct Vec8 {
  uint4 q[BF16 ? 1 : 2];

  __device__ __forceinline__ void load(const void *row, int64_t j) {
    const char *p = (const char *)row + j * (BF16 ? 2 : 4);
    __builtin_memcpy(&q[0], p, 16);
    if constexpr (!BF16) __builtin_memcpy(&q[1], p + 16, 16);
  }
  /* elements j .. j + 7 of which `left` (0 .. 8) are inside, the rest +0 */
  __device__ __forceinline__ void load_some(const void *row, int64_t j, int left) {
    if (left >= 8) {
      load(row, j);
      return;
    }
    uint32_t *w = (uint32_t *)q;
#pragma unroll
    for (int i = 0; i < (BF16 ? 4 : 8); i++) w[i] = 0u;
    if (left <= 0) return;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      if (e >= left) continue;
      if constexpr (BF16)
        w[e / 2] |= (uint32_t)((const uint16_t *)row)[j + e] << 16 * (e % 2);
      else
        w[e] = ((const uint32_t *)row)[j + e];
    }
  }
  __device__ __forceinline__ void values(float *v) const {
    const uint32_t *w = (const uint32_t *)q;
#pragma unroll
    for (int i = 0; i < (BF16 ? 4 : 8); i++) {
      if constexpr (BF16) {
        v[2 * i] = d3s_u2f(w[i] << 16);
        v[2 * i + 1] = d3s_u2f(w[i] & 0xffff0000u);
      } else {
        v[i] = d3s_u2f(w[i]);
      }
    }
  }
};

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

/* elements j .. j + 7 of a row, of which `left` are inside (the rest: `fill`) */
template <bool BF16>
__device__ __forceinline__ void load8(const void *row, int64_t j, int left, float *v, float fill = 0.0f) {
  if (left >= 8) {
    Vec8<BF16> q;
    q.load(row, j);
    q.values(v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = e < left ? load_at<BF16>(row, j + e) : fill;
  }
}

/* PAST: past the caches, for what is not read again soon */
template <bool PAST>
__device__ __forceinline__ void put16(void *p, uint4 q) {
  if constexpr (PAST)
    stream16(p, q);
  else
    __builtin_memcpy(p, &q, 16);
}

template <bool BF16, bool PAST = true>
__device__ __forceinline__ void store8(void *row, int64_t j, int left, const float *v) {
  if (left >= 8) {
    char *p = (char *)row + j * (BF16 ? 2 : 4);
    if constexpr (BF16) {
      put16<PAST>(p, make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])));
    } else {
      put16<PAST>(p, make_uint4(d3s_f2u(v[0]), d3s_f2u(v[1]), d3s_f2u(v[2]), d3s_f2u(v[3])));
      put16<PAST>(p + 16, make_uint4(d3s_f2u(v[4]), d3s_f2u(v[5]), d3s_f2u(v[6]), d3s_f2u(v[7])));
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (e < left) store_at<BF16>(row, j + e, v[e]);
  }
}

}  // namespace
}  // namespace d3s

#endif
