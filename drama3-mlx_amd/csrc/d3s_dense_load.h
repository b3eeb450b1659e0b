/* What the products' kernels load and store at any element.  Device code only. */
#ifndef D3S_DENSE_LOAD_H
#define D3S_DENSE_LOAD_H

#include "d3s_dense.h"
#include "d3s_device.h"
#include "d3s_stream.h"

namespace d3s {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

/* 16 bytes at any element */
__device__ __forceinline__ uint4 load16(const void *p) {
  uint4 q;
  __builtin_memcpy(&q, p, 16);
  return q;
}
/* elements [at, at + 8) of a stored row of `len`, zeros past its end (at < len) */
__device__ __forceinline__ uint4 row_chunk(const uint16_t *row, int64_t at, int64_t len) {
  uint64_t v[2] = {0u, 0u};
  if (len >= 8) { /* near its end the row's last eight, moved down */
    const int64_t from = at < len - 8 ? at : len - 8;
    __builtin_memcpy(v, row + from, 16);
    const int s = (int)(at - from) * 16; /* 0 .. 112 */
    const uint64_t hi = v[1];
    v[1] = s < 64 ? hi >> s : 0u;
    v[0] = s == 0 ? v[0] : s < 64 ? v[0] >> s | hi << (64 - s) : hi >> (s - 64);
  } else {
#pragma nounroll
    for (int64_t e = len - 1; e >= at; e--) {
      v[1] = v[1] << 16 | v[0] >> 48;
      v[0] = v[0] << 16 | row[e];
    }
  }
  return make_uint4((uint32_t)v[0], (uint32_t)(v[0] >> 32), (uint32_t)v[1], (uint32_t)(v[1] >> 32));
}

}  // namespace
}  // namespace d3s

#endif
