/* Stores of outputs, and last reads of inputs.  Device code only. */
#ifndef D3S_STREAM_H
#define D3S_STREAM_H

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace d3s {
namespace {

/* 16 bytes of an output, at any element.  Non-temporal: they do not push out of
 * the caches what the kernel, or the next pass, still reads (ten tensors of 8.4
 * million fp32 gradients clipped: 168 us instead of 201; 4096 x 4097 fp32 logits'
 * gradient 26 instead of 32; 8192 x 2048 x 2048 with everything 84 instead of 93). */
__device__ __forceinline__ void stream16(void *p, uint4 q) {
  typedef uint32_t any4 __attribute__((ext_vector_type(4), aligned(2)));
  const any4 v = {q.x, q.y, q.z, q.w};
  __builtin_nontemporal_store(v, (any4 *)p);
}

/* ... of an input that nothing reads after (the same clipping: 163 us) */
__device__ __forceinline__ uint4 last16(const void *p) {
  typedef uint32_t any4 __attribute__((ext_vector_type(4), aligned(2)));
  const any4 v = __builtin_nontemporal_load((const any4 *)p);
  return make_uint4(v[0], v[1], v[2], v[3]);
}

}  // namespace
}  // namespace d3s

#endif
