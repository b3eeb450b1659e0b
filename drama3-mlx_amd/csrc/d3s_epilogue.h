/* The epilogue of a dense layer and its slopes (include/d3s_train.h), shared by
 * the products' kernels and the activation's gradient.  Device code only. */
#ifndef D3S_EPILOGUE_H
#define D3S_EPILOGUE_H

#include "d3s_dense.h"
#include "d3s_device.h"

namespace d3s {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

/* 1 / (1 + exp(-z)): exp overflows to infinity for z below -88, and 1 / inf is 0 */
__device__ __forceinline__ float logistic(float z) { return 1.0f / (1.0f + __expf(-z)); }

constexpr float GELU_C = 0.7978845608028654f; /* sqrt(2 / pi) */
constexpr float GELU_A = 0.044715f;

__device__ __forceinline__ float tanh_of(float u) { return 1.0f - 2.0f / (1.0f + __expf(2.0f * u)); }

template <int ACT>
__device__ __forceinline__ float activated(float z) {
  /* far below, z times a probability that is 0 in fp32 (-inf times it would be NaN) */
  if (ACT > D3S_ACT_RELU && z < -100.0f) return 0.0f;
  switch (ACT) {
    case D3S_ACT_RELU: return z < 0.0f ? 0.0f : z; /* (a NaN stays one) */
    case D3S_ACT_SILU: return z * logistic(z);
    case D3S_ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
    case D3S_ACT_GELU_TANH: return 0.5f * z * (1.0f + tanh_of(GELU_C * z * fmaf(GELU_A * z, z, 1.0f)));
  }
  return z;
}
template <int ACT, int N>
__device__ __forceinline__ void activate_each(float *z) {
#pragma unroll
  for (int e = 0; e < N; e++) z[e] = activated<ACT>(z[e]);
}
/* (one branch for all N) */
template <int N>
__device__ __forceinline__ void activate(float *z, int act) {
  switch (act) {
    case D3S_ACT_RELU: activate_each<D3S_ACT_RELU, N>(z); break;
    case D3S_ACT_SILU: activate_each<D3S_ACT_SILU, N>(z); break;
    case D3S_ACT_GELU: activate_each<D3S_ACT_GELU, N>(z); break;
    case D3S_ACT_GELU_TANH: activate_each<D3S_ACT_GELU_TANH, N>(z); break;
  }
}

__device__ __forceinline__ float slope(float z, int act) {
  /* far out the slope is 0 or 1 in fp32, and its terms could be 0 times infinity */
  if (act > D3S_ACT_RELU && fabsf(z) > 100.0f) return z > 0.0f ? 1.0f : 0.0f;
  switch (act) {
    case D3S_ACT_RELU: return z > 0.0f ? 1.0f : z == z ? 0.0f : z;
    case D3S_ACT_SILU: {
      const float f = logistic(z);
      return f * fmaf(z, 1.0f - f, 1.0f);
    }
    case D3S_ACT_GELU: /* the normal distribution's function and z times its density */
      return fmaf(z * 0.3989422804014327f, __expf(-0.5f * z * z), 0.5f * (1.0f + erff(z * 0.70710678118654752f)));
    case D3S_ACT_GELU_TANH: {
      const float t = tanh_of(GELU_C * z * fmaf(GELU_A * z, z, 1.0f));
      return 0.5f * (1.0f + t) + 0.5f * z * (1.0f - t * t) * GELU_C * fmaf(3.0f * GELU_A * z, z, 1.0f);
    }
  }
  return 1.0f;
}

__device__ __forceinline__ float bf(uint16_t b) { return d3s_u2f((uint32_t)b << 16); }

/* two rounded to bf16, to nearest even */
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
}
__device__ __forceinline__ uint16_t pack1(float a) { return (uint16_t)pack2(a, 0.0f); }

/* 16 bytes at any element */
__device__ __forceinline__ uint4 load16(const void *p) {
  uint4 q;
  __builtin_memcpy(&q, p, 16);
  return q;
}
__device__ __forceinline__ void store16(void *p, uint4 q) { __builtin_memcpy(p, &q, 16); }

/* output (i, j), its sum s */
__device__ __forceinline__ void put_one(const Out &o, int i, int j, float s) {
  if (o.bias) s += bf(o.bias[j]);
  if (o.z) o.z[(int64_t)i * o.z_stride + j] = pack1(s);
  activate<1>(&s, o.act);
  if (o.f32) {
    if (o.residual) s += ((const float *)o.residual)[(int64_t)i * o.residual_stride + j];
    ((float *)o.y)[(int64_t)i * o.y_stride + j] = s;
  } else {
    if (o.residual) s += bf(((const uint16_t *)o.residual)[(int64_t)i * o.residual_stride + j]);
    ((uint16_t *)o.y)[(int64_t)i * o.y_stride + j] = pack1(s);
  }
}

/* elements of y's type: eight neighbouring ones of a residual */
struct Eight {
  uint4 lo, hi; /* (bf16: lo alone) */
};

/* residual (i, j .. j + 7); nothing where the eight are not all there */
__device__ __forceinline__ void get_eight(const Out &o, int i, int j, Eight &r) {
  r.lo = r.hi = make_uint4(0u, 0u, 0u, 0u);
  if (!o.residual || i >= o.m || j + 8 > o.n) return;
  const int64_t at = (int64_t)i * o.residual_stride + j;
  if (o.f32) {
    r.lo = load16((const float *)o.residual + at);
    r.hi = load16((const float *)o.residual + at + 4);
  } else {
    r.lo = load16((const uint16_t *)o.residual + at);
  }
}

__device__ __forceinline__ void bf_eight(uint4 q, float *v) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int e = 0; e < 4; e++) {
    v[2 * e] = d3s_u2f(w[e] << 16);
    v[2 * e + 1] = d3s_u2f(w[e] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint4 pack_eight(const float *s) {
  return make_uint4(pack2(s[0], s[1]), pack2(s[2], s[3]), pack2(s[4], s[5]), pack2(s[6], s[7]));
}

/* the bias of outputs j .. j + 7, zeros where the eight are not all there */
__device__ __forceinline__ uint4 bias_eight(const Out &o, int j) {
  return o.bias && j + 8 <= o.n ? load16(o.bias + j) : make_uint4(0u, 0u, 0u, 0u);
}

/* Outputs (i, j .. j + 7), in two steps, so that the second, light, can be
 * unrolled over rows whose residuals are in flight: first the sums at `sum` (16-byte
 * aligned) become activations, with the bias as bias_eight gave it ... */
__device__ __forceinline__ void activate_eight(const Out &o, int i, int j, float *sum, uint4 bias) {
  if (i >= o.m || j + 8 > o.n) return;
  float s[8], v[8];
  const f32x4 a = *(const f32x4 *)sum, b = *(const f32x4 *)(sum + 4);
  bf_eight(bias, v);
#pragma unroll
  for (int e = 0; e < 4; e++) s[e] = a[e] + v[e], s[e + 4] = b[e] + v[e + 4];
  if (o.z) store16(o.z + (int64_t)i * o.z_stride + j, pack_eight(s));
  activate<8>(s, o.act);
  *(f32x4 *)sum = f32x4{s[0], s[1], s[2], s[3]};
  *(f32x4 *)(sum + 4) = f32x4{s[4], s[5], s[6], s[7]};
}
/* ... then they are written, with the residual as get_eight gave it.  Where the
 * eight are not all there, `sum` still holds sums. */
__device__ __forceinline__ void put_eight(const Out &o, int i, int j, const float *sum, const Eight &r) {
  if (i >= o.m || j + 8 > o.n) return;
  f32x4 a = *(const f32x4 *)sum, b = *(const f32x4 *)(sum + 4);
  if (o.f32) {
    if (o.residual) a += __builtin_bit_cast(f32x4, r.lo), b += __builtin_bit_cast(f32x4, r.hi);
    float *y = (float *)o.y + (int64_t)i * o.y_stride + j;
    store16(y, __builtin_bit_cast(uint4, a));
    store16(y + 4, __builtin_bit_cast(uint4, b));
  } else {
    float s[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}, v[8];
    bf_eight(r.lo, v);
#pragma unroll
    for (int e = 0; e < 8; e++) s[e] = o.residual ? s[e] + v[e] : s[e];
    store16((uint16_t *)o.y + (int64_t)i * o.y_stride + j, pack_eight(s));
  }
}

}  // namespace
}  // namespace d3s

#endif
