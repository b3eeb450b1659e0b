/* The epilogue of a dense layer and its slopes (include/d3s_train.h), shared by
 * the products' kernels and the activation's gradient.  Device code only. */
#ifndef D3S_EPILOGUE_H
#define D3S_EPILOGUE_H

#include "d3s_device.h"
#include "d3s_train_internal.h"

namespace d3s {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

/* 1 / (1 + exp(-z)): exp overflows to infinity for z below -88, and 1 / inf is 0 */
__device__ __forceinline__ float logistic(float z) { return 1.0f / (1.0f + __expf(-z)); }

constexpr float GELU_C = 0.7978845608028654f; /* sqrt(2 / pi) */
constexpr float GELU_A = 0.044715f;

__device__ __forceinline__ float tanh_of(float u) { return 1.0f - 2.0f / (1.0f + __expf(2.0f * u)); }

__device__ __forceinline__ float activate(float z, int act) {
  /* far below, z times a probability that is 0 in fp32 (-inf times it would be NaN) */
  if (act > D3S_ACT_RELU && z < -100.0f) return 0.0f;
  switch (act) {
    case D3S_ACT_RELU: return z < 0.0f ? 0.0f : z; /* (a NaN stays one) */
    case D3S_ACT_SILU: return z * logistic(z);
    case D3S_ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
    case D3S_ACT_GELU_TANH: return 0.5f * z * (1.0f + tanh_of(GELU_C * z * fmaf(GELU_A * z, z, 1.0f)));
  }
  return z;
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

/* what a product's kernel needs to write its outputs */
struct Out {
  const uint16_t *bias;
  const void *residual;
  uint16_t *z;
  void *y;
  int64_t residual_stride, z_stride, y_stride;
  int m, n, act;
  bool f32;
};

/* output (i, j), its sum s */
__device__ __forceinline__ void put_one(const Out &o, int i, int j, float s) {
  if (o.bias) s += bf(o.bias[j]);
  if (o.z) o.z[(int64_t)i * o.z_stride + j] = d3s_f32_to_bf16_rn(s);
  s = activate(s, o.act);
  if (o.f32) {
    if (o.residual) s += ((const float *)o.residual)[(int64_t)i * o.residual_stride + j];
    ((float *)o.y)[(int64_t)i * o.y_stride + j] = s;
  } else {
    if (o.residual) s += bf(((const uint16_t *)o.residual)[(int64_t)i * o.residual_stride + j]);
    ((uint16_t *)o.y)[(int64_t)i * o.y_stride + j] = d3s_f32_to_bf16_rn(s);
  }
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return (uint32_t)d3s_f32_to_bf16_rn(a) | (uint32_t)d3s_f32_to_bf16_rn(b) << 16;
}

/* outputs (i, j .. j + 3), all inside; the addresses may lie at any element */
__device__ __forceinline__ void put_four(const Out &o, int i, int j, f32x4 s) {
  if (o.bias) {
    uint16_t b[4];
    __builtin_memcpy(b, o.bias + j, 8);
#pragma unroll
    for (int e = 0; e < 4; e++) s[e] += bf(b[e]);
  }
  if (o.z) {
    const uint32_t w[2] = {pack2(s[0], s[1]), pack2(s[2], s[3])};
    __builtin_memcpy(o.z + (int64_t)i * o.z_stride + j, w, 8);
  }
#pragma unroll
  for (int e = 0; e < 4; e++) s[e] = activate(s[e], o.act);
  if (o.f32) {
    if (o.residual) {
      f32x4 r;
      __builtin_memcpy(&r, (const float *)o.residual + (int64_t)i * o.residual_stride + j, 16);
      s += r;
    }
    __builtin_memcpy((float *)o.y + (int64_t)i * o.y_stride + j, &s, 16);
  } else {
    if (o.residual) {
      uint16_t r[4];
      __builtin_memcpy(r, (const uint16_t *)o.residual + (int64_t)i * o.residual_stride + j, 8);
#pragma unroll
      for (int e = 0; e < 4; e++) s[e] += bf(r[e]);
    }
    const uint32_t w[2] = {pack2(s[0], s[1]), pack2(s[2], s[3])};
    __builtin_memcpy((uint16_t *)o.y + (int64_t)i * o.y_stride + j, w, 8);
  }
}

__device__ __forceinline__ void put_edge(const Out &o, int i, int j, f32x4 s) {
  if (i >= o.m) return;
  if (j + 4 <= o.n) {
    put_four(o, i, j, s);
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (j + e < o.n) put_one(o, i, j + e, s[e]);
  }
}

}  // namespace
}  // namespace d3s

#endif
