/* The epilogue of a dense layer and its slopes (include/d3s_train.h), shared by
 * the products' kernels and the activation's gradient.  Device code only. */
#ifndef D3S_EPILOGUE_H
#define D3S_EPILOGUE_H

#include "d3s_dense_load.h"

namespace d3s {
namespace {

/* 2^x and 1 / x of the hardware (one step of 2^-23 off) */
__device__ __forceinline__ float exp2_1(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float rcp_1(float x) { return __builtin_amdgcn_rcpf(x); }

constexpr float LOG2_E = 1.4426950408889634f;

/* 1 / (1 + exp(-z)): exp overflows to infinity for z below -88, and 1 / inf is 0 */
__device__ __forceinline__ float logistic(float z) { return rcp_1(1.0f + exp2_1(-LOG2_E * z)); }

constexpr float GELU_C = 0.7978845608028654f; /* sqrt(2 / pi) */
constexpr float GELU_A = 0.044715f;

/* The normal distribution below -u, 0 <= u <= 15: exp(-u^2 / 2) times a
 * polynomial in t = 1 / (1 + 0.3 u), fitted here to its quotient by the exponential
 * on [0, 14.5] (least squares, reweighted to even the relative error: 1.7e-7, 5e-7
 * with the roundings).  A third of the instructions of erff, no cancellation in
 * the tail.  *e: the exponential. */
__device__ __forceinline__ float normal_below(float u, float *e) {
  const float t = rcp_1(fmaf(0.3f, u, 1.0f));
  float p = 0.03542410947502758f;
  p = fmaf(p, t, -0.15615989033429098f);
  p = fmaf(p, t, 0.20455905705830937f);
  p = fmaf(p, t, -0.052035904466179464f);
  p = fmaf(p, t, 0.12769266076723518f);
  p = fmaf(p, t, 0.10017571147329961f);
  p = fmaf(p, t, 0.12071216892954309f);
  p = fmaf(p, t, 0.11963200540771317f);
  *e = exp2_1(-0.5f * LOG2_E * u * u);
  return p * t * *e;
}

template <int ACT>
__device__ __forceinline__ float activated(float z) {
  if constexpr (ACT == D3S_ACT_GELU) { /* max(z, 0) - |z| P(below -|z|): -1e-48 at 15 is 0 */
    const float u = fminf(fabsf(z), 15.0f);
    float e;
    return fmaf(-u, normal_below(u, &e), __builtin_elementwise_maximum(z, 0.0f));
  }
  /* far below, z times a probability that is 0 in fp32 (-inf times it would be NaN) */
  if (ACT > D3S_ACT_RELU && z < -100.0f) return 0.0f;
  switch (ACT) {
    case D3S_ACT_RELU: return z < 0.0f ? 0.0f : z; /* (a NaN stays one) */
    case D3S_ACT_SILU: return z * logistic(z);
    case D3S_ACT_GELU_TANH: /* (1 + tanh u) / 2 = 1 / (1 + exp(-2 u)) */
      return z * logistic(2.0f * GELU_C * z * fmaf(GELU_A * z, z, 1.0f));
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
    case D3S_ACT_GELU: { /* the normal distribution's function and z times its density */
      const float u = fminf(fabsf(z), 15.0f);
      float e;
      const float q = normal_below(u, &e), z1 = z == z ? copysignf(u, z) : z;
      return fmaf(z1 * 0.3989422804014327f, e, z > 0.0f ? 1.0f - q : q);
    }
    case D3S_ACT_GELU_TANH: { /* f + z f' of the logistic function f of 2 u */
      const float f = logistic(2.0f * GELU_C * z * fmaf(GELU_A * z, z, 1.0f));
      return fmaf(z * f * (1.0f - f), 2.0f * GELU_C * fmaf(3.0f * GELU_A * z, z, 1.0f), f);
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

/* outputs (i, j + skip .. j + N - 1), their sums s: those that are inside */
template <int N>
__device__ __forceinline__ void put_some(const Out &o, int i, int j, int skip, float *s) {
  if (i >= o.m) return;
  const int n = o.n - j;
#pragma unroll
  for (int e = 0; e < N; e++)
    if (o.bias && e >= skip && e < n) s[e] += bf(o.bias[j + e]);
  if (o.z) {
#pragma unroll
    for (int e = 0; e < N; e++)
      if (e >= skip && e < n) o.z[(int64_t)i * o.z_stride + j + e] = pack1(s[e]);
  }
  activate<N>(s, o.act);
  const int64_t y = (int64_t)i * o.y_stride + j, r = (int64_t)i * o.residual_stride + j;
  if (o.f32) {
#pragma unroll
    for (int e = 0; e < N; e++)
      if (e >= skip && e < n) ((float *)o.y)[y + e] = o.residual ? s[e] + ((const float *)o.residual)[r + e] : s[e];
  } else {
#pragma unroll
    for (int e = 0; e < N; e++)
      if (e >= skip && e < n) ((uint16_t *)o.y)[y + e] = pack1(o.residual ? s[e] + bf(((const uint16_t *)o.residual)[r + e]) : s[e]);
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
 * aligned) of rows i and i + down become activations, with the bias as bias_eight
 * gave it ... */
__device__ __forceinline__ void activate_twice_eight(const Out &o, int i, int down, int j, float *sum, int row, uint4 bias) {
  if (i >= o.m || j + 8 > o.n) return;
  float s[16], v[8];
  bf_eight(bias, v);
#pragma unroll
  for (int h = 0; h < 2; h++) { /* (the second row's sums lie `down` rows of LDS further) */
    const f32x4 a = *(const f32x4 *)(sum + h * down * row), b = *(const f32x4 *)(sum + h * down * row + 4);
#pragma unroll
    for (int e = 0; e < 4; e++) s[h * 8 + e] = a[e] + v[e], s[h * 8 + 4 + e] = b[e] + v[e + 4];
  }
  if (o.z) {
    store16(o.z + (int64_t)i * o.z_stride + j, pack_eight(s));
    if (i + down < o.m) store16(o.z + (int64_t)(i + down) * o.z_stride + j, pack_eight(s + 8));
  }
  activate<16>(s, o.act);
#pragma unroll
  for (int h = 0; h < 2; h++) {
    *(f32x4 *)(sum + h * down * row) = f32x4{s[h * 8], s[h * 8 + 1], s[h * 8 + 2], s[h * 8 + 3]};
    *(f32x4 *)(sum + h * down * row + 4) = f32x4{s[h * 8 + 4], s[h * 8 + 5], s[h * 8 + 6], s[h * 8 + 7]};
  }
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
