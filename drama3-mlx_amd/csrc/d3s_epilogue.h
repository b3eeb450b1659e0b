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
  /* (from -100 on down exp overflows and the products are -0; -inf times 0 would be NaN) */
  const float zc = ACT > D3S_ACT_RELU ? __builtin_elementwise_maximum(z, -100.0f) : z;
  switch (ACT) {
    case D3S_ACT_RELU: return __builtin_elementwise_maximum(z, 0.0f); /* (a NaN stays one) */
    case D3S_ACT_SILU: return zc * logistic(zc);
    case D3S_ACT_GELU_TANH: /* (1 + tanh u) / 2 = 1 / (1 + exp(-2 u)) */
      return zc * logistic(2.0f * GELU_C * zc * fmaf(GELU_A * zc, zc, 1.0f));
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

template <int ACT>
__device__ __forceinline__ float slope(float z) {
  /* far out the slope is 0 or 1 in fp32 (and its terms could be 0 times infinity) */
  const float zc = __builtin_elementwise_maximum(__builtin_elementwise_minimum(z, 100.0f), -100.0f);
  switch (ACT) {
    case D3S_ACT_RELU: return z > 0.0f ? 1.0f : z == z ? 0.0f : z;
    case D3S_ACT_SILU: {
      const float f = logistic(zc);
      return f * fmaf(zc, 1.0f - f, 1.0f);
    }
    case D3S_ACT_GELU: { /* the normal distribution's function and z times its density */
      const float u = fminf(fabsf(z), 15.0f);
      float e;
      const float q = normal_below(u, &e), z1 = z == z ? copysignf(u, z) : z;
      return fmaf(z1 * 0.3989422804014327f, e, z > 0.0f ? 1.0f - q : q);
    }
    case D3S_ACT_GELU_TANH: { /* f + z f' of the logistic function f of 2 u */
      const float f = logistic(2.0f * GELU_C * zc * fmaf(GELU_A * zc, zc, 1.0f));
      return fmaf(zc * f * (1.0f - f), 2.0f * GELU_C * fmaf(3.0f * GELU_A * zc, zc, 1.0f), f);
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

/* N neighbouring outputs of row i from j on (DOWN: N neighbouring rows from j on of
 * output i), their sums s: those from `skip` on that are inside */
template <int N, bool DOWN>
__device__ __forceinline__ void put_some(const Out &o, int i, int j, int skip, float *s) {
  if (i >= (DOWN ? o.n : o.m)) return;
  const int n = (DOWN ? o.m : o.n) - j;
  auto at = [&](int64_t stride, int e) { return DOWN ? (int64_t)(j + e) * stride + i : (int64_t)i * stride + j + e; };
#pragma unroll
  for (int e = 0; e < N; e++)
    if (o.bias && e >= skip && e < n) s[e] += bf(o.bias[DOWN ? i : j + e]);
  if (o.z) {
#pragma unroll
    for (int e = 0; e < N; e++)
      if (e >= skip && e < n) o.z[at(o.z_stride, e)] = pack1(s[e]);
  }
  activate<N>(s, o.act);
  if (o.f32) {
#pragma unroll
    for (int e = 0; e < N; e++)
      if (e >= skip && e < n)
        ((float *)o.y)[at(o.y_stride, e)] = o.residual ? s[e] + ((const float *)o.residual)[at(o.residual_stride, e)] : s[e];
  } else {
#pragma unroll
    for (int e = 0; e < N; e++)
      if (e >= skip && e < n)
        ((uint16_t *)o.y)[at(o.y_stride, e)] =
            pack1(o.residual ? s[e] + bf(((const uint16_t *)o.residual)[at(o.residual_stride, e)]) : s[e]);
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

/* A lane's eight neighbouring outputs from j on, of rows i, i + DOWN, ... (ROUNDS
 * of them, from `down` rows below i), whose sums lie ROW floats apart in LDS, 16-byte
 * aligned.  The outputs' addresses may lie at any element. */
template <int ROUNDS, int DOWN, int ROW>
struct Eights {
  const Out &o;
  const int i, j;
  const bool all; /* the eight are inside */
  uint4 bias;
  struct Residual {
    uint4 lo[ROUNDS], hi[ROUNDS]; /* bf16: lo alone */
  };

  __device__ __forceinline__ Eights(const Out &out, int row, int column)
      : o(out), i(row), j(column), all(row < out.m && column + 8 <= out.n) {
    bias = o.bias && all ? load16(o.bias + j) : make_uint4(0u, 0u, 0u, 0u);
  }
  /* rows past the last are the last again */
  __device__ __forceinline__ void get(Residual &r, int down) const {
    if (!o.residual || !all) return;
    if (o.f32) {
      const float *at = (const float *)o.residual + ((int64_t)i * o.residual_stride + j);
#pragma unroll
      for (int c = 0; c < ROUNDS; c++) {
        const float *p = at + (int64_t)min(down + c * DOWN, o.m - 1 - i) * o.residual_stride;
        r.lo[c] = load16(p);
        r.hi[c] = load16(p + 4);
      }
    } else {
      const uint16_t *at = (const uint16_t *)o.residual + ((int64_t)i * o.residual_stride + j);
#pragma unroll
      for (int c = 0; c < ROUNDS; c++) r.lo[c] = load16(at + (int64_t)min(down + c * DOWN, o.m - 1 - i) * o.residual_stride);
    }
  }
  /* sums become activations; z is written */
  __device__ __forceinline__ void activate(float *sums, int down) const {
    if (!all) return;
    uint16_t *z = o.z + ((int64_t)(i + down) * o.z_stride + j);
#pragma nounroll
    for (int c = 0; c < ROUNDS; c++) {
      float s[8], v[8];
      const f32x4 a = *(const f32x4 *)(sums + c * DOWN * ROW), b = *(const f32x4 *)(sums + c * DOWN * ROW + 4);
      bf_eight(bias, v);
#pragma unroll
      for (int e = 0; e < 4; e++) s[e] = a[e] + v[e], s[e + 4] = b[e] + v[e + 4];
      if (o.z && i + down + c * DOWN < o.m) stream16(z + c * (DOWN * o.z_stride), pack_eight(s));
      d3s::activate<8>(s, o.act);
      *(f32x4 *)(sums + c * DOWN * ROW) = f32x4{s[0], s[1], s[2], s[3]};
      *(f32x4 *)(sums + c * DOWN * ROW + 4) = f32x4{s[4], s[5], s[6], s[7]};
    }
  }
  /* y from the activations and the residual */
  __device__ __forceinline__ void put(const float *sums, int down, const Residual &r) const {
    if (!all) return;
    const int64_t y = (int64_t)(i + down) * o.y_stride + j;
    if (o.f32) {
#pragma unroll
      for (int c = 0; c < ROUNDS; c++) {
        f32x4 a = *(const f32x4 *)(sums + c * DOWN * ROW), b = *(const f32x4 *)(sums + c * DOWN * ROW + 4);
        if (o.residual) a += __builtin_bit_cast(f32x4, r.lo[c]), b += __builtin_bit_cast(f32x4, r.hi[c]);
        if (i + down + c * DOWN < o.m) {
          float *at = (float *)o.y + y + c * (DOWN * o.y_stride);
          /* (the caches join the halves of 32 bytes a lane: not past them) */
          __builtin_memcpy(at, &a, 16);
          __builtin_memcpy(at + 4, &b, 16);
        }
      }
    } else {
#pragma unroll
      for (int c = 0; c < ROUNDS; c++) {
        const f32x4 a = *(const f32x4 *)(sums + c * DOWN * ROW), b = *(const f32x4 *)(sums + c * DOWN * ROW + 4);
        float s[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}, v[8];
        if (o.residual) {
          bf_eight(r.lo[c], v);
#pragma unroll
          for (int e = 0; e < 8; e++) s[e] += v[e];
        }
        if (i + down + c * DOWN < o.m) stream16((uint16_t *)o.y + y + c * (DOWN * o.y_stride), pack_eight(s));
      }
    }
  }
  /* columns that are not all there: from the sums, one by one */
  __device__ __forceinline__ void put_rest(const float *sums, int down) const {
    if (all || j >= o.n) return;
#pragma nounroll
    for (int c = 0; c < ROUNDS; c++)
      for (int e = 0; e < o.n - j && i + down + c * DOWN < o.m; e++)
        put_one(o, i + down + c * DOWN, j + e, sums[c * DOWN * ROW + e]);
  }
};

}  // namespace
}  // namespace d3s

#endif
