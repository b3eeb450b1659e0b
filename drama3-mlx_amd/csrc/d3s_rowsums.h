/* Running maximum and sums of a row of logits, a batch of 16-byte chunks at a
 * time: the mathematics is at k_score (d3s_score.hip), which takes log
 * probabilities from them, as k_verify_rows (d3s_verify.hip) does.  Device code
 * only. */
#ifndef D3S_ROWSUMS_H
#define D3S_ROWSUMS_H

#include <float.h>

#include "d3s_device.h"

namespace d3s {
namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
/* the least exponent a term is given: 2^-1000 is 0 in fp32, and 0 times it is 0 where 0 * -inf is not */
constexpr float LEAST = -1000.0f;
/* batches whose shift m c is past this subtract first: it could overflow, and
 * the rounding it leaves (below, at most 1 / 32 here) would too */
constexpr float SHIFT_MOST = 1048576.0f;

__device__ __forceinline__ float maximum(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ bool finite(float T) { return fabsf(T) < __builtin_inff(); }
/* a - b for the exponents of maxima: both may be -FLT_MAX, neither is -inf */
__device__ __forceinline__ float drop(float a, float b, float c) { return fmaxf((a - b) * c, LEAST); }

struct Sums {
  float m, S, A;
};

/* the join of two parts; m, S and A of `a` change */
__device__ __forceinline__ void join(Sums &a, float m, float S, float A, float c) {
  const float M = maximum(a.m, m);
  const float da = drop(a.m, M, c), db = drop(m, M, c);
  const float fa = exp2_hw(da), fb = exp2_hw(db);
  a.A = fa * (a.A + a.S * da) + fb * (A + S * db);
  a.S = fa * a.S + fb * S;
  a.m = M;
}

/* the whole wave's, in every lane */
__device__ __forceinline__ void join_wave(Sums &a, float c) {
  const float M = wave_max_f(a.m);
  const float d = drop(a.m, M, c), f = exp2_hw(d);
  a.A = readlane_f(wave_scan_add_f32(f * (a.A + a.S * d)), 63);
  a.S = readlane_f(wave_scan_add_f32(f * a.S), 63);
  a.m = M;
}

/* Row `row`'s chunks: `base` the 16-byte aligned address at or below its
 * start, `lead` the elements of the first chunk before it. */
template <bool BF16>
struct Row {
  static constexpr int EPC = BF16 ? 8 : 4;
  const uint4 *base;
  int lead, vocab, chunks, banned_chunk, banned;

  __device__ __forceinline__ Row(const void *logits, int64_t stride, int row, int v, int ban) {
    const uintptr_t p = (uintptr_t)logits + (uintptr_t)((int64_t)row * stride) * (BF16 ? 2 : 4);
    base = (const uint4 *)(p & ~(uintptr_t)15);
    lead = (int)(p & 15) / (BF16 ? 2 : 4);
    vocab = v;
    chunks = (lead + v + EPC - 1) / EPC;
    banned = (unsigned)ban < (unsigned)v ? ban : -1;
    banned_chunk = banned < 0 ? -1 : (lead + banned) / EPC;
  }
  __device__ __forceinline__ bool plain(int ch) const { return ch != 0 && ch != chunks - 1 && ch != banned_chunk; }
  /* the chunk's logits, -inf outside the row and at the banned index */
  __device__ __forceinline__ void values(uint4 q, int ch, float *v) const {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if constexpr (BF16) {
        v[2 * i] = d3s_u2f(w[i] << 16);
        v[2 * i + 1] = d3s_u2f(w[i] & 0xffff0000u);
      } else {
        v[i] = d3s_u2f(w[i]);
      }
    }
    if (!plain(ch)) {
#pragma unroll
      for (int i = 0; i < EPC; i++) {
        const int j = ch * EPC + i - lead;
        if (j < 0 || j >= vocab || j == banned) v[i] = -__builtin_inff();
      }
    }
  }
};

template <int N, bool ENT>
__device__ __forceinline__ void add_batch(Sums &s, const float *v, float c) {
  float b = v[0];
#pragma unroll
  for (int i = 1; i < N; i++) b = maximum(b, v[i]);
  const float M = maximum(s.m, b);
  const float d = drop(s.m, M, c), f = exp2_hw(d);
  const float mc = M * c;
  float S[2] = {0.0f, 0.0f}, A[2] = {0.0f, 0.0f};
  float o = 0.0f; /* the terms' exponents are o below (l - M) c */
  if (__any(!(fabsf(mc) < SHIFT_MOST))) { /* huge logits or a mask's lowest value: subtract first */
#pragma unroll
    for (int i = 0; i < N; i++) {
      const float t = fmaxf((v[i] - M) * c, LEAST), e = exp2_hw(t);
      S[i & 1] += e;
      if (ENT) A[i & 1] = fmaf(e, t, A[i & 1]);
    }
  } else {
    o = fmaf(-M, c, mc);
#pragma unroll
    for (int i = 0; i < N; i++) {
      float t = fmaf(v[i], c, -mc);
      if (ENT) t = fmaxf(t, LEAST);
      const float e = exp2_hw(t);
      S[i & 1] += e;
      if (ENT) A[i & 1] = fmaf(e, t, A[i & 1]);
    }
  }
  const float fo = exp2_hw(o), Sb = S[0] + S[1];
  if (ENT) s.A = fmaf(f, fmaf(s.S, d, s.A), fo * fmaf(Sb, o, A[0] + A[1]));
  s.S = fmaf(f, s.S, fo * Sb);
  s.m = M;
}

}  // namespace
}  // namespace d3s

#endif
