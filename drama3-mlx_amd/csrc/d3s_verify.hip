/* k_verify_one, k_verify_ranked: verification of drafted tokens (gfx950, wave64;
 * include/d3s_step.h). */
#include "d3s_rowsums.h"
#include "d3s_step_internal.h"
#include "d3s_vec.h"

namespace d3s {
namespace {

constexpr int VT = 1024;
constexpr int VW = VT / WAVE;
constexpr double LOG2E_64 = 1.4426950408889634074;

__device__ __forceinline__ float least_T(float T) { return T < 1e-5f && T > -__builtin_inff() ? 1e-5f : T; }

/* 2^t for t <= 0 (0 below -1100): the Taylor series of 2^f on |f| <= 1 / 2 to the
 * 11th power (the rest below 2^-46), in 64 bits */
__device__ __forceinline__ double exp2_64(double t) {
  t = fmax(t, -1100.0);
  const double n = rint(t), f = t - n;
  double p = 4.4455382718708116e-10; /* (ln 2)^k / k!, k = 11 .. 0 */
  p = fma(p, f, 7.0549116208011234e-09);
  p = fma(p, f, 1.0178086009239699e-07);
  p = fma(p, f, 1.3215486790144310e-06);
  p = fma(p, f, 1.5252733804059841e-05);
  p = fma(p, f, 1.5403530393381609e-04);
  p = fma(p, f, 1.3333558146428443e-03);
  p = fma(p, f, 9.6181291076284772e-03);
  p = fma(p, f, 5.5504108664821580e-02);
  p = fma(p, f, 2.4022650695910072e-01);
  p = fma(p, f, 6.9314718055994531e-01);
  p = fma(p, f, 1.0);
  return ldexp(p, (int)n);
}

/* a row's greatest logit and sum, and what they say of it */
struct RowStat {
  float m, S;
};
__device__ __forceinline__ bool refused(RowStat r) { return !(r.m < __builtin_inff()); }
/* the probability of a logit (S > 0 unless all is masked) */
__device__ __forceinline__ float prob_of(RowStat r, float l, float T) {
  return r.S > 0.0f ? d3s_expf_nonpos((l - r.m) / T) / r.S : 0.0f;
}

/* What a sequence comes to: its drafts accepted, and how the token after them is drawn */
struct Outcome {
  int accepted;
  bool refuse, rejected;
};

__device__ __forceinline__ float accept_of(float p, float q) { return q > 0.0f ? fminf(p / q, 1.0f) : p > 0.0f ? 1.0f : 0.0f; }

/* p, q (NaN: a refused row) of L drafts; last: p's row behind them is refused */
template <class P, class Q>
__device__ __forceinline__ Outcome decide(int L, const float *u, P p, Q q, bool last_refused) {
  Outcome o{0, false, false};
  for (int i = 0; i < L; i++) {
    const float pi = p(i), qi = q(i);
    if (pi != pi || qi != qi) {
      o.refuse = true;
      return o;
    }
    if (!(u[i] * qi < pi)) {
      o.rejected = true;
      return o;
    }
    o.accepted++;
  }
  o.refuse = last_refused;
  return o;
}

__device__ __forceinline__ void write_tokens(int b, int n_draft, Outcome o, int token, const int32_t *drafted,
                                             int32_t *tokens, int32_t *n_accepted) {
  for (int i = (int)threadIdx.x; i <= n_draft; i += (int)blockDim.x) {
    const size_t at = (size_t)b * (n_draft + 1) + i;
    tokens[at] = i < o.accepted ? drafted[(size_t)b * n_draft + i] : i == o.accepted ? token : -1;
  }
  if (threadIdx.x == 0) n_accepted[b] = o.accepted;
}

__device__ __forceinline__ double shfl_up_f64(double v, int d) { return __shfl_up(v, d); }

struct DrawLds {
  double wave[VW];
  int at;
};

/* the workgroup's sum in one order, in every thread */
__device__ __forceinline__ double block_sum64(double v, DrawLds &L) {
#pragma unroll
  for (int d = 1; d < WAVE; d *= 2) v += __shfl_xor(v, d);
  __syncthreads();
  if (lane_id() == 0) L.wave[threadIdx.x / WAVE] = v;
  __syncthreads();
  double t = 0.0;
  for (int w = 0; w < VW; w++) t += L.wave[w];
  return t;
}

template <bool TB, bool DB>
__global__ __launch_bounds__(VT) void k_verify_one(d3s_verify_params a) {
  __shared__ RowStat stat[2 * D3S_MAX_DRAFT + 1];
  __shared__ float prob[2 * D3S_MAX_DRAFT];
  __shared__ DrawLds L;
  const int b = (int)blockIdx.x, tid = (int)threadIdx.x, V = (int)a.vocab;
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.n_draft) : a.n_draft;
  const float T = least_T(a.temperature ? a.temperature[b] : a.temperature_scalar);
  const float Td = least_T(a.draft_temperature ? a.draft_temperature[b] : a.draft_temperature_scalar);
  const int32_t *x = a.drafted + (size_t)b * a.n_draft;
  const float nan = __builtin_nanf("");

  /* a wave a row: target 0 .. len, then draft 0 .. len - 1 */
  auto row_sums = [&](auto bf16, const void *logits, int64_t stride, int row, float T_) {
    constexpr bool BF16 = decltype(bf16)::value;
    const Row<BF16> R(logits, stride, row, V, -1);
    Sums s{-FLT_MAX, 0.0f, 0.0f};
    const float c = LOG2E / T_;
    for (int ch = lane_id(); ch < R.chunks; ch += WAVE) {
      float v[Row<BF16>::EPC];
      R.values(R.base[ch], ch, v);
      add_batch<Row<BF16>::EPC, false>(s, v, c);
    }
    join_wave(s, c);
    return s;
  };
  const int n_rows = len + 1 + (a.draft ? len : 0);
  for (int r = tid / WAVE; r < n_rows; r += VW) {
    const bool target = r <= len;
    const int i = target ? r : r - len - 1;
    const int row = target ? b * (a.n_draft + 1) + i : b * a.n_draft + i;
    const float Tr = target ? T : Td;
    const Sums s = target ? row_sums(std::integral_constant<bool, TB>{}, a.target, a.target_stride, row, Tr)
                          : row_sums(std::integral_constant<bool, DB>{}, a.draft, a.draft_stride, row, Tr);
    if (lane_id() == 0) {
      RowStat st{s.m, s.S};
      if (!finite(Tr)) st.m = nan;
      stat[r] = st;
      if (i < len) {
        float pr = 0.0f;
        if (refused(st)) {
          pr = nan;
        } else if ((unsigned)x[i] < (unsigned)V) {
          const float l = target ? load_at<TB>(a.target, (int64_t)row * a.target_stride + x[i])
                                 : load_at<DB>(a.draft, (int64_t)row * a.draft_stride + x[i]);
          pr = prob_of(st, l, Tr);
        }
        prob[target ? i : D3S_MAX_DRAFT + i] = pr;
      }
    }
  }
  __syncthreads();
  auto p = [&](int i) { return prob[i]; };
  auto q = [&](int i) { return a.draft ? prob[D3S_MAX_DRAFT + i] : 1.0f; };
  const Outcome o = decide(len, a.u_accept + (size_t)b * a.n_draft, p, q, refused(stat[len]));
  if (a.accept)
    for (int i = tid; i < a.n_draft; i += VT)
      a.accept[(size_t)b * a.n_draft + i] = i >= len ? 0.0f : p(i) != p(i) || q(i) != q(i) ? nan : accept_of(p(i), q(i));
  int token = -1;
  const RowStat sp = stat[o.accepted];
  if (o.refuse) {
    if (tid == 0 && a.counters) atomicAdd(&a.counters[CNT_REFUSED], 1u);
  } else if (sp.S == 0.0f) {
    token = 0;
    if (tid == 0 && a.counters) atomicAdd(&a.counters[CNT_ALL_MASKED], 1u);
  } else {
    /* the draw in 64 bits, a thread a run of the row */
    const int per = ((V + VT - 1) / VT + 7) / 8 * 8, lo = min(V, tid * per), hi = min(V, lo + per);
    const bool pair = o.rejected && a.draft;
    const RowStat sq = pair ? stat[len + 1 + o.accepted] : RowStat{0.0f, 0.0f};
    const int gone = o.rejected && !a.draft ? x[o.accepted] : -1;
    const char *tp = (const char *)a.target + ((int64_t)b * (a.n_draft + 1) + o.accepted) * a.target_stride * (TB ? 2 : 4);
    const char *dp = (const char *)a.draft + ((int64_t)b * a.n_draft + o.accepted) * a.draft_stride * (DB ? 2 : 4);
    const double cp = LOG2E_64 / T, cq = LOG2E_64 / Td;
    auto ep = [&](float l) { return exp2_64(((double)l - sp.m) * cp); };
    auto eq = [&](float l) { return exp2_64(((double)l - sq.m) * cq); };
    double Sp = 0.0, Sq = 0.0;
    for (int j = lo; j < hi; j++) {
      Sp += ep(load_at<TB>(tp, j));
      if (pair) Sq += eq(load_at<DB>(dp, j));
    }
    Sp = 1.0 / block_sum64(Sp, L);
    if (pair) {
      Sq = block_sum64(Sq, L);
      Sq = Sq > 0.0 ? 1.0 / Sq : 0.0;
    }
    bool plain = !o.rejected;
    auto weight = [&](int j) {
      const double w = ep(load_at<TB>(tp, j)) * Sp;
      if (plain) return w;
      if (!pair) return j == gone ? fmax(w - 1.0, 0.0) : w;
      return fmax(w - eq(load_at<DB>(dp, j)) * Sq, 0.0);
    };
    double mine, base, Z;
    for (;;) {
      mine = 0.0;
      for (int j = lo; j < hi; j++) mine += weight(j);
      double incl = mine;
#pragma unroll
      for (int d = 1; d < WAVE; d *= 2) {
        const double t = shfl_up_f64(incl, d);
        if (lane_id() >= d) incl += t;
      }
      __syncthreads();
      if (lane_id() == WAVE - 1) L.wave[tid / WAVE] = incl;
      if (tid == 0) L.at = 0x7fffffff;
      __syncthreads();
      double before = 0.0;
      Z = 0.0;
      for (int w = 0; w < VW; w++) {
        if (w < tid / WAVE) before += L.wave[w];
        Z += L.wave[w];
      }
      base = before + (incl - mine);
      if (Z > 0.0 || plain) break;
      plain = true; /* (p <= q everywhere: rounding alone) */
    }
    const double bar = (double)a.u_draw[b] * Z;
    if (mine > 0.0 && base + mine > bar) atomicMin(&L.at, tid);
    __syncthreads();
    if (L.at == 0x7fffffff) { /* none by rounding: the last that has any */
      __syncthreads();
      if (tid == 0) L.at = -1;
      __syncthreads();
      if (mine > 0.0) atomicMax(&L.at, tid);
      __syncthreads();
    }
    const int who = L.at;
    __syncthreads();
    if (tid == who) {
      int at = -1;
      for (int j = lo; j < hi; j++) {
        const double w = weight(j);
        base += w;
        if (w > 0.0) {
          at = j;
          if (base > bar) break;
        }
      }
      L.at = at;
    }
    __syncthreads();
    token = L.at;
  }
  write_tokens(b, a.n_draft, o, token, a.drafted, a.tokens, a.n_accepted);
}

/* ------------------------------------------------------------------------ */

constexpr int RT = 256;

__global__ __launch_bounds__(RT) void k_verify_ranked(RankedArgs a) {
  __shared__ float prob[2 * D3S_MAX_DRAFT];
  __shared__ int cand[D3S_MAX_RANKED];
  __shared__ float qs[D3S_MAX_RANKED];
  __shared__ float best[RT / WAVE];
  __shared__ int best_at[RT / WAVE];
  const int b = (int)blockIdx.x, tid = (int)threadIdx.x;
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.n_draft) : a.n_draft;
  const int32_t *x = a.drafted + (size_t)b * a.n_draft;
  const size_t t0 = (size_t)b * (a.n_draft + 1) * a.target_k, d0 = (size_t)b * a.n_draft * a.draft_k;
  const float nan = __builtin_nanf("");
  /* (a refused row's candidates are -1; a masked one's probabilities NaN, taken as 0) */
  auto refused_t = [&](int i) { return a.target_cand[t0 + (size_t)i * a.target_k] < 0; };
  for (int i = tid; i < len; i += RT) {
    prob[i] = refused_t(i) ? nan : 0.0f;
    prob[D3S_MAX_DRAFT + i] = !a.draft_cand ? 1.0f : a.draft_cand[d0 + (size_t)i * a.draft_k] < 0 ? nan : 0.0f;
  }
  __syncthreads();
  for (int e = tid; e < len * a.target_k; e += RT) {
    const int i = e / a.target_k;
    if (x[i] >= 0 && a.target_cand[t0 + e] == x[i] && a.target_probs[t0 + e] > 0.0f) prob[i] = a.target_probs[t0 + e];
  }
  if (a.draft_cand)
    for (int e = tid; e < len * a.draft_k; e += RT) {
      const int i = e / a.draft_k;
      if (x[i] >= 0 && a.draft_cand[d0 + e] == x[i] && a.draft_probs[d0 + e] > 0.0f)
        prob[D3S_MAX_DRAFT + i] = a.draft_probs[d0 + e];
    }
  __syncthreads();
  auto p = [&](int i) { return prob[i]; };
  auto q = [&](int i) { return prob[D3S_MAX_DRAFT + i]; };
  const Outcome o = decide(len, a.u_accept + (size_t)b * a.n_draft, p, q, refused_t(len));
  if (a.accept)
    for (int i = tid; i < a.n_draft; i += RT)
      a.accept[(size_t)b * a.n_draft + i] = i >= len ? 0.0f : p(i) != p(i) || q(i) != q(i) ? nan : accept_of(p(i), q(i));
  int token = -1;
  if (o.refuse) {
    if (tid == 0 && a.counters) atomicAdd(&a.counters[CNT_REFUSED], 1u);
  } else {
    const int32_t *tc = a.target_cand + t0 + (size_t)o.accepted * a.target_k;
    const float *tp = a.target_probs + t0 + (size_t)o.accepted * a.target_k;
    if (o.rejected && a.draft_cand)
      for (int e = tid; e < a.draft_k; e += RT) {
        cand[e] = a.draft_cand[d0 + (size_t)o.accepted * a.draft_k + e];
        qs[e] = a.draft_probs[d0 + (size_t)o.accepted * a.draft_k + e];
      }
    __syncthreads();
    bool plain = !o.rejected;
    for (;;) {
      float sc = -2.0f;
      int at = 0x7fffffff;
      for (int r = tid; r < a.target_k; r += RT) {
        float w = tp[r];
        if (!plain && a.draft_cand) {
          for (int e = 0; e < a.draft_k; e++)
            if (cand[e] == tc[r] && qs[e] > 0.0f) w -= qs[e];
        } else if (!plain && tc[r] == x[o.accepted]) {
          w -= 1.0f;
        }
        if (!(w > 0.0f)) continue;
        float score = w / -d3s_logf(1.0f - a.u_draw[(size_t)b * a.target_k + r]);
        score = score > -1.0f ? score : -1.0f; /* (u = 0 gives -inf, as the sampler's race: the last choice) */
        if (score > sc) sc = score, at = r;    /* (a thread's ranks rise) */
      }
      wave_argmax(sc, at);
      __syncthreads();
      if (lane_id() == 0) best[tid / WAVE] = sc, best_at[tid / WAVE] = at;
      __syncthreads();
      for (int w = 0; w < RT / WAVE; w++)
        if (best[w] > sc || (best[w] == sc && best_at[w] < at)) sc = best[w], at = best_at[w];
      if (at != 0x7fffffff) {
        token = tc[at];
        break;
      }
      if (plain) { /* no rank has a probability: a masked row */
        token = 0;
        if (tid == 0 && a.counters) atomicAdd(&a.counters[CNT_ALL_MASKED], 1u);
        break;
      }
      plain = true;
    }
  }
  write_tokens(b, a.n_draft, o, token, a.drafted, a.tokens, a.n_accepted);
}

}  // namespace

size_t verify_workspace_bytes(const d3s_verify_params &) { return 0; }

void launch_verify(const d3s_verify_params &a, void *, hipStream_t s) {
  const dim3 grid((unsigned)a.n_seqs);
  auto go = [&](auto kernel) { kernel<<<grid, VT, 0, s>>>(a); };
  const bool db = a.draft && a.draft_dtype == D3S_DTYPE_BF16;
  if (a.target_dtype == D3S_DTYPE_BF16)
    db ? go(k_verify_one<true, true>) : go(k_verify_one<true, false>);
  else
    db ? go(k_verify_one<false, true>) : go(k_verify_one<false, false>);
}

void launch_verify_ranked(const RankedArgs &args, hipStream_t s) {
  const RankedArgs a = args;
  k_verify_ranked<<<dim3((unsigned)a.n_seqs), RT, 0, s>>>(a);
}

}  // namespace d3s
