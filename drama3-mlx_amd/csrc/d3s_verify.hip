/* k_verify_one, k_verify_rows, k_verify_draw, k_verify_ranked: verification of
 * drafted tokens (gfx950, wave64; include/d3s_step.h).
 *
 * Whether a draft is accepted goes by p and q in fp32: the rows' greatest logits and sums as k_score takes
 * them (d3s_rowsums.h), exp of the draft's logit, u q < p without a quotient.  The token that is drawn
 * goes by sums that meet a border, u Z, and the rows are long: its terms, sums and weights are
 * 64-bit throughout, of the one pair of rows that a sequence draws from (64-bit multiply-adds run at
 * the rate of 32-bit ones here).  All sums are added in an order that the sizes give.
 *
 * Bound: the rows' sums by HBM (64 sequences of 4 drafts over 151936 bf16: 29 us, 6.0 TB/s), the draw by
 * its 64-bit arithmetic (the same: 33 us, of which the decision is 5, the terms 19); short rows
 * by the chain of dependent steps (4097: 10 us; 30 candidates 6.3). */
#include "d3s_rowcore.h"
#include "d3s_rowsums.h"
#include "d3s_step_internal.h"
#include "d3s_vec.h"

namespace d3s {
namespace {

constexpr int VT = 1024;       /* threads of k_verify_one */
constexpr int ST = 256;        /* ... of the split kernels */
constexpr int SU = 4;          /* chunks a lane takes at a time */
constexpr int GRID_MOST = 1 << 22;
constexpr double LOG2E_64 = 1.4426950408889634074;

__device__ __forceinline__ float least_T(float T) { return T < 1e-5f && T > -__builtin_inff() ? 1e-5f : T; }

/* 2^t for t <= 0 (0 from -1100 down): 2^f on |f| <= 1 / 2 by the polynomial that
 * agrees with it at ten Chebyshev nodes (fitted here; 2e-14 relative) */
__device__ __forceinline__ double exp2_64(double t) {
  t = fmax(t, -1100.0);
  const double n = rint(t), f = t - n;
  double p = 1.0205905308574628e-07;
  p = fma(p, f, 1.3259645243778838e-06);
  p = fma(p, f, 1.5252672925435629e-05);
  p = fma(p, f, 0.0001540343375125619);
  p = fma(p, f, 0.0013333558200793471);
  p = fma(p, f, 0.009618129193934302);
  p = fma(p, f, 0.05550410866465168);
  p = fma(p, f, 0.2402265069564034);
  p = fma(p, f, 0.6931471805599462);
  p = fma(p, f, 1.0000000000000135);
  return ldexp(p, (int)n);
}

/* a row's greatest logit and sum (m = NaN: refused) */
struct RowStat {
  float m, S;
};
__device__ __forceinline__ bool refused(RowStat r) { return !(r.m < __builtin_inff()); }

/* what a sequence comes to: its drafts accepted, and how the token after them is drawn */
struct Outcome {
  int accepted;
  bool refuse, rejected;
};

__device__ __forceinline__ float accept_of(float p, float q) {
  return p != p || q != q ? __builtin_nanf("") : q > 0.0f ? fminf(p / q, 1.0f) : p > 0.0f ? 1.0f : 0.0f;
}

/* Lane i of every wave holds u, p and q (NaN: a refused row) of draft i < L <= 64;
 * last_refused: the target's row behind them. */
__device__ __forceinline__ Outcome decide(int L, float u, float p, float q, bool last_refused) {
  const bool inside = lane_id() < L, odd = p != p || q != q;
  const uint64_t refusing = __ballot(inside && odd), stops = __ballot(inside && (odd || !(u * q < p)));
  Outcome o;
  o.accepted = stops ? (int)__builtin_ctzll(stops) : L;
  o.refuse = stops ? (refusing >> o.accepted & 1ull) != 0ull : last_refused;
  o.rejected = stops && !o.refuse;
  return o;
}

/* x: lane i's draft i (a place behind 64 drafts holds none) */
__device__ __forceinline__ void write_tokens(int b, int n_draft, Outcome o, int token, int x, int32_t *tokens, int32_t *n_accepted) {
  const int i = (int)threadIdx.x;
  if (i <= n_draft) tokens[(size_t)b * (n_draft + 1) + i] = i < o.accepted ? x : i == o.accepted ? token : -1;
  if (i == 0) n_accepted[b] = o.accepted;
}

/* A sequence: its length and temperatures, its rows (0 .. n_draft the target's, then the
 * draft model's) */
struct Seq {
  int b, len, rows;
  float T, Td;

  __device__ __forceinline__ Seq(const d3s_verify_params &a, int b_) : b(b_) {
    len = a.lengths ? min(max(a.lengths[b], 0), a.n_draft) : a.n_draft;
    T = least_T(a.temperature ? a.temperature[b] : a.temperature_scalar);
    Td = least_T(a.draft_temperature ? a.draft_temperature[b] : a.draft_temperature_scalar);
    rows = a.n_draft + 1 + (a.draft ? a.n_draft : 0);
  }
  __device__ __forceinline__ bool target(const d3s_verify_params &a, int r) const { return r <= a.n_draft; }
  __device__ __forceinline__ int place(const d3s_verify_params &a, int r) const { return target(a, r) ? r : r - a.n_draft - 1; }
  __device__ __forceinline__ int row(const d3s_verify_params &a, int r) const {
    return target(a, r) ? b * (a.n_draft + 1) + r : b * a.n_draft + r - a.n_draft - 1;
  }
  /* whether the row can count: a target's up to the one behind the drafts */
  __device__ __forceinline__ bool there(const d3s_verify_params &a, int r) const {
    return target(a, r) ? r <= len : place(a, r) < len;
  }
  __device__ __forceinline__ float temperature(const d3s_verify_params &a, int r) const { return target(a, r) ? T : Td; }
};

/* A lane's share of a row's chunks, every `step`-th from `ch` on, up to `hi`; a batch
 * is loaded while the one before it is added, and beside() runs behind the first loads. */
template <bool BF16, class F>
__device__ __forceinline__ void lane_sums(Sums &s, const Row<BF16> &R, int ch, int hi, int step, float c, F beside) {
  constexpr int EPC = Row<BF16>::EPC;
  uint4 q[SU], next[SU];
  bool whole = ch + (SU - 1) * step < hi;
  if (whole) {
#pragma unroll
    for (int u = 0; u < SU; u++) q[u] = R.base[ch + u * step];
  }
  beside();
  while (whole) {
    const int after = ch + SU * step;
    whole = after + (SU - 1) * step < hi;
    if (whole) {
#pragma unroll
      for (int u = 0; u < SU; u++) next[u] = R.base[after + u * step];
    }
    float v[SU * EPC];
#pragma unroll
    for (int u = 0; u < SU; u++) R.values(q[u], ch + u * step, v + u * EPC);
    add_batch<SU * EPC, false>(s, v, c);
#pragma unroll
    for (int u = 0; u < SU; u++) q[u] = next[u];
    ch = after;
  }
  if (__ballot(ch + step < hi) == 0ull) { /* (4097 bf16 over 64 lanes: two batches and a chunk) */
    if (ch >= hi) return;
    float v[EPC];
    R.values(R.base[ch], ch, v);
    add_batch<EPC, false>(s, v, c);
    return;
  }
  if (ch >= hi) return;
  /* the rest, less than a batch: a place past the end is the last chunk again, masked */
  float v[SU * EPC];
#pragma unroll
  for (int u = 0; u < SU; u++) q[u] = R.base[min(ch + u * step, hi - 1)];
#pragma unroll
  for (int u = 0; u < SU; u++) {
    R.values(q[u], min(ch + u * step, hi - 1), v + u * EPC);
    if (ch + u * step >= hi) {
#pragma unroll
      for (int e = 0; e < EPC; e++) v[u * EPC + e] = -__builtin_inff();
    }
  }
  add_batch<SU * EPC, false>(s, v, c);
}

/* LDS of a sequence's decision */
struct Settled {
  RowStat stat[2 * D3S_MAX_DRAFT + 1];
  float prob[2 * D3S_MAX_DRAFT + 1];
};

/* the logit of row r's draft (-inf: not a token, or none) */
template <bool TB, bool DB>
__device__ __forceinline__ float draft_logit(const d3s_verify_params &a, const Seq &q, int r) {
  const int i = q.place(a, r);
  if (r >= q.rows || i >= q.len) return -__builtin_inff();
  const int x = a.drafted[(size_t)q.b * a.n_draft + i];
  if ((unsigned)x >= (unsigned)a.vocab) return -__builtin_inff();
  return q.target(a, r) ? load_at<TB>(a.target, (int64_t)q.row(a, r) * a.target_stride + x)
                        : load_at<DB>(a.draft, (int64_t)q.row(a, r) * a.draft_stride + x);
}

/* A thread a row: the probability of its draft's logit, from the row's statistics (S > 0
 * unless all of the row is masked). */
__device__ __forceinline__ void settle_row(const d3s_verify_params &a, const Seq &q, int r, RowStat st, float l, Settled &L) {
  const float T = q.temperature(a, r);
  if (!finite(T)) st.m = __builtin_nanf("");
  L.stat[r] = st;
  L.prob[r] = refused(st) ? __builtin_nanf("") : st.S > 0.0f ? d3s_expf_nonpos((l - st.m) / T) / st.S : 0.0f;
}

/* lane i's uniform and draft */
__device__ __forceinline__ float lane_u(const d3s_verify_params &a, const Seq &s) {
  return lane_id() < s.len ? a.u_accept[(size_t)s.b * a.n_draft + lane_id()] : 0.0f;
}
__device__ __forceinline__ int lane_draft(const d3s_verify_params &a, const Seq &s) {
  return lane_id() < s.len ? a.drafted[(size_t)s.b * a.n_draft + lane_id()] : -1;
}

/* the whole workgroup, the rows settled; u: lane_u */
__device__ __forceinline__ Outcome settle(const d3s_verify_params &a, const Seq &s, const Settled &L, float u, bool write_accept) {
  const int i = lane_id();
  const bool inside = i < s.len;
  const float p = inside ? L.prob[i] : 0.0f, q = !inside ? 0.0f : a.draft ? L.prob[a.n_draft + 1 + i] : 1.0f;
  if (write_accept && a.accept && (int)threadIdx.x < a.n_draft)
    a.accept[(size_t)s.b * a.n_draft + i] = inside ? accept_of(p, q) : 0.0f;
  return decide(s.len, u, p, q, refused(L.stat[s.len]));
}

/* The weights r_j that a token is drawn from, in 64 bits. */
template <bool TB, bool DB>
struct Weights {
  const char *tp, *dp; /* the rows (dp null: none, or a certain draft) */
  int V, gone;         /* the certain draft's token, or -1 */
  double mp, mq, cp, cq;       /* greatest logits, log2(e) / T */
  double ip, iq;               /* what the terms are multiplied by */

  /* m_p, m_q: the rows' greatest logits; x: lane i's draft i */
  __device__ __forceinline__ Weights(const d3s_verify_params &a, const Seq &s, int accepted, bool rejected, float m_p, float m_q, int x) {
    tp = (const char *)a.target + ((int64_t)s.b * (a.n_draft + 1) + accepted) * a.target_stride * (TB ? 2 : 4);
    dp = rejected && a.draft ? (const char *)a.draft + ((int64_t)s.b * a.n_draft + accepted) * a.draft_stride * (DB ? 2 : 4) : nullptr;
    V = (int)a.vocab;
    gone = rejected && !a.draft ? __builtin_amdgcn_readlane(x, accepted & (WAVE - 1)) : -1;
    mp = m_p, mq = m_q;
    cp = LOG2E_64 / s.T, cq = LOG2E_64 / s.Td;
    ip = iq = 1.0;
  }
  __device__ __forceinline__ int left(int j) const { return min(8, V - j); }
  /* eight terms of each sum from j on (0 past the end), j < V */
  __device__ __forceinline__ void terms(int j, double *p, double *q) const {
    float v[8], w[8];
    load_row<TB, 8>(tp, j, left(j), v);
    if (dp) load_row<DB, 8>(dp, j, left(j), w);
    if (left(j) < 8) {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (e >= left(j)) v[e] = w[e] = -__builtin_inff();
    }
#pragma unroll
    for (int e = 0; e < 8; e++) p[e] = exp2_64(((double)v[e] - mp) * cp);
    if (dp) {
#pragma unroll
      for (int e = 0; e < 8; e++) q[e] = exp2_64(((double)w[e] - mq) * cq);
    }
  }
  /* eight weights from j on; plain: p alone */
  __device__ __forceinline__ void at(int j, bool plain, double *r) const {
    double p[8], q[8];
    terms(j, p, q);
    weights(j, plain, p, q, r);
  }
  __device__ __forceinline__ void weights(int j, bool plain, const double *p, const double *q, double *r) const {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      r[e] = p[e] * ip;
      if (plain) continue;
      if (dp)
        r[e] = fmax(r[e] - q[e] * iq, 0.0);
      else if (j + e == gone) /* (p <= 1) */
        r[e] = 0.0;
    }
  }
};

template <int NT>
struct DrawLds {
  double wave[NT / WAVE];
  double from;
  int at, close;
};

template <int CTRL, int ROWM>
__device__ __forceinline__ double dpp_f64(double v) {
  const uint64_t w = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = dpp_u<CTRL, ROWM>(0u, (uint32_t)w), hi = dpp_u<CTRL, ROWM>(0u, (uint32_t)(w >> 32));
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
/* inclusive sums over the wave (wave_scan_add_f32 in 64 bits) */
__device__ __forceinline__ double wave_scan64(double v) {
  v += dpp_f64<DPP_SHR1, 0xf>(v);
  v += dpp_f64<DPP_SHR2, 0xf>(v);
  v += dpp_f64<DPP_SHR4, 0xf>(v);
  v += dpp_f64<DPP_SHR8, 0xf>(v);
  v += dpp_f64<DPP_BCAST15, 0xa>(v);
  v += dpp_f64<DPP_BCAST31, 0xc>(v);
  return v;
}
template <int NT>
__device__ __forceinline__ double block_sum64(double v, DrawLds<NT> &L) {
  v = wave_scan64(v);
  __syncthreads();
  if (lane_id() == WAVE - 1) L.wave[threadIdx.x / WAVE] = v;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int w = 0; w < NT / WAVE; w++) t += L.wave[w];
  return t;
}
/* the sum of the threads before, and of all */
template <int NT>
__device__ __forceinline__ double block_scan64(double v, DrawLds<NT> &L, double *total) {
  const double incl = wave_scan64(v);
  __syncthreads();
  if (lane_id() == WAVE - 1) L.wave[threadIdx.x / WAVE] = incl;
  __syncthreads();
  double before = 0.0, all = 0.0;
#pragma unroll
  for (int w = 0; w < NT / WAVE; w++) {
    if (w == (int)threadIdx.x / WAVE) before = all;
    all += L.wave[w];
  }
  *total = all;
  return before + (incl - v);
}

/* The first place whose sum passes bar, else (LAST) the last with a weight, else -1, in
 * every thread: a thread's eight weights r follow each other from j on, `before` is the sum of
 * those before them.  L.close is set if a sum is within `doubt` of bar. */
template <int NT>
__device__ __forceinline__ int first_past(const double *r, int j, double before, double bar, bool last_too, DrawLds<NT> &L,
                                          bool ready = false, double doubt = -1.0) {
  int over = 0x7fffffff, last = -1;
  bool close = fabs(before - bar) <= doubt;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    before += r[e];
    close = close || fabs(before - bar) <= doubt;
    last = r[e] > 0.0 ? j + e : last;
    over = min(over, r[e] > 0.0 && before > bar ? j + e : 0x7fffffff);
  }
  if (!ready) { /* (L.at holds it) */
    if (threadIdx.x == 0) L.at = 0x7fffffff;
    __syncthreads();
  }
  /* (places rise with the lanes: the first that has one speaks for its wave) */
  const uint64_t has = __ballot(over != 0x7fffffff);
  if (close) L.close = 1;
  if (has && lane_id() == (int)__builtin_ctzll(has)) atomicMin(&L.at, over);
  __syncthreads();
  int at = L.at;
  if (at != 0x7fffffff || !last_too) {
    if (!ready) __syncthreads();
    return at != 0x7fffffff ? at : -1;
  }
  __syncthreads();
  if (threadIdx.x == 0) L.at = -1;
  __syncthreads();
  if (last >= 0) atomicMax(&L.at, last);
  __syncthreads();
  at = L.at;
  __syncthreads();
  return at;
}

/* the token among [lo, hi), *sum the weights before them, and where there is none those up to hi */
template <int NT, bool TB, bool DB>
__device__ __forceinline__ int pick(const Weights<TB, DB> &W, int lo, int hi, double *sum, double bar, bool plain, DrawLds<NT> &L,
                                    double doubt = -1.0) {
  int last = -1;
  for (int c = lo; c < hi; c += NT * 8) {
    const int j = c + (int)threadIdx.x * 8;
    double r[8] = {0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0}, mine = 0.0, total;
    if (j < hi) W.at(j, plain, r);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      if (j + e >= hi) r[e] = 0.0;
      mine += r[e];
    }
    const double before = *sum + block_scan64(mine, L, &total);
    const int at = first_past(r, j, before, bar, false, L, false, doubt);
    if (at >= 0) return at;
    const int end = first_past(r, j, before, __builtin_inf(), true, L);
    if (end >= 0) last = end;
    *sum += total;
  }
  return last;
}

/* A workgroup a sequence: a wave a row of logits, then the draw.  HELD: rows of which a
 * thread's eight elements are all (VT * 8): their terms stay in registers from the sums to the
 * token; else three passes.  One row of 4097 of four drafts: a chain of dependent steps (loads, sums,
 * decision, loads, 64-bit terms, two sums over the workgroup, the place). */
template <bool TB, bool DB, bool HELD>
__global__ __launch_bounds__(VT) void k_verify_one(d3s_verify_params a, int b0) {
  __shared__ Settled S;
  __shared__ DrawLds<VT> L;
  __shared__ double pair[VT / WAVE][2];
  const int tid = (int)threadIdx.x, V = (int)a.vocab;
  const Seq q(a, b0 + (int)blockIdx.x);
  const float u = lane_u(a, q), ud = a.u_draw[q.b];
  const int x = lane_draft(a, q);
  for (int r = tid / WAVE; r < q.rows; r += VT / WAVE) {
    if (!q.there(a, r)) continue;
    float l;
    Sums s{-FLT_MAX, 0.0f, 0.0f};
    const float c = LOG2E / q.temperature(a, r);
    auto beside = [&] { l = draft_logit<TB, DB>(a, q, r); };
    if (q.target(a, r)) {
      const Row<TB> R(a.target, a.target_stride, q.row(a, r), V, -1);
      lane_sums(s, R, lane_id(), R.chunks, WAVE, c, beside);
    } else {
      const Row<DB> R(a.draft, a.draft_stride, q.row(a, r), V, -1);
      lane_sums(s, R, lane_id(), R.chunks, WAVE, c, beside);
    }
    join_wave(s, c);
    if (lane_id() == 0) settle_row(a, q, r, RowStat{s.m, s.S}, l, S);
  }
  __syncthreads();
  const Outcome o = settle(a, q, S, u, true);
  const RowStat P = S.stat[o.accepted];
  const bool masked = !o.refuse && P.S == 0.0f;
  int token = masked ? 0 : -1;
  if (o.refuse || masked) {
    if (tid == 0 && a.counters) atomicAdd(&a.counters[masked ? CNT_ALL_MASKED : CNT_REFUSED], 1u);
  } else {
    Weights<TB, DB> W(a, q, o.accepted, o.rejected, P.m, S.stat[o.rejected && a.draft ? a.n_draft + 1 + o.accepted : 0].m, x);
    double sp = 0.0, sq = 0.0, p[8], t[8];
    if (HELD) {
#pragma unroll
      for (int e = 0; e < 8; e++) p[e] = t[e] = 0.0;
    }
    for (int j = tid * 8; j < V; j += VT * 8) {
      W.terms(j, p, t);
#pragma unroll
      for (int e = 0; e < 8; e++) sp += p[e];
      if (W.dp) {
#pragma unroll
        for (int e = 0; e < 8; e++) sq += t[e];
      }
      if (HELD) break;
    }
    /* weights p_j - rho q_j: the draw needs no quotient by their sum */
    sp = wave_scan64(sp);
    sq = W.dp ? wave_scan64(sq) : 0.0;
    if (lane_id() == WAVE - 1) pair[tid / WAVE][0] = sp, pair[tid / WAVE][1] = sq;
    if (tid == 0) L.at = 0x7fffffff;
    __syncthreads();
    sp = sq = 0.0;
#pragma unroll
    for (int w = 0; w < VT / WAVE; w++) sp += pair[w][0], sq += pair[w][1];
    W.iq = sq > 0.0 ? sp / sq : 0.0;
    W.ip = 1.0;
    bool plain = !o.rejected;
    double r[8], Z;
    for (;;) {
      if (HELD) {
        double mine = 0.0;
        W.weights(tid * 8, plain, p, t, r);
#pragma unroll
        for (int e = 0; e < 8; e++) mine += r[e];
        const double before = block_scan64(mine, L, &Z);
        if (Z > 0.0 || plain) {
          token = first_past(r, tid * 8, before, (double)ud * Z, true, L, true);
          break;
        }
      } else {
        Z = 0.0;
        for (int j = tid * 8; j < V; j += VT * 8) {
          W.at(j, plain, r);
#pragma unroll
          for (int e = 0; e < 8; e++) Z += r[e];
        }
        Z = block_sum64(Z, L);
        if (Z > 0.0 || plain) {
          double sum = 0.0;
          token = pick<VT>(W, 0, V, &sum, (double)ud * Z, plain, L);
          break;
        }
      }
      plain = true; /* (p <= q everywhere: by rounding alone) */
    }
  }
  write_tokens(q.b, a.n_draft, o, token, x, a.tokens, a.n_accepted);
}

/* ---- long rows: two launches ---- */

constexpr int SWV = ST / WAVE;

/* how the rows are cut: nseg segments of 16-byte chunks for the statistics, nblk blocks for the draw,
 * a part for each of a block's waves, `subs` runs of `sub` elements a part */
struct VerifySplit {
  int nseg, nblk, subs, sub;
};

constexpr int PART = 5;
struct VerifyRoom {
  RowStat *stats; /* [n_seqs, rows, nseg] */
  uint64_t *parts; /* [n_seqs, nblk, SWV, subs, PART]: doubles */
  uint32_t *arrivals;
  int spacing; /* words between two sequences' counters */
};

/* 1: greatest logit and sum of a segment of a row */
template <bool TB, bool DB>
__global__ __launch_bounds__(ST) void k_verify_rows(d3s_verify_params a, VerifySplit sp, VerifyRoom w, int64_t wg0) {
  __shared__ float wm[ST / WAVE], wS[ST / WAVE];
  const int64_t wg = wg0 + blockIdx.x;
  const int rows = a.n_draft + 1 + (a.draft ? a.n_draft : 0);
  const int seg = (int)(wg % sp.nseg), r = (int)(wg / sp.nseg % rows);
  const Seq q(a, (int)(wg / sp.nseg / rows));
  if (!q.there(a, r)) return;
  Sums s{-FLT_MAX, 0.0f, 0.0f};
  const float c = LOG2E / q.temperature(a, r);
  auto go = [&](const auto &R) {
    const int per = (R.chunks + sp.nseg - 1) / sp.nseg;
    lane_sums(s, R, seg * per + (int)threadIdx.x, min(R.chunks, (seg + 1) * per), ST, c, [] {});
  };
  if (q.target(a, r))
    go(Row<TB>(a.target, a.target_stride, q.row(a, r), (int)a.vocab, -1));
  else
    go(Row<DB>(a.draft, a.draft_stride, q.row(a, r), (int)a.vocab, -1));
  join_wave(s, c);
  if (lane_id() == 0) wm[threadIdx.x / WAVE] = s.m, wS[threadIdx.x / WAVE] = s.S;
  __syncthreads();
  if (threadIdx.x != 0) return;
  s = {wm[0], wS[0], 0.0f};
#pragma unroll
  for (int i = 1; i < ST / WAVE; i++) join(s, wm[i], wS[i], 0.0f, c);
  w.stats[wg] = RowStat{s.m, s.S};
}

/* 2: the decision (by every block), and the sums of the rows that the token is drawn from, in 64
 * bits and in one pass.  With P and Q the rows' sums, the weights are p_j / P - q_j / Q =
 * (p_j - rho q_j) / P where that is positive, rho = P / Q.  P and Q are known only behind the pass,
 * but the 32-bit sums give rho0 near it, and with z = sum max(p_j - rho0 q_j, 0) and
 * B = sum of q_j over the same places, z - (rho - rho0) B is the sum at rho, unless p_j - rho q_j is of another sign
 * than p_j - rho0 q_j somewhere: then it is below, by at most |rho - rho0| times these places' q_j.  A is the sum of q_j
 * where that could be, p_j - rho0 q_j being nearer to 0 than BAND rho0 q_j (one place in two rows of 151936).  Each wave
 * leaves P, Q, z, B and A of its runs; the last block of a sequence to arrive finds the run that passes u Z, and the place
 * in it by the weights themselves.  Where what all A allow could decide, their runs are added again from their weights
 * first, and all runs where rho is further than half of BAND from rho0, so that the token is the weights' own.  (A pass for P
 * and Q and another for the weights: 64 sequences of 151936, 49 us where this takes 33.) */
constexpr double BAND = 0x1p-18;

template <bool TB, bool DB>
__global__ __launch_bounds__(ST) void k_verify_draw(d3s_verify_params a, VerifySplit sp, VerifyRoom w) {
  __shared__ Settled S;
  __shared__ DrawLds<ST> L;
  __shared__ double three[3][SWV];
  __shared__ uint32_t last;
  const int tid = (int)threadIdx.x;
  const int blk = (int)(blockIdx.x % (unsigned)sp.nblk);
  const Seq q(a, (int)(blockIdx.x / (unsigned)sp.nblk));
  const float u = lane_u(a, q), ud = a.u_draw[q.b];
  const int x = lane_draft(a, q);
  if (tid < q.rows && q.there(a, tid)) {
    const float l = draft_logit<TB, DB>(a, q, tid);
    const float c = LOG2E / q.temperature(a, tid);
    const RowStat *st = w.stats + ((int64_t)q.b * q.rows + tid) * sp.nseg;
    float m = -FLT_MAX;
    double sum = 0.0; /* (a thousand segments' in 32 bits would be 1e-5 off) */
    constexpr int UN = 8;
    for (int i = 0; i < sp.nseg; i += UN) {
      RowStat part[UN];
#pragma unroll
      for (int u = 0; u < UN; u++) part[u] = st[min(i + u, sp.nseg - 1)];
      float M = m, S = 0.0f;
#pragma unroll
      for (int u = 0; u < UN; u++) M = maximum(M, part[u].m);
#pragma unroll
      for (int u = 0; u < UN; u++) S += i + u < sp.nseg ? part[u].S * exp2_hw(drop(part[u].m, M, c)) : 0.0f;
      sum = sum * (double)exp2_hw(drop(m, M, c)) + (double)S;
      m = M;
    }
    settle_row(a, q, tid, RowStat{m, (float)sum}, l, S);
  }
  __syncthreads();
  const Outcome o = settle(a, q, S, u, blk == 0);
  const RowStat P = S.stat[o.accepted], Q = S.stat[o.rejected && a.draft ? a.n_draft + 1 + o.accepted : 0];
  const bool masked = !o.refuse && P.S == 0.0f;
  if (o.refuse || masked) {
    if (blk != 0) return;
    write_tokens(q.b, a.n_draft, o, masked ? 0 : -1, x, a.tokens, a.n_accepted);
    if (tid == 0 && a.counters) atomicAdd(&a.counters[masked ? CNT_ALL_MASKED : CNT_REFUSED], 1u);
    return;
  }
  Weights<TB, DB> W(a, q, o.accepted, o.rejected, P.m, Q.m, x);
  const double rho0 = W.dp && Q.S > 0.0f ? (double)P.S / Q.S : 0.0, band = rho0 * BAND;
  const int runs = sp.nblk * SWV * sp.subs; /* of the row, in its order */
  uint64_t *parts = w.parts + (int64_t)q.b * runs * PART;
  for (int r = 0; r < sp.subs; r++) {
    const int run = (blk * SWV + tid / WAVE) * sp.subs + r;
    const int64_t lo = (int64_t)run * sp.sub;
    const int hi = (int)min((int64_t)a.vocab, lo + sp.sub);
    double sum[PART] = {0.0, 0.0, 0.0, 0.0, 0.0};
    for (int64_t at = lo + lane_id() * 8; at < hi; at += WAVE * 8) {
      const int j = (int)at;
      double p[8], t[8];
      W.terms(j, p, t);
      if (W.dp) {
        double near = 0.0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const double d = fma(-rho0, t[e], p[e]);
          near = fmin(near, fma(-band, t[e], fabs(d)));
          sum[0] += p[e];
          sum[1] += t[e];
          sum[2] += fmax(d, 0.0);
          sum[3] += d > 0.0 ? t[e] : 0.0;
        }
        if (__builtin_expect(__ballot(near < 0.0) != 0ull, 0)) {
#pragma unroll
          for (int e = 0; e < 8; e++) sum[4] += fabs(fma(-rho0, t[e], p[e])) < band * t[e] ? t[e] : 0.0;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) {
          sum[0] += p[e];
          sum[2] += j + e == W.gone ? 0.0 : p[e];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < PART; i++) { /* (a certain draft's rows have P and z, few runs an A) */
      if (i % 2 && !W.dp) continue;
      if (i == 4 && __builtin_expect(!__ballot(sum[4] > 0.0), 1)) continue;
      sum[i] = wave_scan64(sum[i]);
    }
    if (lane_id() == WAVE - 1) {
#pragma unroll
      for (int i = 0; i < PART; i++) st_agent(parts + run * PART + i, __builtin_bit_cast(uint64_t, sum[i]));
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    uint32_t *cnt = w.arrivals + (int64_t)q.b * w.spacing;
    last = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)(sp.nblk - 1);
    if (last) __hip_atomic_store(cnt, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last) return;
  /* a thread SWV runs (runs <= ST SWV, a multiple of SWV) */
  double at[SWV][PART];
#pragma unroll
  for (int i = 0; i < SWV; i++)
#pragma unroll
    for (int k = 0; k < PART; k++)
      at[i][k] = tid * SWV < runs ? __builtin_bit_cast(double, ld_agent(parts + (tid * SWV + i) * PART + k)) : 0.0;
  /* P, Q and A of the row, by one exchange */
  double row[3] = {0.0, 0.0, 0.0};
#pragma unroll
  for (int i = 0; i < SWV; i++) row[0] += at[i][0], row[1] += at[i][1], row[2] += at[i][4];
#pragma unroll
  for (int k = 0; k < 3; k++) {
    row[k] = wave_scan64(row[k]);
    if (lane_id() == WAVE - 1) three[k][tid / WAVE] = row[k];
  }
  __syncthreads();
  row[0] = row[1] = row[2] = 0.0;
#pragma unroll
  for (int i = 0; i < SWV; i++)
#pragma unroll
    for (int k = 0; k < 3; k++) row[k] += three[k][i];
  const double sum_p = row[0], sum_q = row[1];
  W.ip = 1.0 / sum_p;
  W.iq = sum_q > 0.0 ? 1.0 / sum_q : 0.0;
  const double shift = sum_q > 0.0 ? sum_p / sum_q - rho0 : 0.0;
  /* the runs' weights, the marked ones, and how much these may lack */
  bool plain = !o.rejected, again = !plain && !(fabs(shift) <= 0.5 * band);
  double mine[SWV];
  unsigned marked = 0u;
#pragma unroll
  for (int i = 0; i < SWV; i++) {
    mine[i] = W.ip * (plain ? at[i][0] : fmax(at[i][2] - shift * at[i][3], 0.0));
    if (tid * SWV < runs && (again || at[i][4] > 0.0)) marked |= 1u << i;
  }
  double doubt = plain ? 0.0 : (again ? sum_q : row[2]) * (fabs(shift) * W.ip * (1.0 + 0x1p-20));
  int token;
  for (;;) {
    double all = 0.0, Z;
#pragma unroll
    for (int i = 0; i < SWV; i++) all += mine[i];
    double from = block_scan64(all, L, &Z);
    again = again || (doubt > 0.0 && !(Z > 0.0));
    if (!again && !(Z > 0.0)) { /* p <= q everywhere: p's own draw */
      token = -1;
      if (plain) break; /* (never: the greatest logit has a weight) */
      plain = true;
#pragma unroll
      for (int i = 0; i < SWV; i++) mine[i] = W.ip * at[i][0];
      continue;
    }
    /* the run that passes bar, or the first that is to be added again */
    const double bar = again ? __builtin_inf() : (double)ud * Z;
    int over = again && marked ? tid * SWV + (int)__builtin_ctz(marked) : 0x7fffffff, some = -1;
    double over_from = 0.0, some_from = 0.0;
#pragma unroll
    for (int i = 0; i < SWV; i++) {
      if (mine[i] > 0.0) {
        some = tid * SWV + i, some_from = from;
        if (over == 0x7fffffff && from + mine[i] > bar) over = some, over_from = from;
      }
      from += mine[i];
    }
    if (tid == 0) L.at = 0x7fffffff, L.close = 0;
    __syncthreads();
    if (over != 0x7fffffff) atomicMin(&L.at, over);
    __syncthreads();
    if (L.at == 0x7fffffff) {
      __syncthreads();
      if (again) { /* all are added */
        again = false, doubt = 0.0;
        continue;
      }
      /* none by rounding: the last that has any */
      if (tid == 0) L.at = -1;
      __syncthreads();
      if (some >= 0) atomicMax(&L.at, some);
      over = some, over_from = some_from;
      __syncthreads();
    }
    const int which = L.at;
    if (over == which) L.from = over_from;
    __syncthreads();
    double sum = L.from;
    token = pick<ST>(W, (int)min((int64_t)a.vocab, (int64_t)which * sp.sub), (int)min((int64_t)a.vocab, (int64_t)(which + 1) * sp.sub),
                     &sum, bar, plain, L, again || !(doubt > 0.0) ? -1.0 : doubt);
    const bool close = doubt > 0.0 && L.close; /* (read behind a barrier of pick's) */
    if (!again && !close && token >= 0) break;
    /* (no token: terms below 2^-1022 alone, whose weights are 0 where their sum is not) */
    if (again || !close) {
#pragma unroll
      for (int i = 0; i < SWV; i++)
        if (tid * SWV + i == which) mine[i] = again ? sum : 0.0, marked &= ~(1u << i);
    }
    again = again || close;
  }
  write_tokens(q.b, a.n_draft, o, token, x, a.tokens, a.n_accepted);
}

/* ------------------------------------------------------------------------ */

constexpr int RT = 256;

/* A workgroup a sequence.  All its candidates are loaded at once where HELD entries hold
 * them; else the drawn rows' again. */
__global__ __launch_bounds__(RT) void k_verify_ranked(RankedArgs a) {
  constexpr int HELD = 2048;
  __shared__ float prob[2 * D3S_MAX_DRAFT];
  __shared__ int cand[HELD];
  __shared__ float qs[HELD];
  __shared__ float best[RT / WAVE];
  __shared__ int best_at[RT / WAVE];
  const int b = (int)blockIdx.x, tid = (int)threadIdx.x;
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.n_draft) : a.n_draft;
  const int i = lane_id();
  const int mine = i < a.n_draft ? a.drafted[(size_t)b * a.n_draft + i] : -1; /* lane i: draft i */
  const float u = i < a.n_draft ? a.u_accept[(size_t)b * a.n_draft + i] : 0.0f;
  const float ud = tid < a.target_k ? a.u_draw[(size_t)b * a.target_k + tid] : 0.0f; /* rank tid's */
  const size_t t0 = (size_t)b * (a.n_draft + 1) * a.target_k, d0 = (size_t)b * a.n_draft * a.draft_k;
  const int nt = (len + 1) * a.target_k, nd = a.draft_cand ? len * a.draft_k : 0;
  const bool held = nt + nd <= HELD;
  const float nan = __builtin_nanf("");
  if (tid < 2 * D3S_MAX_DRAFT) prob[tid] = !a.draft_cand && tid >= D3S_MAX_DRAFT ? 1.0f : 0.0f;
  __syncthreads();
  /* (a refused row's candidates are -1; a masked one's probabilities NaN, taken as 0) */
  auto look = [&](const int32_t *c, const float *p, int k, int n, float *out, int at) {
    for (int e0 = 0; e0 < n; e0 += RT) {
      const int e = e0 + tid, row = e / k;
      const int x = __shfl(mine, row & (WAVE - 1)); /* (row <= len <= 64: the row behind 63 drafts has none) */
      if (e >= n) continue;
      const int id = c[e];
      const float pr = p[e];
      if (held) cand[at + e] = id, qs[at + e] = pr;
      if (row < len) {
        if (id < 0) {
          if (e == row * k) out[row] = nan;
        } else if (id == x && pr > 0.0f) {
          out[row] = pr;
        }
      }
    }
  };
  look(a.target_cand + t0, a.target_probs + t0, a.target_k, nt, prob, 0);
  if (a.draft_cand) look(a.draft_cand + d0, a.draft_probs + d0, a.draft_k, nd, prob + D3S_MAX_DRAFT, nt);
  __syncthreads();
  const bool last_refused = (held ? cand[len * a.target_k] : a.target_cand[t0 + (size_t)len * a.target_k]) < 0;
  const float p = i < len ? prob[i] : 0.0f, q = i < len ? prob[D3S_MAX_DRAFT + i] : 0.0f;
  const Outcome o = decide(len, u, p, q, last_refused);
  if (a.accept && tid < a.n_draft) a.accept[(size_t)b * a.n_draft + i] = i < len ? accept_of(p, q) : 0.0f;
  int token = -1;
  if (o.refuse) {
    if (tid == 0 && a.counters) atomicAdd(&a.counters[CNT_REFUSED], 1u);
  } else {
    const int32_t *tc = a.target_cand + t0 + (size_t)o.accepted * a.target_k;
    const float *tp = a.target_probs + t0 + (size_t)o.accepted * a.target_k;
    const bool pair = o.rejected && a.draft_cand;
    const int qa = held ? nt + o.accepted * a.draft_k : 0; /* the draft's row in LDS */
    if (pair && !held) { /* (draft_k <= D3S_MAX_RANKED <= HELD) */
      for (int e = tid; e < a.draft_k; e += RT) {
        cand[e] = a.draft_cand[d0 + (size_t)o.accepted * a.draft_k + e];
        qs[e] = a.draft_probs[d0 + (size_t)o.accepted * a.draft_k + e];
      }
      __syncthreads();
    }
    const int x = o.rejected ? __shfl(mine, o.accepted) : -1;
    bool plain = !o.rejected;
    for (;;) {
      float sc = -2.0f;
      int at = 0x7fffffff;
      for (int r = tid; r < a.target_k; r += RT) {
        const int id = held ? cand[o.accepted * a.target_k + r] : tc[r];
        float w = held ? qs[o.accepted * a.target_k + r] : tp[r];
        if (!plain && pair) {
          float gone = 0.0f; /* (one candidate at most is this one) */
#pragma unroll 8
          for (int e = 0; e < a.draft_k; e++) gone = cand[qa + e] == id ? qs[qa + e] : gone;
          if (gone > 0.0f) w -= gone;
        } else if (!plain && id == x) {
          w -= 1.0f;
        }
        if (!(w > 0.0f)) continue;
        float score = w / -d3s_logf(1.0f - (r < RT ? ud : a.u_draw[(size_t)b * a.target_k + r]));
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
        token = held ? cand[o.accepted * a.target_k + at] : tc[at];
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
  write_tokens(b, a.n_draft, o, token, mine, a.tokens, a.n_accepted);
}

}  // namespace

/* Rows longer than a workgroup holds are split over the chip, unless there are so many sequences that
 * a workgroup for each fills it (16 sequences of 4 drafts over 16384: 14 us, by a workgroup each 38; 300 of
 * 3 over 16000: 39, 68). */
static bool verify_split(const d3s_verify_params &a, bool draft, VerifySplit *sp) {
  if (a.vocab <= VT * 8 || a.n_seqs > 2048) return false;
  const int64_t rows = a.n_seqs * (2 * a.n_draft + 1);
  /* segments of two batches of bf16 chunks a lane, one where there are few */
  const int64_t batches = ((a.vocab + 7) / 8 + SU * ST - 1) / (SU * ST);
  sp->nseg = (int)(rows * batches <= 2048 ? batches : (batches + 1) / 2);
  /* Few enough blocks that the decision, which each makes, is waited for once or little more (256 sequences of one
   * certain draft over 151936: 1024 blocks 79 us, 1280 84, 2560 90; two rows a place, 64 sequences: 1216 blocks 56.6,
   * 960 59.3).  Each run is summed for itself, so that the place is looked for in one of them. */
  const int64_t most = (draft ? 1280 : 1024) / a.n_seqs, blocks = most < 1 ? 1 : most > ST ? ST : most;
  auto up = [](int64_t n, int64_t of, int64_t to) { return ((n + of - 1) / of + to - 1) / to * to; };
  const int64_t part = up(a.vocab, blocks * SWV, WAVE * 8), block = part * SWV;
  sp->nblk = (int)((a.vocab + block - 1) / block);
  const int64_t subs = (part + ST * 8 - 1) / (ST * 8), room = ST / sp->nblk;
  sp->subs = (int)(subs < room ? subs : room);
  sp->sub = (int)up(part, sp->subs, WAVE * 8);
  return true;
}

static size_t verify_layout(const d3s_verify_params &a, const VerifySplit &sp, char *base, VerifyRoom *w) {
  size_t at = split_counter_bytes();
  auto take = [&](size_t bytes) {
    char *p = base + at;
    at += (bytes + 255) / 256 * 256;
    return p;
  };
  const size_t n = (size_t)a.n_seqs;
  w->arrivals = (uint32_t *)base;
  w->spacing = 32;
  w->stats = (RowStat *)take(n * (2 * (size_t)a.n_draft + 1) * sp.nseg * sizeof(RowStat));
  w->parts = (uint64_t *)take(n * sp.nblk * SWV * sp.subs * PART * sizeof(uint64_t));
  return at;
}

size_t verify_workspace_bytes(const d3s_verify_params &a) {
  size_t most = 0; /* with drafts that are certain and without */
  for (const bool draft : {false, true}) {
    VerifySplit sp;
    VerifyRoom w;
    const size_t need = verify_split(a, draft, &sp) ? verify_layout(a, sp, nullptr, &w) : 0;
    most = need > most ? need : most;
  }
  return most;
}

template <bool TB, bool DB>
static void verify_launch(const d3s_verify_params &a, void *ws, hipStream_t s) {
  VerifySplit sp;
  if (!verify_split(a, a.draft != nullptr, &sp)) {
    constexpr int64_t MOST = 1 << 21; /* workgroups a launch: their threads are counted in 32 bits */
    for (int64_t b = 0; b < a.n_seqs; b += MOST) {
      const dim3 grid((unsigned)(a.n_seqs - b < MOST ? a.n_seqs - b : MOST));
      if (a.vocab <= VT * 8)
        k_verify_one<TB, DB, true><<<grid, VT, 0, s>>>(a, (int)b);
      else
        k_verify_one<TB, DB, false><<<grid, VT, 0, s>>>(a, (int)b);
    }
    return;
  }
  VerifyRoom w;
  verify_layout(a, sp, (char *)ws, &w);
  const int64_t wgs = a.n_seqs * (a.n_draft + 1 + (a.draft ? a.n_draft : 0)) * sp.nseg;
  for (int64_t g = 0; g < wgs; g += GRID_MOST)
    k_verify_rows<TB, DB><<<dim3((unsigned)(wgs - g < GRID_MOST ? wgs - g : GRID_MOST)), ST, 0, s>>>(a, sp, w, g);
  const dim3 blocks((unsigned)(a.n_seqs * sp.nblk)); /* (at most 2048 * 256) */
  k_verify_draw<TB, DB><<<blocks, ST, 0, s>>>(a, sp, w);
}

void launch_verify(const d3s_verify_params &params, void *ws, hipStream_t s) {
  const d3s_verify_params a = params;
  const bool db = a.draft && a.draft_dtype == D3S_DTYPE_BF16;
  if (a.target_dtype == D3S_DTYPE_BF16)
    db ? verify_launch<true, true>(a, ws, s) : verify_launch<true, false>(a, ws, s);
  else
    db ? verify_launch<false, true>(a, ws, s) : verify_launch<false, false>(a, ws, s);
}

void launch_verify_ranked(const RankedArgs &args, hipStream_t s) {
  const RankedArgs a = args;
  k_verify_ranked<<<dim3((unsigned)a.n_seqs), RT, 0, s>>>(a);
}

}  // namespace d3s
