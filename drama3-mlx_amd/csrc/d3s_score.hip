/* k_score, k_score_grad: log probabilities of given tokens, entropy and the best
 * alternatives of rows of logits, and their gradient in the logits (gfx950,
 * wave64; include/d3s_train.h).
 *
 * Forward.  One pass over the row: every lane keeps a running maximum m, the
 * sum S of 2^((l - m) c) with c = log2(e) / T and, for the entropy, the sum A of
 * the same terms times their exponents.  A lane takes a batch of 16-byte chunks,
 * raises m to the batch's maximum, rescales (S, A) once and adds the batch:
 *   m' = max(m, batch), f = 2^((m - m') c), A = f (A + S (m - m') c), S = f S.
 * The exponent is one fma(l, c, -RN(m c)): its rounding is relative to the
 * exponent, and what the shift's own rounding leaves, the same for every term
 * of the batch, is put back once a batch (it reaches 0.03 at logits of 10 and a
 * temperature of 1e-5).
 * Lanes, waves and segments join by the same rule; then
 *   logprob = (l - m) / T - log S,  H = log S - ln 2 A / S.
 * Sums are fp32: a lane adds at most V / 256 terms, then a tree.
 * A row of few (long) rows is cut into segments, one workgroup each; the
 * segments' records go to the workspace and the last to arrive joins them (in
 * segment order, so the bits do not depend on who is last).
 *
 * Alternatives.  Of the n best, each of the four waves finds by ballots the
 * ceil(n / 4)-th greatest of its lanes' maxima (its upper 16 bits); at least n
 * logits reach the least of the four, and few others do: a second pass over
 * the segment files those, and the filed keys (order-preserving logit bits, then
 * the complement of the index) are ranked by counting.  More than the list
 * holds (ties, masked rows, logits that agree in their upper 16 bits): the n-th of
 * the filed keys is a bound at least as high, and the pass is run again with it, and
 * with a sample filed where that leaves out too few.  The segment passes through LDS in
 * blocks of 16 KiB; one that is a single block is not loaded again.  The join
 * of the segments bounds their keys the same way and ranks what reaches it.
 *
 * Gradient.  Every element needs its own logit and four numbers of its row:
 * one streaming pass, rows cut into segments that share nothing, stores past the
 * caches (through them: 2 to 20 % slower).
 *
 * Bound: long rows HBM (bf16 [4096, 151936]: 219 us, 5.7 TB/s; fp32 [2048, 151936]
 * 212 us, 5.9 TB/s; the gradient of fp32 [1024, 151936] 233 us, 5.3 TB/s, and of bf16
 * [2048, 151936] 229 us, 5.4 TB/s; of fp32 [4096, 4097] 25 us, 5.3 TB/s); few
 * rows the chain of dependent steps (bf16 [1, 4097] with five alternatives 6.7 us;
 * [64, 151936] with twenty 18.3 us, of which the bytes are 4). */
#include "d3s_rowcore.h"
#include "d3s_rowsums.h"
#include "d3s_stream.h"
#include "d3s_train_internal.h"

namespace d3s {
namespace {

constexpr int ST = 256;        /* threads of a workgroup */
constexpr int SW = ST / WAVE;
constexpr int CUS = 256;
constexpr int GRID_MOST = 1 << 22; /* workgroups a launch: their threads are counted in 32 bits */
constexpr int SU = 4;          /* chunks a lane takes at a time */
constexpr int SCORE_ARRIVALS = 2048; /* rows that have a counter of arrivals */
constexpr int LIST = 512;      /* keys a workgroup files */
constexpr int JOIN = 2048;     /* ... and the segments' that it joins */
constexpr int SEG_MOST = 256;  /* segments a row */
constexpr int SEG_TOP = 64;    /* the same with alternatives: their keys (at most JOIN) are ranked again */
/* a row's temperature; one that is not finite (the row is refused) stays as it is */
__device__ __forceinline__ float row_temperature(const ScoreArgs &a, int row) {
  const float T = a.temperature ? a.temperature[row] : a.temperature_scalar;
  return T < 1e-5f && T > -__builtin_inff() ? 1e-5f : T;
}
struct ScoreLds {
  alignas(16) uint64_t list[LIST + 2]; /* (read in pairs) */
  uint64_t ranked[D3S_MAX_TOP];
  uint32_t least[SW];
  float wm[SW], wS[SW], wA[SW];
  uint64_t bound[SW];
  uint32_t count, last;
};

/* the join of part[0 .. n) (n <= ST, one a thread) in every thread */
__device__ __forceinline__ Sums join_block(ScoreLds &L, Sums s, float c) {
  join_wave(s, c);
  const int wid = threadIdx.x / WAVE;
  if (lane_id() == 0) L.wm[wid] = s.m, L.wS[wid] = s.S, L.wA[wid] = s.A;
  __syncthreads();
  s = {L.wm[0], L.wS[0], L.wA[0]};
#pragma unroll
  for (int w = 1; w < SW; w++) join(s, L.wm[w], L.wS[w], L.wA[w], c);
  return s;
}

/* ranks a list's n keys (two places behind them) and leaves the best k in L.ranked (fewer: the rest 0) */
__device__ __forceinline__ void rank_list(ScoreLds &L, uint64_t *list, uint32_t n, int k) {
  if (threadIdx.x < (unsigned)k) L.ranked[threadIdx.x] = 0ull;
  __syncthreads();
  rank_by_count<ST>(list, n, k, L.ranked);
}

/* the row's outputs, by the whole workgroup: s the row's sums, L.ranked its alternatives */
template <bool BF16>
__device__ __forceinline__ void finish(const ScoreArgs &a, ScoreLds &L, const Row<BF16> &R, int row, Sums s, float T,
                                       float token_logit, int token) {
  const int tid = (int)threadIdx.x;
  const float nan = __builtin_nanf(""), ninf = -__builtin_inff();
  const bool refused = !(s.m < __builtin_inff()) || !finite(T);
  const bool masked = !refused && s.S == 0.0f;
  const float logS = refused ? nan : masked ? ninf : d3s_logf(s.S);
  if (tid == 0) {
    if (a.row_stats) {
      a.row_stats[2 * (size_t)row] = refused ? nan : masked ? ninf : s.m;
      a.row_stats[2 * (size_t)row + 1] = logS;
    }
    /* (a sum that rounds below 1 would make a certain row's entropy negative) */
    if (a.entropy) a.entropy[row] = refused ? nan : masked ? 0.0f : fmaxf(logS - LN2 * (s.A / s.S), 0.0f);
    if (a.counters && (refused || masked)) atomicAdd(&a.counters[masked ? CNT_ALL_MASKED : CNT_REFUSED], 1u);
  }
  auto logprob = [&](float l) { return refused ? nan : masked ? ninf : (l - s.m) / T - logS; };
  if (tid < a.n_tokens) {
    const bool none = (unsigned)token >= (unsigned)a.vocab;
    a.logprobs[(size_t)row * a.n_tokens + tid] = refused ? nan : none ? 0.0f : logprob(token_logit);
  }
  if (tid < a.n_top) {
    const uint64_t key = L.ranked[tid];
    const size_t at = (size_t)row * a.n_top + tid;
    if (a.top_ids) a.top_ids[at] = refused ? -1 : masked ? tid : key_idx(key);
    if (a.top_logprobs) a.top_logprobs[at] = logprob(key_x(key));
  }
}

/* words of a segment's record: (m, S), A, then its alternatives' keys */
__host__ __device__ inline int record_words(int n_top) { return 2 + n_top; }

template <bool BF16, bool ENT, bool TOP>
__global__ __launch_bounds__(ST) void k_score(ScoreArgs a, int nseg, int seg_chunks, uint32_t *arrivals,
                                              uint64_t *records, int row0) {
  constexpr int EPC = Row<BF16>::EPC;
  __shared__ ScoreLds L;
  const int tid = (int)threadIdx.x;
  const int row = row0 + (int)(blockIdx.x / (unsigned)nseg), seg = (int)(blockIdx.x % (unsigned)nseg);
  const float T = row_temperature(a, row);
  const float c = LOG2E / T;
  const Row<BF16> R(a.logits, a.row_stride, row, a.vocab, a.banned ? a.banned[row] : -1);
  int token = -1;
  float token_logit = 0.0f;
  if (tid < a.n_tokens) {
    token = a.tokens[(size_t)row * a.n_tokens + tid];
    if ((unsigned)token < (unsigned)a.vocab) {
      const size_t at = (size_t)((int64_t)row * a.row_stride + token);
      token_logit = token == R.banned ? -__builtin_inff()
                    : BF16 ? d3s_u2f((uint32_t)((const uint16_t *)a.logits)[at] << 16)
                           : ((const float *)a.logits)[at];
    }
  }
  const int lo = seg * seg_chunks, hi = min(R.chunks, lo + seg_chunks);

  Sums s{-FLT_MAX, 0.0f, 0.0f};
  /* With alternatives the segment goes by blocks through LDS (a lane's own
   * places), where the second pass finds it again: rolled loops, since the code of
   * such short work has to be fetched while it runs. */
  __shared__ uint4 block[TOP ? SU * ST + 1 : 1]; /* (later the segments' keys) */
  static_assert(sizeof(uint64_t) * (JOIN + 2) <= sizeof(uint4) * (SU * ST + 1), "the join's list");
  uint4 q[SU];
  auto fetch = [&](int at) {
#pragma unroll
    for (int u = 0; u < SU; u++) q[u] = R.base[min(at + tid + u * ST, hi - 1)];
#pragma unroll
    for (int u = 0; u < SU; u++) block[u * ST + tid] = q[u];
  };
  if (TOP) {
    for (int at = lo; at < hi; at += SU * ST) {
      fetch(at);
      if (at + tid + (SU - 1) * ST < hi) {
        float v[SU * EPC];
#pragma unroll
        for (int u = 0; u < SU; u++) R.values(q[u], at + tid + u * ST, v + u * EPC);
        add_batch<SU * EPC, ENT>(s, v, c);
        continue;
      }
#pragma nounroll
      for (int i = tid; i < min(SU * ST, hi - at); i += ST) {
        float v[EPC];
        R.values(block[i], at + i, v);
        add_batch<EPC, ENT>(s, v, c);
      }
    }
  } else {
    int ch = lo + tid;
    for (; ch + (SU - 1) * ST < hi; ch += SU * ST) {
#pragma unroll
      for (int u = 0; u < SU; u++) q[u] = R.base[ch + u * ST];
      float v[SU * EPC];
#pragma unroll
      for (int u = 0; u < SU; u++) R.values(q[u], ch + u * ST, v + u * EPC);
      add_batch<SU * EPC, ENT>(s, v, c);
    }
    for (; ch < hi; ch += ST) {
      float v[EPC];
      R.values(R.base[ch], ch, v);
      add_batch<EPC, ENT>(s, v, c);
    }
  }
  const uint32_t mine = s.S > 0.0f ? d3s_ordkey(s.m) : 0u; /* (0: below every logit's key) */
  const int k = a.n_top;
  if (TOP) {
    /* the wave's ceil(k / SW)-th greatest lane maximum, its upper 16 bits (0: there
     * are not so many): k logits reach the least wave's */
    const int want = (k + SW - 1) / SW;
    uint32_t t = 0u;
#pragma unroll
    for (int b = 31; b >= 16; b--)
      if (__popcll(__ballot(mine >= (t | 1u << b))) >= want) t |= 1u << b;
    if (lane_id() == 0) L.least[tid / WAVE] = t;
    if (tid == 0) L.count = 0u;
  }
  s = join_block(L, s, c);
  const bool live = s.m < __builtin_inff() && finite(T); /* no NaN or +inf in the segment: the row may be scored */

  if (TOP) {
    uint32_t t = L.least[0];
#pragma unroll
    for (int w = 1; w < SW; w++) t = min(t, L.least[w]);
    uint64_t bound = (uint64_t)t << 32;
    uint32_t n = 0u, shift = 0u, before = ~0u; /* of those that reach, every 2^shift-th to arrive is filed */
    while (live) { /* every thread of the workgroup agrees on `live`, n and shift */
      const float least = (bound >> 32) ? d3s_from_ordkey((uint32_t)(bound >> 32)) : -__builtin_inff();
      for (int at = lo; at < hi; at += SU * ST) {
        if (hi - lo > SU * ST) fetch(at);
        uint32_t reach = 0u; /* a bit an element that may */
#pragma nounroll
        for (int u = 0; u < SU; u++) {
          const int i = u * ST + tid;
          if (at + i >= hi) break;
          float v[EPC];
          R.values(block[i], at + i, v);
#pragma unroll
          for (int e = 0; e < EPC; e++) reach |= (v[e] >= least ? 1u : 0u) << (u * EPC + e);
        }
        while (reach) {
          const int b = __ffs(reach) - 1, i = b / EPC * ST + tid, j = (at + i) * EPC + b % EPC - R.lead;
          reach &= reach - 1u;
          float x = BF16 ? d3s_u2f((uint32_t)((const uint16_t *)&block[i])[b % EPC] << 16) : ((const float *)&block[i])[b % EPC];
          if (j == R.banned) x = -__builtin_inff();
          const uint64_t key = composite_key(x, j);
          if (key >= bound && j >= 0 && j < a.vocab) {
            const uint32_t place = atomicAdd(&L.count, 1u), slot = place >> shift;
            if (slot << shift == place && slot < LIST) L.list[slot] = key;
          }
        }
      }
      __syncthreads();
      n = L.count;
      __syncthreads();
      if (n <= LIST && shift == 0u) break;
      /* at least k of the filed keys reach their k-th: none below it is among the best k */
      const uint32_t filed = min((uint32_t)LIST, ((n - 1u) >> shift) + 1u);
      rank_list(L, L.list, filed, k);
      if (tid == 0) L.count = 0u;
      if (filed >= (uint32_t)k) bound = L.ranked[k - 1];
      /* The first to arrive are a good sample of rows in no order, the best of ties, and
       * the least of a rising row, 448 a pass: where they did not leave out half, every
       * 2^shift-th of all n is filed, which leaves about k << shift. */
      if (shift > 0u && filed >= (uint32_t)k) {
        shift -= min(shift, 31u - __clz(LIST / 2 / k));
      } else if (shift > 0u) { /* (fewer were left) */
        shift = n <= LIST ? 0u : 32u - __clz(n / LIST);
      } else {
        shift = n <= before / 2u ? 0u : 32u - __clz(n / LIST);
        before = n;
      }
      __syncthreads();
    }
    rank_list(L, L.list, n, k);
  }
  if (nseg == 1) {
    finish<BF16>(a, L, R, row, s, T, token_logit, token);
    return;
  }

  /* the record, complete before the arrival is counted (see st_agent) */
  const int words = record_words(k);
  uint64_t *rec = records + ((size_t)row * nseg + seg) * words;
  if (tid == 0) {
    st_agent(rec, (uint64_t)d3s_f2u(s.m) | (uint64_t)d3s_f2u(s.S) << 32);
    st_agent(rec + 1, (uint64_t)d3s_f2u(s.A));
  }
  if (tid < k) st_agent(rec + 2 + tid, L.ranked[tid]);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    uint32_t *cnt = arrivals + (size_t)row * 32;
    L.last = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)(nseg - 1);
    if (L.last) __hip_atomic_store(cnt, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    L.count = 0u;
  }
  __syncthreads();
  if (!L.last) return;
  const uint64_t *rr = records + (size_t)row * nseg * words;
  s = {-FLT_MAX, 0.0f, 0.0f};
  if (tid < nseg) {
    const uint64_t w0 = ld_agent(rr + (size_t)tid * words), w1 = ld_agent(rr + (size_t)tid * words + 1);
    s = {d3s_u2f((uint32_t)w0), d3s_u2f((uint32_t)(w0 >> 32)), d3s_u2f((uint32_t)w1)};
  }
  s = join_block(L, s, c);
  if (TOP) {
    /* a wave's segments, lane i the i-th key (loads together); every segment's
     * ceil(k / nseg)-th key: at least k keys reach the least of them */
    uint64_t *list = (uint64_t *)block;
    const int kc = (k + nseg - 1) / nseg;
    uint64_t key[SEG_TOP / SW], least = ~0ull;
#pragma unroll
    for (int u = 0; u < SEG_TOP / SW; u++) {
      const int q = tid / WAVE + u * SW;
      key[u] = q < nseg && lane_id() < k ? ld_agent(rr + (size_t)q * words + 2 + lane_id()) : 0ull;
    }
#pragma unroll
    for (int u = 0; u < SEG_TOP / SW; u++) {
      const uint64_t at = (uint64_t)readlane_u((uint32_t)(key[u] >> 32), kc - 1) << 32 | readlane_u((uint32_t)key[u], kc - 1);
      if (tid / WAVE + u * SW < nseg) least = min(least, at);
    }
    if (lane_id() == 0) L.bound[tid / WAVE] = least;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SW; w++) least = min(least, L.bound[w]);
#pragma unroll
    for (int u = 0; u < SEG_TOP / SW; u++)
      if (key[u] != 0ull && key[u] >= least) list[atomicAdd(&L.count, 1u)] = key[u];
    __syncthreads();
    rank_list(L, list, L.count, k);
  }
  finish<BF16>(a, L, R, row, s, T, token_logit, token);
}

/* ------------------------------------------------------------------------ */

template <bool BF16>
__device__ __forceinline__ float load_one(const void *p, int64_t at) {
  if constexpr (BF16) return d3s_u2f((uint32_t)((const uint16_t *)p)[at] << 16);
  return ((const float *)p)[at];
}
template <bool BF16>
__device__ __forceinline__ void store_one(void *p, int64_t at, float v) {
  if constexpr (BF16)
    ((uint16_t *)p)[at] = d3s_f32_to_bf16_rn(v);
  else
    ((float *)p)[at] = v;
}

__device__ __forceinline__ uint4 load16(const void *p) {
  uint4 q;
  __builtin_memcpy(&q, p, 16);
  return q;
}

/* one row's numbers */
struct GradRow {
  float m, c, c_lo, inv_S, log2S, G, gH, H, inv_T;
};

/* the gradient at one logit that is no token.  fp32 rows: the exponent in two
 * parts (the product's rounding error and c's own come back by 2^r = 1 + r ln 2),
 * since p is not rounded again; bf16 rows are rounded to 8 bits after. */
template <bool BF16>
__device__ __forceinline__ float grad_at(const GradRow &r, float l) {
  const float d = l - r.m, t = fmaxf(d * r.c, LEAST);
  float p = exp2_hw(t) * r.inv_S;
  float lp;
  if constexpr (BF16) {
    lp = (t - r.log2S) * LN2;
  } else {
    const float e = fmaf(d, r.c, -(d * r.c)) + d * r.c_lo;
    if (t > LEAST) p = fmaf(p, e * LN2, p);
    lp = fmaf(t, LN2, -r.log2S * LN2);
  }
  const float g = -p * fmaf(r.gH, lp + r.H, r.G) * r.inv_T;
  return l == -__builtin_inff() ? 0.0f : g;
}

constexpr int GU = 4; /* chunks a lane takes at a time */

/* Chunks are the gradient's aligned 16 bytes (its stores are whole); the
 * logits' are loaded at whatever offset they lie. */
template <bool BF16>
__global__ __launch_bounds__(ST) void k_score_grad(ScoreArgs a, int nseg, int seg_chunks, int row0) {
  constexpr int EPC = BF16 ? 8 : 4, ES = BF16 ? 2 : 4;
  const int tid = (int)threadIdx.x;
  const int row = row0 + (int)(blockIdx.x / (unsigned)nseg), seg = (int)(blockIdx.x % (unsigned)nseg);
  const int V = a.vocab;
  const char *src = (const char *)a.logits + (int64_t)row * a.row_stride * ES;
  char *dst = (char *)a.grad + (int64_t)row * a.grad_stride * ES;
  const int lead = (int)((uintptr_t)dst & 15) / ES;
  const int chunks = (lead + V + EPC - 1) / EPC;
  const int lo = seg * seg_chunks, hi = min(chunks, lo + seg_chunks);
  const int j0 = max(lo * EPC - lead, 0), j1 = min(hi * EPC - lead, V);
  /* whole chunks, and single elements before and after them: a lane each */
  const int first = max(lo, lead > 0 ? 1 : 0), end = min(hi, (lead + V) / EPC);
  const int head = lead > 0 && lo == 0 ? min(EPC - lead, V) : 0;
  const int tail = lo < chunks && hi == chunks ? max((lead + V) / EPC * EPC - lead, lead > 0 ? min(EPC - lead, V) : 0) : V;
  auto get = [&](int ch) { return load16(src + ((int64_t)ch * EPC - lead) * ES); };

  const float T = row_temperature(a, row);
  const int ban = a.banned ? a.banned[row] : -1;
  GradRow r;
  r.m = a.stats_in[2 * (size_t)row];
  const float logS = a.stats_in[2 * (size_t)row + 1];
  r.gH = a.grad_entropy ? a.grad_entropy[row] : 0.0f;
  r.H = a.grad_entropy ? a.entropy_in[row] : 0.0f;
  /* lane t of every wave: token t and its gradient */
  const int lane = lane_id();
  int token = -1;
  float g = 0.0f;
  if (lane < a.n_tokens) {
    token = a.tokens[(size_t)row * a.n_tokens + lane];
    if ((unsigned)token >= (unsigned)V) token = -1;
    if (token >= 0) g = a.grad_logprobs[(size_t)row * a.n_tokens + lane];
  }
  r.G = 0.0f; /* in token order */
  for (int t = 0; t < a.n_tokens; t++) r.G += readlane_f(g, t);
  const bool zero = __ballot(g != 0.0f) == 0ull && r.gH == 0.0f;
  r.c = LOG2E / T;
  r.c_lo = fmaf(-r.c, T, LOG2E) / T + 1.925963033500e-8f / T; /* log2 e = LOG2E + 1.9e-8 */
  r.inv_S = d3s_expf(-logS);
  r.log2S = logS * LOG2E;
  r.inv_T = 1.0f / T;
  if (!finite(T)) r.inv_T = __builtin_nanf("");

  /* a token's logit, before its place may be overwritten (grad may be logits) */
  const bool here = token >= j0 && token < j1 && threadIdx.x < WAVE;
  const float token_logit = here ? load_one<BF16>(src, token) : 0.0f;
  if (a.n_tokens > 0) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  }
  auto put = [&](int ch, uint4 q) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    uint32_t o[4] = {0u, 0u, 0u, 0u};
    if (!zero) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int j = (ch * EPC - lead) + i * (EPC / 4);
        if constexpr (BF16) {
          float x = grad_at<true>(r, d3s_u2f(w[i] << 16)), y = grad_at<true>(r, d3s_u2f(w[i] & 0xffff0000u));
          if (j == ban) x = 0.0f;
          if (j + 1 == ban) y = 0.0f;
          o[i] = (uint32_t)d3s_f32_to_bf16_rn(x) | (uint32_t)d3s_f32_to_bf16_rn(y) << 16;
        } else {
          o[i] = j == ban ? 0u : d3s_f2u(grad_at<false>(r, d3s_u2f(w[i])));
        }
      }
    }
    stream16(dst + ((int64_t)ch * EPC - lead) * ES, make_uint4(o[0], o[1], o[2], o[3]));
  };
  const int j = tid < head ? tid : tail + (tid - head);
  if (j < V && (tid < head || j >= tail)) {
    float v = 0.0f;
    if (!zero) v = j == ban ? 0.0f : grad_at<BF16>(r, load_one<BF16>(src, j));
    store_one<BF16>(dst, j, v);
  }
  for (int ch = first + tid; ch < end; ch += GU * ST) {
    if (ch + (GU - 1) * ST < end && !zero) {
      uint4 q[GU];
#pragma unroll
      for (int u = 0; u < GU; u++) q[u] = get(ch + u * ST);
#pragma unroll
      for (int u = 0; u < GU; u++) put(ch + u * ST, q[u]);
      continue;
    }
    for (int u = 0; u < GU && ch + u * ST < end; u++)
      put(ch + u * ST, zero ? make_uint4(0u, 0u, 0u, 0u) : get(ch + u * ST));
  }
  if (a.n_tokens == 0 || zero) return;
  /* the tokens' own places, after everything else is there */
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x >= WAVE) return;
  float mine = 0.0f; /* a token given twice has both gradients */
  for (int t = 0; t < a.n_tokens; t++)
    if (__builtin_amdgcn_readlane(token, t) == token) mine += readlane_f(g, t);
  if (here) {
    const bool masked = token == ban || token_logit == -__builtin_inff();
    store_one<BF16>(dst, token, masked ? 0.0f : grad_at<BF16>(r, token_logit) + mine * r.inv_T);
  }
}

template <bool BF16>
int chunks_of(int vocab) {
  constexpr int EPC = Row<BF16>::EPC;
  return (vocab + 2 * EPC - 2) / EPC; /* at the worst offset */
}

}  // namespace

/* Four workgroups a CU, each with at least two chunks a lane (bf16, four and eight
 * a CU: 64 rows of 151936 9.8 and 12.5 us, 1024 of them 53 and 60, 1024 rows of
 * 32000 15 and 20; with ten alternatives 512 rows of 151936 56 and 64).  With alternatives
 * at least a block of LDS, so that filing needs no second read ([16, 151936], twenty
 * alternatives: 14 us, 17 with two chunks a lane), and more of them only while
 * there are few rows (ten alternatives, a block each: 128 rows 27 us, so 24; 512
 * rows 89, so 56). */
int score_segments(Dtype dt, int64_t n_rows, int vocab, int n_top) {
  const int chunks = dt == DT_BF16 ? chunks_of<true>(vocab) : chunks_of<false>(vocab);
  if (n_rows > SCORE_ARRIVALS) return 1;
  const int64_t want = n_rows > 0 ? 4 * CUS / n_rows : 1;
  const int most = n_top > 0 ? min(min(SEG_TOP, JOIN / n_top), (chunks + SU * ST - 1) / (SU * ST)) : min(SEG_MOST, chunks / (2 * ST));
  const int n = (int)(want < most ? want : most);
  return n > 1 ? n : 1;
}

size_t score_workspace_bytes(Dtype dt, int64_t n_rows, int vocab, int n_top) {
  const int nseg = score_segments(dt, n_rows, vocab, n_top);
  if (nseg == 1) return 0;
  return split_counter_bytes() + (size_t)n_rows * nseg * record_words(n_top) * sizeof(uint64_t);
}

template <bool BF16>
static void score_launch(const ScoreArgs &a, void *ws, hipStream_t s) {
  const int nseg = score_segments(BF16 ? DT_BF16 : DT_F32, a.n_rows, a.vocab, a.n_top);
  const int seg_chunks = (chunks_of<BF16>(a.vocab) + nseg - 1) / nseg;
  uint32_t *arrivals = (uint32_t *)ws;
  uint64_t *records = ws ? (uint64_t *)((char *)ws + split_counter_bytes()) : nullptr;
  for (int row0 = 0; row0 < a.n_rows;) {
    const int rows = min(a.n_rows - row0, GRID_MOST / nseg);
    const dim3 grid((unsigned)(rows * nseg));
    auto go = [&](auto kernel) { kernel<<<grid, ST, 0, s>>>(a, nseg, seg_chunks, arrivals, records, row0); };
    if (a.entropy)
      a.n_top > 0 ? go(k_score<BF16, true, true>) : go(k_score<BF16, true, false>);
    else
      a.n_top > 0 ? go(k_score<BF16, false, true>) : go(k_score<BF16, false, false>);
    row0 += rows;
  }
}

void launch_score(const ScoreArgs &a, Dtype dt, void *ws, hipStream_t s) {
  if (dt == DT_BF16)
    score_launch<true>(a, ws, s);
  else
    score_launch<false>(a, ws, s);
}

template <bool BF16>
static void grad_launch(const ScoreArgs &a, hipStream_t s) {
  const int chunks = chunks_of<BF16>(a.vocab);
  /* a segment is two rounds of the workgroup's GU chunks a lane (bf16 [2048, 151936]:
   * 228 us; one 241, four 258, twenty 273), less when there would be fewer than
   * four workgroups a CU ([64, 151936] 9.9 us, 12.8 with sixteen a CU; 1000 rows of
   * 32000 25 and 30.5) */
  const int64_t room = (4 * CUS + a.n_rows - 1) / a.n_rows;
  int64_t nseg = (chunks + 2 * GU * ST - 1) / (2 * GU * ST);
  const int64_t least = (chunks + ST - 1) / ST;
  if (nseg < room) nseg = room < least ? room : least;
  const int seg_chunks = (int)((chunks + nseg - 1) / nseg);
  for (int row0 = 0; row0 < a.n_rows;) {
    const int rows = min(a.n_rows - row0, GRID_MOST / (int)nseg);
    k_score_grad<BF16><<<dim3((unsigned)(rows * nseg)), ST, 0, s>>>(a, (int)nseg, seg_chunks, row0);
    row0 += rows;
  }
}

void launch_score_backward(const ScoreArgs &a, Dtype dt, hipStream_t s) {
  if (dt == DT_BF16)
    grad_launch<true>(a, s);
  else
    grad_launch<false>(a, s);
}

}  // namespace d3s
