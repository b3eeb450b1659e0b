/* k_embed, k_embed_group, k_embed_sum: the rows that ids stand for, and their
 * gradient in the table (gfx950, wave64; include/d3s_step.h).
 *
 * The lookup is bound by HBM, or by what the caches give where rows come again: 8192 tokens of 2048
 * bf16 10.2 us; 4096 frames of ten codes 28 us (6.7 TB/s of the ten rows each); one frame 3.7 us, a launch
 * and two dependent loads.
 * The gradient is bound by the table's writes: 40970 x 2048 fp32 from 40960 codes 79 us (9 of them
 * grouping), 151936 x 1024 bf16 from 16384 tokens 69 us (12 grouping); many ids of few rows by
 * the chains of the frequent rows and their range's grouping (200000 of 512 bf16 119 us). */
#include "d3s_rowcore.h"
#include "d3s_step_internal.h"
#include "d3s_vec.h"

namespace d3s {
namespace {

constexpr int ET = 256;

/* A thread E columns of a row, its ids' rows loaded together (UN at a time).  Rows' chunks are counted
 * through (8192 tokens of 2049 bf16 11.9 us, of 100000 of 129 10.7; a power of two of lanes for each row 18.2
 * and 16.0).  The gradient's rows are not: 151936 x 1025 bf16 take 105 us that way, 90 by lanes. */
template <bool TB, bool YB, int UN>
__global__ __launch_bounds__(ET) void k_embed(EmbedArgs a, Spread c) {
  constexpr int E = YB ? 8 : 4;
  for (int64_t blk = blockIdx.x; blk < c.blocks; blk += gridDim.x) {
    int64_t row, chunk;
    c.find<ET>(blk, &row, &chunk);
    const int64_t j = chunk * E;
    if (row >= a.n_rows) continue;
    const int64_t left = a.width - j;
    const int32_t *ids = a.ids + row * a.n_ids;
    float v[E];
#pragma unroll
    for (int e = 0; e < E; e++) v[e] = 0.0f;
    for (int t = 0; t < a.n_ids; t += UN) {
      int id[UN];
      Vec<TB, E> q[UN];
#pragma unroll
      for (int u = 0; u < UN; u++) id[u] = t + u < a.n_ids ? ids[t + u] : -1;
#pragma unroll
      for (int u = 0; u < UN; u++) {
        const bool live = (uint32_t)id[u] < (uint64_t)a.vocab;
        q[u].load_some((const char *)a.in + ((t + u) * a.slot_rows + (live ? id[u] : 0)) * a.in_stride * (TB ? 2 : 4), j, live ? left : 0);
      }
#pragma unroll
      for (int u = 0; u < UN; u++) {
        float w[E];
        q[u].values(w);
#pragma unroll
        for (int e = 0; e < E; e++) v[e] += w[e];
      }
    }
#pragma unroll
    for (int e = 0; e < E; e++) v[e] *= a.scale;
    store_row<YB, E>((char *)a.out + row * a.out_stride * (YB ? 2 : 4), j, left, v);
  }
}

/* ---- the gradient ----
 * k_embed_group: a workgroup takes a range of the table's rows, looks through all ids (of its
 * slot) and writes the positions of its rows' ids, grouped by row and in their order:
 * the positions follow each other in `order` behind those of lower rows, which it counts
 * as it goes (a counter that each workgroup raises takes 23 ns a workgroup: 26 us for 1187), and seg
 * says for each row where and how many.
 * Many ids are parted first, by range, so that no workgroup looks through all of them (k_part_count,
 * k_part_scan, k_part_move: counts for each block of ids, their sums, the ids' places).
 * k_embed_sum: a row's positions are summed in that order, by lanes across its columns;
 * rows that no id names are filled with zeros.  A row of more than `hot` positions is cut into chunks
 * of twice as many or more, filed in a list; workgroups of their own sum the chunks in fp32, and the last
 * of a row to arrive adds its chunks in order.  No atomics on floating-point values. */

/* threads of k_embed_group: of parted ids more, for the range of the most frequent ones */
template <bool PARTED>
constexpr int group_threads() { return PARTED ? 1024 : 512; }
constexpr int LIST = 512;         /* positions that a wave keeps in LDS (more: the ids are looked through again) */
constexpr int AHEAD = 8;          /* ids that a lane looks at at a time */
constexpr int RANGE_MOST = 1024;  /* rows of the table that a workgroup takes: 32 or 64 KiB of counts */
constexpr int RANGE_LEAST = 4;    /* ... and at least, of parted ids (400000 ids of 300 rows: 222 us; 16 rows 298) */
/* workgroups for the chunks; of parted ids more (100000 ids of 1000 rows, 2048 columns: 146 us, with 512 320), since
 * they are not counted as they end, 23 ns each */
constexpr int HOT_GROUPS = 512;
constexpr int HOT_GROUPS_PARTED = 2048;
/* rows that are cut, at most: a counter of arrivals each (300000 ids of 5000 rows, 64 columns: 126 us; with 4096,
 * which leave rows of 128 ids whole, 226) */
constexpr int HOT_MOST = 32768;
constexpr int HOT_COUNTERS = 64;  /* words before them */

constexpr int PT = 1024;          /* threads of the parting kernels */
constexpr int PW = PT / WAVE;
constexpr int PART_IDS = 8;       /* ids a thread */
constexpr int PART_BLOCK = PT * PART_IDS;
constexpr int PARTS = 1024;       /* ranges that ids are parted into, at most */
/* fewer ids are not parted (40960 ids of 40970 rows: 79 us, parted 98; 20000 of 5000 32 and 42), but half as
 * many are where there are four or more a row, some of them perhaps most of all (50000 of 5000 rows, as often as
 * words in text: 43 us, not parted 116; evenly 38 and 34) */
constexpr int PART_LEAST = 65536;

struct Seg {
  int start, count; /* count < 0: cut into chunks */
};
struct Entry {
  int pos, row; /* the row of dy, the row within its range */
};
struct Chunk {
  int64_t row;
  int start, count, first, chunks, hot, pad; /* first: the row's first chunk */
};
/* chunks, rows cut, workgroups that have ended, and then the rows' arrivals: among the counters that the calls
 * leave at zero; of parted ids, whose first kernel clears them, behind those (no count of workgroups then) */
enum { CNT_CHUNKS = 0, CNT_HOT = 16, CNT_DONE = 32 };

struct GradPlan {
  int64_t slots, rows, n; /* parts of the table, rows in all, ids of each part */
  int range, hot;               /* rows of a range; a row of more positions is cut */
  int64_t ranges;               /* of each part */
  bool parted;
  int bits;                     /* range = 1 << bits */
  int blocks;                   /* of ids to part */
};
struct GradRoom {
  uint32_t *counters;
  Seg *seg;
  int *order;
  Chunk *chunks;
  float *sums; /* a chunk's, [.., width] */
  int *table;  /* [blocks, PARTS]: a block's ids of a range, then those of the blocks before */
  int *begin;  /* [PARTS + 1]: the ranges' first entries */
  Entry *entries;
};

GradPlan grad_plan(int64_t n_rows, int n_ids, int64_t vocab, int64_t slot_rows) {
  GradPlan p;
  p.slots = slot_rows ? n_ids : 1;
  p.rows = vocab + (n_ids - 1) * slot_rows;
  p.n = slot_rows ? n_rows : n_rows * n_ids;
  /* Ranges of 256 rows (16384 ids for 151936 rows: 12 us; 64 and 128 rows 21), wider while looking through the ids
   * for each would read more than 128 MB and there are more ranges than CUs. */
  p.range = 256;
  auto count = [&](int64_t r) { return (vocab + r - 1) / r; };
  while (p.range < RANGE_MOST && p.slots * count(p.range) > 512 && p.slots * count(p.range) * p.n > (int64_t)32 << 20) p.range *= 2;
  /* (ids that do not fit the parts' number are looked through) */
  const int64_t ids = p.n * p.slots;
  p.parted = (ids >= PART_LEAST || (ids >= PART_LEAST / 2 && ids >= 4 * p.rows)) && p.slots * count(RANGE_MOST) <= PARTS;
  if (p.parted)
    for (p.range = RANGE_LEAST; p.slots * count(p.range) > PARTS;) p.range *= 2;
  p.bits = 0;
  while ((1 << p.bits) < p.range) p.bits++;
  p.blocks = p.parted ? (int)((p.n * p.slots + PART_BLOCK - 1) / PART_BLOCK) : 0;
  p.ranges = count(p.range);
  p.hot = 32;
  while ((int64_t)p.hot * HOT_MOST < p.n * p.slots) p.hot *= 2;
  return p;
}
/* chunks at most: a row's one has hot + 1 positions at least, c >= 2 of them 2 hot (c - 1) + 1, which is
 * c (hot + 1 / 2) at least (rows of 2 hot + 1 have two) */
int64_t chunks_most(const GradPlan &p) { return 2 * p.n * p.slots / (2 * p.hot + 1) + 1; }

size_t grad_layout(const GradPlan &p, int64_t width, char *base, GradRoom *w) {
  size_t at = split_counter_bytes();
  auto take = [&](size_t bytes) {
    char *q = base + at;
    at += (bytes + 255) / 256 * 256;
    return q;
  };
  w->counters = (uint32_t *)base;
  w->seg = (Seg *)take((size_t)p.rows * sizeof(Seg));
  w->order = (int *)take((size_t)(p.n * p.slots) * sizeof(int));
  w->chunks = (Chunk *)take((size_t)chunks_most(p) * sizeof(Chunk));
  w->sums = (float *)take((size_t)chunks_most(p) * (size_t)((width + 7) / 8 * 8) * sizeof(float));
  w->table = (int *)take((size_t)p.blocks * PARTS * sizeof(int));
  w->begin = (int *)take(p.parted ? (PARTS + 1) * sizeof(int) : 0);
  if (p.parted) w->counters = (uint32_t *)take((HOT_COUNTERS + HOT_MOST) * sizeof(uint32_t));
  w->entries = (Entry *)take(p.parted ? (size_t)(p.n * p.slots) * sizeof(Entry) : 0);
  return at;
}

/* the range of id number `at`, or -1 */
__device__ __forceinline__ int part_of(const EmbedArgs &a, const GradPlan &p, int at, int id) {
  if ((uint32_t)id >= (uint64_t)a.vocab) return -1;
  return (p.slots > 1 ? at % a.n_ids * (int)p.ranges : 0) + (id >> p.bits);
}

__global__ __launch_bounds__(PT) void k_part_count(EmbedArgs a, GradPlan p, GradRoom w) {
  __shared__ int hist[PARTS];
  const int tid = (int)threadIdx.x, n = (int)(p.n * p.slots);
  if (tid < PARTS) hist[tid] = 0;
  for (int i = (int)blockIdx.x * PT + tid; i < HOT_COUNTERS + HOT_MOST; i += (int)gridDim.x * PT) w.counters[i] = 0u;
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * PART_BLOCK;
  for (int u = 0; u < PART_IDS; u++) {
    const int64_t at = first + u * PT + tid;
    const int r = at < n ? part_of(a, p, (int)at, a.ids[at]) : -1;
    if (r >= 0) atomicAdd(&hist[r], 1);
  }
  __syncthreads();
  if (tid < PARTS) w.table[(int64_t)blockIdx.x * PARTS + tid] = hist[tid];
}

/* a thread a range: its ids in the blocks before each, and the ranges' first places */
__global__ __launch_bounds__(PARTS) void k_part_scan(GradPlan p, GradRoom w) {
  __shared__ int wave_sum[PARTS / WAVE];
  const int r = (int)threadIdx.x;
  int sum = 0, b = 0;
  constexpr int UN = 8;
  for (; b + UN <= p.blocks; b += UN) {
    int c[UN];
#pragma unroll
    for (int u = 0; u < UN; u++) c[u] = w.table[(int64_t)(b + u) * PARTS + r];
#pragma unroll
    for (int u = 0; u < UN; u++) {
      w.table[(int64_t)(b + u) * PARTS + r] = sum;
      sum += c[u];
    }
  }
  for (; b < p.blocks; b++) {
    const int c = w.table[(int64_t)b * PARTS + r];
    w.table[(int64_t)b * PARTS + r] = sum;
    sum += c;
  }
  const int incl = (int)wave_scan_add_u32((uint32_t)sum);
  if (lane_id() == WAVE - 1) wave_sum[r / WAVE] = incl;
  __syncthreads();
  int before = 0;
  for (int g = 0; g < r / WAVE; g++) before += wave_sum[g];
  w.begin[r] = before + incl - sum;
  if (r == PARTS - 1) w.begin[PARTS] = before + incl;
}

/* lanes of one key (`bits` wide) among those of `hits` */
__device__ __forceinline__ uint64_t peers_of(int key, bool hit, uint64_t hits, int bits) {
  uint64_t peers = hits;
  for (int b = 0; b < bits; b++) {
    const uint64_t m = __ballot(hit && (key >> b & 1));
    peers &= key >> b & 1 ? m : ~m;
  }
  return peers;
}
__device__ __forceinline__ int lanes_below(uint64_t m) {
  return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u));
}

/* a block's ids to their ranges' places, in their order */
__global__ __launch_bounds__(PT) void k_part_move(EmbedArgs a, GradPlan p, GradRoom w) {
  __shared__ uint16_t cnt[PW][PARTS]; /* a wave's ids of a range, then those of the waves before (at most 8192) */
  __shared__ int base[PARTS];
  const int tid = (int)threadIdx.x, wid = tid / WAVE, n = (int)(p.n * p.slots);
  for (int i = tid; i < PW * PARTS / 2; i += PT) ((uint32_t *)cnt)[i] = 0u;
  if (tid < PARTS) base[tid] = w.begin[tid] + w.table[(int64_t)blockIdx.x * PARTS + tid];
  const int64_t first = (int64_t)blockIdx.x * PART_BLOCK + wid * (PART_IDS * WAVE) + lane_id();
  int id[PART_IDS], key[PART_IDS];
#pragma unroll
  for (int u = 0; u < PART_IDS; u++) {
    const int64_t at = first + u * WAVE;
    id[u] = at < n ? a.ids[at] : -1;
    key[u] = part_of(a, p, (int)at, id[u]);
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < PART_IDS; u++)
    if (key[u] >= 0) atomicAdd((uint32_t *)&cnt[wid][key[u] & ~1], 1u << 16 * (key[u] & 1));
  __syncthreads();
  if (tid < PARTS) {
    int sum = 0;
    for (int g = 0; g < PW; g++) {
      const int c = cnt[g][tid];
      cnt[g][tid] = (uint16_t)sum;
      sum += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < PART_IDS; u++) {
    const bool hit = key[u] >= 0;
    const uint64_t hits = __ballot(hit), peers = peers_of(key[u], hit, hits, 10);
    const int k = lanes_below(peers);
    int place = 0;
    if (hit) {
      place = cnt[wid][key[u]];
      w.entries[base[key[u]] + place + k] = Entry{(int)((uint32_t)(first + u * WAVE) / (uint32_t)a.n_ids), id[u] & (p.range - 1)};
    }
    wave_lds_sync();
    if (hit && (peers >> lane_id()) >> 1 == 0ull) cnt[wid][key[u]] = (uint16_t)(place + k + 1); /* the last of them */
    wave_lds_sync();
  }
}

template <bool PARTED>
__global__ __launch_bounds__(group_threads<PARTED>()) void k_embed_group(EmbedArgs a, GradPlan p, GradRoom w) {
  constexpr int GT = group_threads<PARTED>(), GW = GT / WAVE;
  extern __shared__ int cnt[]; /* [GW][range]: a wave's count of a row, then its place */
  __shared__ int list_pos[GW][PARTED ? 1 : LIST];
  __shared__ uint16_t list_row[GW][PARTED ? 1 : LIST];
  __shared__ int wave_sum[GW], wave_less[GW];
  const int tid = (int)threadIdx.x, wid = tid / WAVE, lane = lane_id();
  const int step = a.slot_rows ? a.n_ids : 1;                   /* (the last is below 2^31) */
  for (int64_t blk = blockIdx.x; blk < p.slots * p.ranges; blk += gridDim.x) {
    const int64_t slot = blk / p.ranges, v0 = blk % p.ranges * p.range;
    const uint32_t rows = (uint32_t)min((int64_t)p.range, a.vocab - v0);
    /* the wave's ids, of its slot's or of its range's entries */
    const int from = PARTED ? w.begin[blk] : 0, n = PARTED ? w.begin[blk + 1] - from : (int)p.n;
    const int each = (n / GW + WAVE) / WAVE * WAVE;
    const int i0 = min(n, wid * each), i1 = min(n, i0 + each);
    const int32_t *ids = a.slot_rows ? a.ids + slot : a.ids;
    for (int i = tid; i < GW * p.range; i += GT) cnt[i] = 0;
    __syncthreads();
    int *mine = cnt + wid * p.range;
    /* The wave's ids, AHEAD in a row for each lane: those of this range's rows go to its list, those of
     * lower rows are counted (an id below 0 is a row past 2^31 - v0 here).  Most of the kernel's time is this
     * chain; the code has to be short, since it is fetched while it runs (64 ids at a time by ballots,
     * unrolled 16, 32 and 64 times: 15, 26 and 71 us). */
    int less = 0, found = 0;
    int next[AHEAD]; /* (loaded while those before are looked at) */
    auto load = [&](int i) {
      const int at = i + lane * AHEAD;
      if (step == 1 && i1 - i >= AHEAD * WAVE) {
        __builtin_memcpy(next, ids + at, sizeof(next));
      } else if (i < i1) {
        const int32_t *q = ids + (uint32_t)at * (uint32_t)step;
#pragma unroll
        for (int e = 0; e < AHEAD; e++, q += step) next[e] = at + e < i1 ? *q : -1;
      }
    };
    if (!PARTED) load(i0);
    for (int i = i0; !PARTED && i < i1; i += AHEAD * WAVE) {
      const int at = i + lane * AHEAD;
      int id[AHEAD];
#pragma unroll
      for (int e = 0; e < AHEAD; e++) id[e] = next[e];
      load(i + AHEAD * WAVE);
      uint32_t hits = 0u;
#pragma unroll
      for (int e = 0; e < AHEAD; e++) {
        hits |= ((uint32_t)id[e] - (uint32_t)v0 < rows ? 1u : 0u) << e;
        less += (uint32_t)id[e] < (uint32_t)v0 ? 1 : 0;
      }
      if (__ballot(hits != 0u) == 0ull) continue;
      const int mine_here = __popc(hits), incl = (int)wave_scan_add_u32((uint32_t)mine_here);
      int k = found + incl - mine_here;
      found += (int)readlane_u((uint32_t)incl, WAVE - 1);
      for (; hits; hits &= hits - 1u, k++) { /* (loaded again: no register is found by a number) */
        const int e = at + __ffs(hits) - 1;
        if (k < LIST) list_pos[wid][k] = e, list_row[wid][k] = (uint16_t)((uint32_t)ids[(uint32_t)e * (uint32_t)step] - (uint32_t)v0);
      }
    }
    less = (int)wave_sum_u32((uint32_t)less);
    /* f(row of dy, row, whether it is this range's, which lanes' are) for them in their order: from the entries, from
     * the list, or where it does not hold them from the ids again; loads ahead */
    auto each_hit = [&](auto f) {
      if constexpr (PARTED) {
        const Entry *in = w.entries + from;
        constexpr int UN = 4;
        Entry now[UN], next[UN];
        auto get = [&](int e, Entry *q) {
#pragma unroll
          for (int u = 0; u < UN; u++) q[u] = in[min(e + u * WAVE + lane, i1 - 1)];
        };
        if (i0 < i1) get(i0, now);
        for (int e = i0; e < i1; e += UN * WAVE) {
          if (e + UN * WAVE < i1) get(e + UN * WAVE, next);
#pragma unroll
          for (int u = 0; u < UN; u++) {
            const bool hit = e + u * WAVE + lane < i1;
            const uint64_t hits = __ballot(hit);
            if (hits) f(now[u].pos, now[u].row, hit, hits);
          }
#pragma unroll
          for (int u = 0; u < UN; u++) now[u] = next[u];
        }
        return;
      }
      auto row_of = [&](int at) { return a.slot_rows ? at : at / a.n_ids; };
      if (found <= LIST) {
        for (int e = 0; e < found; e += WAVE) {
          const bool hit = e + lane < found;
          f(hit ? row_of(list_pos[wid][e + lane]) : 0, hit ? (int)list_row[wid][e + lane] : 0, hit, __ballot(hit));
        }
        return;
      }
      constexpr int UN = 4;
      for (int i = i0; i < i1; i += UN * WAVE) {
        uint32_t row[UN];
#pragma unroll
        for (int u = 0; u < UN; u++) {
          const int at = i + u * WAVE + lane;
          row[u] = at < i1 ? (uint32_t)ids[(uint32_t)at * (uint32_t)step] - (uint32_t)v0 : rows;
        }
#pragma unroll
        for (int u = 0; u < UN; u++) {
          const uint64_t hits = __ballot(row[u] < rows);
          if (hits) f(row_of(i + u * WAVE + lane), (int)row[u], row[u] < rows, hits);
        }
      }
    };
    each_hit([&](int, int row, bool hit, uint64_t hits) {
      if constexpr (PARTED) { /* (a frequent row's lanes would all add to one place) */
        const uint64_t peers = peers_of(row, hit, hits, p.bits);
        if (hit && lanes_below(peers) == 0) atomicAdd(&mine[row], __popcll(peers));
      } else if (hit) {
        atomicAdd(&mine[row], 1);
      }
    });
    __syncthreads();
    /* the rows' places: a thread `per` rows in a row */
    const int per = (p.range + GT - 1) / GT, r0 = min(p.range, tid * per), r1 = min(p.range, r0 + per);
    int total = 0;
    for (int r = r0; r < r1; r++)
      for (int g = 0; g < GW; g++) total += cnt[g * p.range + r];
    const int incl = (int)wave_scan_add_u32((uint32_t)total);
    if (lane == WAVE - 1) wave_sum[wid] = incl, wave_less[wid] = less;
    __syncthreads();
    int start = (PARTED ? from : (int)(slot * p.n)) + incl - total;
    for (int g = 0; g < GW; g++) start += (PARTED ? 0 : wave_less[g]) + (g < wid ? wave_sum[g] : 0);
    for (int r = r0; r < r1 && (uint32_t)r < rows; r++) {
      const int at = start;
      for (int g = 0; g < GW; g++) {
        const int c = cnt[g * p.range + r];
        cnt[g * p.range + r] = start;
        start += c;
      }
      const int here = start - at;
      const int64_t row = slot * a.slot_rows + v0 + r;
      w.seg[row] = Seg{at, here > p.hot ? -here : here};
      if (here > p.hot) { /* chunks of 2 hot positions, or 64 of them */
        const int size = max(2 * p.hot, (here + 63) / 64), chunks = (here + size - 1) / size;
        const int hot = (int)atomicAdd(&w.counters[CNT_HOT], 1u), first = (int)atomicAdd(&w.counters[CNT_CHUNKS], (uint32_t)chunks);
        for (int c = 0; c < chunks; c++)
          w.chunks[first + c] = Chunk{row, at + c * size, min(size, here - c * size), first, chunks, hot, 0};
      }
    }
    __syncthreads();
    /* the positions: lanes of one row find each other by ballots of its bits */
    each_hit([&](int at, int row, bool hit, uint64_t hits) {
      const uint64_t peers = peers_of(row, hit, hits, p.bits);
      const int k = lanes_below(peers);
      int to = 0;
      if (hit) {
        to = mine[row] + k;
        w.order[to] = at;
      }
      wave_lds_sync();
      if (hit && (peers >> lane) >> 1 == 0ull) mine[row] = to + 1; /* the last of them */
      wave_lds_sync();
    });
    __syncthreads();
  }
}

/* the sum of n rows of dy, at the positions `at`, E columns from j on */
template <bool DB, int E, int UN>
__device__ __forceinline__ void add_rows(const EmbedArgs &a, const int *at, int n, int64_t j, int64_t left, float *v) {
  int k = 0;
  auto row = [&](int i) { return (const char *)a.in + (int64_t)at[i] * a.in_stride * (DB ? 2 : 4); };
  for (; k + UN <= n; k += UN) {
    Vec<DB, E> q[UN];
#pragma unroll
    for (int u = 0; u < UN; u++) q[u].load_some(row(k + u), j, left);
#pragma unroll
    for (int u = 0; u < UN; u++) {
      float d[E];
      q[u].values(d);
#pragma unroll
      for (int e = 0; e < E; e++) v[e] += d[e];
    }
  }
  for (; k < n; k++) {
    float d[E];
    load_row<DB, E>(row(k), j, left, d);
#pragma unroll
    for (int e = 0; e < E; e++) v[e] += d[e];
  }
}

template <bool GB, int E>
__device__ __forceinline__ void put_row(const EmbedArgs &a, int64_t row, int64_t j, int64_t left, float *v) {
  char *out = (char *)a.out + row * a.out_stride * (GB ? 2 : 4);
#pragma unroll
  for (int e = 0; e < E; e++) v[e] *= a.scale;
  if (a.accumulate) {
    float o[E];
    load_row<GB, E>(out, j, left, o);
#pragma unroll
    for (int e = 0; e < E; e++) v[e] += o[e];
  }
  store_row<GB, E>(out, j, left, v);
}

/* SUM_ROWS rows that a thread takes one after the other: a workgroup writes 16 KiB.  (40970 rows of 2048 fp32, the whole
 * gradient: 82 us; two rows 88, one 104.  151936 of 1024 bf16: 79; two rows 81, eight 80.  Through the caches 100 and
 * 144.  A strip of columns for each XCD, so that dy stays in its L2: 84 and more.  Rows without ids filled
 * by k_embed_group instead: 105 and 101.) */
constexpr int FEW_IDS = 4;
/* One row where there are two ids or more a row (300000 ids of 5000 rows: 90 us, four rows 126; of
 * fewer, 200000 for 151936, 165 and 150). */
constexpr int MANY_IDS = 1;
/* (six and eight waves a SIMD: with the registers that the chunks would take, 88 and 84 us, so 78 and 76) */

template <bool DB, bool GB, int SUM_ROWS>
__global__ __launch_bounds__(ET, GB ? 6 : 8) void k_embed_sum(EmbedArgs a, GradPlan p, GradRoom w, int lanes, int64_t strips, int64_t blocks,
                                                  int hot_groups) {
  constexpr int E = GB ? 8 : 4;
  const int tid = (int)threadIdx.x;
  const int across = tid % lanes, down = tid / lanes, at_once = ET / lanes;
  if ((int)blockIdx.x < hot_groups) { /* chunks of rows that are cut, a strip of columns at a time */
    __shared__ uint32_t last;
    __shared__ float part[ET * E];
    const int64_t stride = (a.width + 7) / 8 * 8;
    const int64_t chunks = (int64_t)__hip_atomic_load(w.counters + CNT_CHUNKS, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    /* the groups' values added in their order, in the first */
    auto add_groups = [&](float *v) {
      if (at_once == 1) return;
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E; e++) part[tid * E + e] = v[e];
      __syncthreads();
      if (down != 0) return;
      for (int g = 1; g < at_once; g++)
#pragma unroll
        for (int e = 0; e < E; e++) v[e] += part[(g * lanes + across) * E + e];
    };
    for (int64_t c = blockIdx.x; c < chunks * strips; c += hot_groups) {
      const Chunk k = w.chunks[c / strips];
      const int64_t j = (c % strips * lanes + across) * E;
      /* each group of lanes a run of the positions, then the groups in order */
      const int run = (k.count + at_once - 1) / at_once, e0 = min(k.count, down * run), e1 = min(k.count, e0 + run);
      float v[E];
#pragma unroll
      for (int e = 0; e < E; e++) v[e] = 0.0f;
      if (j < a.width) add_rows<DB, E, DB ? 8 : 4>(a, w.order + k.start + e0, e1 - e0, j, a.width - j, v);
      add_groups(v);
      if (down == 0 && j < a.width) {
        uint64_t *out = (uint64_t *)(w.sums + c / strips * stride + j);
#pragma unroll
        for (int e = 0; e < E / 2; e++) st_agent(out + e, (uint64_t)d3s_f2u(v[2 * e]) | (uint64_t)d3s_f2u(v[2 * e + 1]) << 32);
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (tid == 0) {
        uint32_t *cnt = w.counters + HOT_COUNTERS + k.hot;
        last = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)(k.chunks * strips - 1);
        if (last) __hip_atomic_store(cnt, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      __syncthreads();
      if (last) {
        /* the same for the chunks' sums */
        const int each = (k.chunks + at_once - 1) / at_once, g0 = min(k.chunks, down * each), g1 = min(k.chunks, g0 + each);
        for (int64_t t = 0; t < strips; t++) {
          const int64_t i = (t * lanes + across) * E;
#pragma unroll
          for (int e = 0; e < E; e++) v[e] = 0.0f;
          if (i < a.width) {
#pragma unroll 4
            for (int g = g0; g < g1; g++) {
              const uint64_t *in = (const uint64_t *)(w.sums + (k.first + g) * stride + i);
#pragma unroll
              for (int e = 0; e < E / 2; e++) {
                const uint64_t q = ld_agent(in + e);
                v[2 * e] += d3s_u2f((uint32_t)q);
                v[2 * e + 1] += d3s_u2f((uint32_t)(q >> 32));
              }
            }
          }
          add_groups(v);
          if (down == 0 && i < a.width) put_row<GB, E>(a, k.row, i, a.width - i, v);
        }
      }
      __syncthreads();
    }
    /* the last to end clears what k_embed_group counted */
    if (!p.parted && tid == 0 && __hip_atomic_fetch_add(w.counters + CNT_DONE, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)(hot_groups - 1)) {
      for (int c : {CNT_CHUNKS, CNT_HOT, CNT_DONE})
        __hip_atomic_store(w.counters + c, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    return;
  }
  for (int64_t blk = blockIdx.x - hot_groups; blk < blocks; blk += gridDim.x - hot_groups) {
    const int64_t row0 = blk / strips * (at_once * SUM_ROWS) + down;
    const int64_t j = (blk % strips * lanes + across) * E;
    if (j >= a.width) continue;
    Seg seg[SUM_ROWS];
#pragma unroll
    for (int i = 0; i < SUM_ROWS; i++) {
      const int64_t row = row0 + i * at_once;
      const bool named = row < p.rows && (a.slot_rows == a.vocab || a.slot_rows == 0 || row % a.slot_rows < a.vocab);
      seg[i] = named ? w.seg[row] : Seg{0, 0};
    }
#pragma unroll
    for (int i = 0; i < SUM_ROWS; i++) {
      const int64_t row = row0 + i * at_once;
      if (row >= p.rows || seg[i].count < 0 || (a.accumulate && seg[i].count == 0)) continue;
      float v[E];
#pragma unroll
      for (int e = 0; e < E; e++) v[e] = 0.0f;
      add_rows<DB, E, 4>(a, w.order + seg[i].start, seg[i].count, j, a.width - j, v);
      put_row<GB, E>(a, row, j, a.width - j, v);
    }
  }
}

/* the table's gradient where there are no ids */
template <bool GB>
__global__ __launch_bounds__(ET) void k_embed_zero(EmbedArgs a, int64_t rows, int64_t strips) {
  constexpr int E = GB ? 8 : 4;
  const float zero[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  for (int64_t blk = blockIdx.x; blk < rows * strips; blk += gridDim.x) {
    const int64_t j = (blk % strips * ET + threadIdx.x) * E;
    if (j < a.width) store_row<GB, E>((char *)a.out + blk / strips * a.out_stride * (GB ? 2 : 4), j, a.width - j, zero);
  }
}

}  // namespace

void launch_embed(const EmbedArgs &args, Dtype in, Dtype out, hipStream_t s) {
  const EmbedArgs a = args;
  const Spread c = Spread::of<ET>(a.n_rows, a.width, out == DT_BF16 ? 8 : 4);
  const dim3 grid((unsigned)(c.blocks < STEP_GRID ? c.blocks : STEP_GRID));
  auto go = [&](auto kernel) { kernel<<<grid, ET, 0, s>>>(a, c); };
  auto many = [&](auto tb, auto yb) {
    constexpr bool T = decltype(tb)::value, Y = decltype(yb)::value;
    a.n_ids == 1 ? go(k_embed<T, Y, 1>) : go(k_embed<T, Y, 4>);
  };
  if (in == DT_BF16)
    out == DT_BF16 ? many(std::true_type{}, std::true_type{}) : many(std::true_type{}, std::false_type{});
  else
    out == DT_BF16 ? many(std::false_type{}, std::true_type{}) : many(std::false_type{}, std::false_type{});
}

size_t embed_grad_workspace_bytes(int64_t n_rows, int n_ids, int64_t vocab, int64_t slot_rows, int64_t width) {
  if (n_rows == 0 || width == 0) return 0;
  GradRoom w;
  return grad_layout(grad_plan(n_rows, n_ids, vocab, slot_rows), width, nullptr, &w);
}

void launch_embed_grad(const EmbedArgs &args, Dtype in, Dtype out, void *ws, hipStream_t s) {
  const EmbedArgs a = args;
  auto grid = [](int64_t n) { return dim3((unsigned)(n < STEP_GRID ? n : STEP_GRID)); };
  const GradPlan p = grad_plan(a.n_rows, a.n_ids, a.vocab, a.slot_rows);
  const int E = out == DT_BF16 ? 8 : 4;
  if (a.n_rows == 0) {
    const int64_t strips = (a.width + ET * E - 1) / (ET * E);
    if (out == DT_BF16)
      k_embed_zero<true><<<grid(p.rows * strips), ET, 0, s>>>(a, p.rows, strips);
    else
      k_embed_zero<false><<<grid(p.rows * strips), ET, 0, s>>>(a, p.rows, strips);
    return;
  }
  GradRoom w;
  grad_layout(p, a.width, (char *)ws, &w);
  auto counts = [&](int threads) { return threads / WAVE * p.range * sizeof(int); };
  if (p.parted) {
    k_part_count<<<dim3((unsigned)p.blocks), PT, 0, s>>>(a, p, w);
    k_part_scan<<<1, PARTS, 0, s>>>(p, w);
    k_part_move<<<dim3((unsigned)p.blocks), PT, 0, s>>>(a, p, w);
    k_embed_group<true><<<grid(p.slots * p.ranges), group_threads<true>(), counts(group_threads<true>()), s>>>(a, p, w);
  } else {
    k_embed_group<false><<<grid(p.slots * p.ranges), group_threads<false>(), counts(group_threads<false>()), s>>>(a, p, w);
  }
  int lanes = 1;
  while (lanes < ET && (int64_t)lanes * E < a.width) lanes *= 2;
  const int together = p.n * p.slots >= 2 * p.rows ? MANY_IDS : FEW_IDS;
  const int64_t strips = (a.width + lanes * E - 1) / (lanes * E), rows = ET / lanes * together;
  const int64_t blocks = strips * ((p.rows + rows - 1) / rows);
  const int64_t most = chunks_most(p);
  const int at_most = p.parted ? HOT_GROUPS_PARTED : HOT_GROUPS, hot_groups = (int)(most < at_most ? most : at_most);
  auto go = [&](auto kernel) {
    kernel<<<dim3((unsigned)(hot_groups + (blocks < STEP_GRID ? blocks : STEP_GRID))), ET, 0, s>>>(a, p, w, lanes, strips, blocks, hot_groups);
  };
  auto typed = [&](auto db, auto gb) {
    constexpr bool D = decltype(db)::value, G = decltype(gb)::value;
    together == MANY_IDS ? go(k_embed_sum<D, G, MANY_IDS>) : go(k_embed_sum<D, G, FEW_IDS>);
  };
  if (in == DT_BF16)
    out == DT_BF16 ? typed(std::true_type{}, std::true_type{}) : typed(std::true_type{}, std::false_type{});
  else
    out == DT_BF16 ? typed(std::false_type{}, std::true_type{}) : typed(std::false_type{}, std::false_type{});
}

}  // namespace d3s
