// Token rows to their experts and back, for expert products outside this library, and the gradients of
// both. With row(t, j) the permuted row of pair (t, j) (wm_permute's inverse, -1 where the pair's id is
// no expert):
//   sort              rows[row(t, j)] = x[t]                    (rows behind the last pair: zero)
//   its gradient      dx[t] = sum_j drows[row(t, j)]
//   back              y[t] = add[t] + sum_j w[t, j] rows[row(t, j)]
//   its gradients     drows[row(t, j)] = w[t, j] dy[t],  dw[t, j] = dy[t] . rows[row(t, j)]
// (qwen4_exp.py:865-904: the gather, the inverse gather and the weighted sum of the reference's grouped
// experts; it has no gradients.)
//
// All four are bound by HBM and walk the tokens, not the permuted rows: a token's row is read or written
// once and its k permuted rows once each. Sums are fp32 in j order, so a result does not depend on the
// grid, and are rounded once. 4096 tokens x 8 of 7168 in bf16: the sort 102 us (529 MB, 5.2 TB/s), back 107 us
// (578 MB, 5.4 TB/s); 2048 x 6 of 5120 in fp32: the gradients of back 98 us (545 MB, 5.6 TB/s). Rows of 512 bytes and
// less are two to four times their bytes' time: neighbouring tokens write parts of one 128-byte line, and the
// gradients of back leave most lanes of a wave without a unit.
#include "permute_device.h"
#include "row_units.h"

namespace wm {

constexpr int SORT_MAX_K = 64;

// How permuted rows are stored: through the 256 MB cache, past it, or the first `through` rows through it and the others
// past it. Their reader starts with the first; what a call leaves in the cache, the next work has to write back.
//
// Up to 192 MB all stay for the reader. Up to 256 MB the first 96 MB do. Call and a pass that reads its rows, behind a
// pass over other memory (in brackets one of many calls in a row), us, with none / 96 MB / all through:
//   sort       200 MB of 14 KB rows   131 (48)    121 (42)    94 (60)
//              240 MB of 20 KB        151 (57)    118 (57)   115 (65)
//              240 MB of 2002 bytes   212 (94)    188 (82)   171 (108)
//   gradients  200 MB of 14 KB        165 (87)    151 (74)   118 (95)
//              240 MB of 20 KB        198 (108)   164 (97)   151 (118)
//              240 MB of 2002 bytes   286 (170)   269 (170)  254 (174)
// Larger ones go past it: with 64 or 96 MB through, calls in a row of more than two sets of tensors evict each other's
// (sort of 470 MB 101 us, with 64 MB 119), and for the reader there is less to win:
//   sort       448 MB of 14 KB        244 (101)   242 (119)  246 (120)
//              640 MB of 20 KB        315 (142)   308 (168)  338 (167)
//   gradients  448 MB of 14 KB        333 (194)   324 (198)  315 (209)
//              640 MB of 20 KB        437 (268)   429 (284)  443 (292)
// Short rows that are no whole 128-byte lines always stay, since their lines are written in parts: 256 MB of 500-byte
// rows sorted and read 242, past the cache 265, their gradients 340 and 382; of 384 MB 384 and 393, 518 and 574.
enum RowStore { THROUGH, PAST, SPLIT };
struct RowStores {
  RowStore how;
  int64_t through;
};
static RowStores row_stores(int64_t pairs, int64_t row_bytes) {
  const int64_t bytes = pairs * row_bytes;
  if (bytes <= 192ll << 20 || (row_bytes <= 512 && row_bytes % 128 != 0)) return {THROUGH, pairs};
  if (bytes <= 256ll << 20) return {SPLIT, (96ll << 20) / row_bytes};
  return {PAST, 0};
}

// A unit of a permuted row; `past` where the call splits them. The empty statements keep the two stores apart, of
// which the compiler would make one that goes through the cache.
template <typename Unit, int STORE>
__device__ __forceinline__ void store_row_unit(typename Unit::Elem* p, typename Unit::Raw v, bool past) {
  if (STORE == PAST) {
    Unit::store_once(p, v);
  } else if (STORE == SPLIT && past) {
    asm volatile("");
    Unit::store_once(p, v);
    asm volatile("");
  } else {
    Unit::store(p, v);
  }
}

// ---- sort. A workgroup owns a chunk of tokens (256 pairs at most) and a range of units. It finds its
// pairs' rows in LDS, and moves the tokens' units to them. Three ways to the rows, by the number of pairs:
//   up to 256     (sort_few_kernel) a workgroup a token; each has all ids in LDS and counts, for each of its
//                 pairs, the pairs before it in expert order. The token's units are on their way meanwhile.
//   up to 16384   (sort_kernel) every workgroup counts all pairs by expert, those before its chunk apart, so it
//                 knows the first row of each expert for this chunk; a pair's row is that plus its place
//                 among the chunk's earlier pairs of its expert. One launch and no workspace, the counting
//                 repeated by every workgroup.
//   more          a launch before counts the pairs of spans (sort_spans_kernel); a workgroup adds up the spans'
//                 counts and counts only the pairs of its own span before its chunk. Past 64 spans of 8192 pairs
//                 a second launch adds them up for all (sort_bases_kernel), so that a workgroup's counting has
//                 an end however many pairs there are.
// Each has one workgroup more, for the lists that belong to no pair.
constexpr int SORT_THREADS = 512;
constexpr int SORT_CHUNK = 256;

struct SortArgs {
  const void* x;
  const int32_t* indices;
  int64_t tokens, length;  // a row's length in 2-byte elements: rows are moved, whatever they hold
  RowUnits row;
  int k, experts, tile_rows;
  int chunk_tokens, split_units;
  void* rows;
  int32_t *order, *inverse, *offsets, *tiles, *tile_count;
  int64_t max_tiles;
  int64_t through;             // of SPLIT
  const int32_t* span_counts;  // [spans][experts], null where there is one span
  const int32_t* totals;       // [experts], where span_counts are those of the spans before; else null
  int64_t span_pairs;
  int spans;
};

// Exclusive prefix sums over the workgroup's threads, and the total. Every thread calls it.
__device__ __forceinline__ int32_t sort_scan(int32_t v, int32_t* total) {
  __shared__ int32_t wave_sum[SORT_THREADS / 64];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  int32_t incl = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int32_t o = __shfl_up(incl, d, 64);
    if (lane >= d) incl += o;
  }
  if (lane == 63) wave_sum[wave] = incl;
  __syncthreads();
  int32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < SORT_THREADS / 64; ++w) {
    before += w < wave ? wave_sum[w] : 0;
    all += wave_sum[w];
  }
  __syncthreads();  // wave_sum is free again
  *total = all;
  return before + incl - v;
}

// Adds the pairs q0 .. q1 by expert: before p0 to `before`, from p0 on to `later` (null: nowhere). Every thread
// calls it, between barriers.
__device__ __forceinline__ void sort_count(const SortArgs& a, int64_t q0, int64_t q1, int64_t p0, int32_t* before,
                                           int32_t* later) {
  // 16 ids in flight a thread, by 16 bytes at any alignment
  for (int64_t q = q0 + 4 * threadIdx.x; q < q1; q += 16 * SORT_THREADS) {
    int32_t e[4][4];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int64_t at = q + b * 4 * SORT_THREADS;
      if (at + 4 <= q1) {
        const wm_u32x4 v = load16(a.indices + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) e[b][i] = (int32_t)v[i];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) e[b][i] = at + i < q1 ? a.indices[at + i] : -1;
      }
    }
#pragma unroll
    for (int b = 0; b < 4; ++b) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        int32_t* to = q + b * 4 * SORT_THREADS + i < p0 ? before : later;
        if ((uint32_t)e[b][i] < (uint32_t)a.experts && to) atomicAdd(&to[e[b][i]], 1);
      }
    }
  }
}

// The pairs of every expert before p0 and in all (`before`, `all`: an entry an expert). Every thread calls it;
// ends with a barrier.
__device__ __forceinline__ void sort_counts(const SortArgs& a, int64_t p0, int32_t* before, int32_t* all) {
  const int E = a.experts;
  if (a.totals) {
    const int64_t span = p0 / a.span_pairs;
    for (int e = threadIdx.x; e < E; e += SORT_THREADS) before[e] = a.span_counts[span * E + e], all[e] = a.totals[e];
    __syncthreads();
    sort_count(a, span * a.span_pairs, p0, p0, before, nullptr);
    __syncthreads();
    return;
  }
  for (int e = threadIdx.x; e < E; e += SORT_THREADS) before[e] = all[e] = 0;
  __syncthreads();
  if (!a.span_counts) {
    sort_count(a, 0, a.tokens * a.k, p0, before, all);
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += SORT_THREADS) all[e] += before[e];
  } else {
    const int span = (int)(p0 / a.span_pairs), n = a.spans * E;
    constexpr int BATCH = 8;
    for (int i0 = threadIdx.x; i0 < n; i0 += BATCH * SORT_THREADS) {
      int32_t v[BATCH];
#pragma unroll
      for (int b = 0; b < BATCH; ++b) v[b] = i0 + b * SORT_THREADS < n ? a.span_counts[i0 + b * SORT_THREADS] : 0;
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        const int i = i0 + b * SORT_THREADS, e = i % E;
        if (v[b]) {
          atomicAdd(&all[e], v[b]);
          if (i / E < span) atomicAdd(&before[e], v[b]);
        }
      }
    }
    sort_count(a, span * a.span_pairs, p0, p0, before, nullptr);
  }
  __syncthreads();
}

__global__ void __launch_bounds__(SORT_THREADS) sort_spans_kernel(SortArgs a, int32_t* __restrict__ counts) {
  __shared__ int32_t count[PERMUTE_MAX_EXPERTS];
  for (int e = threadIdx.x; e < a.experts; e += SORT_THREADS) count[e] = 0;
  __syncthreads();
  const int64_t q0 = blockIdx.x * a.span_pairs, q1 = min(a.tokens * a.k, q0 + a.span_pairs);
  sort_count(a, q0, q1, q1, count, nullptr);
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += SORT_THREADS) counts[(int64_t)blockIdx.x * a.experts + e] = count[e];
}

// The spans' counts [spans][experts] become those of the spans before, and the row behind them the totals. A lane has an
// expert, the waves slices of the spans in order; 64 experts a workgroup.
constexpr int BASES_WAVES = 16;
__global__ void __launch_bounds__(64 * BASES_WAVES) sort_bases_kernel(int32_t* counts, int spans, int experts) {
  __shared__ int32_t slice_sum[BASES_WAVES][64];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, e = blockIdx.x * 64 + lane;
  const int per = (spans + BASES_WAVES - 1) / BASES_WAVES;
  const int64_t s0 = min((int64_t)spans, (int64_t)wave * per), s1 = min((int64_t)spans, s0 + per);
  int32_t sum = 0;
  if (e < experts) {
#pragma unroll 8
    for (int64_t s = s0; s < s1; ++s) sum += counts[s * experts + e];
  }
  slice_sum[wave][lane] = sum;
  __syncthreads();
  int32_t at = 0;
  for (int w = 0; w < wave; ++w) at += slice_sum[w][lane];
  if (e >= experts) return;
  constexpr int BATCH = 8;  // loaded before any is written
  for (int64_t s = s0; s < s1; s += BATCH) {
    int32_t n[BATCH];
#pragma unroll
    for (int b = 0; b < BATCH; ++b) n[b] = s + b < s1 ? counts[(s + b) * experts + e] : 0;
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      if (s + b < s1) counts[(s + b) * experts + e] = at;
      at += n[b];
    }
  }
  if (wave == BASES_WAVES - 1) counts[(int64_t)spans * experts + e] = at;
}

// The lists that belong to no pair: offsets, tiles, their number. One workgroup; count and first are LDS of an
// entry an expert.
__device__ __forceinline__ void sort_lists(const SortArgs& a, int32_t* count, int32_t* first) {
  __shared__ int32_t tile_start[PERMUTE_MAX_EXPERTS];
  const int E = a.experts;
  sort_counts(a, 0, first, count);
  const int e0 = 2 * threadIdx.x, e1 = e0 + 1;  // two experts a thread
  const int32_t n0 = e0 < E ? count[e0] : 0, n1 = e1 < E ? count[e1] : 0;
  int32_t present, tiles;
  const int32_t row = sort_scan(n0 + n1, &present);
  const uint32_t per = a.tile_rows;  // the sums below pass 31 bits
  const int32_t t0 = (int32_t)((n0 + per - 1) / per), t1 = (int32_t)((n1 + per - 1) / per);
  const int32_t tile = sort_scan(t0 + t1, &tiles);
  if (e0 < E) a.offsets[e0] = first[e0] = row, tile_start[e0] = tile;
  if (e1 < E) a.offsets[e1] = first[e1] = row + n0, tile_start[e1] = tile + t0;
  if (threadIdx.x == 0) {
    a.offsets[E] = present;
    a.tile_count[0] = tiles;
  }
  __syncthreads();
  // Tile i belongs to the last expert whose first tile is <= i: experts without tiles share their start with
  // the next one that has some, and come before it.
  for (int64_t i = threadIdx.x; i < a.max_tiles; i += SORT_THREADS) {
    int2 t = make_int2(-1, -1);
    if (i < tiles) {
      int lo = 0, hi = E - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (tile_start[mid] <= i) lo = mid; else hi = mid - 1;
      }
      t = make_int2(lo, first[lo] + ((int32_t)i - tile_start[lo]) * a.tile_rows);
    }
    reinterpret_cast<int2*>(a.tiles)[i] = t;
  }
}

// One unit of a row: from x's element `at`, to the same place of a token's k rows.
template <typename Unit, int STORE>
__device__ __forceinline__ void sort_store(const SortArgs& a, int64_t at, const int32_t* row, typename Unit::Raw v) {
  uint16_t* rows = (uint16_t*)a.rows;
#pragma unroll 4
  for (int j = 0; j < a.k; ++j)
    if (row[j] >= 0) store_row_unit<Unit, STORE>(rows + row[j] * a.length + at, v, row[j] >= a.through);
}

// Zeros in the rows from `present` on, every step-th from the me-th, units c0 .. c1.
__device__ __forceinline__ void sort_clear(const SortArgs& a, int32_t present, int64_t me, int64_t step, int c0, int c1) {
  uint16_t* rows = (uint16_t*)a.rows;
  for (int64_t r = present + me; r < a.tokens * a.k; r += step) {
    for (int c = c0 + threadIdx.x; c < c1; c += SORT_THREADS) {
      if (c < a.row.wide) store16_nt(rows + r * a.length + 8 * (int64_t)c, wm_u32x4{0, 0, 0, 0});
      else rows[r * a.length + 8 * (int64_t)a.row.wide + c - a.row.wide] = 0;
    }
  }
}

// A workgroup a token, and the last one for the lists; columns by SORT_THREADS units.
__global__ void __launch_bounds__(SORT_THREADS) sort_few_kernel(SortArgs a) {
  __shared__ int32_t scratch[2][PERMUTE_MAX_EXPERTS];
  __shared__ int32_t row[SORT_MAX_K], present_;
  if (blockIdx.x == a.tokens) {
    if (blockIdx.y == 0) sort_lists(a, scratch[0], scratch[1]);
    return;
  }
  int32_t* key = scratch[0];
  const int t = blockIdx.x, pairs = (int)a.tokens * a.k, p0 = t * a.k;
  const int c = blockIdx.y * SORT_THREADS + threadIdx.x;
  if ((int)threadIdx.x < pairs) {
    const int32_t e = a.indices[threadIdx.x];
    key[threadIdx.x] = (uint32_t)e < (uint32_t)a.experts ? e : 0x7fffffff;
  }
  const uint16_t* x = (const uint16_t*)a.x + t * a.length;
  const int64_t at = c < a.row.wide ? 8 * (int64_t)c : 8 * (int64_t)a.row.wide + c - a.row.wide;
  wm_u32x4 v = {0, 0, 0, 0};
  uint16_t one = 0;
  if (c < a.row.wide) v = load16(x + at);
  else if (c < a.row.units) one = x[at];
  __syncthreads();
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  for (int j = wave; j < a.k + 1; j += SORT_THREADS / 64) {  // the last one counts the pairs that are there
    const int p = p0 + j;
    const int32_t e = j < a.k ? key[p] : 0x7fffffff;
    int32_t before = 0;
    for (int q0 = 0; q0 < pairs; q0 += 64) {
      const int q = q0 + lane;
      before += __popcll(__ballot(q < pairs && (key[q] < e || (j < a.k && key[q] == e && q < p))));
    }
    if (lane == 0) {
      if (j == a.k) {
        present_ = before;
      } else {
        const int32_t r = e == 0x7fffffff ? -1 : before;
        row[j] = r;
        if (blockIdx.y == 0) {
          a.inverse[p] = r;
          if (r >= 0) a.order[r] = p;
        }
      }
    }
  }
  __syncthreads();
  const int32_t present = present_;
  if (blockIdx.y == 0 && (int)threadIdx.x < a.k && p0 + (int)threadIdx.x >= present) a.order[p0 + threadIdx.x] = -1;
  if (c < a.row.wide) sort_store<RowUnit<false, true>, THROUGH>(a, at, row, v);
  else if (c < a.row.units) sort_store<RowUnit<false, false>, THROUGH>(a, at, row, one);
  const int c0 = blockIdx.y * SORT_THREADS;
  sort_clear(a, present, t, a.tokens, c0, min(a.row.units, c0 + SORT_THREADS));
}

template <int STORE>
__global__ void __launch_bounds__(SORT_THREADS) sort_kernel(SortArgs a) {
  // base: the chunk's first row of each expert
  __shared__ int32_t base[PERMUTE_MAX_EXPERTS], all[PERMUTE_MAX_EXPERTS];
  __shared__ __align__(16) int32_t key[SORT_CHUNK];
  __shared__ int32_t row[SORT_CHUNK];
  const int64_t t0 = (int64_t)blockIdx.x * a.chunk_tokens;
  const int64_t p0 = t0 * a.k;
  if (t0 >= a.tokens) {
    if (blockIdx.y == 0) sort_lists(a, base, all);
    return;
  }
  const int tokens = (int)min((int64_t)a.chunk_tokens, a.tokens - t0);
  const int n = tokens * a.k;
  const int E = a.experts;
  if (threadIdx.x < n) {
    const int32_t e = a.indices[p0 + threadIdx.x];
    key[threadIdx.x] = (uint32_t)e < (uint32_t)E ? e : -1;
  }
  sort_counts(a, p0, base, all);
  const int e0 = 2 * threadIdx.x, e1 = e0 + 1;  // two experts a thread
  const int32_t n0 = e0 < E ? all[e0] : 0, n1 = e1 < E ? all[e1] : 0;
  int32_t present;
  const int32_t first = sort_scan(n0 + n1, &present);
  if (e0 < E) base[e0] += first;
  if (e1 < E) base[e1] += first + n0;
  __syncthreads();
  if (threadIdx.x < SORT_CHUNK) {  // whole waves: ballots
    const bool in_range = threadIdx.x < n;
    const int32_t e = in_range ? key[threadIdx.x] : -1;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int bits = 32 - __clz(E);
    uint64_t peers = __ballot(e >= 0);  // the wave's pairs of the same expert
    for (int bit = 0; bit < bits; ++bit) {
      const uint64_t set = __ballot((e >> bit) & 1);
      peers &= ((e >> bit) & 1) ? set : ~set;
    }
    int32_t r = __popcll(peers & (lane == 0 ? 0ull : ~0ull >> (64 - lane)));
    const int4* earlier = reinterpret_cast<const int4*>(key);
#pragma unroll 4
    for (int j = 0; j < 16 * wave; ++j) {  // the pairs of the waves before, all of the chunk
      const int4 v = earlier[j];
      r += (v.x == e) + (v.y == e) + (v.z == e) + (v.w == e);
    }
    if (in_range) {
      if (e >= 0) r += base[e];
      else r = -1;
      row[threadIdx.x] = r;
      const int64_t p = p0 + threadIdx.x;
      if (blockIdx.y == 0) {
        a.inverse[p] = r;
        if (r >= 0) a.order[r] = (int32_t)p;
        if (p >= present) a.order[p] = -1;
      }
    }
  }
  __syncthreads();
  const uint16_t* x = (const uint16_t*)a.x;
  const int c0 = blockIdx.y * a.split_units, c1 = min(a.row.units, c0 + a.split_units);
  // Units of all the chunk's tokens one behind the other: no thread without one but at the end.
  const int width = c1 - c0;
  for (int i = threadIdx.x; i < tokens * width; i += SORT_THREADS) {
    const int t = (int)((uint32_t)i / (uint32_t)width), c = c0 + i - t * width;
    const uint16_t* from = x + (t0 + t) * a.length;
    const int64_t at = c < a.row.wide ? 8 * (int64_t)c : 8 * (int64_t)a.row.wide + c - a.row.wide;
    if (c < a.row.wide) sort_store<RowUnit<false, true>, STORE>(a, at, row + t * a.k, load16(from + at));
    else sort_store<RowUnit<false, false>, STORE>(a, at, row + t * a.k, from[at]);
  }
  // The rows behind the last pair, spread over the workgroups: the few that own the last pairs would take
  // twice as long (4096 tokens x 8, hidden 7168, 2% of the pairs absent: 112 us, spread 103).
  sort_clear(a, present, blockIdx.x, (a.tokens + a.chunk_tokens - 1) / a.chunk_tokens, c0, c1);
}

// Up to this many pairs each way is taken. 8 tokens x 10 of 2560, captured: a workgroup a token 4.3 us, the
// counting workgroups 7.3. Captured, 8 of 256 experts a token, some far busier than others, of 136 and of 1000 columns:
// 16384 pairs in one launch 10.4 and 14.1 us, with the spans' launch 11.6 and 16.4; 32768 pairs 14.7 and 23.3, with it
// 12.7 and 22.4 (evenly routed 11.5 and 21.4, with it 12.8 and 22.7).
constexpr int64_t SORT_FEW_MAX = 256, SORT_ONE_MAX = 16384;

// Spans that are counted apart: each a multiple of the chunk, of 2048 to 8192 pairs (and less than a chunk more).
// Up to SORT_SPANS_ADDED of them every workgroup adds up itself.
constexpr int SORT_SPANS_ADDED = 64;
struct SortSpans {
  int64_t pairs;
  int spans;
};
static int sort_chunk_tokens(int64_t tokens, int k) {
  const int most = SORT_CHUNK / k > 0 ? SORT_CHUNK / k : 1;
  const int64_t want = (tokens + 255) / 256;  // few tokens: a workgroup each
  return (int)(want < 1 ? 1 : want < most ? want : most);
}
static SortSpans sort_spans(int64_t tokens, int k) {
  const int64_t pairs = tokens * k, chunk = (int64_t)sort_chunk_tokens(tokens, k) * k;
  if (pairs <= SORT_ONE_MAX) return {pairs, 1};
  const int64_t part = (pairs + SORT_SPANS_ADDED - 1) / SORT_SPANS_ADDED;
  const int64_t least = part < 2048 ? 2048 : part > 8192 ? 8192 : part, span = (least + chunk - 1) / chunk * chunk;
  return {span, (int)((pairs + span - 1) / span)};
}

static void sort_launch(SortArgs a, int32_t* workspace, hipStream_t s) {
  const int64_t pairs = a.tokens * a.k;
  if (pairs <= SORT_FEW_MAX) {
    const dim3 grid((unsigned)a.tokens + 1, (unsigned)((a.row.units + SORT_THREADS - 1) / SORT_THREADS));
    hipLaunchKernelGGL(sort_few_kernel, grid, dim3(SORT_THREADS), 0, s, a);
    check_launch("sort_few");
    return;
  }
  const int64_t chunks = (a.tokens + a.chunk_tokens - 1) / a.chunk_tokens;
  const unsigned blocks = grid_of("sort", chunks + 1, SORT_THREADS);
  if (a.spans > 1) {
    hipLaunchKernelGGL(sort_spans_kernel, dim3(a.spans), dim3(SORT_THREADS), 0, s, a, workspace);
    check_launch("sort_spans");
    a.span_counts = workspace;
    if (a.spans > SORT_SPANS_ADDED) {
      hipLaunchKernelGGL(sort_bases_kernel, dim3((a.experts + 63) / 64), dim3(64 * BASES_WAVES), 0, s, workspace, a.spans, a.experts);
      check_launch("sort_bases");
      a.totals = workspace + (int64_t)a.spans * a.experts;
    }
  }
  // columns are split, by whole waves, until the chip has work for every CU
  const int64_t most = (a.row.units + 255) / 256;
  int64_t splits = chunks >= 512 ? 1 : (511 + chunks) / chunks;
  if (splits > most) splits = most;
  a.split_units = (int)(((a.row.units + splits - 1) / splits + 63) / 64 * 64);
  const dim3 grid(blocks, (unsigned)((a.row.units + a.split_units - 1) / a.split_units));
  const RowStores stores = row_stores(pairs, a.length * 2);
  a.through = stores.through;
  if (stores.how == THROUGH) hipLaunchKernelGGL(sort_kernel<THROUGH>, grid, dim3(SORT_THREADS), 0, s, a);
  else if (stores.how == PAST) hipLaunchKernelGGL(sort_kernel<PAST>, grid, dim3(SORT_THREADS), 0, s, a);
  else hipLaunchKernelGGL(sort_kernel<SPLIT>, grid, dim3(SORT_THREADS), 0, s, a);
  check_launch("sort");
}

// ---- back (WEIGHTED) and the sort's gradient: a thread owns one unit of a token, sums its k rows.
// A row is read once and not again, so past the cache.
constexpr int GATHER_BATCH = 8;  // rows in flight

template <typename U, bool WEIGHTED>
__device__ __forceinline__ void gather_unit(const typename U::Elem* __restrict__ rows, const float* __restrict__ weights,
                                            const int32_t* __restrict__ inverse, uint32_t pairs, int64_t hidden, int64_t t,
                                            int64_t at, int k, const typename U::Elem* add, typename U::Elem* y) {
  float acc[U::N] = {};
  for (int j0 = 0; j0 < k; j0 += GATHER_BATCH) {
    uint32_t r[GATHER_BATCH];
    typename U::Raw v[GATHER_BATCH];
#pragma unroll
    for (int q = 0; q < GATHER_BATCH; ++q) r[q] = j0 + q < k ? (uint32_t)inverse[t * k + j0 + q] : 0xffffffffu;
#pragma unroll
    for (int q = 0; q < GATHER_BATCH; ++q)
      if (r[q] < pairs) v[q] = U::load_once(rows + r[q] * hidden + at);
#pragma unroll
    for (int q = 0; q < GATHER_BATCH; ++q) {
      if (r[q] < pairs) {
        const float w = WEIGHTED ? weights[t * k + j0 + q] : 1.0f;
        float f[U::N];
        U::unpack(v[q], f);
#pragma unroll
        for (int i = 0; i < U::N; ++i) acc[i] = WEIGHTED ? fmaf(w, f[i], acc[i]) : acc[i] + f[i];
      }
    }
  }
  if (add) {
    float f[U::N];
    U::unpack(U::load(add + t * hidden + at), f);
#pragma unroll
    for (int i = 0; i < U::N; ++i) acc[i] += f[i];
  }
  U::store(y + t * hidden + at, U::pack(acc));
}

template <bool F32, bool WEIGHTED>
__global__ void __launch_bounds__(256) gather_sum_kernel(const void* __restrict__ rows_, const float* __restrict__ weights,
                                                        const int32_t* __restrict__ inverse, int64_t tokens, int64_t hidden,
                                                        RowUnits row, int log2, int k, const void* add_, void* y_) {
  typedef typename RowUnit<F32, true>::Elem Elem;
  const int64_t t = (int64_t)blockIdx.x * (256 >> log2) + (threadIdx.x >> log2);
  const int c = ((int)blockIdx.y << log2) + (threadIdx.x & ((1 << log2) - 1));
  if (t >= tokens || c >= row.units) return;
  constexpr int N = RowUnit<F32, true>::N;
  const uint32_t pairs = (uint32_t)(tokens * k);
  const Elem *rows = (const Elem*)rows_, *add = (const Elem*)add_;
  if (c < row.wide)
    gather_unit<RowUnit<F32, true>, WEIGHTED>(rows, weights, inverse, pairs, hidden, t, (int64_t)c * N, k, add, (Elem*)y_);
  else
    gather_unit<RowUnit<F32, false>, WEIGHTED>(rows, weights, inverse, pairs, hidden, t, (int64_t)row.wide * N + c - row.wide, k,
                                               add, (Elem*)y_);
}

template <bool WEIGHTED>
static void gather_sum(const void* rows, bool f32, const float* weights, const int32_t* inverse, int64_t tokens, int k,
                       int64_t hidden, const void* add, void* y, hipStream_t s) {
  const RowUnits row = row_units(hidden, f32);
  const RowGrid g = row_grid("gather_sum", tokens, row.units);
  if (f32)
    hipLaunchKernelGGL((gather_sum_kernel<true, WEIGHTED>), g.grid, dim3(256), 0, s, rows, weights, inverse, tokens, hidden, row,
                       g.log2, k, add, y);
  else
    hipLaunchKernelGGL((gather_sum_kernel<false, WEIGHTED>), g.grid, dim3(256), 0, s, rows, weights, inverse, tokens, hidden, row,
                       g.log2, k, add, y);
  check_launch("gather_sum");
}

// ---- the gradients of back: GROUP threads a token, a wave or a workgroup of 256 or 1024. Each thread holds the same units of dy
// for a batch of pairs, so a pair's row is read once, its gradient written, and its dot product summed over the
// group.
constexpr int BACK_BATCH = 8;

template <bool F32, int STORE, int GROUP, int THREADS>
__global__ void __launch_bounds__(THREADS) back_grad_kernel(const void* __restrict__ dy_, const void* __restrict__ rows_,
                                                       const float* __restrict__ weights, const int32_t* __restrict__ inverse,
                                                       const int32_t* __restrict__ present_, int64_t tokens, int64_t hidden,
                                                       RowUnits row, int k, int64_t through, void* __restrict__ drows_,
                                                       float* __restrict__ dweights) {
  typedef typename RowUnit<F32, true>::Elem Elem;
  constexpr int N = RowUnit<F32, true>::N;
  __shared__ float part[BACK_BATCH][GROUP / 64];
  const int64_t t = blockIdx.x * (THREADS / GROUP) + threadIdx.x / GROUP;
  const int me = threadIdx.x % GROUP, lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  if (t >= tokens) return;  // a whole wave, where a token has one: no barrier is ahead
  const Elem* dy = (const Elem*)dy_ + t * hidden;
  const Elem* rows = (const Elem*)rows_;
  Elem* drows = (Elem*)drows_;
  const uint32_t pairs = (uint32_t)(tokens * k);
  // the rows without a pair, spread over the tokens
  for (int64_t r = max(*present_, 0) + t; r < tokens * k; r += tokens) {
    for (int c = me; c < row.units; c += GROUP) {
      if (c < row.wide) store16_nt(drows + r * hidden + (int64_t)c * N, wm_u32x4{0, 0, 0, 0});
      else drows[r * hidden + (int64_t)row.wide * N + c - row.wide] = 0;
    }
  }
  for (int j0 = 0; j0 < k; j0 += BACK_BATCH) {
    uint32_t r[BACK_BATCH];
    float w[BACK_BATCH], dot[BACK_BATCH] = {};
#pragma unroll
    for (int q = 0; q < BACK_BATCH; ++q) {
      const int64_t p = t * k + j0 + q;
      r[q] = j0 + q < k ? (uint32_t)inverse[p] : 0xffffffffu;
      w[q] = j0 + q < k ? weights[p] : 0.0f;
    }
    auto unit = [&](auto u, int64_t at) {
      typedef decltype(u) U;
      float d[U::N];
      typename U::Raw v[BACK_BATCH];
      U::unpack(U::load(dy + at), d);
#pragma unroll
      for (int q = 0; q < BACK_BATCH; ++q)
        if (r[q] < pairs) v[q] = U::load_once(rows + r[q] * hidden + at);
#pragma unroll
      for (int q = 0; q < BACK_BATCH; ++q) {
        if (r[q] < pairs) {
          float f[U::N], o[U::N];
          U::unpack(v[q], f);
#pragma unroll
          for (int i = 0; i < U::N; ++i) {
            dot[q] = fmaf(d[i], f[i], dot[q]);
            o[i] = w[q] * d[i];
          }
          store_row_unit<U, STORE>(drows + r[q] * hidden + at, U::pack(o), r[q] >= through);
        }
      }
    };
    for (int c = me; c < row.wide; c += GROUP) unit(RowUnit<F32, true>(), (int64_t)c * N);
    if (me < row.units - row.wide) unit(RowUnit<F32, false>(), (int64_t)row.wide * N + me);
    if (GROUP == 64) {
#pragma unroll
      for (int q = 0; q < BACK_BATCH; ++q) {
        const float v = segment_sum<64>(dot[q]);
        if (lane == q && j0 + q < k) dweights[t * k + j0 + q] = v;
      }
      continue;
    }
#pragma unroll
    for (int q = 0; q < BACK_BATCH; ++q) {
      const float v = segment_sum<64>(dot[q]);
      if (lane == 0) part[q][wave] = v;
    }
    __syncthreads();
    if (threadIdx.x < BACK_BATCH && j0 + (int)threadIdx.x < k) {
      const float* v = part[threadIdx.x];
      float sum = 0.0f;
#pragma unroll
      for (int q = 0; q + 4 <= GROUP / 64; q += 4) sum += (v[q] + v[q + 1]) + (v[q + 2] + v[q + 3]);
      dweights[t * k + j0 + threadIdx.x] = sum;
    }
    __syncthreads();
  }
}

template <bool F32, int STORE>
static void back_grad(const void* dy, const void* rows, const float* weights, const int32_t* inverse, const int32_t* present,
                      int64_t tokens, int64_t hidden, int k, int64_t through, void* drows, float* dweights, hipStream_t s) {
  const RowUnits row = row_units(hidden, F32);
  if (row.units <= 64)  // 16000 tokens x 8 of 100 in bf16: 39 us, with a workgroup a token 102; of 1000 95 and 92
    hipLaunchKernelGGL((back_grad_kernel<F32, STORE, 64, 256>), dim3(grid_of("back_grad", (tokens + 3) / 4, 256)), dim3(256), 0, s, dy, rows, weights,
                       inverse, present, tokens, hidden, row, k, through, drows, dweights);
  else if (tokens <= 256 && row.units > 256)  // a CU a token: 11 x 7 of 6016 in fp32 7.2 us, with 256 threads 10.7
    hipLaunchKernelGGL((back_grad_kernel<F32, STORE, 1024, 1024>), dim3((unsigned)tokens), dim3(1024), 0, s, dy, rows, weights, inverse,
                       present, tokens, hidden, row, k, through, drows, dweights);
  else
    hipLaunchKernelGGL((back_grad_kernel<F32, STORE, 256, 256>), dim3(grid_of("back_grad", tokens, 256)), dim3(256), 0, s, dy, rows, weights, inverse,
                       present, tokens, hidden, row, k, through, drows, dweights);
  check_launch("back_grad");
}

static void check_rows(const char* name, int64_t tokens, int k, int64_t hidden, int f32) {
  const std::string n(name);
  if (tokens < 0) fail(n + ": tokens must not be negative");
  if (k < 1 || k > SORT_MAX_K) fail(n + ": k must be in 1..64");
  if (tokens * k > (int64_t)0x7fffffff) fail(n + ": tokens * k must be below 2^31");
  if (hidden < 1 || hidden > 1 << 20) fail(n + ": hidden must be in 1..1048576");
  if (f32 != 0 && f32 != 1) fail(n + ": fp32 must be 0 (bf16 rows) or 1");
}

}  // namespace wm

using namespace wm;

extern "C" {

WM_EXPORT size_t wm_sort_tokens_workspace_size(int32_t tokens, int32_t k, int32_t experts) {
  const int64_t pairs = (int64_t)tokens * k;
  if (tokens < 0 || k < 1 || k > SORT_MAX_K || experts < 1 || pairs <= SORT_ONE_MAX) return 0;
  const int spans = sort_spans(tokens, k).spans;
  return (size_t)(spans + (spans > SORT_SPANS_ADDED)) * experts * sizeof(int32_t);
}

WM_EXPORT int wm_sort_tokens(const void* x, int32_t fp32, int32_t tokens, int32_t hidden, const int32_t* indices, int32_t k,
                             int32_t experts, int32_t tile_rows, void* rows, int32_t* order, int32_t* inverse,
                             int32_t* offsets, int32_t* tiles, int32_t* tile_count, void* workspace, size_t workspace_bytes,
                             void* stream) {
  return guarded([&] {
    check_rows("wm_sort_tokens", tokens, k, hidden, fp32);
    const int64_t pairs = (int64_t)tokens * k;
    if (experts < 1 || experts > PERMUTE_MAX_EXPERTS) fail("wm_sort_tokens: experts must be in 1..1024");
    if (tile_rows < 1) fail("wm_sort_tokens: tile_rows must be positive");
    const size_t need = wm_sort_tokens_workspace_size(tokens, k, experts);
    if (!offsets || !tiles || !tile_count || (need > 0 && !workspace) || (pairs > 0 && (!x || !indices || !rows || !order || !inverse)))
      fail("wm_sort_tokens: null pointer");
    if (((uintptr_t)x | (uintptr_t)rows) % (fp32 ? 4 : 2) || (uintptr_t)tiles % 8)
      fail("wm_sort_tokens: rows must be aligned to their elements and tiles to 8 bytes");
    if (workspace_bytes < need || (uintptr_t)workspace % 4) fail("wm_sort_tokens: workspace too small or misaligned");
    hipStream_t s = as_stream(stream);
    SortArgs a = {};
    a.x = x, a.indices = indices, a.tokens = tokens, a.k = k, a.experts = experts, a.tile_rows = tile_rows;
    a.chunk_tokens = sort_chunk_tokens(tokens, k);
    a.rows = rows, a.order = order, a.inverse = inverse, a.offsets = offsets, a.tiles = tiles, a.tile_count = tile_count;
    a.max_tiles = (pairs + tile_rows - 1) / tile_rows + experts;
    const SortSpans spans = sort_spans(tokens, k);
    a.span_pairs = spans.pairs, a.spans = spans.spans;
    a.length = (int64_t)hidden * (fp32 ? 2 : 1);
    a.row = row_units(a.length, false);
    sort_launch(a, (int32_t*)workspace, s);
  });
}

WM_EXPORT int wm_sort_tokens_backward(const void* drows, int32_t fp32, const int32_t* inverse, int32_t tokens, int32_t k,
                                      int32_t hidden, void* dx, void* stream) {
  return guarded([&] {
    check_rows("wm_sort_tokens_backward", tokens, k, hidden, fp32);
    if (tokens == 0) return;
    if (!drows || !inverse || !dx) fail("wm_sort_tokens_backward: null pointer");
    if (((uintptr_t)drows | (uintptr_t)dx) % (fp32 ? 4 : 2)) fail("wm_sort_tokens_backward: rows must be aligned to their elements");
    gather_sum<false>(drows, fp32 != 0, nullptr, inverse, tokens, k, hidden, nullptr, dx, as_stream(stream));
  });
}

WM_EXPORT int wm_combine_rows(const void* rows, int32_t fp32, const float* weights, const int32_t* inverse, int32_t tokens,
                              int32_t k, int32_t hidden, const void* add, void* y, void* stream) {
  return guarded([&] {
    check_rows("wm_combine_rows", tokens, k, hidden, fp32);
    if (tokens == 0) return;
    if (!rows || !weights || !inverse || !y) fail("wm_combine_rows: null pointer");
    if (((uintptr_t)rows | (uintptr_t)add | (uintptr_t)y) % (fp32 ? 4 : 2))
      fail("wm_combine_rows: rows must be aligned to their elements");
    gather_sum<true>(rows, fp32 != 0, weights, inverse, tokens, k, hidden, add, y, as_stream(stream));
  });
}

WM_EXPORT int wm_combine_rows_backward(const void* dy, const void* rows, int32_t fp32, const float* weights,
                                       const int32_t* inverse, const int32_t* present, int32_t tokens, int32_t k,
                                       int32_t hidden, void* drows, float* dweights, void* stream) {
  return guarded([&] {
    check_rows("wm_combine_rows_backward", tokens, k, hidden, fp32);
    if (tokens == 0) return;
    if (!dy || !rows || !weights || !inverse || !present || !drows || !dweights) fail("wm_combine_rows_backward: null pointer");
    if (((uintptr_t)dy | (uintptr_t)rows | (uintptr_t)drows) % (fp32 ? 4 : 2))
      fail("wm_combine_rows_backward: rows must be aligned to their elements");
    hipStream_t s = as_stream(stream);
    const RowStores stores = row_stores((int64_t)tokens * k, (int64_t)hidden * (fp32 ? 4 : 2));
#define WM_BACK(F, S) back_grad<F, S>(dy, rows, weights, inverse, present, tokens, hidden, k, stores.through, drows, dweights, s)
#define WM_BACKS(F)                                     \
  if (stores.how == THROUGH) WM_BACK(F, THROUGH);       \
  else if (stores.how == PAST) WM_BACK(F, PAST);        \
  else WM_BACK(F, SPLIT);
    if (fp32) { WM_BACKS(true) } else { WM_BACKS(false) }
#undef WM_BACKS
#undef WM_BACK
  });
}

}  // extern "C"
