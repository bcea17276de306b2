// The draw of a token from logits: temperature, top-k, top-p, min-p and the inverse of the distribution's running
// sum at a given number. Per row, with T its temperature and L its largest logit:
//   e[v] = exp((l[v] - L) / T)                      the token's weight; 0 where l is -inf
//   top-k: the k tokens of the largest logits stay, of equal ones those of the lower ids
//   top-p: of these, in that order, the ones stay before which less than p of their weights lies (the first always)
//   min-p: of these, the ones with e >= p
//   token: the lowest id of those left whose running sum, in the order of the ids, is above u times the whole sum
// Where a cut or the draw falls between two tokens is decided by sums over a whole vocabulary, which fp32 or sums in
// another order would move. So weights are fixed point: e in fp64, rounded to a multiple of 2^-s, s from
// the vocabulary's size so that no sum passes 2^62. Sums of integers do not depend on their order; every token
// is off by at most 2^-(s + 1) of the largest one's weight (2^-46 for 129,280 tokens).
//
// A few rows are bound by dependent launches and, in the last one, by a workgroup's chain of barriers (1 row of 129,280 fp32
// logits, top-k and top-p: 17 to 20 us, of it 9 to 13 the last launch; 5 rows with top-p alone 28); many rows by the instructions a token
// takes where there is no small top-k (512 rows of fp32 314 us with top-p alone), and by HBM where there is (256 rows of fp32 with
// top-k 50 47 us, 2.8 TB/s). Rows whose cut falls among more than CANDIDATES tokens of one bin take up to 35 times a row's
// usual time (below).
#include <cmath>

#include "norm_rows.h"

namespace wm {
namespace smp {

constexpr int MAX_VOCAB = 1 << 22;
// One row of 129,280 tokens with top-k 48: 16.2 us, with 256 threads 19.7, with 1024 18.2 (k 256: 26.7, 41.5, 24.8).
constexpr int THREADS = 512, WAVES = THREADS / 64;
constexpr int PARTS = 1024;  // a row's chunks at most
constexpr int MOST = 2;      // units of a chunk at most
// Tokens of a vocabulary that one workgroup takes in one launch, passing them several times from its L2. With top-k 48 and top-p 0.9,
// top-p alone and neither, one row: 22, 18 and 9 us of 2048 tokens (in chunks 22, 22 and 14), 24, 21 and 10 of 3000 (23, 23
// and 15), 28, 24 and 10 of 4096 (16, 24 and 15), 48, 39 and 15 of 8192 (15, 25 and 15); 512 rows likewise.
constexpr int SMALL = 2048;

struct Args {
  const void* logits;
  int rows, vocab, shift;  // shift: s
  const float *uniforms, *temperature;
  const int32_t* top_k;
  const float *top_p, *min_p;
  int32_t* tokens;
  float* logp;
};

// The order of fp32 values as the order of unsigned integers.
__device__ __forceinline__ uint32_t key_of(float l) {
  const uint32_t b = __float_as_uint(l);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// Logit i of a row; -0 is 0.
template <bool F32>
__device__ __forceinline__ float logit(const void* row, int i) {
  return (F32 ? ((const float*)row)[i] : bf16_bits_to_f32(((const uint16_t*)row)[i])) + 0.0f;
}

// A row's rules. k: 0 is off; p: 1 and more is off; a greedy row is top-k 1.
struct Rules {
  float top;      // L
  double scale;   // log2(e) / T
  int k;
  float p, m;
  // Loaded before the row's largest logit is known, which `top` is set to.
  __device__ __forceinline__ Rules(const Args& a, int row) : top(0.0f) {
    float t = a.temperature ? a.temperature[row] : 1.0f;
    k = a.top_k ? a.top_k[row] : 0;
    p = a.top_p ? a.top_p[row] : 1.0f;
    m = a.min_p ? a.min_p[row] : 0.0f;
    if (!(t > 0.0f)) t = 1.0f, k = 1;  // greedy: 0, below, NaN
    if (k < 0 || k >= a.vocab) k = 0;
    if (!(p < 1.0f)) p = 1.0f;
    if (!(m > 0.0f)) m = 0.0f;
    m = fminf(m, 1.0f);
    scale = 1.4426950408889634 / (double)t;
  }
};

// e of a logit, to 2^-51 of it, without a branch. With x = (l - L) log2(e) / T, n the whole number next to it and f = x - n
//   e = 2^n sum_j (f ln 2)^j / j!     |f| <= 1/2, so that what lies behind j = 12 is below 2^-52
// x ends at -100, far below what a weight's integer holds; a masked logit is there too, where T is infinite (NaN) as well.
__device__ __forceinline__ double weight_of(float l, const Rules& r) {
  constexpr double L1 = 0.6931471805599453, L2 = L1 * L1, L3 = L2 * L1, L4 = L2 * L2, L6 = L4 * L2, L8 = L4 * L4;
  constexpr double WHOLE = 0x1.8p52;  // added to x it leaves n in the sum's low bits
  const double x = fmax(((double)l - (double)r.top) * r.scale, -100.0);
  const double t = x + WHOLE, f = x - (t - WHOLE);
  double s = L8 * L4 / 479001600.0;
  s = fma(s, f, L8 * L3 / 39916800.0);
  s = fma(s, f, L8 * L2 / 3628800.0);
  s = fma(s, f, L8 * L1 / 362880.0);
  s = fma(s, f, L8 / 40320.0);
  s = fma(s, f, L6 * L1 / 5040.0);
  s = fma(s, f, L6 / 720.0);
  s = fma(s, f, L4 * L1 / 120.0);
  s = fma(s, f, L4 / 24.0);
  s = fma(s, f, L3 / 6.0);
  s = fma(s, f, L2 / 2.0);
  s = fma(s, f, L1);
  s = fma(s, f, 1.0);
  const double e = __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, s) + (__builtin_bit_cast(uint64_t, t) << 52));
  return l == r.top ? 1.0 : e;  // also where both are infinite
}
// e to a multiple of 2^-shift, as an integer: adding 2^52 leaves it in the sum's low bits (shift is at most 51).
__device__ __forceinline__ uint64_t fixed_of(double e, int shift) {
  const double v = __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, e) + ((uint64_t)shift << 52)) + 0x1p52;
  return __builtin_bit_cast(uint64_t, v) & ((1ull << 52) - 1);
}

// Tokens that stay: logits above the key, and of those at it the ones up to id.
struct Cut {
  uint32_t key;
  int id;
  __device__ __forceinline__ bool keeps(uint32_t k, int i) const { return k > key || (k == key && i <= id); }
};

// ---------------------------------------------------------------------------------- sums over a workgroup

struct Shared {
  uint64_t sums[256];
  uint64_t part[WAVES];
  float top[WAVES];
  uint64_t chunk[PARTS];  // the chunks' sums
  uint64_t bcast[3];
};

template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t add_dpp(uint64_t v) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xf, false);
  return v + ((uint64_t)hi << 32 | lo);
}
// Sum of the lanes up to this one, by moves within rows of 16 lanes and from row to row.
__device__ __forceinline__ uint64_t wave_scan(uint64_t v) {
  v = add_dpp<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8
  v = add_dpp<0x112, 0xf>(v);
  v = add_dpp<0x114, 0xf>(v);
  v = add_dpp<0x118, 0xf>(v);
  v = add_dpp<0x142, 0xa>(v);  // row_bcast 15 to rows 1 and 3
  v = add_dpp<0x143, 0xc>(v);  // row_bcast 31 to rows 2 and 3
  return v;
}
// Room for `n` of this lane in a list: the first place, after the wave's lanes before. One addition a wave, whose lanes all
// call it.
__device__ __forceinline__ uint32_t reserve(uint32_t* counter, uint32_t n) {
  uint32_t s = n;
#define WM_SCAN_STEP(CTRL, ROWS) s += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)s, CTRL, ROWS, 0xf, false)
  WM_SCAN_STEP(0x111, 0xf);
  WM_SCAN_STEP(0x112, 0xf);
  WM_SCAN_STEP(0x114, 0xf);
  WM_SCAN_STEP(0x118, 0xf);
  WM_SCAN_STEP(0x142, 0xa);
  WM_SCAN_STEP(0x143, 0xc);
#undef WM_SCAN_STEP
  const uint32_t all = (uint32_t)__builtin_amdgcn_readlane((int)s, 63);
  uint32_t first = 0;
  if (all > 0) {
    if (threadIdx.x % 64 == 0) first = atomicAdd(counter, all);
    first = (uint32_t)__builtin_amdgcn_readfirstlane((int)first);
  }
  return first + s - n;
}
// Sum of the threads before this one; `total` of all. Every thread calls it.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t* part, uint64_t& total) {
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const uint64_t s = wave_scan(v);
  __syncthreads();
  if (lane == 63) part[wave] = s;
  __syncthreads();
  uint64_t before = 0;
  total = 0;
  for (int w = 0; w < WAVES; ++w) {
    if (w < wave) before += part[w];
    total += part[w];
  }
  return before + s - v;
}

// ---------------------------------------------------------------------------------- the cut of one row by one workgroup
//
// The key of the token at which a sum over the tokens in order of their logits reaches `want`: eight bits at a time from the
// top, by a histogram of the tokens that agree so far. WEIGHTS: sums of weights of the tokens that `k` keeps, else
// counts. Returns what lies above the key in `above`. The sum over all reaches `want`.
template <bool F32, bool WEIGHTS>
__device__ uint32_t select_key(const Args& a, const void* row, const Rules& r, Shared& s, const Cut& k, uint64_t want, uint64_t& above) {
  uint32_t key = 0;
  above = 0;
  for (int bit = 24; bit >= 0; bit -= 8) {
    __syncthreads();
    if (threadIdx.x < 256) s.sums[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < a.vocab; i += THREADS) {
      const float l = logit<F32>(row, i);
      const uint32_t at = key_of(l);
      if (bit < 24 && (at ^ key) >> (bit + 8)) continue;
      if (WEIGHTS && !k.keeps(at, i)) continue;
      const uint64_t v = WEIGHTS ? fixed_of(weight_of(l, r), a.shift) : 1;
      if (v) atomicAdd((unsigned long long*)&s.sums[at >> bit & 255], (unsigned long long)v);
    }
    __syncthreads();
    if (threadIdx.x < 64) {  // lane l: bins 255 - 4 l and the three below
      uint64_t v[4], sum = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) sum += v[j] = s.sums[255 - 4 * (int)threadIdx.x - j];
      uint64_t before = above + wave_scan(sum) - sum;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (before < want && before + v[j] >= want) {
          s.bcast[0] = 255 - 4 * threadIdx.x - j;
          s.bcast[1] = before;
        }
        before += v[j];
      }
    }
    __syncthreads();
    key |= (uint32_t)s.bcast[0] << bit;
    above = s.bcast[1];
  }
  return key;
}

// The id of token n (from 1 on) of those at `key`.
template <bool F32>
__device__ int nth_id(const Args& a, const void* row, Shared& s, uint32_t key, uint64_t n) {
  uint64_t before = 0;
  for (int lo = 0; lo < a.vocab; lo += THREADS) {
    const int i = lo + (int)threadIdx.x;
    const bool is = i < a.vocab && key_of(logit<F32>(row, i)) == key;
    uint64_t total;
    const uint64_t at = before + block_scan(is, s.part, total) + 1;
    if (is && at == n) s.bcast[2] = i;
    before += total;
    if (before >= n) break;  // the same for all threads
  }
  __syncthreads();
  return (int)s.bcast[2];
}

// The sum of the weights that `cut` keeps.
template <bool F32>
__device__ uint64_t kept_sum(const Args& a, const void* row, const Rules& r, Shared& s, const Cut& cut) {
  uint64_t v = 0, total;
  for (int i = threadIdx.x; i < a.vocab; i += THREADS) {
    const float l = logit<F32>(row, i);
    if (cut.keeps(key_of(l), i)) v += fixed_of(weight_of(l, r), a.shift);
  }
  block_scan(v, s.part, total);
  return total;
}

// ceil(p z) for 0 <= p < 1, at least 1: what must lie before a token for it to go.
__device__ __forceinline__ uint64_t part_of(float p, uint64_t z) {
  const uint64_t f = (uint64_t)(fmaxf(p, 0.0f) * 0x1p64f);  // exact down to 2^-41, below that p z is less than 2^22 units
  const uint64_t hi = __umul64hi(f, z);
  return max(hi + (f * z != 0), (uint64_t)1);
}

template <bool F32>
__device__ Cut row_cut(const Args& a, const void* row, const Rules& r, Shared& s) {
  Cut cut = {0, a.vocab};  // everything: no logit has the key 0 but a NaN
  uint64_t above;
  if (r.k > 0) {
    cut.key = select_key<F32, false>(a, row, r, s, cut, r.k, above);
    cut.id = nth_id<F32>(a, row, s, cut.key, r.k - above);
  }
  if (r.p < 1.0f) {
    const uint64_t want = part_of(r.p, kept_sum<F32>(a, row, r, s, cut));
    const uint32_t key = select_key<F32, true>(a, row, r, s, cut, want, above);
    const uint64_t each = fixed_of(weight_of(value_of(key), r), a.shift);
    // the tokens at the key weigh the same: the ones stay before which less than `want` lies
    const int id = nth_id<F32>(a, row, s, key, (want - above + each - 1) / each);
    cut = {key, id};
  }
  return cut;
}

// ---------------------------------------------------------------------------------- the draw
//
// floor(u whole), below the whole.
__device__ __forceinline__ uint64_t place_of(float u, uint64_t whole) {
  return __umul64hi((uint64_t)((u > 0.0f ? fminf(u, 1.0f - 0x1p-24f) : 0.0f) * 0x1p64f), whole);
}

// The part of `parts` that holds the draw's place, into s.bcast[0]; returns the place, the sum of all and of the parts before.
// Every thread calls it, behind a barrier; ends with one.
__device__ __forceinline__ uint64_t find_part(const Args& a, int row, Shared& s, int parts, uint64_t& whole, uint64_t& before) {
  constexpr int EACH = PARTS / THREADS;
  uint64_t v[EACH], sum = 0;
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const int c = threadIdx.x * EACH + j;
    sum += v[j] = c < parts ? s.chunk[c] : 0;
  }
  uint64_t at = block_scan(sum, s.part, whole);
  const uint64_t place = place_of(a.uniforms[row], whole);
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    if (place >= at && place < at + v[j]) {
      s.bcast[0] = threadIdx.x * EACH + j;
      s.bcast[1] = at;
    }
    at += v[j];
  }
  __syncthreads();
  before = s.bcast[1];
  return place;
}

// The row's results: token i of logit l, drawn among weights of this sum.
__device__ __forceinline__ void write_token(const Args& a, int row, const Rules& r, int i, float l, uint64_t whole) {
  const double t = l == r.top ? 0.0 : ((double)l - (double)r.top) * r.scale;
  a.tokens[row] = i;
  a.logp[row] = (float)((t - log2(ldexp((double)whole, -a.shift))) * 0.6931471805599453);
}

// Eight logits of a chunk from token i on, `n` of them there; the others are -inf.
template <bool F32>
struct Eight {
  Row8<F32> raw;
  __device__ __forceinline__ void load(const void* logits, int64_t base, int i, int n) {
    raw.clear();
    if (n > 0) raw.template load<false>(logits, base + i, n);
  }
  __device__ __forceinline__ float get(int e, int n) const { return e < n ? raw.get(e) + 0.0f : -INFINITY; }
};

// Writes the token whose running sum passes the draw's place, given the chunks' sums in s.chunk. left(l, i): the weight of
// logit l with id i, 0 if it goes. `size` is a chunk's tokens, MOST * 8 * THREADS at most and a multiple of 4 * THREADS. Every
// thread calls it.
template <bool F32, typename Left>
__device__ void draw(const Args& a, int row, const Rules& r, Shared& s, int chunks, int size, Left left) {
  uint64_t whole, first_of;
  __syncthreads();
  const uint64_t want = find_part(a, row, s, chunks, whole, first_of) - first_of;
  const int c = (int)s.bcast[0], each = size / THREADS;
  const int first = c * size + (int)threadIdx.x * each, end = min(first + each, a.vocab);
  float l[8 * MOST];
  uint64_t w[8 * MOST], mine = 0, total;
#pragma unroll
  for (int u = 0; u < MOST; ++u) {
    Eight<F32> raw;
    const int i = first + 8 * u;
    raw.load(a.logits, (int64_t)row * a.vocab, i, end - i);
#pragma unroll
    for (int e = 0; e < 8; ++e) l[8 * u + e] = raw.get(e, end - i);
  }
#pragma unroll
  for (int j = 0; j < 8 * MOST; ++j) mine += w[j] = l[j] == -INFINITY ? 0 : left(l[j], first + j);
  uint64_t before = block_scan(mine, s.part, total);
#pragma unroll
  for (int j = 0; j < 8 * MOST; ++j) {
    if (want >= before && want < before + w[j]) write_token(a, row, r, first + j, l[j], whole);
    before += w[j];
  }
}

// The weight of a logit that a row's cut keeps, if min-p does.
__device__ __forceinline__ uint64_t left_of(const Args& a, const Rules& r, float l) {
  const double e = weight_of(l, r);
  return e >= (double)r.m ? fixed_of(e, a.shift) : 0;
}

// The draw of a row from its cut, which is found here, and the chunks' sums.
template <bool F32>
__device__ void draw_cut(const Args& a, const void* p, int row, const Rules& r, Shared& s, int chunks, int size) {
  const Cut cut = row_cut<F32>(a, p, r, s);
  auto left = [&](float l, int i) -> uint64_t { return cut.keeps(key_of(l), i) ? left_of(a, r, l) : 0; };
  for (int c = 0; c < chunks; ++c) {
    uint64_t v = 0, total;
    for (int i = c * size + threadIdx.x; i < min((c + 1) * size, a.vocab); i += THREADS) v += left(logit<F32>(p, i), i);
    block_scan(v, s.part, total);
    if (threadIdx.x == 0) s.chunk[c] = total;
  }
  draw<F32>(a, row, r, s, chunks, size, left);
}

// Vocabularies of one chunk: a workgroup a row does all of it.
template <bool F32>
__global__ void __launch_bounds__(THREADS) sample_row_kernel(Args a) {
  __shared__ Shared s;
  const int row = blockIdx.x;
  const void* p = (const uint8_t*)a.logits + (int64_t)row * a.vocab * (F32 ? 4 : 2);
  Rules r(a, row);
  // the largest logit; a NaN's key is the largest or the smallest
  uint32_t high = 0;
  bool nan = false;
  for (int i = threadIdx.x; i < a.vocab; i += THREADS) {
    const float l = logit<F32>(p, i);
    high = max(high, key_of(l));
    nan |= l != l;
  }
  for (int d = 32; d > 0; d /= 2) high = max(high, (uint32_t)__shfl_xor((int)high, d, 64));
  if (threadIdx.x % 64 == 0) s.part[threadIdx.x / 64] = high;
  const bool any = __syncthreads_or(nan);
  for (int w = 0; w < WAVES; ++w) high = max(high, (uint32_t)s.part[w]);
  const float top = value_of(high);
  if (any || top == -INFINITY) {
    if (threadIdx.x == 0) a.tokens[row] = -1, a.logp[row] = NAN;
    return;
  }
  r.top = top;
  draw_cut<F32>(a, p, row, r, s, 1, SMALL);
}

// ---------------------------------------------------------------------------------- larger vocabularies
//
// Chunks of the rows, and then a workgroup a row. A first launch finds each chunk's largest logit, and each group's of 64
// tokens.
//
// With a small k (LIST_K) a row needs no other pass: of the groups' largest logits the k largest are k tokens, so
// the tokens that top-k may keep are no smaller than the k-th of these, and lie in the few groups that reach it.
//
// Otherwise two more launches go over the chunks: weights and counts by bins of the distance from the row's largest logit; and
// the tokens in the bins that a cut may fall into (candidates), with the chunks' sums of those above. A bin is
// 1/32 of a factor of 2, so that a cut has some hundreds of candidates where it falls among the bulk of the tokens and a few
// where it does not.
//
// Either way the last launch sorts the candidates, cuts and draws. Rows of more candidates than there is room for are
// cut by radix selection as above: their one workgroup passes the row seven times for top-p and twelve with top-k too. That
// is not rare for bf16: values of magnitude 8 to 16 are 1/16 apart, so that one value alone can be thousands of tokens of the tail.
// Normal logits of mean -10 and deviation 1.5 have 2100 candidates of 129,280 at top-p 0.9 and T 1, fp32 ones of
// deviation 1 at T 2 and top-p 0.8 as many; equal logits have all of them, for a greedy row as well. One row of 129,280 in
// bf16 with top-p 0.9: 25 us a head's logits, 56 the normal ones below the limit, 400 to 540 above it, 716 equal ones (greedy
// 565); 192 rows 104, 159, 876 and 952 (657).
constexpr int BINS = 2048, BIN_THREADS = 512, UNIT = 8 * BIN_THREADS, CANDIDATES = 2048;

// A row's candidates come from its groups while k is small and at most 3/4 of the groups: beyond, the groups' bound sinks fast.
// By the groups and by the bins, one row of 129,280 tokens: k 48 16.4 and 21 us, 128 20.5 and 21.6, 256 26 and 22; 256 rows 47
// and 108, 51 and 106, 60 and 109. One row of 8192 (128 groups): k 96 18.6 and 21.8, 128 28 and 23.
constexpr int GROUP = 64, LIST_K = 256;
__device__ __forceinline__ bool listed(const Args& a, const Rules& r) { return r.k > 0 && r.k <= min(LIST_K, a.vocab / GROUP * 3 / 4); }

// Rows whose cut takes bins.
__device__ __forceinline__ bool binned(const Args& a, const Rules& r) { return !listed(a, r) && (r.k > 0 || r.p < 1.0f); }

struct RowInfo {
  uint64_t below_lo, between;  // weights of the bins below lo, and of those between hi and kbin
  int32_t lo, hi;              // bins below lo stay, bins above hi go by top-p
  int32_t kbin, kleft;         // top-k ends in kbin, which has kleft tokens that stay (BINS: nowhere)
};

struct Work {
  float* tops;          // [rows][chunks]; NaN where the chunk has one
  uint64_t* sums;       // [rows][chunks]
  RowInfo* info;        // [rows]
  uint64_t* weights;    // [rows][BINS]
  uint32_t* counts;     // [rows][BINS]
  uint64_t* list;       // [rows][CANDIDATES]: key and the complement of the id
  uint32_t* listed;     // [rows]
  float* groups;        // [rows][chunks * size / GROUP]: each group's largest logit
  int chunks, size;
};

__device__ __forceinline__ uint64_t entry_of(float l, int i) { return (uint64_t)key_of(l) << 32 | (uint32_t)~i; }

// A row's bins: monotone in the logit, BINS - 1 where the weight is 0 (from 2^-63.9 on). Distances are taken h times, h a power
// of two, so that neither they nor the scale leave fp32 where the weight is not 0: a quarter for temperatures of 0.7 and more
// (the types' largest values are 2^129 apart), 2^60 for ones below 2^-60 (differences of 2^-149 count there) among logits below 2^60;
// larger logits are 2^36 apart or equal. Between, h is 1, and a distance past fp32 has weight 0.
struct Bins {
  float top, h, top_h, scale;
  __device__ __forceinline__ explicit Bins(const Rules& r) : top(r.top) {
    const double s = 32.0 * r.scale;
    const bool large = s <= 64.0, small = s >= 0x1p66 && fabsf(top) < 0x1p60f;
    h = large ? 0.25f : small ? 0x1p60f : 1.0f;
    top_h = top * h;
    scale = (float)(large ? 4.0 * s : small ? 0x1p-60 * s : s);
  }
  __device__ __forceinline__ int of(float l) const { return l == top ? 0 : (int)fminf(fmaf(-l, h, top_h) * scale, (float)(BINS - 1)); }
};

// The row's largest logit from its chunks'; false for a row that has nothing to draw. Every thread calls it.
template <int N>
__device__ __forceinline__ bool row_top(const float* tops, int chunks, float* part, float& top) {
  float t = -INFINITY;
  bool nan = false;
  for (int c = threadIdx.x; c < chunks; c += N) {
    const float v = tops[c];
    nan |= v != v;
    t = fmaxf(t, v);
  }
  t = segment_max<64>(t);
  if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = t;
  nan = __syncthreads_or(nan);
#pragma unroll
  for (int w = 0; w < N / 64; ++w) t = fmaxf(t, part[w]);
  top = t;
  return !nan && t != -INFINITY;
}

// A thread's logits of a chunk, all on their way at once: before what the launch has to know of the row.
template <bool F32>
struct ChunkLogits {
  Eight<F32> l[MOST];
  __device__ __forceinline__ void load(const void* logits, int64_t base, int lo, int end, int size) {
#pragma unroll
    for (int u = 0; u < MOST; ++u)
      if (u * UNIT < size) {
        const int i = lo + u * UNIT + 8 * (int)threadIdx.x;
        l[u].load(logits, base, i, end - i);
      }
  }
};

template <bool F32>
__global__ void __launch_bounds__(BIN_THREADS) sample_tops_kernel(Args a, Work w) {
  __shared__ float part[BIN_THREADS / 64];
  const int row = blockIdx.x / w.chunks, c = blockIdx.x % w.chunks;
  const int64_t base = (int64_t)row * a.vocab;
  const int lo = c * w.size, end = min(lo + w.size, a.vocab);
  ChunkLogits<F32> here;
  here.load(a.logits, base, lo, end, w.size);
  if (binned(a, Rules(a, row))) {
    for (int i = c * BIN_THREADS + threadIdx.x; i < BINS; i += w.chunks * BIN_THREADS) {
      w.weights[(int64_t)row * BINS + i] = 0;
      w.counts[(int64_t)row * BINS + i] = 0;
    }
  }
  if (c == 0 && threadIdx.x == 0) w.listed[row] = 0;
  float t = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int u = 0; u < MOST; ++u) {
    if (u * UNIT >= w.size) break;
    const int i = lo + u * UNIT + 8 * (int)threadIdx.x;  // whole waves, also behind the vocabulary's end
    float mine = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = here.l[u].get(e, end - i);
      nan |= v != v;
      mine = fmaxf(mine, v);
    }
    t = fmaxf(t, mine);
    mine = fmaxf(mine, dpp_f<0xB1>(mine));   // over 8 lanes, a group's
    mine = fmaxf(mine, dpp_f<0x4E>(mine));
    mine = fmaxf(mine, dpp_f<0x141>(mine));
    if (threadIdx.x % 8 == 0) w.groups[((int64_t)row * w.chunks * w.size + i) / GROUP] = mine;
  }
  t = segment_max<64>(t);
  if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = t;
  nan = __syncthreads_or(nan);
  if (threadIdx.x == 0) {
#pragma unroll
    for (int q = 1; q < BIN_THREADS / 64; ++q) t = fmaxf(t, part[q]);
    w.tops[blockIdx.x] = nan ? NAN : t;
  }
}

template <bool F32>
__global__ void __launch_bounds__(BIN_THREADS) sample_bins_kernel(Args a, Work w) {
  __shared__ uint64_t weights[BINS];
  __shared__ uint32_t counts[BINS];
  __shared__ float part[BIN_THREADS / 64];
  const int row = blockIdx.x / w.chunks, c = blockIdx.x % w.chunks;
  Rules r(a, row);
  const bool by_weight = r.p < 1.0f, by_count = r.k > 0;
  if (!binned(a, r)) return;
  const int64_t base = (int64_t)row * a.vocab;
  const int lo = c * w.size, end = min(lo + w.size, a.vocab);
  ChunkLogits<F32> here;
  here.load(a.logits, base, lo, end, w.size);
  if (!row_top<BIN_THREADS>(w.tops + (int64_t)row * w.chunks, w.chunks, part, r.top)) return;
  const Bins bins(r);
  for (int i = threadIdx.x; i < BINS; i += BIN_THREADS) {
    if (by_weight) weights[i] = 0;
    if (by_count) counts[i] = 0;
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < MOST; ++u) {
    const int i = lo + u * UNIT + 8 * (int)threadIdx.x;
    if (u * UNIT >= w.size || i >= end) break;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = here.l[u].get(e, end - i);
      const int b = bins.of(v);
      if (b == BINS - 1) continue;
      if (by_count) atomicAdd(&counts[b], 1u);
      if (by_weight) atomicAdd((unsigned long long*)&weights[b], (unsigned long long)fixed_of(weight_of(v, r), a.shift));
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += BIN_THREADS) {
    if (by_weight && weights[i])
      atomicAdd((unsigned long long*)&w.weights[(int64_t)row * BINS + i], (unsigned long long)weights[i]);
    if (by_count && counts[i]) atomicAdd(&w.counts[(int64_t)row * BINS + i], counts[i]);
  }
}

// Sum of the threads before this one over a workgroup of N threads.
template <int N>
__device__ __forceinline__ uint64_t scan_of(uint64_t v, uint64_t* part, uint64_t& total) {
  const uint64_t s = wave_scan(v);
  __syncthreads();
  if (threadIdx.x % 64 == 63) part[threadIdx.x / 64] = s;
  __syncthreads();
  uint64_t before = 0;
  total = 0;
#pragma unroll
  for (int q = 0; q < N / 64; ++q) {
    if (q < (int)threadIdx.x / 64) before += part[q];
    total += part[q];
  }
  return before + s - v;
}

template <bool F32>
__global__ void __launch_bounds__(BIN_THREADS) sample_gather_kernel(Args a, Work w) {
  constexpr int EACH = BINS / BIN_THREADS;
  __shared__ uint64_t part[BIN_THREADS / 64];
  __shared__ float top_part[BIN_THREADS / 64];
  __shared__ RowInfo info;
  __shared__ uint64_t k_below, k_in;  // weights below kbin, and in it
  __shared__ uint64_t list[CANDIDATES];
  __shared__ uint32_t found, first;
  const int row = blockIdx.x / w.chunks, c = blockIdx.x % w.chunks;
  Rules r(a, row);
  if (listed(a, r)) return;
  const int64_t base = (int64_t)row * a.vocab;
  const int lo = c * w.size, end = min(lo + w.size, a.vocab);
  ChunkLogits<F32> here;
  here.load(a.logits, base, lo, end, w.size);
  if (!row_top<BIN_THREADS>(w.tops + (int64_t)row * w.chunks, w.chunks, top_part, r.top)) return;
  const Bins bins(r);
  if (threadIdx.x == 0) info = {0, 0, BINS, BINS, BINS, 0}, found = 0;
  if (binned(a, r)) {
    uint64_t weight[EACH], sum = 0, total, before;
    uint32_t count[EACH], n = 0;
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      const int64_t at = (int64_t)row * BINS + threadIdx.x * EACH + j;
      sum += weight[j] = w.weights[at];
      n += count[j] = w.counts[at];
    }
    before = scan_of<BIN_THREADS>(sum, part, total);
    if (threadIdx.x == 0) k_below = total, k_in = 0;
    if (r.k > 0) {
      uint64_t counted;
      uint64_t at = scan_of<BIN_THREADS>(n, part, counted), below = before;
#pragma unroll
      for (int j = 0; j < EACH; ++j) {
        if (at < (uint64_t)r.k && at + count[j] >= (uint64_t)r.k) {
          info.kbin = threadIdx.x * EACH + j;
          info.kleft = r.k - (int)at;
          k_below = below;
          k_in = info.kleft == (int)count[j] ? 0 : weight[j];
          if (!k_in) k_below += weight[j];
        }
        at += count[j];
        below += weight[j];
      }
    }
    __syncthreads();
    if (r.p < 1.0f) {
      // the weights that top-k leaves are k_below to k_below + k_in
      const uint64_t least = part_of(r.p, k_below > 0 ? k_below : 1), most = part_of(r.p, k_below + k_in);
      uint64_t at = before;
#pragma unroll
      for (int j = 0; j < EACH; ++j) {
        const int b = threadIdx.x * EACH + j;
        if (at < least && at + weight[j] >= least) info.lo = b, info.below_lo = at;
        if (at < most && at + weight[j] >= most) info.hi = b;
        at += weight[j];
      }
      __syncthreads();
      const int hi = info.hi, kbin = info.kbin;
      uint64_t v = 0;
#pragma unroll
      for (int j = 0; j < EACH; ++j) {
        const int b = threadIdx.x * EACH + j;
        if (b > hi && b < kbin) v += weight[j];
      }
      scan_of<BIN_THREADS>(v, part, total);
      if (threadIdx.x == 0) info.between = total;
    } else if (threadIdx.x == 0) {
      info.lo = info.hi = info.kbin;
    }
  }
  __syncthreads();
  if (c == 0 && threadIdx.x == 0) w.info[row] = info;
  const int stay = info.lo, hi = info.hi, kbin = info.kbin;
  uint64_t sum = 0;
#pragma unroll
  for (int u = 0; u < MOST; ++u) {
    if (u * UNIT >= w.size) break;
    const int i = lo + u * UNIT + 8 * (int)threadIdx.x;  // whole waves, also behind the vocabulary's end
    uint32_t hits = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = here.l[u].get(e, end - i);
      const int b = bins.of(v);
      if (b == BINS - 1) continue;
      if (b < stay) sum += left_of(a, r, v);
      else if (b <= hi || b == kbin) hits |= 1u << e;
    }
    uint32_t at = reserve(&found, __popc(hits));
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (hits >> e & 1) {
        if (at < CANDIDATES) list[at] = entry_of(here.l[u].get(e, end - i), i + e);
        ++at;
      }
  }
  uint64_t total;
  scan_of<BIN_THREADS>(sum, part, total);  // and a barrier
  if (threadIdx.x == 0) {
    w.sums[blockIdx.x] = total;
    first = found ? atomicAdd(&w.listed[row], found) : 0;
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < found && first + i < CANDIDATES; i += BIN_THREADS)
    w.list[(int64_t)row * CANDIDATES + first + i] = list[i];
}

// Descending, in LDS; n a power of two.
__device__ __forceinline__ void sort_entries(uint64_t* v, int n) {
  for (int k = 2; k <= n; k *= 2)
    for (int j = k / 2; j > 0; j /= 2) {
      __syncthreads();
      for (int t = threadIdx.x; t < n / 2; t += THREADS) {
        const int i = 2 * t - (t & (j - 1)), o = i + j;  // the pair's lower place
        const uint64_t x = v[i], y = v[o];
        if ((x < y) == ((i & k) == 0)) v[i] = y, v[o] = x;
      }
    }
  __syncthreads();
}

// The same for up to THREADS entries, each put in its place by how many are above it. Ends with a barrier.
__device__ __forceinline__ void rank_entries(uint64_t* v, uint64_t* other, int n) {
  const int t = threadIdx.x;
  if (t < 8) v[n + t] = 0;  // below every entry
  __syncthreads();
  if (t < n) {
    const uint64_t mine = v[t];
    int above = 0;
    for (int i = 0; i < n; i += 8) {
      uint64_t o[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = v[i + j];
#pragma unroll
      for (int j = 0; j < 8; ++j) above += o[j] > mine;
    }
    other[above] = mine;
  }
  __syncthreads();
  if (t < n) v[t] = other[t];
  __syncthreads();
}

// The first groups' largest logits, a thread's own in registers: requested before anything else is known of the row.
struct Groups {
  static constexpr int KEPT = 4;
  float kept[KEPT];
  const float* tops;
  int groups;
  __device__ __forceinline__ Groups(const Args& a, const Work& w, int row)
      : tops(w.groups + (int64_t)row * w.chunks * w.size / GROUP), groups((a.vocab + GROUP - 1) / GROUP) {
#pragma unroll
    for (int j = 0; j < KEPT; ++j) {
      const int g = THREADS * j + (int)threadIdx.x;
      kept[j] = g < groups ? tops[g] : -INFINITY;
    }
  }
  // f(group, its largest logit) for whole waves; groups behind the last are -inf.
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll
    for (int j = 0; j < KEPT; ++j)
      if (THREADS * j < groups) f(THREADS * j + (int)threadIdx.x, kept[j]);
#pragma unroll 1
    for (int g0 = THREADS * KEPT; g0 < groups; g0 += THREADS) {
      const int g = g0 + (int)threadIdx.x;
      f(g, g < groups ? tops[g] : -INFINITY);
    }
  }
};

// The entries of a row that a small k may keep, into `entry`, and how many there are: more than CANDIDATES where they do not
// fit. A bin that k groups' largest logits reach bounds the tokens; `counts` is BINS + CANDIDATES words.
template <bool F32>
__device__ int list_row(const Args& a, const Groups& groups, const void* p, const Rules& r, const Bins& bins, Shared& s,
                        uint64_t* entry, uint32_t* counts, uint32_t* found) {
  constexpr int EACH = BINS / THREADS, AHEAD = 8;
  uint32_t* which = counts + BINS;
  for (int i = threadIdx.x; i < BINS; i += THREADS) counts[i] = 0;
  if (threadIdx.x < 2) found[threadIdx.x] = 0;
  if (threadIdx.x == 0) s.bcast[0] = BINS - 2;
  __syncthreads();
  groups.each([&](int, float top) {
    const int b = bins.of(top);
    if (b < BINS - 1) atomicAdd(&counts[b], 1u);
  });
  __syncthreads();
  uint64_t n = 0, total;
#pragma unroll
  for (int j = 0; j < EACH; ++j) n += counts[threadIdx.x * EACH + j];
  uint64_t at = block_scan(n, s.part, total);
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const uint64_t next = at + counts[threadIdx.x * EACH + j];
    if (at < (uint64_t)r.k && next >= (uint64_t)r.k) s.bcast[0] = threadIdx.x * EACH + j;
    at = next;
  }
  __syncthreads();
  const int bound = (int)s.bcast[0];
  groups.each([&](int g, float top) {
    const bool is = bins.of(top) <= bound;
    const uint32_t i = reserve(&found[0], is);
    if (is && i < CANDIDATES) which[i] = g;
  });
  __syncthreads();
  const uint32_t hits = found[0];
  if (hits > CANDIDATES) return CANDIDATES + 1;
  for (uint32_t e0 = 0; e0 < hits * GROUP; e0 += THREADS * AHEAD) {
    float l[AHEAD];
    int id[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const uint32_t e = e0 + THREADS * j + threadIdx.x;
      id[j] = e < hits * GROUP ? (int)(which[e / GROUP] * GROUP + e % GROUP) : a.vocab;
      l[j] = id[j] < a.vocab ? logit<F32>(p, id[j]) : -INFINITY;
    }
    uint32_t in = 0;
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) in |= (uint32_t)(bins.of(l[j]) <= bound) << j;
    uint32_t i = reserve(&found[1], __popc(in));
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (in >> j & 1) {
        if (i < CANDIDATES) entry[i] = entry_of(l[j], id[j]);
        ++i;
      }
  }
  __syncthreads();
  return (int)found[1];
}

template <bool F32>
__global__ void __launch_bounds__(THREADS) sample_draw_kernel(Args a, Work w) {
  __shared__ Shared s;
  // the candidates, their weights, and what lies ahead of each
  __shared__ uint64_t entry[CANDIDATES], weight[CANDIDATES], ahead[CANDIDATES];
  __shared__ int in_part;
  __shared__ uint32_t found[2];
  const int row = blockIdx.x;
  const void* p = (const uint8_t*)a.logits + (int64_t)row * a.vocab * (F32 ? 4 : 2);
  Rules r(a, row);
  const Groups groups(a, w, row);
  if (!row_top<THREADS>(w.tops + (int64_t)row * w.chunks, w.chunks, s.top, r.top)) {
    if (threadIdx.x == 0) a.tokens[row] = -1, a.logp[row] = NAN;
    return;
  }
  const Bins bins(r);
  const bool list = listed(a, r);
  RowInfo info = {0, 0, 0, BINS, BINS, 0};
  int n;
  if (list) {
    n = list_row<F32>(a, groups, p, r, bins, s, entry, (uint32_t*)weight, found);
  } else {
    n = (int)w.listed[row];
    info = w.info[row];
  }
  if (n > CANDIDATES) {  // the same for all threads
    draw_cut<F32>(a, p, row, r, s, w.chunks, w.size);
    return;
  }
  // the weights by id: in parts of the chunks' size, or, where the list is all there is, a thousand
  int part = w.size;
  if (list) part = (a.vocab + PARTS - 1) / PARTS;
  if (threadIdx.x == 0) in_part = 0;
  for (int c = threadIdx.x; c < PARTS; c += THREADS) s.chunk[c] = !list && c < w.chunks ? w.sums[(int64_t)row * w.chunks + c] : 0;
  if (!list)
    for (int i = threadIdx.x; i < n; i += THREADS) entry[i] = w.list[(int64_t)row * CANDIDATES + i];
  if (n <= THREADS) {  // (a row of 129,280 tokens with top-k 48 16 us so and 28 by the sort, 256 26 and 35)
    rank_entries(entry, weight, n);
  } else {
    int places = 2 * THREADS;
    while (places < n) places *= 2;
    for (int i = n + threadIdx.x; i < places; i += THREADS) entry[i] = 0;
    sort_entries(entry, places);
  }
  // In order: the bins from lo to hi, then kbin's, if that is behind them. Entries ahead of kbin's:
  int before_k = 0;
  if (!list) {
#pragma unroll 1
    for (int i0 = 0; i0 < n; i0 += THREADS) {
      const int i = i0 + (int)threadIdx.x;
      before_k += __syncthreads_count(i < n && bins.of(value_of((uint32_t)(entry[i] >> 32))) < info.kbin);
    }
  }
  uint64_t sum = info.below_lo;
#pragma unroll 1
  for (int i0 = 0; i0 < n; i0 += THREADS) {
    const int i = i0 + (int)threadIdx.x;
    uint64_t v = 0, total;
    bool stays = false;
    if (i < n) {
      const float l = value_of((uint32_t)(entry[i] >> 32));
      const int b = bins.of(l);
      const double e = weight_of(l, r);
      stays = e >= (double)r.m;
      if (list ? i < r.k : b < info.kbin || (b == info.kbin && i < before_k + info.kleft)) v = fixed_of(e, a.shift);
    }
    const uint64_t before = sum + block_scan(v, s.part, total);
    if (i < n) {
      weight[i] = v | (uint64_t)stays << 63;
      ahead[i] = before;
    }
    sum += total;
  }
  const uint64_t want = r.p < 1.0f ? part_of(r.p, sum + info.between) : ~0ull;
  int kept = 0;
#pragma unroll 1
  for (int i0 = 0; i0 < n; i0 += THREADS) {
    const int i = i0 + (int)threadIdx.x;
    const uint64_t v = i < n ? weight[i] : 0;
    // a token of top-k whose weight is 0 does not matter, nor does one between hi and kbin: it has more than `want` ahead
    const bool keep = (v << 1) != 0 && ahead[i] < want;
    kept += __syncthreads_count(keep);
    if (i < n) weight[i] = keep && v >> 63 ? v << 1 >> 1 : 0;
    if (keep && v >> 63) atomicAdd((unsigned long long*)&s.chunk[(int)~(uint32_t)entry[i] / part], (unsigned long long)(v << 1 >> 1));
  }
  __syncthreads();
  if (!list) {
    const uint64_t last = kept > 0 ? entry[kept - 1] : ~0ull;  // the last entry that stays
    draw<F32>(a, row, r, s, w.chunks, w.size, [&](float l, int i) -> uint64_t {
      const int b = bins.of(l);
      return b < BINS - 1 && (b < info.lo || entry_of(l, i) >= last) ? left_of(a, r, l) : 0;
    });
    return;
  }
  // the part of the ids that holds the draw's place, its entries, and of these the one
  uint64_t whole, first;
  const uint64_t place = find_part(a, row, s, PARTS, whole, first);
  const int at = (int)s.bcast[0];
#pragma unroll 1
  for (int i = threadIdx.x; i < n; i += THREADS)
    if (weight[i] && (int)~(uint32_t)entry[i] / part == at) ahead[atomicAdd(&in_part, 1)] = i;
  __syncthreads();
  const int few = in_part;
#pragma unroll 1
  for (int j = threadIdx.x; j < few; j += THREADS) {
    const int i = (int)ahead[j], id = (int)~(uint32_t)entry[i];
    uint64_t before = first;
#pragma unroll 1
    for (int q = 0; q < few; ++q) {
      const int o = (int)ahead[q];
      if ((int)~(uint32_t)entry[o] < id) before += weight[o];
    }
    if (place >= before && place < before + weight[i]) write_token(a, row, r, id, value_of((uint32_t)(entry[i] >> 32)), whole);
  }
}

// Tokens of a chunk: whole units, so many that the launches have about three workgroups a CU, two at most: more of them make the
// draw's part of one chunk longer, fewer add work a chunk. At most 1, 2 and 4 take, with top-p alone, 390, 313
// and 328 us for 512 rows of 129,280 tokens and 118, 109 and 132 for 512 of 32,768; with no rule 180, 177, 200 and 57, 62, 87.
static int chunk_size(int64_t rows, int vocab) {
  const int64_t units = (vocab + UNIT - 1) / UNIT, each = rows * units / 768;
  return (int)(each < 1 ? 1 : each > MOST ? MOST : each) * UNIT;
}
struct Layout {
  int chunks, size;
  size_t tops, sums, info, weights, counts, list, listed, groups, bytes;
  Layout(int64_t rows, int vocab) {
    size = chunk_size(rows, vocab);
    chunks = (vocab + size - 1) / size;
    bytes = 0;
    auto part = [&](size_t n) {
      const size_t at = bytes;
      bytes += (n + 15) / 16 * 16;
      return at;
    };
    sums = part(rows * chunks * sizeof(uint64_t));
    info = part(rows * sizeof(RowInfo));
    weights = part(rows * BINS * sizeof(uint64_t));
    list = part(rows * CANDIDATES * sizeof(uint64_t));
    counts = part(rows * BINS * sizeof(uint32_t));
    tops = part(rows * chunks * sizeof(float));
    groups = part(rows * chunks * (size / GROUP) * sizeof(float));
    listed = part(rows * sizeof(uint32_t));
  }
};

// Rows that one set of launches takes, which bounds the workspace: a row has 41 KB, vocab / 16 bytes of groups and 12 bytes a
// chunk (49 KB of 129,280 tokens, 309 KB of 4,194,304, and so 316 MB at most).
constexpr int BATCH = 1024;

template <bool F32>
static void launch(Args a, void* workspace, hipStream_t st) {
  if (a.vocab <= SMALL) {
    hipLaunchKernelGGL((sample_row_kernel<F32>), dim3(a.rows), dim3(THREADS), 0, st, a);
    check_launch("sample_row");
    return;
  }
  const Layout at(a.rows < BATCH ? a.rows : BATCH, a.vocab);
  uint8_t* base = (uint8_t*)workspace;
  const Work w = {(float*)(base + at.tops),       (uint64_t*)(base + at.sums),   (RowInfo*)(base + at.info),
                  (uint64_t*)(base + at.weights), (uint32_t*)(base + at.counts), (uint64_t*)(base + at.list),
                  (uint32_t*)(base + at.listed),  (float*)(base + at.groups),    at.chunks,
                  at.size};
  for (int left = a.rows; left > 0; left -= BATCH) {
    a.rows = left < BATCH ? left : BATCH;
    const dim3 grid((unsigned)(a.rows * at.chunks));
    hipLaunchKernelGGL((sample_tops_kernel<F32>), grid, dim3(BIN_THREADS), 0, st, a, w);
    check_launch("sample_tops");
    if (a.top_k || a.top_p) {  // else no row takes bins: a greedy row's k of 1 is listed
      hipLaunchKernelGGL((sample_bins_kernel<F32>), grid, dim3(BIN_THREADS), 0, st, a, w);
      check_launch("sample_bins");
    }
    hipLaunchKernelGGL((sample_gather_kernel<F32>), grid, dim3(BIN_THREADS), 0, st, a, w);
    check_launch("sample_gather");
    hipLaunchKernelGGL((sample_draw_kernel<F32>), dim3(a.rows), dim3(THREADS), 0, st, a, w);
    check_launch("sample_draw");
    a.logits = (const uint8_t*)a.logits + (int64_t)BATCH * a.vocab * (F32 ? 4 : 2);
    a.uniforms += BATCH;
    if (a.temperature) a.temperature += BATCH;
    if (a.top_k) a.top_k += BATCH;
    if (a.top_p) a.top_p += BATCH;
    if (a.min_p) a.min_p += BATCH;
    a.tokens += BATCH;
    a.logp += BATCH;
  }
}

}  // namespace smp
}  // namespace wm

using namespace wm;

extern "C" {

WM_EXPORT size_t wm_sample_logits_workspace_size(int32_t rows, int32_t vocab) {
  if (rows < 0 || vocab <= smp::SMALL || vocab > smp::MAX_VOCAB) return 0;
  return smp::Layout(rows < smp::BATCH ? rows : smp::BATCH, vocab).bytes;
}

WM_EXPORT int wm_sample_logits(const void* logits, int32_t fp32, int32_t rows, int32_t vocab, const float* uniforms,
                               const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                               int32_t* tokens, float* logp, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded([&] {
    if (rows < 0) fail("wm_sample_logits: rows must not be negative");
    if (vocab < 1 || vocab > smp::MAX_VOCAB) fail("wm_sample_logits: vocab must be in 1..4194304");
    if (fp32 != 0 && fp32 != 1) fail("wm_sample_logits: fp32 must be 0 (bf16 logits) or 1");
    grid_of("wm_sample_logits", rows, smp::THREADS);
    if (rows == 0) return;
    if (!logits || !uniforms || !tokens || !logp) fail("wm_sample_logits: null pointer");
    if ((uintptr_t)logits % (fp32 ? 4 : 2) ||
        ((uintptr_t)uniforms | (uintptr_t)temperature | (uintptr_t)top_k | (uintptr_t)top_p | (uintptr_t)min_p | (uintptr_t)tokens |
         (uintptr_t)logp) % 4)
      fail("wm_sample_logits: tensors must be aligned to their elements");
    const size_t need = wm_sample_logits_workspace_size(rows, vocab);
    if (need > 0 && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
      fail("wm_sample_logits: workspace too small or misaligned");
    int bits = 0;
    while ((1 << bits) < vocab) ++bits;
    const smp::Args a = {logits, rows, vocab, 62 - bits < 51 ? 62 - bits : 51, uniforms, temperature, top_k, top_p, min_p, tokens, logp};
    if (fp32) smp::launch<true>(a, workspace, as_stream(stream));
    else smp::launch<false>(a, workspace, as_stream(stream));
  });
}

}  // extern "C"
