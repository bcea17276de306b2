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
#include <cmath>

#include "row_units.h"

namespace wm {
namespace smp {

constexpr int MAX_VOCAB = 1 << 22;
constexpr int THREADS = 1024, WAVES = THREADS / 64;
constexpr int CHUNK = 8192;  // tokens whose weights are added up before the draw looks for its place

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
  __device__ __forceinline__ Rules(const Args& a, int row, float top_) : top(top_) {
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

// 2^x for x <= 0, to 2^-51 of it: x split into a whole number and a rest of at most 1/2, whose power is its
// series in the rest times ln 2. 0 from 2^-64 on, which no fixed-point weight holds.
__device__ __forceinline__ double exp2_f64(double x) {
  if (!(x > -64.0)) return 0.0;
  constexpr double LN2 = 0.6931471805599453;
  const double n = rint(x), f = (x - n) * LN2;
  double s = 1.0 / 479001600.0;
  s = fma(s, f, 1.0 / 39916800.0);
  s = fma(s, f, 1.0 / 3628800.0);
  s = fma(s, f, 1.0 / 362880.0);
  s = fma(s, f, 1.0 / 40320.0);
  s = fma(s, f, 1.0 / 5040.0);
  s = fma(s, f, 1.0 / 720.0);
  s = fma(s, f, 1.0 / 120.0);
  s = fma(s, f, 1.0 / 24.0);
  s = fma(s, f, 1.0 / 6.0);
  s = fma(s, f, 0.5);
  s = fma(s, f, 1.0);
  s = fma(s, f, 1.0);
  return ldexp(s, (int)n);
}

// e of a logit.
__device__ __forceinline__ double weight_of(float l, const Rules& r) {
  if (l == r.top) return 1.0;
  if (l == -INFINITY || r.top == INFINITY) return 0.0;
  return exp2_f64(((double)l - (double)r.top) * r.scale);
}
// e to a multiple of 2^-shift, as an integer: adding 2^52 leaves it in the sum's low bits (shift is at most 51).
__device__ __forceinline__ uint64_t fixed_of(double e, int shift) {
  const double v = ldexp(e, shift) + 0x1p52;
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
  uint32_t counts[256];
  uint64_t part[WAVES];
  float top[WAVES];
  uint64_t chunk[MAX_VOCAB / CHUNK];
  uint64_t bcast[3];
};

__device__ __forceinline__ uint64_t shfl_u64(uint64_t v, int from) {
  const uint32_t lo = __shfl((uint32_t)v, from, 64), hi = __shfl((uint32_t)(v >> 32), from, 64);
  return (uint64_t)hi << 32 | lo;
}
// Sum of the lanes up to this one.
__device__ __forceinline__ uint64_t wave_scan(uint64_t v) {
  const int lane = threadIdx.x % 64;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint64_t o = shfl_u64(v, lane >= d ? lane - d : lane);
    if (lane >= d) v += o;
  }
  return v;
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

template <bool F32>
__global__ void __launch_bounds__(THREADS) sample_kernel(Args a) {
  __shared__ Shared s;
  const int row = blockIdx.x;
  const void* p = (const uint8_t*)a.logits + (int64_t)row * a.vocab * (F32 ? 4 : 2);
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  // the largest logit; a NaN's key is the largest or the smallest
  uint32_t high = 0;
  bool nan = false;
  for (int i = threadIdx.x; i < a.vocab; i += THREADS) {
    const float l = logit<F32>(p, i);
    high = max(high, key_of(l));
    nan |= l != l;
  }
  for (int d = 32; d > 0; d /= 2) high = max(high, (uint32_t)__shfl_xor((int)high, d, 64));
  if (lane == 0) s.part[wave] = high;
  const bool any = __syncthreads_or(nan);
  for (int w = 0; w < WAVES; ++w) high = max(high, (uint32_t)s.part[w]);
  const float top = value_of(high);
  if (any || top == -INFINITY) {
    if (threadIdx.x == 0) a.tokens[row] = -1, a.logp[row] = NAN;
    return;
  }
  const Rules r(a, row, top);
  const Cut cut = row_cut<F32>(a, p, r, s);
  auto kept = [&](int i) -> uint64_t {
    const float l = logit<F32>(p, i);
    if (!cut.keeps(key_of(l), i)) return 0;
    const double e = weight_of(l, r);
    return e >= (double)r.m ? fixed_of(e, a.shift) : 0;
  };
  const int chunks = (a.vocab + CHUNK - 1) / CHUNK;
  uint64_t whole = 0;
  for (int c = 0; c < chunks; ++c) {
    uint64_t v = 0, total;
    for (int i = c * CHUNK + threadIdx.x; i < min((c + 1) * CHUNK, a.vocab); i += THREADS) v += kept(i);
    block_scan(v, s.part, total);
    if (threadIdx.x == 0) s.chunk[c] = total;
    whole += total;
  }
  const float u = a.uniforms[row];
  const uint64_t f = (uint64_t)((u > 0.0f ? fminf(u, 1.0f - 0x1p-24f) : 0.0f) * 0x1p64f);
  uint64_t want = __umul64hi(f, whole);  // floor(u whole), below the whole
  __syncthreads();
  int c = 0;
  while (want >= s.chunk[c]) want -= s.chunk[c++];
  constexpr int EACH = CHUNK / THREADS;
  const int first = c * CHUNK + (int)threadIdx.x * EACH;
  uint64_t v[EACH], mine = 0, total;
#pragma unroll
  for (int j = 0; j < EACH; ++j) mine += v[j] = first + j < a.vocab ? kept(first + j) : 0;
  uint64_t before = block_scan(mine, s.part, total);
  if (want >= before && want < before + mine) {
    int j = 0;
#pragma unroll
    for (int q = 0; q < EACH; ++q)
      if (want >= before + v[q] && j == q) before += v[q], j = q + 1;
    a.tokens[row] = first + j;
    const float l = logit<F32>(p, first + j);
    const double t = l == top ? 0.0 : ((double)l - (double)top) * r.scale;
    a.logp[row] = (float)((t - log2(ldexp((double)whole, -a.shift))) * 0.6931471805599453);
  }
}

}  // namespace smp
}  // namespace wm

using namespace wm;

extern "C" {

WM_EXPORT size_t wm_sample_logits_workspace_size(int32_t rows, int32_t vocab) { return 0; }

WM_EXPORT int wm_sample_logits(const void* logits, int32_t fp32, int32_t rows, int32_t vocab, const float* uniforms,
                               const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                               int32_t* tokens, float* logp, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded([&] {
    if (rows < 0) fail("wm_sample_logits: rows must not be negative");
    if (vocab < 1 || vocab > smp::MAX_VOCAB) fail("wm_sample_logits: vocab must be in 1..4194304");
    if (fp32 != 0 && fp32 != 1) fail("wm_sample_logits: fp32 must be 0 (bf16 logits) or 1");
    const unsigned grid = grid_of("wm_sample_logits", rows, smp::THREADS);
    if (rows == 0) return;
    if (!logits || !uniforms || !tokens || !logp) fail("wm_sample_logits: null pointer");
    if ((uintptr_t)logits % (fp32 ? 4 : 2) ||
        ((uintptr_t)uniforms | (uintptr_t)temperature | (uintptr_t)top_k | (uintptr_t)top_p | (uintptr_t)min_p | (uintptr_t)tokens |
         (uintptr_t)logp) % 4)
      fail("wm_sample_logits: tensors must be aligned to their elements");
    int bits = 0;
    while ((1 << bits) < vocab) ++bits;
    const smp::Args a = {logits, rows, vocab, 62 - bits < 51 ? 62 - bits : 51, uniforms, temperature, top_k, top_p, min_p, tokens, logp};
    if (fp32) hipLaunchKernelGGL((smp::sample_kernel<true>), dim3(grid), dim3(smp::THREADS), 0, as_stream(stream), a);
    else hipLaunchKernelGGL((smp::sample_kernel<false>), dim3(grid), dim3(smp::THREADS), 0, as_stream(stream), a);
    check_launch("sample_logits");
  });
}

}  // extern "C"
