// From a model's logits to what sampling and acceptance take (wm_mtp_verify_greedy reads logits,
// wm_mtp_verify_rejection log-probabilities; the reference's sampler does these steps on the host before
// Sampler.verify, native_qwen.py:389-408). Per row, with c[v] how often token v is in the answer so far
// and seen[v] whether it is anywhere in the history:
//   l = seen[v] ? (l > 0 ? l / repetition : l * repetition) : l
//   l = l - frequency c[v] - presence [c[v] > 0] + bias[v]
//   l = allowed[v] ? l / temperature : -inf
//   log-probabilities: l - max l - log sum exp(l - max l), where -inf stays -inf
//
// The launch that writes is bound by HBM: the logits are read and the results written. Log-probabilities read the
// logits twice, once for the rows' maxima and sums (a chunk's go to the workspace) and once to write, which is
// less than writing the processed logits and going over them again. A workgroup owns a chunk of a row's
// vocabulary, a thread units of 4 tokens, so that a wave's stores are 1 KB without a gap (with 8 tokens a thread,
// 16 bytes in every 32 a store, 192 rows of 129,280 take 34 us to write, so 23). 192 rows of bf16 logits to
// log-probabilities with 2000 ids, 64 biases and a mask each take 49 us: 28 to write (50 MB read, 99 written; 22.5
// without lists and mask) and 24 for the maxima, which is no HBM time (50 MB, 2.1 TB/s): 15 are the chunks' own,
// each workgroup waiting for its 16 KB and then reducing them, three workgroups in turn a place, 2 the mask, and
// 8 the counting of 2000 ids by each of a row's 16 chunks.
//
// A workgroup counts its row's whole history (a few thousand tokens, from L2 after the first workgroup) into one
// LDS word per token of the chunk, so no count table exists in memory and nothing is left to clear; only for long
// histories of few rows the first launch keeps the words for the second. A word holds the answer's count (20 bits),
// whether a prompt holds the token (1) and the place of its bias in the list (11, the last one where a token is
// listed twice): integer additions and maxima, so the result does not depend on their order.
//
// The lists cost latency, not work: the ids' way from memory, three barriers, then the logits'. So the chunk's
// logits, the first ids of the history and the biases are all loaded before the first barrier. A history
// names a few percent of the tokens, which is enough for most waves to hold one and take the penalties' way:
// they are products with the penalty or its reciprocal, no divisions.
#include <cmath>

#include "row_units.h"

namespace wm {

// 256 threads read a long history twice as often: log-probabilities of 15 rows with 18000 ids each 19.5 us, with 512
// 15.3, with 1024 13.6, but these take 95 us for 192 rows of 300 ids, 512 56.
constexpr int LOGIT_THREADS = 512;
constexpr int LOGIT_UNIT = 4;  // a wave's units are 1 KB of results without a gap
constexpr int LOGIT_MAX_HISTORY = (1 << 20) - 1;
constexpr int LOGIT_MAX_BIASES = (1 << 11) - 1;
constexpr uint32_t LOGIT_COUNT = (1u << 20) - 1, LOGIT_PROMPT = 1u << 20;
constexpr int LOGIT_BIAS_SHIFT = 21;
constexpr float LOG2E = 1.4426950408889634f;

// The maximum of some values and their sum of exp(l - top). Of nothing but -inf the sum is 0; a NaN, which no
// maximum sees, makes the sum NaN.
struct LogitPart {
  float top, sum;
};

__device__ __forceinline__ float finite_top(float top) { return top == -INFINITY ? 0.0f : top; }

// Over a wave, in every lane.
__device__ __forceinline__ LogitPart wave_part(LogitPart p) {
  const float top = segment_max<64>(p.top);
  const float sum = p.sum * __builtin_amdgcn_exp2f((p.top - finite_top(top)) * LOG2E);
  return {top, segment_sum<64>(sum)};
}

// A row's values that do not depend on the token.
struct LogitRow {
  float rep, inv_rep, freq, pres, inv_temp;
  const float* bias;
  const uint8_t* mask;
};
__device__ __forceinline__ LogitRow logit_row(const wm_logit_rules& r, int row) {
  const float temp = r.temperature ? r.temperature[row] : 1.0f;
  // temperatures whose reciprocal is a normal number
  const bool scaled = temp >= 0x1p-126f && temp <= 0x1p126f;
  const float rep = r.repetition ? r.repetition[row] : 1.0f;
  return {rep, 1.0f / rep, r.frequency ? r.frequency[row] : 0.0f,
          r.presence ? r.presence[row] : 0.0f, scaled ? 1.0f / temp : 1.0f,
          r.bias_values ? r.bias_values + row * r.bias_stride : nullptr,
          r.mask ? (const uint8_t*)((const uint32_t*)r.mask + row * r.mask_stride) : nullptr};
}

// A unit's raw logits, `n` of them there.
template <bool F32>
struct LogitRaw;
template <>
struct LogitRaw<true> {
  wm_u32x4 a;
  __device__ __forceinline__ void load(const void* logits, int64_t at) { a = load16((const float*)logits + at); }
  __device__ __forceinline__ void load_part(const void* logits, int64_t at, int n) {
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] = e < n ? ((const uint32_t*)logits)[at + e] : 0u;
  }
  __device__ __forceinline__ void unpack(float l[LOGIT_UNIT]) const { RowUnit<true, true>::unpack(a, l); }
};
template <>
struct LogitRaw<false> {
  wm_u32x2 a;
  __device__ __forceinline__ void load(const void* logits, int64_t at) { a = load8((const uint16_t*)logits + at); }
  __device__ __forceinline__ void load_part(const void* logits, int64_t at, int n) {
    const uint16_t* p = (const uint16_t*)logits + at;
    a[0] = p[0] | (n > 1 ? (uint32_t)p[1] << 16 : 0u);
    a[1] = n > 2 ? p[2] : 0u;
  }
  __device__ __forceinline__ void unpack(float l[LOGIT_UNIT]) const {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      l[2 * m] = __uint_as_float(a[m] << 16);
      l[2 * m + 1] = __uint_as_float(a[m] & 0xffff0000u);
    }
  }
};

template <int CHUNK>
struct LogitWords {
  uint32_t word[CHUNK];
  float bias[LOGIT_THREADS];  // the first biases' values, for the threads that meet them
};

// A row's lists, and the first of them a thread has in flight: 16 ids by 16 bytes at any alignment, -1 where there
// are none, one of the last ids that make no 16 bytes, and a bias. Loaded before the logits, since a wait
// for a load is a wait for those before it, and without a use of what is loaded.
struct LogitIds {
  const int32_t *ids, *bias_ids;
  int len, prompt, biases, bias_id;
  float bias_value;
  uint32_t last;
  wm_u32x4 v[4];

  __device__ __forceinline__ void fetch(int j0) {
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int j = j0 + b * 4 * LOGIT_THREADS;
      v[b] = wm_u32x4{0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
      if (j + 4 <= len) v[b] = load16(ids + j);
    }
  }
  __device__ __forceinline__ void load(const wm_logit_rules& r, int row) {
    ids = r.history ? r.history + row * r.history_stride : nullptr;
    len = !ids ? 0 : r.lengths ? max(0, min(r.lengths[row], r.history_len)) : r.history_len;
    prompt = r.prompt_lengths ? r.prompt_lengths[row] : 0;
    bias_ids = r.bias_ids ? r.bias_ids + row * r.bias_stride : nullptr;
    biases = bias_ids ? r.biases : 0;
    bias_id = -1;
    bias_value = 0.0f;
    if ((int)threadIdx.x < biases) {
      bias_id = bias_ids[threadIdx.x];
      bias_value = r.bias_values[row * r.bias_stride + threadIdx.x];
    }
    last = 0xffffffffu;
    if ((int)threadIdx.x < len % 4) last = (uint32_t)ids[len - len % 4 + threadIdx.x];
    fetch(4 * threadIdx.x);
  }
};

// The words of a chunk of n tokens from lo on. Every thread of the workgroup calls it; ends with a barrier.
template <int CHUNK>
__device__ __forceinline__ void count_words(LogitIds& f, int lo, int n, LogitWords<CHUNK>& s) {
  uint32_t(&word)[CHUNK] = s.word;
#pragma unroll
  for (int i = 4 * threadIdx.x; i < CHUNK; i += 4 * LOGIT_THREADS) *reinterpret_cast<uint4*>(&word[i]) = make_uint4(0, 0, 0, 0);
  s.bias[threadIdx.x] = f.bias_value;
  __syncthreads();
  if (f.biases > 0) {
    for (int j = threadIdx.x; j < f.biases; j += LOGIT_THREADS) {
      const int id = j < LOGIT_THREADS ? f.bias_id : f.bias_ids[j];
      const uint32_t at = (uint32_t)id - (uint32_t)lo;  // a negative id is beyond every chunk's end
      if (at < (uint32_t)n) atomicMax(&word[at], (uint32_t)(j + 1) << LOGIT_BIAS_SHIFT);
    }
    __syncthreads();  // the words' lower bits are 0 until here
  }
  auto count = [&](uint32_t id, int j) {
    const uint32_t at = id - (uint32_t)lo;
    if (at < (uint32_t)n) {
      if (j < f.prompt) atomicOr(&word[at], LOGIT_PROMPT);
      else atomicAdd(&word[at], 1u);
    }
  };
  for (int j0 = 4 * threadIdx.x; j0 + 4 <= f.len; j0 += 16 * LOGIT_THREADS) {
    if (j0 >= 16 * LOGIT_THREADS) f.fetch(j0);  // (fetched a round ahead: more registers, 192 rows 62.3 -> 66.3 us)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int j = j0 + b * 4 * LOGIT_THREADS;
      if (j + 4 > f.len) break;
#pragma unroll
      for (int i = 0; i < 4; ++i) count(f.v[b][i], j + i);
    }
  }
  count(f.last, f.len - f.len % 4 + threadIdx.x);
  __syncthreads();
}

// Penalties and bias of a unit's logits, by their words.
__device__ __forceinline__ void apply_words(const uint4& a, const float* biases, const LogitRow& r, float l[LOGIT_UNIT]) {
  if ((a.x | a.y | a.z | a.w) == 0) return;
  const uint32_t w[LOGIT_UNIT] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int e = 0; e < LOGIT_UNIT; ++e) {
    const uint32_t count = w[e] & LOGIT_COUNT;
    if (w[e] & (LOGIT_COUNT | LOGIT_PROMPT)) l[e] *= l[e] > 0.0f ? r.inv_rep : r.rep;
    if (count) l[e] = l[e] - r.freq * (float)count - r.pres;
    const uint32_t j = w[e] >> LOGIT_BIAS_SHIFT;
    if (j) l[e] += biases && j <= LOGIT_THREADS ? biases[j - 1] : r.bias[j - 1];
  }
}

// Mask and temperature of a unit's logits; `bits` says which are allowed.
__device__ __forceinline__ void mask_and_scale(uint32_t bits, bool masked, float inv_temp, float l[LOGIT_UNIT]) {
  if (masked) {
#pragma unroll
    for (int e = 0; e < LOGIT_UNIT; ++e) {
      const uint32_t keep = (uint32_t)((int32_t)(bits << (31 - e)) >> 31);  // all ones where the token is allowed
      l[e] = __uint_as_float((__float_as_uint(l[e]) & keep) | (0xff800000u & ~keep));
    }
  }
#pragma unroll
  for (int e = 0; e < LOGIT_UNIT; ++e) l[e] *= inv_temp;  // finite and above 0: -inf stays
}

// A unit's results to out, `n` of them there.
__device__ __forceinline__ void store_unit(float* out, int64_t at, int n, const float l[LOGIT_UNIT]) {
  if (n >= LOGIT_UNIT) {
    store16_nt(out + at, RowUnit<true, true>::pack(l));
  } else {
#pragma unroll
    for (int e = 0; e < LOGIT_UNIT; ++e)
      if (e < n) out[at + e] = l[e];
  }
}

// A workgroup's chunk: the raw logits, and the mask's bytes that hold their tokens' bits. WHOLE: a chunk that the
// vocabulary does not end in, without a branch between the loads.
template <bool F32, int PER, bool WHOLE>
struct LogitChunk {
  LogitRaw<F32> raw[PER];
  uint8_t mask[PER];
  static constexpr int STEP = LOGIT_THREADS * LOGIT_UNIT;
  __device__ __forceinline__ void load(const void* logits, int64_t base, int lo, int n, const uint8_t* bytes) {
    const int at = threadIdx.x * LOGIT_UNIT;
    if (bytes) {
#pragma unroll
      for (int k = 0; k < PER; ++k)
        if (WHOLE || k * STEP + at < n) mask[k] = bytes[(lo + k * STEP + at) / 8];
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = k * STEP + at;
      if (WHOLE || i + LOGIT_UNIT <= n) raw[k].load(logits, base + i);
      else if (i < n) raw[k].load_part(logits, base + i, n - i);
    }
  }
  // The words of unit k.
  static __device__ __forceinline__ uint4 words_of(const uint32_t* words, int k) {
    return *reinterpret_cast<const uint4*>(words + k * STEP + threadIdx.x * LOGIT_UNIT);
  }
  // Logits of unit k after the rules, by its words; biases null: not in LDS.
  __device__ __forceinline__ void apply(int k, const uint4& words, const float* biases, const LogitRow& r,
                                        float l[LOGIT_UNIT]) const {
    raw[k].unpack(l);
    apply_words(words, biases, r, l);
    mask_and_scale((uint32_t)mask[k] >> (threadIdx.x % 2 * LOGIT_UNIT), r.mask != nullptr, r.inv_temp, l);
  }
};

// The maximum and the sum of a chunk: in part[0] .. of the waves.
template <bool F32, int PER, bool WHOLE, bool KEPT>
__device__ __forceinline__ void chunk_stats(const void* logits, int vocab, const wm_logit_rules& r, int row, int lo, int n,
                                            LogitWords<LOGIT_THREADS * LOGIT_UNIT * PER>& s, LogitPart* part,
                                            uint32_t* __restrict__ kept) {
  const bool lists = r.history || r.bias_ids;
  const LogitRow lr = logit_row(r, row);
  LogitIds f;
  if (lists) f.load(r, row);
  LogitChunk<F32, PER, WHOLE> c;
  c.load(logits, (int64_t)row * vocab + lo, lo, n, lr.mask);
  if (lists) count_words(f, lo, n, s);
  float l[PER][LOGIT_UNIT];
  LogitPart p = {-INFINITY, 0.0f};
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int i = (k * LOGIT_THREADS + threadIdx.x) * LOGIT_UNIT;
    if (WHOLE || i < n) {
      const uint4 w = lists ? c.words_of(s.word, k) : make_uint4(0, 0, 0, 0);
      if (KEPT) *reinterpret_cast<uint4*>(kept + i) = w;
      c.apply(k, w, s.bias, lr, l[k]);
#pragma unroll
      for (int e = 0; e < LOGIT_UNIT; ++e) {
        if (!WHOLE && i + e >= n) l[k][e] = -INFINITY;
        p.top = fmaxf(p.top, l[k][e]);
      }
    }
  }
  const float top = finite_top(p.top);
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    if (WHOLE || (k * LOGIT_THREADS + (int)threadIdx.x) * LOGIT_UNIT < n) {
#pragma unroll
      for (int e = 0; e < LOGIT_UNIT; ++e) p.sum += __builtin_amdgcn_exp2f((l[k][e] - top) * LOG2E);
    }
  }
  p = wave_part(p);
  if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = p;
}

// The chunks' maxima and sums, and their words where the write kernel takes them (KEPT).
template <bool F32, int PER, bool KEPT>
__global__ void __launch_bounds__(LOGIT_THREADS) logit_stats_kernel(const void* __restrict__ logits, int vocab, int chunks,
                                                                   wm_logit_rules r, LogitPart* __restrict__ parts,
                                                                   uint32_t* kept) {
  constexpr int CHUNK = LOGIT_THREADS * LOGIT_UNIT * PER;
  __shared__ __align__(16) LogitWords<CHUNK> s;
  __shared__ LogitPart part[LOGIT_THREADS / 64];
  const int row = blockIdx.x / chunks, lo = blockIdx.x % chunks * CHUNK, n = min(CHUNK, vocab - lo);
  if (KEPT) kept += (int64_t)blockIdx.x * CHUNK;
  if (n == CHUNK) chunk_stats<F32, PER, true, KEPT>(logits, vocab, r, row, lo, n, s, part, kept);
  else chunk_stats<F32, PER, false, KEPT>(logits, vocab, r, row, lo, n, s, part, kept);
  __syncthreads();
  if (threadIdx.x < 64) {
    LogitPart p = threadIdx.x < LOGIT_THREADS / 64 ? part[threadIdx.x] : LogitPart{-INFINITY, 0.0f};
    p = wave_part(p);
    if (threadIdx.x == 0) parts[blockIdx.x] = p;
  }
}

// A chunk's results. parts (nullable): the row's chunks, for log-probabilities. KEPT: the words are in memory.
template <bool F32, int PER, bool WHOLE, bool KEPT>
__device__ __forceinline__ void chunk_write(const void* logits, int vocab, int chunks, const wm_logit_rules& r, int row, int lo,
                                            int n, const LogitPart* __restrict__ parts, float* out,
                                            LogitWords<LOGIT_THREADS * LOGIT_UNIT * PER>& s, LogitPart* whole, const uint32_t* kept) {
  const int64_t base = (int64_t)row * vocab + lo;
  const bool lists = r.history || r.bias_ids;
  const LogitRow lr = logit_row(r, row);
  LogitIds f;
  if (!KEPT && lists) f.load(r, row);
  LogitPart o = {-INFINITY, 0.0f};
  if (parts && threadIdx.x < 64 && (int)threadIdx.x < chunks) o = parts[threadIdx.x];
  LogitChunk<F32, PER, WHOLE> c;
  uint4 words[PER];
  if (KEPT) {
#pragma unroll
    for (int k = 0; k < PER; ++k)
      if (WHOLE || (k * LOGIT_THREADS + (int)threadIdx.x) * LOGIT_UNIT < n) words[k] = c.words_of(kept, k);
  }
  c.load(logits, base, lo, n, lr.mask);
  if (parts && threadIdx.x < 64) {
    LogitPart p = o;
    for (int q = 64 + threadIdx.x; q < chunks; q += 64) {
      o = parts[q];
      const float top = fmaxf(p.top, o.top);
      p.sum = p.sum * __builtin_amdgcn_exp2f((p.top - finite_top(top)) * LOG2E) +
              o.sum * __builtin_amdgcn_exp2f((o.top - finite_top(top)) * LOG2E);
      p.top = top;
    }
    p = wave_part(p);
    if (threadIdx.x == 0) *whole = p;
  }
  if (!KEPT && lists) count_words(f, lo, n, s);
  else __syncthreads();
  const float top = parts ? finite_top(whole->top) : 0.0f, log_sum = parts ? logf(whole->sum) : 0.0f;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int i = (k * LOGIT_THREADS + threadIdx.x) * LOGIT_UNIT;
    if (!WHOLE && i >= n) break;
    float l[LOGIT_UNIT];
    if (!KEPT) words[k] = lists ? c.words_of(s.word, k) : make_uint4(0, 0, 0, 0);
    c.apply(k, words[k], KEPT ? nullptr : s.bias, lr, l);
    if (parts) {
#pragma unroll
      for (int e = 0; e < LOGIT_UNIT; ++e) l[e] = l[e] == -INFINITY ? l[e] : (l[e] - top) - log_sum;
    }
    store_unit(out, base + i, WHOLE ? LOGIT_UNIT : n - i, l);
  }
}

template <bool F32, int PER, bool KEPT>
__global__ void __launch_bounds__(LOGIT_THREADS) logit_write_kernel(const void* logits, int vocab, int chunks, wm_logit_rules r,
                                                                   const LogitPart* __restrict__ parts, float* out,
                                                                   const uint32_t* __restrict__ kept) {
  constexpr int CHUNK = LOGIT_THREADS * LOGIT_UNIT * PER;
  __shared__ __align__(16) LogitWords<CHUNK> s;
  __shared__ LogitPart whole;
  const int row = blockIdx.x / chunks, lo = blockIdx.x % chunks * CHUNK, n = min(CHUNK, vocab - lo);
  const LogitPart* mine = parts ? parts + (int64_t)row * chunks : nullptr;
  if (KEPT) kept += (int64_t)blockIdx.x * CHUNK;
  if (n == CHUNK) chunk_write<F32, PER, true, KEPT>(logits, vocab, chunks, r, row, lo, n, mine, out, s, &whole, kept);
  else chunk_write<F32, PER, false, KEPT>(logits, vocab, chunks, r, row, lo, n, mine, out, s, &whole, kept);
}

// Units of a thread, by how many workgroups the rows make: 64 rows of 129,280 23.2 us with four, 26.0 with two; one row
// 5.9 and 5.2.
static int logit_per(int64_t rows, int64_t vocab) {
  return rows * ((vocab + 8191) / 8192) >= 512 ? 4 : 2;
}
static int64_t logit_chunks(int64_t rows, int64_t vocab) {
  const int64_t chunk = LOGIT_THREADS * LOGIT_UNIT * logit_per(rows, vocab);
  return (vocab + chunk - 1) / chunk;
}

// Words that the chunks' statistics keep for the write kernel, which then reads no list: where a history is longer
// than a round of ids and the words are few. Log-probabilities of 4 rows with 32768 ids 12.4 us, counted twice 16.6;
// 15 rows of 18000 13.3 and 15.3, of 4000 11.9 and 11.7; 64 rows of 4096 32.9 and 27.7.
constexpr int LOGIT_KEEP_HISTORY = 16 * LOGIT_THREADS;
static int64_t logit_kept(int64_t rows, int64_t vocab) {
  const int64_t words = logit_chunks(rows, vocab) * rows * LOGIT_THREADS * LOGIT_UNIT * logit_per(rows, vocab);
  return words <= 1 << 22 ? words : 0;
}

template <bool F32, int PER>
static void process_logits(const void* logits, int rows, int vocab, const wm_logit_rules& r, float* out, LogitPart* parts,
                           uint32_t* kept, hipStream_t s) {
  const int chunks = (int)logit_chunks(rows, vocab);
  const dim3 grid((unsigned)(rows * chunks));
  if (parts) {
    if (kept)
      hipLaunchKernelGGL((logit_stats_kernel<F32, PER, true>), grid, dim3(LOGIT_THREADS), 0, s, logits, vocab, chunks, r, parts, kept);
    else
      hipLaunchKernelGGL((logit_stats_kernel<F32, PER, false>), grid, dim3(LOGIT_THREADS), 0, s, logits, vocab, chunks, r, parts, kept);
    check_launch("logit_stats");
  }
  if (kept)
    hipLaunchKernelGGL((logit_write_kernel<F32, PER, true>), grid, dim3(LOGIT_THREADS), 0, s, logits, vocab, chunks, r, parts, out,
                       kept);
  else
    hipLaunchKernelGGL((logit_write_kernel<F32, PER, false>), grid, dim3(LOGIT_THREADS), 0, s, logits, vocab, chunks, r, parts,
                       out, kept);
  check_launch("logit_write");
}

}  // namespace wm

using namespace wm;

extern "C" {

WM_EXPORT size_t wm_process_logits_workspace_size(int32_t rows, int32_t vocab) {
  if (rows < 0 || vocab < 1) return 0;
  return (size_t)(rows * logit_chunks(rows, vocab)) * sizeof(LogitPart) + 8 + logit_kept(rows, vocab) * sizeof(uint32_t);
}

WM_EXPORT int wm_process_logits(const void* logits, int32_t fp32, int32_t rows, int32_t vocab, const wm_logit_rules* rules,
                                int32_t log_probs, float* out, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded([&] {
    if (!rules) fail("wm_process_logits: null rules");
    if (rows < 0) fail("wm_process_logits: rows must not be negative");
    if (vocab < 1 || vocab > 1 << 22) fail("wm_process_logits: vocab must be in 1..4194304");
    grid_of("wm_process_logits", rows * logit_chunks(rows, vocab), LOGIT_THREADS);
    if (fp32 != 0 && fp32 != 1) fail("wm_process_logits: fp32 must be 0 (bf16 logits) or 1");
    const wm_logit_rules& r = *rules;
    if (r.history_len < 0 || r.history_len > LOGIT_MAX_HISTORY) fail("wm_process_logits: history_len must be in 0..1048575");
    if (r.biases < 0 || r.biases > LOGIT_MAX_BIASES) fail("wm_process_logits: biases must be in 0..2047");
    if (r.history_stride < 0 || r.bias_stride < 0 || r.mask_stride < 0) fail("wm_process_logits: strides must not be negative");
    if (!r.history && (r.lengths || r.prompt_lengths)) fail("wm_process_logits: lengths without a history");
    if ((r.bias_ids != nullptr) != (r.bias_values != nullptr)) fail("wm_process_logits: bias ids and values go together");
    if (rows == 0) return;
    if (!logits || !out) fail("wm_process_logits: null pointer");
    if ((uintptr_t)logits % (fp32 ? 4 : 2) || (uintptr_t)out % 4 || (uintptr_t)r.mask % 4)
      fail("wm_process_logits: tensors must be aligned to their elements");
    if (log_probs && (!workspace || workspace_bytes < wm_process_logits_workspace_size(rows, vocab) || (uintptr_t)workspace % 8))
      fail("wm_process_logits: workspace too small or misaligned");
    LogitPart* parts = log_probs ? (LogitPart*)workspace : nullptr;
    uint32_t* kept = nullptr;  // behind the parts, at 16 bytes
    if (log_probs && r.history && r.history_len > LOGIT_KEEP_HISTORY && logit_kept(rows, vocab) > 0)
      kept = (uint32_t*)(((uintptr_t)(parts + rows * logit_chunks(rows, vocab)) + 15) / 16 * 16);
    hipStream_t s = as_stream(stream);
    const int per = logit_per(rows, vocab);
#define WM_LOGITS(F, P) process_logits<F, P>(logits, rows, vocab, r, out, parts, kept, s)
    if (fp32) {
      if (per == 4) WM_LOGITS(true, 4); else WM_LOGITS(true, 2);
    } else {
      if (per == 4) WM_LOGITS(false, 4); else WM_LOGITS(false, 2);
    }
#undef WM_LOGITS
  });
}

}  // extern "C"
