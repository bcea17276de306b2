// From a model's logits to what sampling and acceptance take (wm_mtp_verify_greedy reads logits,
// wm_mtp_verify_rejection log-probabilities; the reference's sampler does these steps on the host before
// Sampler.verify, native_qwen.py:389-408). Per row, with c[v] how often token v is in the answer so far
// and seen[v] whether it is anywhere in the history:
//   l = seen[v] ? (l > 0 ? l / repetition : l * repetition) : l
//   l = l - frequency c[v] - presence [c[v] > 0] + bias[v]
//   l = allowed[v] ? l / temperature : -inf
//   log-probabilities: l - max l - log sum exp(l - max l), where -inf stays -inf
//
// Bound by HBM: the logits are read and the results written. A workgroup owns a chunk of a row's
// vocabulary. It counts the row's whole history (a few thousand tokens, from L2 after the first
// workgroup) into one LDS word per token of the chunk, so no count table exists in memory and nothing
// is left to clear. A word holds the answer's count (20 bits), whether a prompt holds the token (1) and
// the place of its bias in the list (11, the last one where a token is listed twice): integer
// additions and maxima, so the result does not depend on their order.
#include "row_units.h"

namespace wm {

constexpr int LOGIT_CHUNK = 4096;
constexpr int LOGIT_THREADS = 256;
constexpr int LOGIT_MAX_HISTORY = (1 << 20) - 1;
constexpr int LOGIT_MAX_BIASES = (1 << 11) - 1;
constexpr uint32_t LOGIT_COUNT = (1u << 20) - 1, LOGIT_PROMPT = 1u << 20;
constexpr int LOGIT_BIAS_SHIFT = 21;

struct LogitPart {
  float top, sum;  // the chunk's maximum and its sum of exp(l - top)
};

__device__ __forceinline__ float block_max(float v, float* part) {
  v = segment_max<64>(v);
  if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = v;
  __syncthreads();
  v = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
  __syncthreads();
  return v;
}
__device__ __forceinline__ float block_sum(float v, float* part) {
  v = segment_sum<64>(v);
  if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = v;
  __syncthreads();
  v = (part[0] + part[1]) + (part[2] + part[3]);
  __syncthreads();
  return v;
}

template <bool F32, bool WIDE>
__global__ void __launch_bounds__(LOGIT_THREADS) logit_chunk_kernel(const void* logits, int vocab, int chunks,
                                                                   wm_logit_rules r, float* out,
                                                                   LogitPart* __restrict__ parts) {
  __shared__ uint32_t word[LOGIT_CHUNK];
  __shared__ float part[4];
  const int row = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
  const int lo = chunk * LOGIT_CHUNK, n = min(LOGIT_CHUNK, vocab - lo);
  for (int i = threadIdx.x; i < LOGIT_CHUNK; i += LOGIT_THREADS) word[i] = 0;
  __syncthreads();
  const float* bias = nullptr;
  if (r.bias_ids) {
    const int32_t* ids = r.bias_ids + row * r.bias_stride;
    bias = r.bias_values + row * r.bias_stride;
    for (int j = threadIdx.x; j < r.biases; j += LOGIT_THREADS) {
      const int id = ids[j];
      const uint32_t at = (uint32_t)id - (uint32_t)lo;
      if (id >= 0 && at < (uint32_t)n) atomicMax(&word[at], (uint32_t)(j + 1) << LOGIT_BIAS_SHIFT);
    }
    __syncthreads();
  }
  if (r.history) {
    const int32_t* ids = r.history + row * r.history_stride;
    const int len = r.lengths ? max(0, min(r.lengths[row], r.history_len)) : r.history_len;
    const int prompt = r.prompt_lengths ? r.prompt_lengths[row] : 0;
    for (int j = threadIdx.x; j < len; j += LOGIT_THREADS) {
      const int id = ids[j];
      const uint32_t at = (uint32_t)id - (uint32_t)lo;
      if (id >= 0 && at < (uint32_t)n) {
        if (j < prompt) atomicOr(&word[at], LOGIT_PROMPT);
        else atomicAdd(&word[at], 1u);
      }
    }
    __syncthreads();
  }
  const float rep = r.repetition ? r.repetition[row] : 1.0f;
  const float freq = r.frequency ? r.frequency[row] : 0.0f;
  const float pres = r.presence ? r.presence[row] : 0.0f;
  float temp = r.temperature ? r.temperature[row] : 1.0f;
  if (!(temp > 0.0f)) temp = 1.0f;
  const uint32_t* mask = r.mask ? (const uint32_t*)r.mask + row * r.mask_stride : nullptr;
  typedef RowUnit<F32, WIDE> U;
  typedef typename U::Raw Raw;
  constexpr int N = U::N, PER = LOGIT_CHUNK / LOGIT_THREADS / N;
  float v[PER][N];
  const int64_t base = (int64_t)row * vocab + lo;
  float top = -INFINITY;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int i = (k * LOGIT_THREADS + threadIdx.x) * N;
    if (i < n) {
      U::unpack(((const Raw*)((const typename U::Elem*)logits + base))[i / N], v[k]);
      const uint32_t bits = mask ? mask[(lo + i) / 32] >> ((lo + i) % 32) : 0xffffffffu;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const uint32_t w = word[i + e];
        const uint32_t count = w & LOGIT_COUNT;
        float l = v[k][e];
        if (w & (LOGIT_COUNT | LOGIT_PROMPT)) {
          l = l > 0.0f ? l / rep : l * rep;
          if (count) l = l - freq * (float)count - pres;
        }
        if (w >> LOGIT_BIAS_SHIFT) l += bias[(w >> LOGIT_BIAS_SHIFT) - 1];
        l = (bits >> e) & 1u ? l / temp : -INFINITY;
        v[k][e] = l;
        top = fmaxf(top, l);
      }
      if constexpr (N == 1) {
        out[base + i] = v[k][0];
      } else {
#pragma unroll
        for (int q = 0; q < N; q += 4)
          *reinterpret_cast<float4*>(out + base + i + q) = make_float4(v[k][q], v[k][q + 1], v[k][q + 2], v[k][q + 3]);
      }
    }
  }
  if (!parts) return;
  top = block_max(top, part);
  float sum = 0.0f;
  if (top > -INFINITY) {
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      if ((k * LOGIT_THREADS + threadIdx.x) * N < n) {
#pragma unroll
        for (int e = 0; e < N; ++e) sum += expf(v[k][e] - top);
      }
    }
  } else {
    // a chunk without an allowed token adds nothing, one of NaN (which no maximum sees) spoils its row
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      if ((k * LOGIT_THREADS + threadIdx.x) * N < n) {
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (isnan(v[k][e])) sum = v[k][e];
      }
    }
  }
  sum = block_sum(sum, part);
  if (threadIdx.x == 0) parts[blockIdx.x] = LogitPart{top, sum};
}

// The rows' logarithms of the sum, from their chunks, and out -= them.
__global__ void __launch_bounds__(LOGIT_THREADS) logit_norm_kernel(float* __restrict__ out, int vocab, int chunks,
                                                                  const LogitPart* __restrict__ parts) {
  __shared__ float part[4];
  const int row = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
  const LogitPart* mine = parts + (int64_t)row * chunks;
  float top = -INFINITY, sum = 0.0f;
  for (int c = threadIdx.x; c < chunks; c += LOGIT_THREADS) top = fmaxf(top, mine[c].top);
  top = block_max(top, part);
  for (int c = threadIdx.x; c < chunks; c += LOGIT_THREADS)
    sum += mine[c].top > -INFINITY ? mine[c].sum * expf(mine[c].top - top) : mine[c].sum;
  sum = block_sum(sum, part);
  const float log_sum = logf(sum);
  const int lo = chunk * LOGIT_CHUNK, n = min(LOGIT_CHUNK, vocab - lo);
  float* o = out + (int64_t)row * vocab + lo;
  for (int i = threadIdx.x; i < n; i += LOGIT_THREADS) {
    const float l = o[i];
    if (l != -INFINITY) o[i] = l - top - log_sum;
  }
}

}  // namespace wm

using namespace wm;

extern "C" {

WM_EXPORT size_t wm_process_logits_workspace_size(int32_t rows, int32_t vocab) {
  if (rows < 0 || vocab < 1) return 0;
  return (size_t)rows * ((vocab + LOGIT_CHUNK - 1) / LOGIT_CHUNK) * sizeof(LogitPart);
}

WM_EXPORT int wm_process_logits(const void* logits, int32_t fp32, int32_t rows, int32_t vocab, const wm_logit_rules* rules,
                                int32_t log_probs, float* out, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded([&] {
    if (!rules) fail("wm_process_logits: null rules");
    if (rows < 0) fail("wm_process_logits: rows must not be negative");
    if (vocab < 1 || vocab > 1 << 22) fail("wm_process_logits: vocab must be in 1..4194304");
    const int64_t chunks = (vocab + LOGIT_CHUNK - 1) / LOGIT_CHUNK;
    if (rows * chunks > (int64_t)0x7fffffff) fail("wm_process_logits: too many rows");
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
    const bool wide = rows_wide(vocab, fp32 != 0, {logits, out});
    LogitPart* parts = log_probs ? (LogitPart*)workspace : nullptr;
    hipStream_t s = as_stream(stream);
#define WM_LOGITS(F, W)                                                                                                      \
  hipLaunchKernelGGL((logit_chunk_kernel<F, W>), dim3((unsigned)(rows * chunks)), dim3(LOGIT_THREADS), 0, s, logits, vocab, \
                     (int)chunks, r, out, parts)
    if (fp32) {
      if (wide) WM_LOGITS(true, true); else WM_LOGITS(true, false);
    } else {
      if (wide) WM_LOGITS(false, true); else WM_LOGITS(false, false);
    }
#undef WM_LOGITS
    check_launch("logit_chunk");
    if (log_probs) {
      hipLaunchKernelGGL(logit_norm_kernel, dim3((unsigned)(rows * chunks)), dim3(LOGIT_THREADS), 0, s, out, vocab, (int)chunks,
                         parts);
      check_launch("logit_norm");
    }
  });
}

}  // extern "C"
