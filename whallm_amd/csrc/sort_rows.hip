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
// grid, and are rounded once.
#include <initializer_list>

#include "moe_internal.h"
#include "permute_device.h"
#include "row_units.h"

namespace wm {

constexpr int SORT_MAX_K = 64;

// ---- sort: the lists are there, x's rows go to theirs. Block (t / rows a block, unit block).
template <typename Unit>
__global__ void __launch_bounds__(256) sort_move_kernel(const Unit* __restrict__ x, int64_t tokens, int64_t units, int log2,
                                                       int k, int experts, const int32_t* __restrict__ inverse,
                                                       const int32_t* __restrict__ offsets, Unit* __restrict__ rows,
                                                       int32_t* __restrict__ order, int32_t* __restrict__ tiles,
                                                       const int32_t* __restrict__ tile_count, int64_t max_tiles) {
  const int64_t t = (int64_t)blockIdx.x * (256 >> log2) + (threadIdx.x >> log2);
  const int64_t c = ((int64_t)blockIdx.y << log2) + (threadIdx.x & ((1 << log2) - 1));
  const int64_t pairs = tokens * k;
  // Behind the ends: -1 in the lists (first unit block), zero rows.
  const int32_t present = offsets[experts];
  if (blockIdx.y == 0) {
    const int64_t step = (int64_t)gridDim.x * 256;
    const int64_t me = (int64_t)blockIdx.x * 256 + threadIdx.x;
    for (int64_t r = present + me; r < pairs; r += step) order[r] = -1;
    for (int64_t i = tile_count[0] + me; i < max_tiles; i += step) reinterpret_cast<int2*>(tiles)[i] = make_int2(-1, -1);
  }
  if (t >= tokens || c >= units) return;
  const Unit v = x[t * units + c];
  for (int j = 0; j < k; ++j) {
    const int64_t p = t * k + j;
    const int32_t r = inverse[p];
    if (r >= 0) rows[r * units + c] = v;
    if (p >= present) rows[p * units + c] = Unit{};
  }
}

template <typename Unit>
static void sort_move(const void* x, int64_t tokens, int64_t units, int k, int experts, int32_t* order, const int32_t* inverse,
                      const int32_t* offsets, void* rows, int32_t* tiles, const int32_t* tile_count, int64_t max_tiles,
                      hipStream_t s) {
  const RowGrid g = row_grid(tokens > 0 ? tokens : 1, units);  // without tokens the list of tiles still ends
  hipLaunchKernelGGL(sort_move_kernel<Unit>, g.grid, dim3(256), 0, s, (const Unit*)x, tokens, units, g.log2, k, experts,
                     inverse, offsets, (Unit*)rows, order, tiles, tile_count, max_tiles);
  check_launch("sort_move");
}

// ---- back (WEIGHTED) and the sort's gradient: a thread owns one unit of a token, sums its k rows.
template <bool F32, bool WIDE, bool WEIGHTED>
__global__ void __launch_bounds__(256) gather_sum_kernel(const void* __restrict__ rows_, const float* __restrict__ weights,
                                                        const int32_t* __restrict__ inverse, int64_t tokens, int64_t units,
                                                        int log2, int k, const void* add_, void* y_) {
  typedef RowUnit<F32, WIDE> U;
  typedef typename U::Raw Raw;
  const int64_t t = (int64_t)blockIdx.x * (256 >> log2) + (threadIdx.x >> log2);
  const int64_t c = ((int64_t)blockIdx.y << log2) + (threadIdx.x & ((1 << log2) - 1));
  if (t >= tokens || c >= units) return;
  const Raw* rows = (const Raw*)rows_;
  const uint32_t pairs = (uint32_t)(tokens * k);
  float acc[U::N] = {};
  for (int j = 0; j < k; ++j) {
    const int64_t p = t * k + j;
    const uint32_t r = (uint32_t)inverse[p];
    if (r >= pairs) continue;
    float f[U::N];
    U::unpack(rows[r * units + c], f);
    const float w = WEIGHTED ? weights[p] : 1.0f;
#pragma unroll
    for (int i = 0; i < U::N; ++i) acc[i] = WEIGHTED ? fmaf(w, f[i], acc[i]) : acc[i] + f[i];
  }
  if (add_) {
    float f[U::N];
    U::unpack(((const Raw*)add_)[t * units + c], f);
#pragma unroll
    for (int i = 0; i < U::N; ++i) acc[i] += f[i];
  }
  ((Raw*)y_)[t * units + c] = U::pack(acc);
}

template <bool WEIGHTED>
static void gather_sum(const void* rows, bool f32, const float* weights, const int32_t* inverse, int64_t tokens, int k,
                       int64_t hidden, const void* add, void* y, hipStream_t s) {
  const bool wide = rows_wide(hidden, f32, {rows, add, y});
  const int64_t units = wide ? hidden / (f32 ? 4 : 8) : hidden;
  const RowGrid g = row_grid(tokens, units);
#define WM_GS(F, W)                                                                                                     \
  hipLaunchKernelGGL((gather_sum_kernel<F, W, WEIGHTED>), g.grid, dim3(256), 0, s, rows, weights, inverse, tokens, units, \
                     g.log2, k, add, y)
  if (f32) {
    if (wide) WM_GS(true, true); else WM_GS(true, false);
  } else {
    if (wide) WM_GS(false, true); else WM_GS(false, false);
  }
#undef WM_GS
  check_launch("gather_sum");
}

// ---- the gradients of back: a block per token. Each thread holds the same units of dy for a batch of
// pairs, so a pair's row is read once, its gradient written, and its dot product summed over the block.
constexpr int BACK_BATCH = 8;

template <bool F32, bool WIDE>
__global__ void __launch_bounds__(256) back_grad_kernel(const void* __restrict__ dy_, const void* __restrict__ rows_,
                                                       const float* __restrict__ weights, const int32_t* __restrict__ inverse,
                                                       const int32_t* __restrict__ present_, int64_t tokens, int64_t units,
                                                       int k, void* __restrict__ drows_, float* __restrict__ dweights) {
  typedef RowUnit<F32, WIDE> U;
  typedef typename U::Raw Raw;
  __shared__ float part[BACK_BATCH][4];
  const int64_t t = blockIdx.x;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const Raw* dy = (const Raw*)dy_ + t * units;
  const Raw* rows = (const Raw*)rows_;
  Raw* drows = (Raw*)drows_;
  const uint32_t pairs = (uint32_t)(tokens * k);
  const int32_t present = *present_;
  for (int j0 = 0; j0 < k; j0 += BACK_BATCH) {
    uint32_t r[BACK_BATCH];
    float w[BACK_BATCH], dot[BACK_BATCH] = {};
#pragma unroll
    for (int q = 0; q < BACK_BATCH; ++q) {
      const int64_t p = t * k + j0 + q;
      r[q] = j0 + q < k ? (uint32_t)inverse[p] : 0xffffffffu;
      w[q] = j0 + q < k ? weights[p] : 0.0f;
    }
    for (int64_t c = threadIdx.x; c < units; c += 256) {
      float d[U::N];
      U::unpack(dy[c], d);
#pragma unroll
      for (int q = 0; q < BACK_BATCH; ++q) {
        if (r[q] < pairs) {
          float f[U::N], o[U::N];
          U::unpack(rows[r[q] * units + c], f);
#pragma unroll
          for (int i = 0; i < U::N; ++i) {
            dot[q] = fmaf(d[i], f[i], dot[q]);
            o[i] = w[q] * d[i];
          }
          drows[r[q] * units + c] = U::pack(o);
        }
        if (j0 + q < k && t * k + j0 + q >= present) drows[(t * k + j0 + q) * units + c] = U::zero();
      }
    }
#pragma unroll
    for (int q = 0; q < BACK_BATCH; ++q) {
      const float v = segment_sum<64>(dot[q]);
      if (lane == 0) part[q][wave] = v;
    }
    __syncthreads();
    if (threadIdx.x < BACK_BATCH && j0 + (int)threadIdx.x < k) {
      const float* v = part[threadIdx.x];
      dweights[t * k + j0 + threadIdx.x] = (v[0] + v[1]) + (v[2] + v[3]);
    }
    __syncthreads();
  }
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
  if (tokens < 0 || k < 1 || experts < 1) return 0;
  return wm_permute_workspace_size((int64_t)tokens * k, experts);
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
    if (!offsets || !tiles || !tile_count || !workspace || (pairs > 0 && (!x || !indices || !rows || !order || !inverse)))
      fail("wm_sort_tokens: null pointer");
    if (((uintptr_t)x | (uintptr_t)rows) % (fp32 ? 4 : 2) || (uintptr_t)tiles % 8)
      fail("wm_sort_tokens: rows must be aligned to their elements and tiles to 8 bytes");
    if (workspace_bytes < wm_sort_tokens_workspace_size(tokens, k, experts)) fail("wm_sort_tokens: workspace too small");
    hipStream_t s = as_stream(stream);
    const PermuteWorkspace ws = permute_workspace(workspace, pairs, experts);
    permute_count(indices, pairs, experts, ws, s);
    permute_lists(indices, pairs, experts, tile_rows, 0, order, inverse, nullptr, 1, offsets, tiles, nullptr, tile_count, ws, s);
    const int64_t bytes = (int64_t)hidden * (fp32 ? 4 : 2);
    const int64_t max_tiles = (pairs + tile_rows - 1) / tile_rows + experts;
    const uintptr_t at = (uintptr_t)x | (uintptr_t)rows | (uintptr_t)bytes;
    if (at % 16 == 0)
      sort_move<uint4>(x, tokens, bytes / 16, k, experts, order, inverse, offsets, rows, tiles, tile_count, max_tiles, s);
    else if (at % 4 == 0)
      sort_move<uint32_t>(x, tokens, bytes / 4, k, experts, order, inverse, offsets, rows, tiles, tile_count, max_tiles, s);
    else
      sort_move<uint16_t>(x, tokens, bytes / 2, k, experts, order, inverse, offsets, rows, tiles, tile_count, max_tiles, s);
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
    const bool f32 = fp32 != 0, wide = rows_wide(hidden, f32, {dy, rows, drows});
    const int64_t units = wide ? hidden / (f32 ? 4 : 8) : hidden;
    hipStream_t s = as_stream(stream);
#define WM_BG(F, W)                                                                                                      \
  hipLaunchKernelGGL((back_grad_kernel<F, W>), dim3((unsigned)tokens), dim3(256), 0, s, dy, rows, weights, inverse, present, \
                     (int64_t)tokens, units, k, drows, dweights)
    if (f32) {
      if (wide) WM_BG(true, true); else WM_BG(true, false);
    } else {
      if (wide) WM_BG(false, true); else WM_BG(false, false);
    }
#undef WM_BG
    check_launch("back_grad");
  });
}

}  // extern "C"
