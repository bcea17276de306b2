// What the norm kernels share: eight elements of a row, sums over the threads that hold a row, a row's mean, a thread's
// place among the rows, and the launch shapes.
#pragma once

#include "row_units.h"

namespace wm {

constexpr int NORM_MAX_HIDDEN = 16384;

// Eight consecutive elements of a row as they are stored, from an address aligned to the elements; `n` of
// them are there, the others 0. WHOLE: all are, which the launch knows from hidden % 8 == 0.
template <bool F32>
struct Row8;
template <>
struct Row8<false> {
  wm_u32x4 a;
  template <bool WHOLE>
  __device__ __forceinline__ void load(const void* p, int64_t i, int n) {
    const uint16_t* q = (const uint16_t*)p + i;
    if (WHOLE || n >= 8) {
      a = load16(q);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) a[e] = (2 * e < n ? q[2 * e] : 0u) | (2 * e + 1 < n ? (uint32_t)q[2 * e + 1] << 16 : 0u);
    }
  }
  __device__ __forceinline__ void clear() { a = wm_u32x4{0, 0, 0, 0}; }
  // The compiler must not keep what it unpacked before this: the packed words are half the registers.
  __device__ __forceinline__ void repack() { asm volatile("" : "+v"(a)); }
  __device__ __forceinline__ float get(int i) const { return __uint_as_float(i % 2 ? a[i / 2] & 0xffff0000u : a[i / 2] << 16); }
};
template <>
struct Row8<true> {
  wm_u32x4 a, b;
  template <bool WHOLE>
  __device__ __forceinline__ void load(const void* p, int64_t i, int n) {
    const float* q = (const float*)p + i;
    if (WHOLE || n >= 8) {
      a = load16(q);
      b = load16(q + 4);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[e] = e < n ? __float_as_uint(q[e]) : 0u;
        b[e] = 4 + e < n ? __float_as_uint(q[4 + e]) : 0u;
      }
    }
  }
  __device__ __forceinline__ void clear() { a = b = wm_u32x4{0, 0, 0, 0}; }
  __device__ __forceinline__ void repack() {}
  __device__ __forceinline__ float get(int i) const { return __uint_as_float(i < 4 ? a[i] : b[i - 4]); }
};
template <bool WHOLE>
__device__ __forceinline__ void store8(void* p, bool f32, int64_t i, int n, const float f[8]) {
  if (f32) {
    float* q = (float*)p + i;
    if (WHOLE || n >= 8) {
      store16(q, RowUnit<true, true>::pack(f));
      store16(q + 4, RowUnit<true, true>::pack(f + 4));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n) q[e] = f[e];
    }
  } else {
    uint16_t* q = (uint16_t*)p + i;
    if (WHOLE || n >= 8) {
      store16(q, RowUnit<false, true>::pack(f));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n) q[e] = (uint16_t)pack_bf16(f[e], 0.0f);
    }
  }
}

// Sums N values over the group in a fixed order; every thread gets them. GROUP 0 is the workgroup (whole waves,
// 16 at most): `part` holds zeros behind the waves, and is written again only behind another sum's barrier:
// the callers alternate between two or three.
template <int N, int GROUP>
__device__ __forceinline__ void group_sums(float v[N], float (*part)[16]) {
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    v[n] = segment_sum<GROUP == 16 ? 16 : 64>(v[n]);
    if (GROUP == 0 && lane == 0) part[n][wave] = v[n];
  }
  if (GROUP != 0) return;
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) v[n] = segment_sum<16>(part[n][lane % 16]);
}
__device__ __forceinline__ void clear_parts(float* part, int n) {
  for (int i = threadIdx.x; i < n; i += blockDim.x) part[i] = 0.0f;
  __syncthreads();
}

// A row's mean from its threads' sums. They are added as parts of 2^-k, 2^k the power of two from `hidden` on: exact, and
// the row's sum is then not past fp32 where the mean is not.
struct RowMean {
  float part, n;  // n: hidden 2^-k
  __device__ __forceinline__ explicit RowMean(int hidden) {
    part = __uint_as_float((uint32_t)(127 - (hidden > 1 ? 32 - __clz(hidden - 1) : 0)) << 23);
    n = (float)hidden * part;
  }
};

// A thread's place: group g of all has tokens g, g + groups, ..; the thread columns 8 (v size + me) .. + 7 of each,
// v < V.
template <int GROUP>
struct NormGroup {
  int me, size;
  int64_t g, groups;
  __device__ __forceinline__ NormGroup() {
    size = GROUP == 0 ? (int)blockDim.x : GROUP;
    me = GROUP == 0 ? (int)threadIdx.x : (int)threadIdx.x % GROUP;
    g = GROUP == 0 ? blockIdx.x : blockIdx.x * (int64_t)(blockDim.x / GROUP) + threadIdx.x / GROUP;
    groups = GROUP == 0 ? gridDim.x : gridDim.x * (int64_t)(blockDim.x / GROUP);
  }
  __device__ __forceinline__ int column(int v) const { return (v * size + me) * 8; }
};

// The weights of a thread's columns as they are stored: ones without weights, which then have no offset.
struct Weight8 {
  Row8<false> w;
  template <bool WHOLE>
  __device__ __forceinline__ void load(const uint16_t* p, int c, int n) {
    w.a = wm_u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
    if (p) w.template load<WHOLE>(p, c, n);
  }
  __device__ __forceinline__ float get(float offset, int i) const { return w.get(i) + offset; }
};

// How a row is held: by `group` threads (0: a workgroup of `threads`), 8 v columns each. Short rows have 16 threads
// or a wave, four waves a workgroup (16000 tokens of 100, captured, 5.5 us and the gradients 12.6, with a workgroup a
// row 12.0 and 42); rows of more than 8192 columns 16 columns a thread, since a workgroup has 1024.
struct NormShape {
  int group, v, threads;
};
inline NormShape norm_shape(int hidden) {
  const int units = (hidden + 7) / 8;
  if (units <= 64) return {units <= 16 ? 16 : 64, 1, 256};
  const int v = units <= 1024 ? 1 : 2;
  return {0, v, ((units + v - 1) / v + 63) / 64 * 64};
}
inline int norm_groups_of_block(const NormShape& s) { return s.group ? s.threads / s.group : 1; }

// Workgroups of a pass by the waves a CU gets, `least` at least. (The forward pass with 64, twice what a CU holds,
// 152 us for 16384 tokens of 4096, with 32 157 us, with a workgroup a token 218.)
inline int norm_blocks(int64_t tokens, const NormShape& s, int waves, int least) {
  const int64_t per_cu = waves * 64 / s.threads, want = 256 * (per_cu > least ? per_cu : least);
  const int64_t most = (tokens + norm_groups_of_block(s) - 1) / norm_groups_of_block(s);
  return (int)(most < want ? most : want);
}

}  // namespace wm
