// Runs of consecutive row elements, bf16 or fp32, moved 16 bytes at a time and computed with as fp32. Rows may
// start at any address that is aligned to their elements: the global 16-byte accesses of this GPU need no more
// than that, and aligned ones run as fast as through a type that promises 16 bytes. A row's elements behind
// its last whole 16 bytes are units of one element.
#pragma once

#include "wm_common.h"

namespace wm {

typedef uint32_t wm_u32x4_any __attribute__((ext_vector_type(4), aligned(2)));  // 16 bytes at 2-byte alignment

// The non-temporal forms are for rows that pass once and are more than the caches hold.
__device__ __forceinline__ wm_u32x4 load16(const void* p) {
  return *(const __attribute__((address_space(1))) wm_u32x4_any*)(p);
}
__device__ __forceinline__ wm_u32x4 load16_nt(const void* p) {
  return __builtin_nontemporal_load((const __attribute__((address_space(1))) wm_u32x4_any*)(p));
}
__device__ __forceinline__ void store16(void* p, wm_u32x4 v) { *(__attribute__((address_space(1))) wm_u32x4_any*)(p) = v; }
__device__ __forceinline__ void store16_nt(void* p, wm_u32x4 v) {
  __builtin_nontemporal_store((wm_u32x4_any)v, (__attribute__((address_space(1))) wm_u32x4_any*)(p));
}

typedef uint32_t wm_u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t wm_u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
__device__ __forceinline__ wm_u32x2 load8(const void* p) {
  return *(const __attribute__((address_space(1))) wm_u32x2_any*)(p);
}

// Two fp32 to bf16, to nearest even, by the one instruction that does it (V_CVT_PK_BF16_F32).
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const wm_bf16x2 v = {(__bf16)lo, (__bf16)hi};
  return bf16x2_to_bits(v);
}

// Sixteen bytes of a row (WIDE) or one element.
template <bool F32, bool WIDE>
struct RowUnit;

template <>
struct RowUnit<false, true> {
  static constexpr int N = 8;
  typedef uint16_t Elem;
  typedef wm_u32x4 Raw;
  static __device__ __forceinline__ Raw load(const Elem* p) { return load16(p); }
  static __device__ __forceinline__ Raw load_once(const Elem* p) { return load16_nt(p); }
  static __device__ __forceinline__ void store(Elem* p, Raw v) { store16(p, v); }
  static __device__ __forceinline__ void store_once(Elem* p, Raw v) { store16_nt(p, v); }
  static __device__ __forceinline__ void unpack(Raw v, float f[N]) {
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      f[2 * m] = __uint_as_float(v[m] << 16);
      f[2 * m + 1] = __uint_as_float(v[m] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ Raw pack(const float f[N]) {
    const Raw v = {pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7])};
    return v;
  }
};

template <>
struct RowUnit<false, false> {
  static constexpr int N = 1;
  typedef uint16_t Elem;
  typedef uint16_t Raw;
  static __device__ __forceinline__ Raw load(const Elem* p) { return *p; }
  static __device__ __forceinline__ Raw load_once(const Elem* p) { return *p; }
  static __device__ __forceinline__ void store(Elem* p, Raw v) { *p = v; }
  static __device__ __forceinline__ void store_once(Elem* p, Raw v) { *p = v; }
  static __device__ __forceinline__ void unpack(Raw v, float f[N]) { f[0] = bf16_bits_to_f32(v); }
  static __device__ __forceinline__ Raw pack(const float f[N]) { return (Raw)pack_bf16(f[0], 0.0f); }
};

template <>
struct RowUnit<true, true> {
  static constexpr int N = 4;
  typedef float Elem;
  typedef wm_u32x4 Raw;
  static __device__ __forceinline__ Raw load(const Elem* p) { return load16(p); }
  static __device__ __forceinline__ Raw load_once(const Elem* p) { return load16_nt(p); }
  static __device__ __forceinline__ void store(Elem* p, Raw v) { store16(p, v); }
  static __device__ __forceinline__ void store_once(Elem* p, Raw v) { store16_nt(p, v); }
  static __device__ __forceinline__ void unpack(Raw v, float f[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = __uint_as_float(v[i]);
  }
  static __device__ __forceinline__ Raw pack(const float f[N]) {
    const Raw v = {__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
    return v;
  }
};

template <>
struct RowUnit<true, false> {
  static constexpr int N = 1;
  typedef float Elem;
  typedef float Raw;
  static __device__ __forceinline__ Raw load(const Elem* p) { return *p; }
  static __device__ __forceinline__ Raw load_once(const Elem* p) { return *p; }
  static __device__ __forceinline__ void store(Elem* p, Raw v) { *p = v; }
  static __device__ __forceinline__ void store_once(Elem* p, Raw v) { *p = v; }
  static __device__ __forceinline__ void unpack(Raw v, float f[N]) { f[0] = v; }
  static __device__ __forceinline__ Raw pack(const float f[N]) { return f[0]; }
};

// A row of `hidden` elements as 16-byte units and the single elements behind them: unit c of `units` starts at
// element c < wide ? c * n : wide * n + c - wide.
struct RowUnits {
  int32_t wide, units;
};
inline RowUnits row_units(int64_t hidden, bool f32) {
  const int64_t n = f32 ? 4 : 8;
  return {(int32_t)(hidden / n), (int32_t)(hidden / n + hidden % n)};
}

// A launch of 256 threads over rows of `units` units: 2^log2 threads side by side in a row, 256 >> log2
// rows a block; grid (row blocks, unit blocks).
struct RowGrid {
  int log2;
  dim3 grid;
};
// Workgroups of one launch dimension, whose threads HIP counts in 32 bits.
inline unsigned grid_of(const char* name, int64_t blocks, int threads) {
  if (blocks * threads > 0xffffffffll) fail(std::string(name) + ": too many rows for one launch");
  return (unsigned)blocks;
}
inline RowGrid row_grid(const char* name, int64_t rows, int64_t units) {
  int log2 = 0;
  while (log2 < 8 && (1 << log2) < units) ++log2;
  const int64_t per = 256 >> log2;
  return {log2, dim3(grid_of(name, (rows + per - 1) / per, 256), (unsigned)((units + (1 << log2) - 1) >> log2))};
}

}  // namespace wm
