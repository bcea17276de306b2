// Runs of consecutive row elements, bf16 or fp32, as 16-byte units or one by one (rows whose length or
// address does not allow 16 bytes), computed with as fp32.
#pragma once

#include "wm_common.h"

namespace wm {

template <bool F32, bool WIDE>
struct RowUnit;

template <>
struct RowUnit<false, true> {
  static constexpr int N = 8;
  typedef uint16_t Elem;
  typedef uint4 Raw;
  static __device__ __forceinline__ void unpack(const Raw& v, float f[N]) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      f[2 * m] = __uint_as_float(u[m] << 16);
      f[2 * m + 1] = __uint_as_float(u[m] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ Raw pack(const float f[N]) {
    uint32_t u[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) u[m] = f32_to_bf16_bits(f[2 * m]) | ((uint32_t)f32_to_bf16_bits(f[2 * m + 1]) << 16);
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
  static __device__ __forceinline__ Raw zero() { return make_uint4(0, 0, 0, 0); }
};

template <>
struct RowUnit<false, false> {
  static constexpr int N = 1;
  typedef uint16_t Elem;
  typedef uint16_t Raw;
  static __device__ __forceinline__ void unpack(const Raw& v, float f[N]) { f[0] = bf16_bits_to_f32(v); }
  static __device__ __forceinline__ Raw pack(const float f[N]) { return f32_to_bf16_bits(f[0]); }
  static __device__ __forceinline__ Raw zero() { return 0; }
};

template <>
struct RowUnit<true, true> {
  static constexpr int N = 4;
  typedef float Elem;
  typedef float4 Raw;
  static __device__ __forceinline__ void unpack(const Raw& v, float f[N]) {
    f[0] = v.x;
    f[1] = v.y;
    f[2] = v.z;
    f[3] = v.w;
  }
  static __device__ __forceinline__ Raw pack(const float f[N]) { return make_float4(f[0], f[1], f[2], f[3]); }
  static __device__ __forceinline__ Raw zero() { return make_float4(0, 0, 0, 0); }
};

template <>
struct RowUnit<true, false> {
  static constexpr int N = 1;
  typedef float Elem;
  typedef float Raw;
  static __device__ __forceinline__ void unpack(const Raw& v, float f[N]) { f[0] = v; }
  static __device__ __forceinline__ Raw pack(const float f[N]) { return f[0]; }
  static __device__ __forceinline__ Raw zero() { return 0.0f; }
};

// A unit with the non-temporal hint, for rows that pass once.
__device__ __forceinline__ uint4 load_once(const uint4* p) { return gload16_nt(p); }
__device__ __forceinline__ float4 load_once(const float4* p) {
  const uint4 v = gload16_nt(p);
  return make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
}
template <typename T>
__device__ __forceinline__ T load_once(const T* p) {
  return __builtin_nontemporal_load(p);
}
__device__ __forceinline__ void store_once(uint4* p, uint4 v) {
  const wm_u32x4 u = {v.x, v.y, v.z, v.w};
  __builtin_nontemporal_store(u, (__attribute__((address_space(1))) wm_u32x4*)(p));
}
__device__ __forceinline__ void store_once(float4* p, float4 v) {
  store_once(reinterpret_cast<uint4*>(p), make_uint4(__float_as_uint(v.x), __float_as_uint(v.y), __float_as_uint(v.z), __float_as_uint(v.w)));
}
__device__ __forceinline__ void store_once(uint32_t* p, uint32_t v) { __builtin_nontemporal_store(v, p); }
__device__ __forceinline__ void store_once(uint16_t* p, uint16_t v) { __builtin_nontemporal_store(v, p); }
__device__ __forceinline__ void store_once(float* p, float v) { __builtin_nontemporal_store(v, p); }

// A launch of 256 threads over rows of `units` units: 2^log2 threads side by side in a row, 256 >> log2
// rows a block; grid (row blocks, unit blocks).
struct RowGrid {
  int log2;
  dim3 grid;
};
inline RowGrid row_grid(int64_t rows, int64_t units) {
  int log2 = 0;
  while (log2 < 8 && (1 << log2) < units) ++log2;
  const int64_t per = 256 >> log2;
  return {log2, dim3((unsigned)((rows + per - 1) / per), (unsigned)((units + (1 << log2) - 1) >> log2))};
}

// Whether rows of `hidden` elements at these addresses can be moved in 16-byte units.
inline bool rows_wide(int64_t hidden, bool f32, std::initializer_list<const void*> rows) {
  uintptr_t all = 0;
  for (const void* p : rows) all |= (uintptr_t)p;
  return all % 16 == 0 && hidden % (f32 ? 4 : 8) == 0;
}

}  // namespace wm
