// Rows in E4M3 with an fp32 scale for each 128 values, as the FP8 products take them: of rows as they are, of gated
// activations, and of the norm between a block's output and the next projection. For a block of 128 values v
//   s = max(max |v| / 448, 2^-126)           (pow2: the next power of two from that on)
//   q = e4m3(v / s), to nearest even         v / s as v times the reciprocal of s
// so that |q| <= 448, a block of zeros has q = 0, and a block with a NaN or an infinity has that scale. The values are
//   silu(g) u                                g, u clamped where there is a limit (the experts' activation)
//   r' rsqrt(mean(r'^2) + eps) (o + w)       r' = r + y, as it is stored
// in fp32 and rounded once, to E4M3: no bf16 row in between (x is a copy in bf16, for readers that take that).
// Dividing by a reciprocal moves a value by 2^-23 of it, which can only change q next to a rounding border.
//
// The silu is 0 for gates below -87.3, where it is less than 1.2e-36 and its exponential below the normal numbers.
//
// All are bound by HBM and pass every tensor once (kernels alone: 16,384 rows of 7168 bf16 62 us, 5.7 TB/s; the norm of 4001 tokens
// of 5120 with a bf16 residual and x 33 us, 5.6 TB/s; captured, 16,384 rows of 2 x 2048 to SwiGLU 44 us in bf16, 3.9 TB/s, and 59 in
// fp32, 5.1), the small ones by a launch and a chain of loads (one token of 7168
// 3.0 us, 64 rows of 2 x 2048 2.6). Sixteen lanes hold a block, 8 values a lane, so that the maximum is
// four moves within a row of lanes. The norm holds a token's row in registers like block_norm.
#include "norm_rows.h"

namespace wm {

constexpr float E4M3_MAX = 448.0f;
constexpr int FP8_BLOCK = 128;

typedef uint32_t wm_u32x2_byte __attribute__((ext_vector_type(2), aligned(1)));

// The largest of 16 lanes' bits. As integers a NaN's are above infinity's, and these above every number's.
__device__ __forceinline__ uint32_t block_max(uint32_t v) {
#define WM_MAX_STEP(CTRL) v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, false))
  WM_MAX_STEP(0xB1);   // quad_perm [1,0,3,2]: pairs
  WM_MAX_STEP(0x4E);   // quad_perm [2,3,0,1]: quads
  WM_MAX_STEP(0x141);  // row_half_mirror: 8 lanes
  WM_MAX_STEP(0x140);  // row_mirror: 16 lanes
#undef WM_MAX_STEP
  return v;
}

// The scale of a block from each lane's eight values; values behind a row's end are 0.
__device__ __forceinline__ float block_scale(const float v[8], bool pow2) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  top = block_max(top);
  uint32_t s = max(__float_as_uint(__uint_as_float(top) / E4M3_MAX), 0x00800000u);
  if (pow2 && s < 0x7f800000u) s = (s + 0x007fffffu) & 0x7f800000u;
  return __uint_as_float(s);
}

// Eight values in E4M3 (OCP), to nearest even.
__device__ __forceinline__ wm_u32x2 to_e4m3(const float v[8], float inv) {
  wm_u32x2 q;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    int w = 0;
    w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h] * inv, v[4 * h + 1] * inv, w, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h + 2] * inv, v[4 * h + 3] * inv, w, true);
    q[h] = (uint32_t)w;
  }
  return q;
}

template <bool WHOLE>
__device__ __forceinline__ void store_e4m3(uint8_t* p, int n, wm_u32x2 q) {
  if (WHOLE || n >= 8) {
    *(__attribute__((address_space(1))) wm_u32x2_byte*)(p) = q;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = (uint8_t)(q[i / 4] >> (8 * (i % 4)));
  }
}

struct Fp8Out {
  uint8_t* q;
  float* scales;
  int pow2;
};

// ---------------------------------------------------------------------------------- rows and gated activations

struct RowArgs {
  const void* x;    // [rows][width], or [rows][2 width]: the gate's half at gate_at, the other one's at width - gate_at
  int width, blocks, gate_at;
  float limit;      // 0: none
  int64_t units;    // rows * blocks
};

// 16 lanes a block. (Four blocks a group of lanes, their loads in flight together, took 4.0 us for 256 rows of 7168 and 65.2 for
// 16,384; one 3.3 and 64.5.)
template <bool F32, bool SWIGLU, bool WHOLE>
__global__ void __launch_bounds__(256) fp8_rows_kernel(RowArgs a, Fp8Out o) {
  const int lane = threadIdx.x % 16;
  const int64_t unit = (int64_t)blockIdx.x * 16 + threadIdx.x / 16;
  const int64_t row = unit / a.blocks;
  const int col = (int)(unit - row * a.blocks) * FP8_BLOCK + 8 * lane, n = a.width - col;
  const bool in = unit < a.units && n > 0;
  Row8<F32> x, up;
  x.clear();
  if (SWIGLU) up.clear();
  if (in) {
    if (SWIGLU) {
      const int64_t at = row * 2 * a.width + col;
      x.template load<WHOLE>(a.x, at + a.gate_at, n);
      up.template load<WHOLE>(a.x, at + (a.width - a.gate_at), n);
    } else {
      x.template load<WHOLE>(a.x, row * a.width + col, n);
    }
  }
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = x.get(i);
    if (SWIGLU) {
      float u = up.get(i);
      if (a.limit > 0.0f) {  // NaN passes
        v[i] = __builtin_elementwise_minimum(v[i], a.limit);
        u = __builtin_elementwise_maximum(__builtin_elementwise_minimum(u, a.limit), -a.limit);
      }
      v[i] = v[i] * sigmoid_f32(v[i]) * u;
    }
  }
  const float s = block_scale(v, o.pow2);
  if (in) {
    store_e4m3<WHOLE>(o.q + row * a.width + col, n, to_e4m3(v, 1.0f / s));
    if (lane == 0) o.scales[unit] = s;
  }
}

// ---------------------------------------------------------------------------------- norm

struct Fp8NormArgs {
  const void* residual;
  const uint16_t* y;       // null: nothing is added
  const uint16_t* weight;  // null: ones
  float offset, eps;
  int64_t tokens;
  int hidden;
  void* residual_out;  // null: not written
  uint16_t* x;         // null: not written
};

template <bool F32, int V, bool WHOLE, int GROUP, int THREADS>
__global__ void __launch_bounds__(THREADS) norm_fp8_kernel(Fp8NormArgs a, Fp8Out o) {
  __shared__ float part[2][1][16];
  if (GROUP == 0) clear_parts(&part[0][0][0], 32);
  const NormGroup<GROUP> at;
  const int H = a.hidden, blocks = (H + FP8_BLOCK - 1) / FP8_BLOCK;
  const RowMean mean(H);
  const float offset = a.weight ? a.offset : 0.0f;
  Weight8 w[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = at.column(v);
    if (c < H) w[v].template load<WHOLE>(a.weight, c, H - c);
  }
  int odd = 0;
  for (int64_t t = at.g; t < a.tokens; t += at.groups, odd ^= 1) {
    Row8<F32> raw[V];
    Row8<false> y[V];
    float r[V][8];
    float sum[1] = {0.0f};
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = at.column(v);
      raw[v].clear();
      y[v].clear();
      if (c < H) {
        raw[v].template load<WHOLE>(a.residual, t * H + c, H - c);
        if (a.y) y[v].template load<WHOLE>(a.y, t * H + c, H - c);
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = at.column(v);
#pragma unroll
      for (int i = 0; i < 8; ++i) r[v][i] = raw[v].get(i) + y[v].get(i);
      if (!F32) RowUnit<false, true>::unpack(RowUnit<false, true>::pack(r[v]), r[v]);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[0] = fmaf(r[v][i], r[v][i], sum[0]);
      if (a.residual_out && c < H) store8<WHOLE>(a.residual_out, F32, t * H + c, H - c, r[v]);
    }
    sum[0] *= mean.part;
    group_sums<1, GROUP>(sum, part[odd]);
    const float q = rsqrtf(sum[0] / mean.n + a.eps);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = at.column(v);
#pragma unroll
      for (int i = 0; i < 8; ++i) r[v][i] = c < H ? r[v][i] * (q * w[v].get(offset, i)) : 0.0f;
      if (!WHOLE) {
#pragma unroll
        for (int i = 0; i < 8; ++i) r[v][i] = c + i < H ? r[v][i] : 0.0f;  // 0 times a weight of infinity
      }
      const float s = block_scale(r[v], o.pow2);
      if (c < H) {
        store_e4m3<WHOLE>(o.q + t * H + c, H - c, to_e4m3(r[v], 1.0f / s));
        if (c % FP8_BLOCK == 0) o.scales[t * blocks + c / FP8_BLOCK] = s;
        if (a.x) store8<WHOLE>(a.x, false, t * H + c, H - c, r[v]);
      }
    }
  }
}

template <bool F32>
static void norm_fp8(const Fp8NormArgs& a, const Fp8Out& o, hipStream_t s) {
  const NormShape shape = norm_shape(a.hidden);
  const dim3 grid((unsigned)norm_blocks(a.tokens, shape, 64, 2)), threads(shape.threads);
#define WM_NORM_FP8(V, G, N)                                                                              \
  if (a.hidden % 8 == 0) hipLaunchKernelGGL((norm_fp8_kernel<F32, V, true, G, N>), grid, threads, 0, s, a, o); \
  else hipLaunchKernelGGL((norm_fp8_kernel<F32, V, false, G, N>), grid, threads, 0, s, a, o)
  if (shape.group == 16) { WM_NORM_FP8(1, 16, 256); }
  else if (shape.group == 64) { WM_NORM_FP8(1, 64, 256); }
  else if (shape.v == 2) { WM_NORM_FP8(2, 0, 1024); }
  else if (shape.threads > 512) { WM_NORM_FP8(1, 0, 1024); }
  else { WM_NORM_FP8(1, 0, 512); }
#undef WM_NORM_FP8
  check_launch("norm_fp8");
}

template <bool F32, bool SWIGLU, bool WHOLE>
static void fp8_rows(const RowArgs& a, const Fp8Out& o, hipStream_t s) {
  const dim3 grid(grid_of("wm_fp8_rows", (a.units + 15) / 16, 256));
  hipLaunchKernelGGL((fp8_rows_kernel<F32, SWIGLU, WHOLE>), grid, dim3(256), 0, s, a, o);
  check_launch("fp8_rows");
}

}  // namespace wm

using namespace wm;

extern "C" {

WM_EXPORT int wm_norm_fp8(const void* residual, int32_t fp32, const void* y, const void* weight, float weight_offset, float eps,
                          int32_t tokens, int32_t hidden, int32_t pow2, void* residual_out, void* q, float* scales, void* x,
                          void* stream) {
  return guarded([&] {
    if (tokens < 0) fail("wm_norm_fp8: tokens must not be negative");
    if (hidden < 1 || hidden > NORM_MAX_HIDDEN) fail("wm_norm_fp8: hidden must be in 1..16384");
    if (fp32 != 0 && fp32 != 1) fail("wm_norm_fp8: fp32 must be 0 (bf16 residual) or 1");
    if (pow2 != 0 && pow2 != 1) fail("wm_norm_fp8: pow2 must be 0 or 1");
    if (!(eps >= 0.0f)) fail("wm_norm_fp8: eps must not be negative");
    if (tokens == 0) return;
    if (!residual || !q || !scales) fail("wm_norm_fp8: null pointer");
    if (((uintptr_t)residual | (uintptr_t)residual_out) % (fp32 ? 4 : 2) || (uintptr_t)scales % 4 ||
        ((uintptr_t)y | (uintptr_t)weight | (uintptr_t)x) % 2)
      fail("wm_norm_fp8: tensors must be aligned to their elements");
    const Fp8NormArgs a = {residual, (const uint16_t*)y, (const uint16_t*)weight, weight_offset, eps, tokens, hidden, residual_out,
                           (uint16_t*)x};
    const Fp8Out o = {(uint8_t*)q, scales, pow2};
    if (fp32) norm_fp8<true>(a, o, as_stream(stream));
    else norm_fp8<false>(a, o, as_stream(stream));
  });
}

WM_EXPORT int wm_fp8_rows(const void* x, int32_t fp32, int32_t rows, int32_t width, int32_t swiglu, int32_t up_first, float limit,
                          int32_t pow2, void* q, float* scales, void* stream) {
  return guarded([&] {
    if (rows < 0) fail("wm_fp8_rows: rows must not be negative");
    if (width < 1 || width > 1 << 20) fail("wm_fp8_rows: width must be in 1..1048576");
    if (fp32 != 0 && fp32 != 1) fail("wm_fp8_rows: fp32 must be 0 (bf16) or 1");
    if (swiglu != 0 && swiglu != 1) fail("wm_fp8_rows: swiglu must be 0 or 1");
    if (up_first != 0 && up_first != 1) fail("wm_fp8_rows: up_first must be 0 or 1");
    if (pow2 != 0 && pow2 != 1) fail("wm_fp8_rows: pow2 must be 0 or 1");
    if (!(limit >= 0.0f)) fail("wm_fp8_rows: limit must not be negative");
    const int64_t blocks = (width + FP8_BLOCK - 1) / FP8_BLOCK, units = rows * blocks;
    grid_of("wm_fp8_rows", (units + 15) / 16, 256);
    if (rows == 0) return;
    if (!x || !q || !scales) fail("wm_fp8_rows: null pointer");
    if ((uintptr_t)x % (fp32 ? 4 : 2) || (uintptr_t)scales % 4) fail("wm_fp8_rows: tensors must be aligned to their elements");
    const RowArgs a = {x, width, (int)blocks, up_first ? width : 0, limit, units};
    const Fp8Out o = {(uint8_t*)q, scales, pow2};
    hipStream_t s = as_stream(stream);
#define WM_FP8_ROWS(F, G) if (width % 8 == 0) fp8_rows<F, G, true>(a, o, s); else fp8_rows<F, G, false>(a, o, s)
    if (fp32) {
      if (swiglu) { WM_FP8_ROWS(true, true); } else { WM_FP8_ROWS(true, false); }
    } else {
      if (swiglu) { WM_FP8_ROWS(false, true); } else { WM_FP8_ROWS(false, false); }
    }
#undef WM_FP8_ROWS
  });
}

}  // extern "C"
