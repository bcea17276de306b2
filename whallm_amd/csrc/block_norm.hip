// The norms around a block, with its gate and residual scale, and their gradients. For a token with
// residual r and block output y, o the weights' offset:
//   z = y rsqrt(mean(y^2) + eps) (o + w_post)      (or z = y)
//   r' = r + s g z                                 g: 1, or per token, channel or element, plain or sigmoid
//   x = r' rsqrt(mean(r'^2) + eps) (o + w_pre)     r' as it is stored
// the residual add and norm of a decoder layer (DecoderLayer.feed_forward, qwen4_exp.py:1127-1149) for
// layers that also norm, gate or scale what a block adds. With q and p the two reciprocal roots and
// a = dx (o + w_pre):
//   dr' = dr_out + q a - r' q^3 mean(a r')         dr = dr'         dw_pre = sum_t dx r' q
//   b = s g dr',  c = b (o + w_post)               dy = p c - y p^3 mean(c y)     dw_post = sum_t b y p
//   dg = s dr' z (by sigmoid'), summed over what g is broadcast over
//
// Bound by HBM: every tensor passes once. A workgroup holds a token's row in registers (a thread has VEC
// consecutive columns, V times), sums over the row twice at most, and goes on to the next token with the
// weights still in registers. Sums over tokens (weight gradients) stay in the threads' registers, go to
// the workspace once per workgroup and are added up by a second launch in the workgroups' order. All
// arithmetic is fp32; bf16 outputs are rounded once, from values that no earlier rounding touched but
// r''s own (x is the norm of the residual that the next block reads).
#include "wm_common.h"

namespace wm {

constexpr int NORM_MAX_HIDDEN = 16384;
enum { GATE_NONE = 0, GATE_TOKEN = 1, GATE_CHANNEL = 2, GATE_FULL = 3 };

// VEC consecutive elements from index i: bf16, or fp32.
template <int VEC>
__device__ __forceinline__ void load_bf16(const void* p, int64_t i, float f[VEC]) {
  if constexpr (VEC == 8) {
    const uint4 v = *reinterpret_cast<const uint4*>((const uint16_t*)p + i);
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      f[2 * m] = __uint_as_float(u[m] << 16);
      f[2 * m + 1] = __uint_as_float(u[m] & 0xffff0000u);
    }
  } else {
    f[0] = bf16_bits_to_f32(((const uint16_t*)p)[i]);
  }
}
template <int VEC>
__device__ __forceinline__ void load_f32(const void* p, int64_t i, float f[VEC]) {
  if constexpr (VEC == 8) {
    const float4 a = *reinterpret_cast<const float4*>((const float*)p + i);
    const float4 b = *reinterpret_cast<const float4*>((const float*)p + i + 4);
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  } else {
    f[0] = ((const float*)p)[i];
  }
}
template <int VEC>
__device__ __forceinline__ void load_any(const void* p, bool f32, int64_t i, float f[VEC]) {
  if (f32) load_f32<VEC>(p, i, f); else load_bf16<VEC>(p, i, f);
}
template <int VEC>
__device__ __forceinline__ void store_bf16(void* p, int64_t i, const float f[VEC]) {
  if constexpr (VEC == 8) {
    uint32_t u[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) u[m] = f32_to_bf16_bits(f[2 * m]) | ((uint32_t)f32_to_bf16_bits(f[2 * m + 1]) << 16);
    *reinterpret_cast<uint4*>((uint16_t*)p + i) = make_uint4(u[0], u[1], u[2], u[3]);
  } else {
    ((uint16_t*)p)[i] = f32_to_bf16_bits(f[0]);
  }
}
template <int VEC>
__device__ __forceinline__ void store_any(void* p, bool f32, int64_t i, const float f[VEC]) {
  if (!f32) {
    store_bf16<VEC>(p, i, f);
  } else if constexpr (VEC == 8) {
    *reinterpret_cast<float4*>((float*)p + i) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4*>((float*)p + i + 4) = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    ((float*)p)[i] = f[0];
  }
}

__device__ __forceinline__ float sigmoid_f32(float v) { return 1.0f / (1.0f + expf(-v)); }

// Sums N values over the workgroup (whole waves, 16 at most) in a fixed order; every thread gets them.
// `part` is not used again before every thread is past this sum: the caller alternates two.
template <int N>
__device__ __forceinline__ void block_sums(float v[N], float (*part)[16]) {
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, waves = blockDim.x / 64;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    v[n] = segment_sum<64>(v[n]);
    if (lane == 0) part[n][wave] = v[n];
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    float s = part[n][0];
    for (int w = 1; w < waves; ++w) s += part[n][w];
    v[n] = s;
  }
}

struct NormArgs {
  const void* residual;  // forward: r; backward: r' (residual_out)
  const uint16_t* y;
  const uint16_t* post;
  const uint16_t* pre;
  const void* gate;
  float offset, scale, eps;
  int post_norm, gate_kind, gate_f32, gate_sigmoid;
  int64_t tokens;
  int hidden;
};

// The gate of a thread's columns: its value (through the sigmoid) for element (t, c).
template <int VEC>
__device__ __forceinline__ void gate_values(const NormArgs& a, int64_t t, int c, float g[VEC]) {
  if (a.gate_kind == GATE_NONE) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) g[i] = 1.0f;
    return;
  }
  if (a.gate_kind == GATE_TOKEN) {
    float v[1];
    load_any<1>(a.gate, a.gate_f32, t, v);
    if (a.gate_sigmoid) v[0] = sigmoid_f32(v[0]);
#pragma unroll
    for (int i = 0; i < VEC; ++i) g[i] = v[0];
    return;
  }
  load_any<VEC>(a.gate, a.gate_f32, (a.gate_kind == GATE_FULL ? t * a.hidden : 0) + c, g);
  if (a.gate_sigmoid) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) g[i] = sigmoid_f32(g[i]);
  }
}

// o + w for a thread's columns, 1 without weights.
template <int VEC>
__device__ __forceinline__ void norm_weights(const uint16_t* w, float offset, int c, float f[VEC]) {
  if (!w) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = 1.0f;
    return;
  }
  load_bf16<VEC>(w, c, f);
#pragma unroll
  for (int i = 0; i < VEC; ++i) f[i] += offset;
}

template <bool F32, int VEC, int V>
__global__ void __launch_bounds__(1024) block_norm_kernel(NormArgs a, void* residual_out, uint16_t* __restrict__ x) {
  __shared__ float part[2][1][16];
  const int H = a.hidden;
  float wpost[V][VEC], wpre[V][VEC];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = (v * blockDim.x + threadIdx.x) * VEC;
    if (c < H) {
      norm_weights<VEC>(a.post, a.offset, c, wpost[v]);
      norm_weights<VEC>(a.pre, a.offset, c, wpre[v]);
    }
  }
  for (int64_t t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    float r[V][VEC], y[V][VEC];
    float sum[1] = {0.0f};
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (v * blockDim.x + threadIdx.x) * VEC;
      if (c < H) {
        load_any<VEC>(a.residual, F32, t * H + c, r[v]);
        load_bf16<VEC>(a.y, t * H + c, y[v]);
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum[0] = fmaf(y[v][i], y[v][i], sum[0]);
      }
    }
    float p = 1.0f;
    if (a.post_norm) {
      block_sums<1>(sum, part[0]);
      p = rsqrtf(sum[0] / (float)H + a.eps);
    }
    sum[0] = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (v * blockDim.x + threadIdx.x) * VEC;
      if (c < H) {
        float g[VEC];
        gate_values<VEC>(a, t, c, g);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          r[v][i] = fmaf(a.scale * g[i], y[v][i] * p * wpost[v][i], r[v][i]);
          if (!F32) r[v][i] = bf16_bits_to_f32(f32_to_bf16_bits(r[v][i]));
          sum[0] = fmaf(r[v][i], r[v][i], sum[0]);
        }
        store_any<VEC>(residual_out, F32, t * H + c, r[v]);
      }
    }
    block_sums<1>(sum, part[1]);
    const float q = rsqrtf(sum[0] / (float)H + a.eps);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (v * blockDim.x + threadIdx.x) * VEC;
      if (c < H) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) r[v][i] *= q * wpre[v][i];
        store_bf16<VEC>(x, t * H + c, r[v]);
      }
    }
    __syncthreads();  // part is free again
  }
}

struct NormGrads {
  const uint16_t* dx;
  const void* dres;  // null: zero
  void* dr;
  uint16_t* dy;
  void* dgate;    // token: fp32 [T]; full: in the gate's type
  float* partial;  // [workgroups][3][H]: post, pre, channel gate
};

template <bool F32, int VEC, int V>
__global__ void __launch_bounds__(1024) block_norm_grad_kernel(NormArgs a, NormGrads d) {
  __shared__ float part[2][3][16];
  const int H = a.hidden;
  float wpost[V][VEC], wpre[V][VEC], dpost[V][VEC], dpre[V][VEC], dch[V][VEC];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = (v * blockDim.x + threadIdx.x) * VEC;
    if (c < H) {
      norm_weights<VEC>(a.post, a.offset, c, wpost[v]);
      norm_weights<VEC>(a.pre, a.offset, c, wpre[v]);
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) dpost[v][i] = dpre[v][i] = dch[v][i] = 0.0f;
  }
  const float inv = 1.0f / (float)H;
  for (int64_t t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    float r[V][VEC], y[V][VEC], dx[V][VEC], dr[V][VEC];
    float sum[3] = {0.0f, 0.0f, 0.0f};  // r'^2, a r', y^2
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (v * blockDim.x + threadIdx.x) * VEC;
      if (c < H) {
        load_any<VEC>(a.residual, F32, t * H + c, r[v]);
        load_bf16<VEC>(d.dx, t * H + c, dx[v]);
        load_bf16<VEC>(a.y, t * H + c, y[v]);
        if (d.dres) {
          load_any<VEC>(d.dres, F32, t * H + c, dr[v]);
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i) dr[v][i] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          sum[0] = fmaf(r[v][i], r[v][i], sum[0]);
          sum[1] = fmaf(dx[v][i] * wpre[v][i], r[v][i], sum[1]);
          sum[2] = fmaf(y[v][i], y[v][i], sum[2]);
        }
      }
    }
    block_sums<3>(sum, part[0]);
    const float q = rsqrtf(sum[0] * inv + a.eps);
    const float p = a.post_norm ? rsqrtf(sum[2] * inv + a.eps) : 1.0f;
    const float k1 = q * q * q * (sum[1] * inv);
    float sum2[2] = {0.0f, 0.0f};  // c y, the token's gate gradient
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (v * blockDim.x + threadIdx.x) * VEC;
      if (c < H) {
        float g[VEC], dg[VEC];
        gate_values<VEC>(a, t, c, g);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          dr[v][i] += fmaf(q, dx[v][i] * wpre[v][i], -r[v][i] * k1);
          dpre[v][i] = fmaf(dx[v][i] * q, r[v][i], dpre[v][i]);
          const float n = y[v][i] * p;
          const float sdr = a.scale * dr[v][i];
          dg[i] = sdr * n * wpost[v][i] * (a.gate_sigmoid ? g[i] * (1.0f - g[i]) : 1.0f);
          const float b = sdr * g[i];
          dpost[v][i] = fmaf(b, n, dpost[v][i]);
          dch[v][i] += dg[i];
          sum2[1] += dg[i];
          dx[v][i] = b * wpost[v][i];  // c from here on
          sum2[0] = fmaf(dx[v][i], y[v][i], sum2[0]);
        }
        store_any<VEC>(d.dr, F32, t * H + c, dr[v]);
        if (a.gate_kind == GATE_FULL) store_any<VEC>(d.dgate, a.gate_f32, t * H + c, dg);
      }
    }
    block_sums<2>(sum2, part[1]);
    const float k2 = a.post_norm ? p * p * p * (sum2[0] * inv) : 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (v * blockDim.x + threadIdx.x) * VEC;
      if (c < H) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) dx[v][i] = fmaf(p, dx[v][i], -y[v][i] * k2);
        store_bf16<VEC>(d.dy, t * H + c, dx[v]);
      }
    }
    if (a.gate_kind == GATE_TOKEN && threadIdx.x == 0) ((float*)d.dgate)[t] = sum2[1];
    __syncthreads();  // part is free again
  }
  float* out = d.partial + (int64_t)blockIdx.x * 3 * H;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = (v * blockDim.x + threadIdx.x) * VEC;
    if (c < H) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        if (a.post) out[c + i] = dpost[v][i];
        if (a.pre) out[H + c + i] = dpre[v][i];
        if (a.gate_kind == GATE_CHANNEL) out[2 * H + c + i] = dch[v][i];
      }
    }
  }
}

// out[which][c] = the sum of partial[b][which][c] over the workgroups: 16 columns x 16 slices of workgroups
// a block, then the slices in order.
__global__ void __launch_bounds__(256) norm_columns_kernel(const float* __restrict__ partial, int blocks, int hidden,
                                                          float* dpost, float* dpre, float* dgate) {
  __shared__ float slice[16][17];
  float* out = blockIdx.y == 0 ? dpost : blockIdx.y == 1 ? dpre : dgate;
  if (!out) return;
  const int col = threadIdx.x % 16, part = threadIdx.x / 16;
  const int c = blockIdx.x * 16 + col;
  float sum = 0.0f;
  if (c < hidden)
    for (int b = part; b < blocks; b += 16) sum += partial[((int64_t)b * 3 + blockIdx.y) * hidden + c];
  slice[part][col] = sum;
  __syncthreads();
  if (part == 0 && c < hidden) {
    for (int s = 1; s < 16; ++s) sum += slice[s][col];
    out[c] = sum;
  }
}

// Workgroups of the gradient pass: each adds a row to the second launch's work.
static int norm_grad_blocks(int64_t tokens) { return (int)(tokens < 512 ? tokens : 512); }

static NormArgs norm_args(const char* name, const wm_block_norm_form* f, const void* residual, const void* y, int tokens,
                          int hidden) {
  const std::string n(name);
  if (!f) fail(n + ": null form");
  if (tokens < 0) fail(n + ": tokens must not be negative");
  if (hidden < 1 || hidden > NORM_MAX_HIDDEN) fail(n + ": hidden must be in 1..16384");
  if (f->gate_kind < GATE_NONE || f->gate_kind > GATE_FULL) fail(n + ": gate_kind must be in 0..3");
  const bool empty = tokens == 0 && (f->gate_kind == GATE_TOKEN || f->gate_kind == GATE_FULL);  // a gate of no values
  if (!empty && (f->gate_kind != GATE_NONE) != (f->gate != nullptr)) fail(n + ": a gate and its kind go together");
  if (f->post_weight && !f->post_norm) fail(n + ": a post weight needs the post norm");
  if (!(f->eps >= 0.0f)) fail(n + ": eps must not be negative");
  if (tokens > 0 && (!residual || !y)) fail(n + ": null pointer");
  return {residual, (const uint16_t*)y, (const uint16_t*)f->post_weight, (const uint16_t*)f->pre_weight, f->gate,
          f->weight_offset, f->scale, f->eps, f->post_norm != 0, f->gate_kind, f->gate_fp32 != 0, f->gate_sigmoid != 0,
          tokens, hidden};
}

// Elements of `f32` tensors aligned to themselves; returns whether all rows can be read 16 bytes at a time.
static bool norm_aligned(const char* name, const wm_block_norm_form* f, int hidden, std::initializer_list<const void*> bf16,
                         std::initializer_list<const void*> residuals, const void* f32_or_null, const void* gate2) {
  uintptr_t all = (uintptr_t)f->post_weight | (uintptr_t)f->pre_weight, wide = all;
  for (const void* p : bf16) all |= (uintptr_t)p;
  wide |= all;
  uintptr_t res = 0, gate = (uintptr_t)f->gate | (uintptr_t)gate2;
  for (const void* p : residuals) res |= (uintptr_t)p;
  if (all % 2 || res % (f->residual_fp32 ? 4 : 2) || gate % (f->gate_fp32 ? 4 : 2) || (uintptr_t)f32_or_null % 4)
    fail(std::string(name) + ": tensors must be aligned to their elements");
  wide |= res;
  if (f->gate_kind >= GATE_CHANNEL) wide |= gate;
  return hidden % 8 == 0 && wide % 16 == 0;
}

// Threads of a workgroup: a thread has V runs of VEC columns of the row.
struct NormShape {
  int vec, v, threads;
};
static NormShape norm_shape(int hidden, bool wide) {
  const int units = wide ? hidden / 8 : hidden;
  const int v = wide ? (units <= 1024 ? 1 : 2) : (units <= 1024 ? 1 : units <= 4096 ? 4 : 16);
  const int threads = (units + v - 1) / v;
  return {wide ? 8 : 1, v, (threads + 63) / 64 * 64};
}

#define WM_NORM_SHAPES(F32, LAUNCH)                 \
  if (s.vec == 8) {                                 \
    if (s.v == 1) LAUNCH(F32, 8, 1); else LAUNCH(F32, 8, 2); \
  } else if (s.v == 1) {                            \
    LAUNCH(F32, 1, 1);                              \
  } else if (s.v == 4) {                            \
    LAUNCH(F32, 1, 4);                              \
  } else {                                          \
    LAUNCH(F32, 1, 16);                             \
  }

}  // namespace wm

using namespace wm;

extern "C" {

WM_EXPORT int wm_block_norm(const wm_block_norm_form* form, const void* residual, const void* y, int32_t tokens,
                            int32_t hidden, void* residual_out, void* x, void* stream) {
  return guarded([&] {
    const NormArgs a = norm_args("wm_block_norm", form, residual, y, tokens, hidden);
    if (tokens == 0) return;
    if (!residual_out || !x) fail("wm_block_norm: null pointer");
    const NormShape s = norm_shape(hidden, norm_aligned("wm_block_norm", form, hidden, {y, x}, {residual, residual_out}, nullptr,
                                                        nullptr));
    const unsigned blocks = (unsigned)(tokens < 2048 ? tokens : 2048);
#define WM_NORM(F, VEC, V)                                                                                          \
  hipLaunchKernelGGL((block_norm_kernel<F, VEC, V>), dim3(blocks), dim3(s.threads), 0, as_stream(stream), a, residual_out, \
                     (uint16_t*)x)
    if (form->residual_fp32) {
      WM_NORM_SHAPES(true, WM_NORM)
    } else {
      WM_NORM_SHAPES(false, WM_NORM)
    }
#undef WM_NORM
    check_launch("block_norm");
  });
}

WM_EXPORT size_t wm_block_norm_backward_workspace_size(int32_t tokens, int32_t hidden) {
  if (tokens < 0 || hidden < 1) return 0;
  return (size_t)norm_grad_blocks(tokens) * 3 * hidden * sizeof(float);
}

WM_EXPORT int wm_block_norm_backward(const wm_block_norm_form* form, const void* dx, const void* dresidual_out,
                                     const void* residual_out, const void* y, int32_t tokens, int32_t hidden, void* dresidual,
                                     void* dy, float* dpost_weight, float* dpre_weight, void* dgate, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  return guarded([&] {
    const NormArgs a = norm_args("wm_block_norm_backward", form, residual_out, y, tokens, hidden);
    if ((form->post_weight != nullptr) != (dpost_weight != nullptr) || (form->pre_weight != nullptr) != (dpre_weight != nullptr) ||
        (form->gate != nullptr) != (dgate != nullptr))
      fail("wm_block_norm_backward: each weight and the gate go with their gradients");
    if (tokens > 0 && (!dx || !dresidual || !dy || !workspace)) fail("wm_block_norm_backward: null pointer");
    if (workspace_bytes < wm_block_norm_backward_workspace_size(tokens, hidden) || (uintptr_t)workspace % 16)
      fail("wm_block_norm_backward: workspace too small or misaligned");
    const bool wide = norm_aligned("wm_block_norm_backward", form, hidden, {y, dx, dy}, {residual_out, dresidual_out, dresidual},
                                   (const void*)((uintptr_t)dpost_weight | (uintptr_t)dpre_weight |
                                                 (form->gate_kind == GATE_FULL ? 0 : (uintptr_t)dgate)),
                                   form->gate_kind == GATE_FULL ? dgate : nullptr);
    const NormShape s = norm_shape(hidden, wide);
    const int blocks = norm_grad_blocks(tokens);
    const NormGrads d = {(const uint16_t*)dx, dresidual_out, dresidual, (uint16_t*)dy, dgate, (float*)workspace};
    if (blocks > 0) {
#define WM_NORM(F, VEC, V) \
  hipLaunchKernelGGL((block_norm_grad_kernel<F, VEC, V>), dim3(blocks), dim3(s.threads), 0, as_stream(stream), a, d)
      if (form->residual_fp32) {
        WM_NORM_SHAPES(true, WM_NORM)
      } else {
        WM_NORM_SHAPES(false, WM_NORM)
      }
#undef WM_NORM
      check_launch("block_norm_grad");
    }
    float* dchannel = form->gate_kind == GATE_CHANNEL ? (float*)dgate : nullptr;
    if (dpost_weight || dpre_weight || dchannel) {
      hipLaunchKernelGGL(norm_columns_kernel, dim3((hidden + 15) / 16, 3), dim3(256), 0, as_stream(stream), d.partial, blocks,
                         hidden, dpost_weight, dpre_weight, dchannel);
      check_launch("norm_columns");
    }
  });
}

}  // extern "C"
