// The norms around a block, with its gate and residual scale, and their gradients. For a token with
// residual r and block output y, o the weights' offset:
//   z = y rsqrt(mean(y^2) + eps) (o + w_post)      (or z = y)
//   r' = r + s g z                                 g: 1, or per token, channel or element, plain or sigmoid
//   x = r' rsqrt(mean(r'^2) + eps) (o + w_pre)     r' as it is stored
// the residual add and norm of a decoder layer (DecoderLayer.feed_forward, qwen4_exp.py:1127-1149) for
// layers that also norm, gate or scale what a block adds. With q and p the two reciprocal roots and
// a = dx (o + w_pre):
//   dr' = dr_out + q (a - r' q^2 mean(a r'))       dr = dr'         dw_pre = sum_t dx r' q
//   b = s g dr',  c = b (o + w_post)               dy = p c - y p p mean(c y p)   dw_post = sum_t b y p
//   dg = s dr' z (by sigmoid'), summed over what g is broadcast over
//
// Bound by HBM: every tensor passes once. A group of threads holds a token's row in registers, 8 or 16 columns
// a thread, sums over the row twice at most, and goes on to its next token with the weights still in
// registers. A group is 16 threads or a wave for short rows, whose sums need no barrier, else a workgroup. Sums
// over tokens (weight gradients) stay with the group, go to the workspace once per workgroup and are added up
// by a second launch in the workgroups' order. All arithmetic is fp32; bf16 outputs are rounded once, from
// values that no earlier rounding touched but r''s own (x is the norm of the residual that the next block
// reads). Rows may have any magnitude whose squares fp32 holds (about 1e-17 to 1e18). 16384 tokens of 4096 in fp32
// take 152 us (805 MB, 5.3 TB/s), the gradients of 4001 tokens of 5120 in bf16 with a full gate 68 + 5 us (328 MB,
// 4.8 TB/s in the first launch).
#include <initializer_list>

#include "row_units.h"

namespace wm {

constexpr int NORM_MAX_HIDDEN = 16384;
enum { GATE_NONE = 0, GATE_TOKEN = 1, GATE_CHANNEL = 2, GATE_FULL = 3, GATE_FULL_F32 = 4 };  // 4: kernels only

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

// 1 / (1 + exp(-v)) to a few units: exp2 of the product with log2 e, whose rounding and the constant's rest come in as
// a factor. v is held between the ends first, so that product and rest are finite for infinite v and the types'
// largest values, too; NaN passes. From 88 on the result is 1; below -87.34 it would be less than the smallest normal
// number, and the reciprocal makes it 0.
__device__ __forceinline__ float sigmoid_f32(float v) {
  constexpr float LOG2E = 1.44269502162933349609375f, REST = 1.925963033500011079e-8f, LN2 = 0.693147182464599609375f;
  const float c = __builtin_elementwise_maximum(__builtin_elementwise_minimum(v, 88.0f), -88.7f);  // e below 2^128
  const float h = -c * LOG2E;
  const float l = fmaf(-c, LOG2E, -h) - c * REST;
  float e = __builtin_amdgcn_exp2f(h);
  e = fmaf(e, l * LN2, e);
  return __builtin_amdgcn_rcpf(1.0f + e);
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

// One value of a gate (through the sigmoid).
__device__ __forceinline__ float gate_value(const NormArgs& a, int64_t i) {
  const float g = a.gate_f32 ? ((const float*)a.gate)[i] : bf16_bits_to_f32(((const uint16_t*)a.gate)[i]);
  return a.gate_sigmoid ? sigmoid_f32(g) : g;
}

template <bool F32, int V, bool WHOLE, int GATE, int GROUP, int THREADS>
__global__ void __launch_bounds__(THREADS) block_norm_kernel(NormArgs a, void* residual_out, uint16_t* __restrict__ x) {
  __shared__ float part[3][1][16];
  if (GROUP == 0) clear_parts(&part[0][0][0], 48);
  const NormGroup<GROUP> at;
  const int H = a.hidden;
  const RowMean mean(H);
  const float opost = a.post ? a.offset : 0.0f, opre = a.pre ? a.offset : 0.0f;
  Weight8 wpost[V], wpre[V];
  float channel[V][8];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = at.column(v);
    if (c < H) {
      wpost[v].template load<WHOLE>(a.post, c, H - c);
      wpre[v].template load<WHOLE>(a.pre, c, H - c);
      if (GATE == GATE_CHANNEL) {
#pragma unroll
        for (int i = 0; i < 8; ++i) channel[v][i] = WHOLE || i < H - c ? a.scale * gate_value(a, c + i) : 0.0f;
      }
    }
  }
  int odd = 0;
  for (int64_t t = at.g; t < a.tokens; t += at.groups, odd ^= 1) {
    Row8<F32> raw[V];
    Row8<false> y[V];
    Row8<GATE == GATE_FULL_F32> gate[V];
    float r[V][8];
    float sum[1] = {0.0f};
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = at.column(v);
      if (c < H) {
        y[v].template load<WHOLE>(a.y, t * H + c, H - c);
        raw[v].template load<WHOLE>(a.residual, t * H + c, H - c);
        if (GATE >= GATE_FULL) gate[v].template load<WHOLE>(a.gate, t * H + c, H - c);
      }
    }
    const float g1 = GATE == GATE_TOKEN ? a.scale * gate_value(a, t) : a.scale;
    float p = 1.0f;
    if (a.post_norm) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (at.column(v) < H) {
#pragma unroll
          for (int i = 0; i < 8; ++i) sum[0] = fmaf(y[v].get(i), y[v].get(i), sum[0]);
        }
      }
      sum[0] *= mean.part;
      group_sums<1, GROUP>(sum, part[0]);
      p = rsqrtf(sum[0] / mean.n + a.eps);
    }
    sum[0] = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = at.column(v);
      if (c < H) {
        float g[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = GATE == GATE_CHANNEL ? channel[v][i] : g1;
        if (GATE >= GATE_FULL) {
#pragma unroll
          for (int i = 0; i < 8; ++i) g[i] = a.gate_sigmoid ? sigmoid_f32(gate[v].get(i)) : gate[v].get(i);
#pragma unroll
          for (int i = 0; i < 8; ++i) g[i] *= a.scale;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
          r[v][i] = fmaf(g[i], y[v].get(i) * p * wpost[v].get(opost, i), raw[v].get(i));
        if (!F32) RowUnit<false, true>::unpack(RowUnit<false, true>::pack(r[v]), r[v]);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (WHOLE || i < H - c) sum[0] = fmaf(r[v][i], r[v][i], sum[0]);
        store8<WHOLE>(residual_out, F32, t * H + c, H - c, r[v]);
      }
    }
    sum[0] *= mean.part;
    group_sums<1, GROUP>(sum, part[1 + odd]);  // without the post norm no other barrier stands between two of these
    const float q = rsqrtf(sum[0] / mean.n + a.eps);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = at.column(v);
      if (c < H) {
#pragma unroll
        for (int i = 0; i < 8; ++i) r[v][i] *= q * wpre[v].get(opre, i);
        store8<WHOLE>(x, false, t * H + c, H - c, r[v]);
      }
    }
  }
}

struct NormGrads {
  const uint16_t* dx;
  const void* dres;  // null: zero
  void* dr;
  uint16_t* dy;
  void* dgate;     // token: fp32 [T]; full: in the gate's type
  float* partial;  // [3][workgroups][H]: post, pre, channel gate
};

// What a thread loads of a token's row. A workgroup that has a CU to itself loads the next token's behind the first
// sums, while it works on this one's: 4001 tokens of 5120 with a full gate 69.7 us, without 72.4. (Workgroups that
// share one do so for each other; they unpack the weights anew for each token, since more registers make them
// fewer: 16000 of 2051 with a channel's gate 136 us, with the weights kept 183.)
template <bool F32, int V, bool WHOLE, int GATE>
struct NormRow {
  Row8<F32> r[V], dr[V];
  Row8<false> y[V], dx[V];
  Row8<GATE == GATE_FULL_F32> gate[V];
  template <int GROUP>
  __device__ __forceinline__ void load(const NormArgs& a, const NormGrads& d, const NormGroup<GROUP>& at, int64_t t) {
    const int H = a.hidden;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = at.column(v);
      if (c < H) {
        r[v].template load<WHOLE>(a.residual, t * H + c, H - c);
        dx[v].template load<WHOLE>(d.dx, t * H + c, H - c);
        y[v].template load<WHOLE>(a.y, t * H + c, H - c);
        if (d.dres) dr[v].template load<WHOLE>(d.dres, t * H + c, H - c);
        if (GATE >= GATE_FULL) gate[v].template load<WHOLE>(a.gate, t * H + c, H - c);
      }
    }
  }
};

// A thread's sums over its tokens, of the post weight (or of what its gradient and a channel gate's have in
// common) and of the pre weight. With 16 columns they are in LDS: registers would not hold them.
template <int V, int THREADS>
struct NormSums {
  float post_[8], pre_[8];
  __device__ __forceinline__ void clear(float*) {
#pragma unroll
    for (int i = 0; i < 8; ++i) post_[i] = pre_[i] = 0.0f;
  }
  __device__ __forceinline__ void post(float*, int, int i, float x, float y) { post_[i] = fmaf(x, y, post_[i]); }
  __device__ __forceinline__ void pre(float*, int, int i, float x, float y) { pre_[i] = fmaf(x, y, pre_[i]); }
  __device__ __forceinline__ float post(const float*, int, int i) const { return post_[i]; }
  __device__ __forceinline__ float pre(const float*, int, int i) const { return pre_[i]; }
};
template <int THREADS>
struct NormSums<2, THREADS> {
  static constexpr int PRE = 16 * THREADS;
  static __device__ __forceinline__ int place(int v, int i) { return (8 * v + i) * THREADS + threadIdx.x; }
  __device__ __forceinline__ void clear(float* s) {
    for (int i = 0; i < 32; ++i) s[i * THREADS + threadIdx.x] = 0.0f;
  }
  __device__ __forceinline__ void post(float* s, int v, int i, float x, float y) { s[place(v, i)] = fmaf(x, y, s[place(v, i)]); }
  __device__ __forceinline__ void pre(float* s, int v, int i, float x, float y) {
    s[PRE + place(v, i)] = fmaf(x, y, s[PRE + place(v, i)]);
  }
  __device__ __forceinline__ float post(const float* s, int v, int i) const { return s[place(v, i)]; }
  __device__ __forceinline__ float pre(const float* s, int v, int i) const { return s[PRE + place(v, i)]; }
};

template <bool F32, int V, bool WHOLE, int GATE, int GROUP, int THREADS>
__global__ void __launch_bounds__(THREADS, 4) block_norm_grad_kernel(NormArgs a, NormGrads d) {
  __shared__ float part[2][3][16];
  __shared__ float lds[V == 2 ? 32 * THREADS : GROUP != 0 ? 8 * THREADS : 1];
  if (GROUP == 0) clear_parts(&part[0][0][0], 96);
  const NormGroup<GROUP> at;
  const int H = a.hidden;
  const float opost = a.post ? a.offset : 0.0f, opre = a.pre ? a.offset : 0.0f;
  Weight8 wpost[V], wpre[V];
  float channel[V][8];
  NormSums<V, THREADS> sums;
  sums.clear(lds);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = at.column(v);
    if (c < H) {
      wpost[v].template load<WHOLE>(a.post, c, H - c);
      wpre[v].template load<WHOLE>(a.pre, c, H - c);
      if (GATE == GATE_CHANNEL) {
#pragma unroll
        for (int i = 0; i < 8; ++i) channel[v][i] = WHOLE || i < H - c ? gate_value(a, c + i) : 0.0f;
      }
    }
  }
  const RowMean mean(H);
  const float inv = 1.0f / mean.n;
  NormRow<F32, V, WHOLE, GATE> row;
#pragma unroll
  for (int v = 0; v < V; ++v) row.dr[v].clear();
  constexpr bool AHEAD = THREADS == 1024 && V == 1;
  NormRow<F32, V, WHOLE, GATE> next = row;
  if (AHEAD) next.load(a, d, at, at.g);
  for (int64_t t = at.g; t < a.tokens; t += at.groups) {
    if (AHEAD) row = next;
    else row.load(a, d, at, t);
    const float g1 = GATE == GATE_TOKEN ? gate_value(a, t) : 1.0f;
    float sum[3] = {0.0f, 0.0f, 0.0f};  // r'^2, a r', y^2
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (at.column(v) < H) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {  // behind a row's end r', dx and y are 0
          const float r = row.r[v].get(i), y = row.y[v].get(i);
          sum[0] = fmaf(r, r, sum[0]);
          sum[1] = fmaf(row.dx[v].get(i) * wpre[v].get(opre, i), r, sum[1]);
          sum[2] = fmaf(y, y, sum[2]);
        }
      }
    }
#pragma unroll
    for (int n = 0; n < 3; ++n) sum[n] *= mean.part;
    group_sums<3, GROUP>(sum, part[0]);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      row.r[v].repack();
      row.dx[v].repack();
      row.y[v].repack();
      if (THREADS < 1024 || V == 2) wpre[v].w.repack(), wpost[v].w.repack();
    }
    if (AHEAD && t + at.groups < a.tokens) next.load(a, d, at, t + at.groups);
    const float q = rsqrtf(sum[0] * inv + a.eps);
    const float p = a.post_norm ? rsqrtf(sum[2] * inv + a.eps) : 1.0f;
    const float k1 = q * (q * (sum[1] * inv));  // the third q comes last: q^3 leaves fp32 for rows of 1e13 or 1e-13
    float sum2[2] = {0.0f, 0.0f};  // c y p, the token's gate gradient
    float cc[V][8];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = at.column(v);
      if (c < H) {
        float dr[8], dg[8];
#pragma unroll
        for (int h = 0; h < 8; h += 4) {
          float g[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            g[j] = GATE == GATE_CHANNEL ? channel[v][h + j] : GATE >= GATE_FULL ? row.gate[v].get(h + j) : g1;
          if (GATE >= GATE_FULL && a.gate_sigmoid) {
#pragma unroll
            for (int j = 0; j < 4; ++j) g[j] = sigmoid_f32(g[j]);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int i = h + j;
            const float r = row.r[v].get(i), dx = row.dx[v].get(i), n = row.y[v].get(i) * p;
            dr[i] = fmaf(q, fmaf(dx, wpre[v].get(opre, i), -r * k1), row.dr[v].get(i));
            sums.pre(lds, v, i, q * dx, r);
            const float sdr = a.scale * dr[i], w = wpost[v].get(opost, i);
            const float b = sdr * g[j];
            sums.post(lds, v, i, GATE == GATE_CHANNEL ? sdr : b, n);
            if (GATE != GATE_NONE && GATE != GATE_CHANNEL) dg[i] = sdr * (n * w);
            if (GATE >= GATE_FULL && a.gate_sigmoid) dg[i] *= g[j] * (1.0f - g[j]);
            if (GATE == GATE_TOKEN) sum2[1] += dg[i];
            cc[v][i] = b * w;
            sum2[0] = fmaf(cc[v][i], n, sum2[0]);
          }
          if (V == 2) __builtin_amdgcn_sched_barrier(0);  // fewer values at once: there are no registers for more
        }
        store8<WHOLE>(d.dr, F32, t * H + c, H - c, dr);
        if (GATE >= GATE_FULL) store8<WHOLE>(d.dgate, GATE == GATE_FULL_F32, t * H + c, H - c, dg);
      }
    }
    sum2[0] *= mean.part;
    if (GROUP != 0 || a.post_norm || GATE == GATE_TOKEN) group_sums<GATE == GATE_TOKEN ? 2 : 1, GROUP>(sum2, part[1]);
    else __syncthreads();
    const float k2 = a.post_norm ? p * (sum2[0] * inv) : 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = at.column(v);
      row.y[v].repack();
      if (c < H) {
#pragma unroll
        for (int i = 0; i < 8; ++i) cc[v][i] = fmaf(p, cc[v][i], -(row.y[v].get(i) * p) * k2);
        store8<WHOLE>(d.dy, false, t * H + c, H - c, cc[v]);
      }
    }
    if (GATE == GATE_TOKEN && at.me == 0) ((float*)d.dgate)[t] = a.gate_sigmoid ? sum2[1] * (g1 * (1.0f - g1)) : sum2[1];
  }
  // A workgroup's row of each sum.
  auto emit = [&](int which, auto value) {
    float* out = d.partial + ((int64_t)which * gridDim.x + blockIdx.x) * H;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = at.column(v);
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = c < H ? value(v, i) : 0.0f;
      if (GROUP == 0) {
        if (c < H) store8<WHOLE>(out, true, c, H - c, f);
      } else {  // its groups' sums, in their order
        float* mine = &lds[threadIdx.x * 8];
#pragma unroll
        for (int i = 0; i < 8; ++i) mine[i] = f[i];
        __syncthreads();
        for (int j = threadIdx.x; j < H; j += THREADS) {
          float sum = 0.0f;
          for (int g = 0; g < THREADS; g += GROUP) sum += lds[g * 8 + j];
          out[j] = sum;
        }
        __syncthreads();
      }
    }
  };
  if (a.post) emit(0, [&](int v, int i) { return sums.post(lds, v, i) * (GATE == GATE_CHANNEL ? channel[v][i] : 1.0f); });
  if (a.pre) emit(1, [&](int v, int i) { return sums.pre(lds, v, i); });
  if (GATE == GATE_CHANNEL) {
    emit(2, [&](int v, int i) {
      const float g = channel[v][i];
      return sums.post(lds, v, i) * wpost[v].get(opost, i) * (a.gate_sigmoid ? g * (1.0f - g) : 1.0f);
    });
  }
}

// out[which][c] = the sum of partial[which][b][c] over the workgroups b: a workgroup has 64 columns, each of its
// 16 waves every 16th b, and the waves' sums are added in their order.
__global__ void __launch_bounds__(1024) norm_columns_kernel(const float* __restrict__ partial, int blocks, int hidden,
                                                           float* dpost, float* dpre, float* dgate) {
  __shared__ float wave_sum[16][64];
  float* out = blockIdx.y == 0 ? dpost : blockIdx.y == 1 ? dpre : dgate;
  if (!out) return;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int c = blockIdx.x * 64 + lane;
  const float* mine = partial + (int64_t)blockIdx.y * blocks * hidden + c;
  float sum = 0.0f;
  if (c < hidden) {
#pragma unroll 8
    for (int b = wave; b < blocks; b += 16) sum += mine[(int64_t)b * hidden];
  }
  wave_sum[wave][lane] = sum;
  __syncthreads();
  if (wave == 0 && c < hidden) {
    for (int w = 1; w < 16; ++w) sum += wave_sum[w][lane];
    out[c] = sum;
  }
}

// How a row is held: by `group` threads (0: a workgroup of `threads`), 8 v columns each. Short rows have 16 threads
// or a wave, four waves a workgroup (16000 tokens of 100, captured, 5.5 us and the gradients 12.6, with a workgroup a
// row 12.0 and 42); rows of more than 8192 columns 16 columns a thread, since a workgroup has 1024.
struct NormShape {
  int group, v, threads;
};
static NormShape norm_shape(int hidden) {
  const int units = (hidden + 7) / 8;
  if (units <= 64) return {units <= 16 ? 16 : 64, 1, 256};
  const int v = units <= 1024 ? 1 : 2;
  return {0, v, ((units + v - 1) / v + 63) / 64 * 64};
}
static int norm_groups_of_block(const NormShape& s) { return s.group ? s.threads / s.group : 1; }

// Workgroups of a pass by the waves a CU gets, `least` at least. (The forward pass with 64, twice what a CU holds,
// 152 us for 16384 tokens of 4096, with 32 157 us, with a workgroup a token 218.)
static int norm_blocks(int64_t tokens, const NormShape& s, int waves, int least) {
  const int64_t per_cu = waves * 64 / s.threads, want = 256 * (per_cu > least ? per_cu : least);
  const int64_t most = (tokens + norm_groups_of_block(s) - 1) / norm_groups_of_block(s);
  return (int)(most < want ? most : want);
}
// The gradient pass has what a CU holds at once, one workgroup of long rows (4001 tokens of 5120: 69.7 us, two in turn
// 74.8), and adds a row a workgroup to the second launch's work: 8 tokens a group or more, 4 where rows are
// short and no eights (their loads take longer), unless that leaves CUs without one: 18775 tokens of 479 with a
// channel's gate 60 us with 8, 46 with 4; 16000 of 512 in fp32 28 and 32.
static int norm_grad_blocks(int64_t tokens, int hidden) {
  const NormShape s = norm_shape(hidden);
  const int64_t each = (s.group && hidden % 8 ? 4 : 8) * norm_groups_of_block(s), most = tokens / each > 512 ? tokens / each : 512;
  const int64_t blocks = norm_blocks(tokens, s, 16, 1);
  return (int)(blocks < most ? blocks : most);
}
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

// Every tensor is aligned to its elements.
static void norm_aligned(const char* name, const wm_block_norm_form* f, std::initializer_list<const void*> bf16,
                         std::initializer_list<const void*> residuals, std::initializer_list<const void*> f32,
                         const void* full_gate) {
  uintptr_t two = (uintptr_t)f->post_weight | (uintptr_t)f->pre_weight, res = 0, four = 0;
  for (const void* p : bf16) two |= (uintptr_t)p;
  for (const void* p : residuals) res |= (uintptr_t)p;
  for (const void* p : f32) four |= (uintptr_t)p;
  const uintptr_t gate = (uintptr_t)f->gate | (uintptr_t)full_gate;
  if (two % 2 || res % (f->residual_fp32 ? 4 : 2) || gate % (f->gate_fp32 ? 4 : 2) || four % 4)
    fail(std::string(name) + ": tensors must be aligned to their elements");
}

// The kernels' instances: the residual's type, the gate, whole rows of eights or not, and the shapes that
// norm_shape gives; fewer threads a workgroup leave each more registers.
#define WM_NORM_GATES(KERNEL, F, V, W, G, N, ...)                                                          \
  switch (gate) {                                                                                         \
    case GATE_NONE: hipLaunchKernelGGL((KERNEL<F, V, W, GATE_NONE, G, N>), __VA_ARGS__); break;           \
    case GATE_TOKEN: hipLaunchKernelGGL((KERNEL<F, V, W, GATE_TOKEN, G, N>), __VA_ARGS__); break;         \
    case GATE_CHANNEL: hipLaunchKernelGGL((KERNEL<F, V, W, GATE_CHANNEL, G, N>), __VA_ARGS__); break;     \
    case GATE_FULL: hipLaunchKernelGGL((KERNEL<F, V, W, GATE_FULL, G, N>), __VA_ARGS__); break;           \
    default: hipLaunchKernelGGL((KERNEL<F, V, W, GATE_FULL_F32, G, N>), __VA_ARGS__);                     \
  }
#define WM_NORM_WHOLE(KERNEL, F, V, G, N, ...)                                    \
  if (a.hidden % 8 == 0) { WM_NORM_GATES(KERNEL, F, V, true, G, N, __VA_ARGS__) } \
  else { WM_NORM_GATES(KERNEL, F, V, false, G, N, __VA_ARGS__) }
#define WM_NORM_SHAPES(KERNEL, F, ...)                                                     \
  if (shape.group == 16) { WM_NORM_WHOLE(KERNEL, F, 1, 16, 256, __VA_ARGS__) }             \
  else if (shape.group == 64) { WM_NORM_WHOLE(KERNEL, F, 1, 64, 256, __VA_ARGS__) }        \
  else if (shape.v == 2) { WM_NORM_WHOLE(KERNEL, F, 2, 0, 1024, __VA_ARGS__) }             \
  else if (shape.threads > 512) { WM_NORM_WHOLE(KERNEL, F, 1, 0, 1024, __VA_ARGS__) }      \
  else { WM_NORM_WHOLE(KERNEL, F, 1, 0, 512, __VA_ARGS__) }
#define WM_NORM_LAUNCH(KERNEL, ...)                                                       \
  const int gate = a.gate_kind == GATE_FULL && a.gate_f32 ? GATE_FULL_F32 : a.gate_kind;  \
  const dim3 threads(shape.threads);                                                      \
  if (f32) { WM_NORM_SHAPES(KERNEL, true, __VA_ARGS__) } else { WM_NORM_SHAPES(KERNEL, false, __VA_ARGS__) }

static void norm_forward(const NormArgs& a, bool f32, void* residual_out, uint16_t* x, hipStream_t s) {
  const NormShape shape = norm_shape(a.hidden);
  const dim3 blocks((unsigned)norm_blocks(a.tokens, shape, 64, 2));
  WM_NORM_LAUNCH(block_norm_kernel, blocks, threads, 0, s, a, residual_out, x)
  check_launch("block_norm");
}

static void norm_grad(const NormArgs& a, bool f32, const NormGrads& d, int grid, hipStream_t s) {
  const NormShape shape = norm_shape(a.hidden);
  const dim3 blocks((unsigned)grid);
  WM_NORM_LAUNCH(block_norm_grad_kernel, blocks, threads, 0, s, a, d)
  check_launch("block_norm_grad");
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
    norm_aligned("wm_block_norm", form, {y, x}, {residual, residual_out}, {}, nullptr);
    norm_forward(a, form->residual_fp32 != 0, residual_out, (uint16_t*)x, as_stream(stream));
  });
}

WM_EXPORT size_t wm_block_norm_backward_workspace_size(int32_t tokens, int32_t hidden) {
  if (tokens < 0 || hidden < 1 || hidden > NORM_MAX_HIDDEN) return 0;
  return (size_t)norm_grad_blocks(tokens, hidden) * 3 * hidden * sizeof(float);
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
    norm_aligned("wm_block_norm_backward", form, {y, dx, dy}, {residual_out, dresidual_out, dresidual},
                 {dpost_weight, dpre_weight, form->gate_kind == GATE_FULL ? nullptr : dgate},
                 form->gate_kind == GATE_FULL ? dgate : nullptr);
    const int blocks = norm_grad_blocks(tokens, hidden);
    const NormGrads d = {(const uint16_t*)dx, dresidual_out, dresidual, (uint16_t*)dy, dgate, (float*)workspace};
    hipStream_t s = as_stream(stream);
    if (blocks > 0) norm_grad(a, form->residual_fp32 != 0, d, blocks, s);
    float* dchannel = form->gate_kind == GATE_CHANNEL ? (float*)dgate : nullptr;
    if (dpost_weight || dpre_weight || dchannel) {
      hipLaunchKernelGGL(norm_columns_kernel, dim3((hidden + 63) / 64, 3), dim3(1024), 0, s, d.partial, blocks, hidden,
                         dpost_weight, dpre_weight, dchannel);
      check_launch("norm_columns");
    }
  });
}

}  // extern "C"
