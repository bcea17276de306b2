// Products of 8-bit rows: E4M3 on both sides, an fp32 scale for each 128 values of a token's row and for each
// 128 x 128 block of the weights. With b the blocks along K
//   y[t, n] = add[t, n] + sum_b xs[t, b] ws[n / 128, b] sum_{k in b} x[t, k] w[n, k]
// The inner sum is one matrix instruction (K 128) from zero; its 4 results a lane go to the fp32 accumulators by one
// multiply-add each, with the product of the two scales. The weights are the A operand, so that a lane's results belong to one
// token (column lane % 16) and 4 weight rows of one block: one scale a lane and token tile. The 4 multiply-adds take 16 of
// the instruction's 32 cycles, and run beside another's.
//
// The FP8 matrix instructions line products up with their group's largest and drop what falls below about 2^-13 of
// it (measured: 1.3e-5 of a sum of normal values, 1.4e-4 of the sum of magnitudes at worst). That is far below a bf16
// output's rounding (2^-8) but not below fp32's: for fp32 outputs the bytes, which are bf16 values, are
// converted to bf16 in registers, exactly, and multiplied by the bf16 instructions, whose sums are fp32's (2^-21 of the
// magnitudes), at half the rate.
#include <type_traits>

#include "lds_dma.h"
#include "row_units.h"

namespace wm {
namespace g8 {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int BLOCK = 128;  // K values of a scale and of a step

struct Args {
  const uint8_t* x;
  const float* xs;
  const uint8_t* w;
  const float* ws;
  const void* add;
  void* out;
  int tokens, n, k, blocks;
};

// A lane's 32 bytes of a row's block: the pieces g and 4 + g of 16 bytes, g = lane / 16, of row lane % 16 of a
// tile. Both operands take the same pieces, so that the sum is the whole block's whatever the instruction's own
// order is.
struct Frag {
  uint4 lo, hi;
};
__device__ __forceinline__ void zero_behind(Frag& f, int g, int pieces) {  // the pieces from `pieces` on
  const uint4 z = make_uint4(0, 0, 0, 0);
  if (g >= pieces) f.lo = z;
  if (4 + g >= pieces) f.hi = z;
}

// Eight bytes to bf16, exactly.
__device__ __forceinline__ bf16x8 widen(uint32_t a, uint32_t b) {
  const wm_bf16x2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true),
                          __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true)};
  return __builtin_bit_cast(bf16x8, v);
}

// An operand as the matrix instruction takes it.
template <bool EXACT>
struct Operand;
template <>
struct Operand<false> {
  i32x8 v;
  Operand() = default;
  __device__ __forceinline__ explicit Operand(const Frag& f) {
    v = i32x8{(int)f.lo.x, (int)f.lo.y, (int)f.lo.z, (int)f.lo.w, (int)f.hi.x, (int)f.hi.y, (int)f.hi.z, (int)f.hi.w};
  }
  // The block's sums, weights first.
  static __device__ __forceinline__ f32x4 product(const Operand& w, const Operand& x) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v, x.v, f32x4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0, 127, 0, 127);
  }
};
template <>
struct Operand<true> {
  bf16x8 v[4];
  Operand() = default;
  __device__ __forceinline__ explicit Operand(const Frag& f)
      : v{widen(f.lo.x, f.lo.y), widen(f.lo.z, f.lo.w), widen(f.hi.x, f.hi.y), widen(f.hi.z, f.hi.w)} {}
  static __device__ __forceinline__ f32x4 product(const Operand& w, const Operand& x) {
    f32x4 d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.v[i], x.v[i], d, 0, 0, 0);
    return d;
  }
};

// Output (token t, weight row n), fp32 or bf16.
template <bool F32>
__device__ __forceinline__ void store_one(const Args& a, int t, int n, float v) {
  const int64_t at = (int64_t)t * a.n + n;
  if (F32) {
    if (a.add) v += ((const float*)a.add)[at];
    ((float*)a.out)[at] = v;
  } else {
    if (a.add) v += bf16_bits_to_f32(((const uint16_t*)a.add)[at]);
    ((uint16_t*)a.out)[at] = (uint16_t)pack_bf16(v, 0.0f);
  }
}
// Weight rows n .. n + 3 of token t, with what is to be added.
template <bool F32>
__device__ __forceinline__ f32x4 added(const Args& a, int t, int n, f32x4 v) {
  if (!a.add || t >= a.tokens) return v;
  const int64_t at = (int64_t)t * a.n + n;
  if (n + 4 <= a.n) {
    if (F32) {
      const wm_u32x4 d = load16((const float*)a.add + at);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += __uint_as_float(d[i]);
    } else {
      const wm_u32x2 d = load8((const uint16_t*)a.add + at);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += __uint_as_float(i % 2 ? d[i / 2] & 0xffff0000u : d[i / 2] << 16);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.n) v[i] += F32 ? ((const float*)a.add)[at + i] : bf16_bits_to_f32(((const uint16_t*)a.add)[at + i]);
  }
  return v;
}

// ---------------------------------------------------------------------------------
// stream: few tokens. A block of 8 waves owns 16 NT weight rows x 16 MT tokens; the waves take the blocks of K in turn,
// operands straight from memory, DEPTH blocks in flight a wave, and their sums meet in LDS, added in wave order.
constexpr int SW = 8;

template <int NT, int MT>
struct StreamSlot {
  Frag w[NT], x[MT];
  float xs[MT], ws[NT];
};

template <int NT, int MT, int DEPTH, bool F32, bool TAIL>
__global__ void __launch_bounds__(64 * SW) stream_kernel(Args a) {
  __shared__ float red[SW][NT * MT][4][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int c = lane % 16, g = lane / 16;
  const int n0 = blockIdx.x * (16 * NT), t0 = blockIdx.y * (16 * MT);
  const uint8_t *wp[NT], *xp[MT];
  const float *xsp[MT], *wsp[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    wp[j] = a.w + (int64_t)min(n0 + 16 * j + c, a.n - 1) * a.k + 16 * g;
    wsp[j] = a.ws + (int64_t)(min(n0 + 16 * j, a.n - 1) / BLOCK) * a.blocks;
  }
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int64_t t = min(t0 + 16 * m + c, a.tokens - 1);
    xp[m] = a.x + t * a.k + 16 * g;
    xsp[m] = a.xs + t * a.blocks;
  }
  f32x4 acc[NT][MT];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[j][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  StreamSlot<NT, MT> s[DEPTH];
  auto load = [&](StreamSlot<NT, MT>& s, int b) {
    int64_t lo = (int64_t)b * BLOCK, hi = lo + 64;
    if (TAIL) {  // pieces behind the row's end read its first bytes and count as zero
      lo = lo + 16 * g < a.k ? lo : -16 * g;
      hi = hi + 16 * g < a.k ? hi : -16 * g;
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) s.w[j] = {gload16_nt(wp[j] + lo), gload16_nt(wp[j] + hi)};
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      s.x[m] = {gload16(xp[m] + lo), gload16(xp[m] + hi)};
      s.xs[m] = gload<float>(xsp[m] + b);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) s.ws[j] = wsp[j][b];
  };
  auto multiply = [&](StreamSlot<NT, MT>& s, int b) {
    if (TAIL && b == a.blocks - 1) {
      const int pieces = (a.k - b * BLOCK) / 16;
#pragma unroll
      for (int j = 0; j < NT; ++j) zero_behind(s.w[j], g, pieces);
#pragma unroll
      for (int m = 0; m < MT; ++m) zero_behind(s.x[m], g, pieces);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const Operand<F32> x(s.x[m]);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const f32x4 d = Operand<F32>::product(Operand<F32>(s.w[j]), x);
        const float f = s.xs[m] * s.ws[j];
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][m][i] = fmaf(d[i], f, acc[j][m][i]);
      }
    }
  };
  int b = wave;
#pragma unroll
  for (int u = 0; u < DEPTH; ++u) load(s[u], min(b + SW * u, a.blocks - 1));
  for (; b + SW * DEPTH < a.blocks; b += SW * DEPTH) {
#pragma unroll
    for (int u = 0; u < DEPTH; ++u) {
      multiply(s[u], b + SW * u);
      load(s[u], min(b + SW * (DEPTH + u), a.blocks - 1));
    }
  }
#pragma unroll
  for (int u = 0; u < DEPTH; ++u)
    if (b + SW * u < a.blocks) multiply(s[u], b + SW * u);  // wave-uniform

#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) red[wave][j * MT + m][i][lane] = acc[j][m][i];
  __syncthreads();
  for (int e = threadIdx.x; e < 256 * NT * MT; e += 64 * SW) {
    const int o = e % (16 * NT), tc = e / (16 * NT);  // weight row and token of the tile
    const int at = o / 16 * MT + tc / 16, i = o % 4, l = 16 * (o % 16 / 4) + tc % 16;
    float v = red[0][at][i][l];
#pragma unroll
    for (int q = 1; q < SW; ++q) v += red[q][at][i][l];
    if (t0 + tc < a.tokens && n0 + o < a.n) store_one<F32>(a, t0 + tc, n0 + o, v);
  }
}

// ---------------------------------------------------------------------------------
// tiled: WN x WM waves, each 16 TN weight rows x 16 TM tokens. A step is a block of K: its rows of 128 bytes and its scales go
// straight to LDS, STAGES steps at once, pieces of 16 bytes XOR-swizzled by row, so that the 8 rows of a
// ds_read_b128 cycle fall on distinct banks.
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}
template <int PER, int MOST>
__device__ __forceinline__ void wait_step(int ahead) {
  if (ahead >= MOST) {
    wait_loads<PER * MOST>();
  } else if constexpr (MOST > 0) {
    wait_step<PER, MOST - 1>(ahead);
  }
}

template <int TN_, int TM_, int WN_, int WM_, int STAGES_>
struct Tile {
  static constexpr int TN = TN_, TM = TM_, WN = WN_, WM = WM_, STAGES = STAGES_, WAVES = WN * WM;
  static constexpr int BN = 16 * TN * WN, BM = 16 * TM * WM;
  static constexpr int W = BN * BLOCK, X = BM * BLOCK, SCALES = W + X, STAGE = SCALES + 4 * BM + 256;
  static constexpr int WL = BN / 8 / WAVES, XL = BM / 8 / WAVES;  // row loads of a wave
  static constexpr int LOADS = WL + XL + 1;                       // and one of scales
  static_assert(BN % (8 * WAVES) == 0 && BM % (8 * WAVES) == 0 && BM / 64 < WAVES && BM % 64 == 0 && BN <= 64 * BLOCK && 128 % (16 * TN) == 0);
  static_assert(STAGES * STAGE <= 160 * 1024);
};

// Tiles of 8 token tiles at a time, these innermost: an XCD (block b runs on XCD b % 8) works on a patch of 8 token tiles and a
// few weight tiles at once, whose rows stay in its L2.
__device__ __forceinline__ bool tile_of(int n_tiles, int t_tiles, int& nt, int& tt) {
  const int64_t total = (int64_t)n_tiles * t_tiles, tile = blockIdx.x % 8 * ((total + 7) / 8) + blockIdx.x / 8;
  if (tile >= total) return false;
  const int64_t group = tile / (8 * (int64_t)n_tiles), rest = tile - group * 8 * n_tiles;
  const int high = min(8, t_tiles - 8 * (int)group);
  tt = 8 * (int)group + (int)(rest % high);
  nt = (int)(rest / high);
  return true;
}

template <typename T, bool F32, bool TAIL>
__global__ void __launch_bounds__(64 * T::WAVES) tiled_kernel(Args a, int n_tiles, int t_tiles) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[T::STAGES * T::STAGE];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  int nt, tt;
  if (!tile_of(n_tiles, t_tiles, nt, tt)) return;
  const int n0 = nt * T::BN, t0 = tt * T::BM;
  const int wn = wave % T::WN, wm = wave / T::WN;

  // A load fills 8 rows of 128 bytes: lane l row l / 8, position l % 8 with the piece (l % 8) ^ (row % 8). Rows past the
  // end read the last one.
  const int lrow = lane / 8, piece = (lane % 8) ^ lrow;
  const uint8_t* wbase = a.w + (int64_t)n0 * a.k;
  const uint8_t* xbase = a.x + (int64_t)t0 * a.k;
  uint32_t woff[T::WL], xoff[T::XL], soff;
#pragma unroll
  for (int i = 0; i < T::WL; ++i)
    woff[i] = (uint32_t)(min(n0 + 8 * (wave + T::WAVES * i) + lrow, a.n - 1) - n0) * (uint32_t)a.k + 16u * piece;
#pragma unroll
  for (int i = 0; i < T::XL; ++i)
    xoff[i] = (uint32_t)(min(t0 + 8 * (wave + T::WAVES * i) + lrow, a.tokens - 1) - t0) * (uint32_t)a.k + 16u * piece;
  // waves below BM / 64 load 64 tokens' scales each, the others those of the weights
  const bool tokens_scales = wave < T::BM / 64;
  const float* sbase = tokens_scales ? a.xs + (int64_t)t0 * a.blocks : a.ws + (int64_t)(n0 / BLOCK) * a.blocks;
  const uint32_t sdst = T::SCALES + (tokens_scales ? 256u * wave : 4u * T::BM);
  soff = (uint32_t)(tokens_scales ? min(t0 + 64 * wave + lane, a.tokens - 1) - t0
                                  : min(lane, (a.n - 1) / BLOCK - n0 / BLOCK)) * (uint32_t)a.blocks * 4u;
  // Load i of block b's LOADS.
  auto issue = [&](int b, int i) {
    const uint32_t slot = lds_addr(lds + b % T::STAGES * T::STAGE);
    // pieces behind the rows' end read the block's first one
    const uint32_t off = (uint32_t)BLOCK * b - (TAIL && BLOCK * b + 16 * piece >= a.k ? 16u * piece : 0u);
    if (i < T::WL) dma16(wbase, woff[i] + off, slot + 1024 * (wave + T::WAVES * i));
    else if (i < T::WL + T::XL) dma16(xbase, xoff[i - T::WL] + off, slot + T::W + 1024 * (wave + T::WAVES * (i - T::WL)));
    else dma4(sbase, soff + 4u * b, slot + sdst);
  };

  f32x4 acc[T::TN][T::TM];
#pragma unroll
  for (int i = 0; i < T::TN; ++i)
#pragma unroll
    for (int m = 0; m < T::TM; ++m) acc[i][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const int c = lane % 16, g = lane / 16;
  const uint32_t pos = 16u * (uint32_t)(g ^ (c % 8));
  const uint32_t wrow = (uint32_t)(16 * T::TN * wn + c) * BLOCK + pos, xrow = T::W + (uint32_t)(16 * T::TM * wm + c) * BLOCK + pos;
  const uint32_t xscale = T::SCALES + 4u * (16 * T::TM * wm + c), wscale = T::SCALES + 4u * (T::BM + 16 * T::TN * wn / BLOCK);

  // Block b's sums. The multiply-adds of a matrix instruction's results stand beside the instruction TM later, so that
  // none waits for them (the last ones of a block beside the next block's first). With AHEAD the loads of the block STAGES - 1
  // behind it go out between the instructions of the block's first half.
  f32x4 d[T::TM];
  float f[T::TM];
#pragma unroll
  for (int m = 0; m < T::TM; ++m) d[m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f[m] = 0.0f;
  auto step = [&](int b, auto ahead, auto last) {
    constexpr bool AHEAD = decltype(ahead)::value, LAST = decltype(last)::value;
    const uint8_t* s = lds + b % T::STAGES * T::STAGE;
    const int pieces = (a.k - b * BLOCK) / 16;
    auto frag = [&](uint32_t at) {
      Frag f = {*reinterpret_cast<const uint4*>(s + at), *reinterpret_cast<const uint4*>(s + (at ^ 64u))};
      if (TAIL && LAST) zero_behind(f, g, pieces);
      return Operand<F32>(f);
    };
    Operand<F32> x[T::TM], w[2];
    w[0] = frag(wrow);
#pragma unroll
    for (int m = 0; m < T::TM; ++m) x[m] = frag(xrow + 16 * BLOCK * m);
    const float ws = *reinterpret_cast<const float*>(s + wscale);
    float xs[T::TM];
#pragma unroll
    for (int m = 0; m < T::TM; ++m) xs[m] = *reinterpret_cast<const float*>(s + xscale + 64 * m);
#pragma unroll
    for (int i = 0; i < T::TN; ++i) {
      if (i + 1 < T::TN) w[(i + 1) % 2] = frag(wrow + 16 * BLOCK * (i + 1));
      if (AHEAD) {
        constexpr int PER = (2 * T::LOADS + T::TN - 1) / T::TN;  // in the first half
#pragma unroll
        for (int q = i * PER; q < (i + 1) * PER && q < T::LOADS; ++q) issue(b + T::STAGES - 1, q);
      }
#pragma unroll
      for (int m = 0; m < T::TM; ++m) {
        const f32x4 p = Operand<F32>::product(w[i % 2], x[m]);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[(i + T::TN - 1) % T::TN][m][e] = fmaf(d[m][e], f[m], acc[(i + T::TN - 1) % T::TN][m][e]);
        if (i == 0) f[m] = ws * xs[m];
        d[m] = p;
        __builtin_amdgcn_sched_barrier(0);  // the order as it is written
      }
    }
  };
  const std::true_type yes;
  const std::false_type no;
  int b = 0;
  for (; b < T::STAGES - 1 && b < a.blocks; ++b)
#pragma unroll
    for (int i = 0; i < T::LOADS; ++i) issue(b, i);
  // at the top of a block its loads have landed in every wave, and every wave is done with the slot that the next
  // loads overwrite
  for (b = 0; b + T::STAGES - 1 < a.blocks; ++b) {
    wait_loads<T::LOADS * (T::STAGES - 2)>();
    step(b, yes, no);
  }
  for (; b + 1 < a.blocks; ++b) {
    wait_step<T::LOADS, T::STAGES - 2>(a.blocks - 1 - b);
    step(b, no, no);
  }
  wait_loads<0>();
  step(b, no, yes);
#pragma unroll
  for (int m = 0; m < T::TM; ++m)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[T::TN - 1][m][e] = fmaf(d[m][e], f[m], acc[T::TN - 1][m][e]);
  // Results by way of LDS, so that stores are whole runs of a row: a wave has ROWS tokens at a time there, its 16 TN weight rows
  // each as pieces of 16 bytes, the piece's place XOR the token's.
  wait_loads<0>();
  constexpr int WIDE = 16 * T::TN, SIZE = F32 ? 4 : 2, EACH = 16 / SIZE, PIECES = WIDE / EACH, BYTES = 16 * WIDE * SIZE;
  constexpr int MASK = PIECES < 16 ? PIECES - 1 : 15;
  uint8_t* mine = lds + wave * BYTES;
  static_assert(T::WAVES * BYTES <= T::STAGES * T::STAGE);
#pragma unroll
  for (int m = 0; m < T::TM; ++m) {
    if (m > 0) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // its own reads
#pragma unroll
    for (int i = 0; i < T::TN; ++i) {
      const f32x4 v = added<F32>(a, t0 + 16 * (T::TM * wm + m) + c, n0 + WIDE * wn + 16 * i + 4 * g, acc[i][m]);
      if constexpr (F32) {
        *reinterpret_cast<f32x4*>(mine + c * WIDE * 4 + 16 * ((4 * i + g) ^ (c & MASK))) = v;
      } else {
        *reinterpret_cast<wm_u32x2*>(mine + c * WIDE * 2 + 16 * ((2 * i + g / 2) ^ (c & MASK)) + 8 * (g % 2)) =
            wm_u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int j = 0; j < PIECES / 4; ++j) {
      const int at = 64 * j + lane, row = at / PIECES, q = at % PIECES;
      const int t = t0 + 16 * (T::TM * wm + m) + row, n = n0 + WIDE * wn + EACH * q;
      const wm_u32x4 v = *reinterpret_cast<const wm_u32x4*>(mine + row * WIDE * SIZE + 16 * (q ^ (row & MASK)));
      if (t >= a.tokens || n >= a.n) continue;
      uint8_t* to = (uint8_t*)a.out + ((int64_t)t * a.n + n) * SIZE;
      if (n + EACH <= a.n) {
        store16(to, v);
      } else {
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
          if (n + e >= a.n) continue;
          if (F32) ((uint32_t*)to)[e] = v[e % 4];
          else ((uint16_t*)to)[e] = (uint16_t)(v[e / 2 % 4] >> (16 * (e % 2)));
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------------

template <int NT, int MT, int DEPTH, bool F32>
static void launch_stream(const Args& a, hipStream_t s) {
  const dim3 grid((a.n + 16 * NT - 1) / (16 * NT), (a.tokens + 16 * MT - 1) / (16 * MT));
  if (a.k % BLOCK) hipLaunchKernelGGL((stream_kernel<NT, MT, DEPTH, F32, true>), grid, dim3(64 * SW), 0, s, a);
  else hipLaunchKernelGGL((stream_kernel<NT, MT, DEPTH, F32, false>), grid, dim3(64 * SW), 0, s, a);
  check_launch("linear_fp8 (stream)");
}

template <typename T, bool F32>
static void launch_tiled(const Args& a, hipStream_t s) {
  const int64_t n_tiles = (a.n + T::BN - 1) / T::BN, t_tiles = (a.tokens + T::BM - 1) / T::BM;
  const dim3 grid(grid_of("wm_linear_fp8", 8 * ((n_tiles * t_tiles + 7) / 8), 64 * T::WAVES));
  if (a.k % BLOCK) hipLaunchKernelGGL((tiled_kernel<T, F32, true>), grid, dim3(64 * T::WAVES), 0, s, a, (int)n_tiles, (int)t_tiles);
  else hipLaunchKernelGGL((tiled_kernel<T, F32, false>), grid, dim3(64 * T::WAVES), 0, s, a, (int)n_tiles, (int)t_tiles);
  check_launch("linear_fp8 (tiled)");
}

using Large = Tile<8, 4, 2, 4, 2>;   // 256 x 256
using Wide = Tile<4, 4, 2, 4, 3>;    // 128 x 256, for bf16 operands, which are twice the registers
using Middle = Tile<4, 4, 2, 2, 2>;  // 128 x 128
using Small = Tile<2, 2, 2, 2, 4>;   // 64 x 64

template <bool F32>
static void launch(const Args& a, hipStream_t s) {
  if (a.tokens <= 16) {
    if (a.n >= 16384) return launch_stream<2, 1, 3, F32>(a, s);
    return launch_stream<1, 1, 4, F32>(a, s);
  }
  if (a.tokens <= 32) return launch_stream<1, 2, 3, F32>(a, s);
  if (a.tokens <= 64) return launch_stream<1, 4, 2, F32>(a, s);
  auto blocks = [&](int64_t n, int64_t t) { return ((a.n + n - 1) / n) * ((a.tokens + t - 1) / t); };
  if constexpr (F32) {
    if (blocks(128, 256) >= 256) return launch_tiled<Wide, F32>(a, s);
  } else {
    if (blocks(256, 256) >= 256) return launch_tiled<Large, F32>(a, s);
  }
  if (blocks(128, 128) >= 256) return launch_tiled<Middle, F32>(a, s);
  launch_tiled<Small, F32>(a, s);
}

}  // namespace g8
}  // namespace wm

using namespace wm;

extern "C" {

WM_EXPORT int wm_linear_fp8(const void* x, const float* x_scales, int32_t tokens, int32_t k, const void* weight,
                            const float* weight_scales, int32_t n, const void* add, int32_t out_fp32, void* out, void* stream) {
  return guarded([&] {
    constexpr int MOST = INT32_MAX - 65535;
    if (tokens < 0 || tokens > MOST) fail("wm_linear_fp8: tokens must be in 0..2147418112");
    if (k < 1 || k % 16 || k > 1 << 20) fail("wm_linear_fp8: k must be a multiple of 16 in 16..1048576");
    if (n < 1 || n > MOST) fail("wm_linear_fp8: n must be in 1..2147418112");
    if (out_fp32 != 0 && out_fp32 != 1) fail("wm_linear_fp8: out_fp32 must be 0 (bf16) or 1");
    if (tokens == 0) return;
    if (!x || !x_scales || !weight || !weight_scales || !out) fail("wm_linear_fp8: null pointer");
    if (((uintptr_t)x | (uintptr_t)weight) % 16) fail("wm_linear_fp8: x and weight must be 16-byte aligned");
    if (((uintptr_t)x_scales | (uintptr_t)weight_scales) % 4 || ((uintptr_t)add | (uintptr_t)out) % (out_fp32 ? 4 : 2))
      fail("wm_linear_fp8: tensors must be aligned to their elements");
    const g8::Args a = {(const uint8_t*)x, x_scales, (const uint8_t*)weight, weight_scales, add, out, tokens, n, k, (k + 127) / 128};
    if (out_fp32) g8::launch<true>(a, as_stream(stream));
    else g8::launch<false>(a, as_stream(stream));
  });
}

}  // extern "C"
