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
//
// Few tokens are bound by the weights' bytes (captured calls, 1 token of 7168 to 4096: 4.7 us with the weights in the caches,
// 6.8 from memory, 4.3 TB/s; 6 tokens to 129,280 in fp32 141 us, 6.6 TB/s), many by the matrix units and what a tile does
// before and behind its loop (16,384 tokens of 7168 to 4096 452 us, 2.13 PFLOP/s; 8192^3 524 us, 2.10).
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
// stream: few tokens, where the weights' way from memory is what counts. A block of W waves owns 16 TN weight rows x 16 TM
// tokens; the waves take the blocks of K in turn, each through a ring of its own of D slots in LDS, so that no wave waits
// for another one until the sums meet at the end, added in wave order. A block of K comes as direct loads of
// 8 rows of 128 bytes, whole lines: X rows of tokens (8 where that is all). A wave's scales come for eight of its blocks at
// once, 8 tokens a load: a block's alone would be a line for each token.
template <int N>
__device__ __forceinline__ void wait_own() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
template <int PER, int MOST>
__device__ __forceinline__ void wait_own_steps(int ahead) {
  if (ahead >= MOST) {
    wait_own<PER * MOST>();
  } else if constexpr (MOST > 0) {
    wait_own_steps<PER, MOST - 1>(ahead);
  }
}

template <int TN_, int TM_, int X_, int W_, int D_>
struct Stream {
  static constexpr int TN = TN_, TM = TM_, X = X_, W = W_, D = D_;
  static constexpr int BN = 16 * TN, BM = 16 * TM;
  static constexpr int WEIGHTS = BN * BLOCK, SLOT = WEIGHTS + X * BLOCK;
  static constexpr int SCALES = 32 * X + 256;  // of eight blocks: [token][8], and the weights'
  static constexpr int LOADS = 2 * TN + X / 8;
  static constexpr int OWN = D * SLOT + 2 * SCALES, RING = W * OWN, SUMS = W * TN * TM * 1024, LDS = RING > SUMS ? RING : SUMS;
  static_assert(BLOCK % BN == 0 && X % 8 == 0 && (X == BM || (X == 8 && TM == 1)) && D <= 8 && LDS <= 160 * 1024 &&
                LOADS * (D - 1) <= 63);
};

template <typename T, bool F32, bool TAIL>
__global__ void __launch_bounds__(64 * T::W) stream_kernel(Args a, int n_tiles) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[T::LDS];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int n0 = blockIdx.x % n_tiles * T::BN, t0 = blockIdx.x / n_tiles * T::BM;
  // lane l fills row l / 8, position l % 8 with the piece (l % 8) ^ (row % 8); rows past the end read the last one
  const int lrow = lane / 8, piece = (lane % 8) ^ lrow;
  const uint8_t* wbase = a.w + (int64_t)n0 * a.k;
  const uint8_t* xbase = a.x + (int64_t)t0 * a.k;
  uint32_t woff[2 * T::TN], xoff[T::X / 8];
#pragma unroll
  for (int i = 0; i < 2 * T::TN; ++i) woff[i] = (uint32_t)(min(n0 + 8 * i + lrow, a.n - 1) - n0) * (uint32_t)a.k + 16u * piece;
#pragma unroll
  for (int i = 0; i < T::X / 8; ++i) xoff[i] = (uint32_t)(min(t0 + 8 * i + lrow, a.tokens - 1) - t0) * (uint32_t)a.k + 16u * piece;
  const float* xsbase = a.xs + (int64_t)t0 * a.blocks;
  const float* wsbase = a.ws + (int64_t)(n0 / BLOCK) * a.blocks;
  uint8_t* ring = lds + wave * T::OWN;
  uint8_t* scales = ring + T::D * T::SLOT;
  // the scales of this wave's blocks j .. j + 7, j a multiple of 8
  auto issue_scales = [&](int j) {
    const uint32_t to = lds_addr(scales + j / 8 % 2 * T::SCALES);
    const uint32_t block = (uint32_t)min(wave + T::W * (j + lane % 8), a.blocks - 1);
#pragma unroll
    for (int i = 0; i < T::X / 8; ++i)
      dma4(xsbase, 4u * ((uint32_t)(min(t0 + 8 * i + lrow, a.tokens - 1) - t0) * (uint32_t)a.blocks + block), to + 256 * i);
    dma4(wsbase, 4u * block, to + 32 * T::X);
  };
  auto issue = [&](int b, int slot) {
    const uint32_t to = lds_addr(ring + slot * T::SLOT);
    // pieces behind the rows' end read the block's first one
    const uint32_t off = (uint32_t)BLOCK * b - (TAIL && BLOCK * b + 16 * piece >= a.k ? 16u * piece : 0u);
#pragma unroll
    for (int i = 0; i < 2 * T::TN; ++i) dma16<(T::X <= 16)>(wbase, woff[i] + off, to + 1024 * i);
#pragma unroll
    for (int i = 0; i < T::X / 8; ++i) dma16(xbase, xoff[i] + off, to + T::WEIGHTS + 1024 * i);
  };
  f32x4 acc[T::TN][T::TM];
#pragma unroll
  for (int j = 0; j < T::TN; ++j)
#pragma unroll
    for (int m = 0; m < T::TM; ++m) acc[j][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const int c = lane % 16, g = lane / 16, xc = c % T::X;
  const uint32_t pos = 16u * (uint32_t)(g ^ (c % 8));
  auto multiply = [&](int j, int slot) {
    const int b = wave + T::W * j;
    const uint8_t* s = ring + slot * T::SLOT;
    const float* sc = reinterpret_cast<const float*>(scales + j / 8 % 2 * T::SCALES) + j % 8;
    auto frag = [&](uint32_t at) {
      Frag f = {*reinterpret_cast<const uint4*>(s + at), *reinterpret_cast<const uint4*>(s + (at ^ 64u))};
      if (TAIL && b == a.blocks - 1) zero_behind(f, g, (a.k - b * BLOCK) / 16);
      return Operand<F32>(f);
    };
    const float ws = sc[8 * T::X];
    Operand<F32> w[T::TN];
#pragma unroll
    for (int i = 0; i < T::TN; ++i) w[i] = frag((16 * i + c) * BLOCK + pos);
#pragma unroll
    for (int m = 0; m < T::TM; ++m) {
      const Operand<F32> x = frag(T::WEIGHTS + (16 * m + xc) * BLOCK + pos);
      const float f = ws * sc[8 * (16 * m + xc)];
#pragma unroll
      for (int i = 0; i < T::TN; ++i) {
        const f32x4 d = Operand<F32>::product(w[i], x);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][m][e] = fmaf(d[e], f, acc[i][m][e]);
      }
    }
  };
  const int mine = (a.blocks - wave + T::W - 1) / T::W;  // this wave's blocks: wave, wave + W, ..
#pragma unroll
  for (int p = 0; p < T::D; ++p)
    if (p < mine) {
      if (p == 0) issue_scales(0);
      issue(wave + T::W * p, p);
    }
  int slot = 0;
  for (int j = 0; j < mine; ++j) {
    wait_own_steps<T::LOADS, T::D - 1>(mine - 1 - j);  // scales among the loads ahead make it wait for more than it must
    multiply(j, slot);
    if (j + T::D < mine) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the slot's reads have come back
      if ((j + T::D) % 8 == 0) issue_scales(j + T::D);
      issue(wave + T::W * (j + T::D), slot);
    }
    slot = slot + 1 == T::D ? 0 : slot + 1;
  }

  __syncthreads();  // the sums lie over the rings
  float(*red)[T::TN * T::TM][4][64] = reinterpret_cast<float(*)[T::TN * T::TM][4][64]>(lds);
#pragma unroll
  for (int j = 0; j < T::TN; ++j)
#pragma unroll
    for (int m = 0; m < T::TM; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) red[wave][j * T::TM + m][i][lane] = acc[j][m][i];
  __syncthreads();
  for (int e = threadIdx.x; e < 256 * T::TN * T::TM; e += 64 * T::W) {
    const int o = e % T::BN, tc = e / T::BN;  // weight row and token of the tile
    const int at = o / 16 * T::TM + tc / 16, i = o % 4, l = 16 * (o % 16 / 4) + tc % 16;
    float v = red[0][at][i][l];
#pragma unroll
    for (int q = 1; q < T::W; ++q) v += red[q][at][i][l];
    if (t0 + tc < a.tokens && n0 + o < a.n) store_one<F32>(a, t0 + tc, n0 + o, v);
  }
}

// ---------------------------------------------------------------------------------
// tiled: WN x WM waves, each 16 TN weight rows x 16 TM tokens. A step is KB blocks of K: their rows of 128 bytes and their scales
// go straight to LDS, STAGES steps at once, pieces of 16 bytes XOR-swizzled by row, so that the 8 rows of a
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

template <int TN_, int TM_, int WN_, int WM_, int KB_, int STAGES_, bool ONCE_ = false>
struct Tile {
  static constexpr bool ONCE = ONCE_;  // the weights pass once: loads with the non-temporal hint
  static constexpr int TN = TN_, TM = TM_, WN = WN_, WM = WM_, KB = KB_, STAGES = STAGES_, WAVES = WN * WM;
  static constexpr int BN = 16 * TN * WN, BM = 16 * TM * WM;
  static constexpr int W = BN * BLOCK, X = BM * BLOCK, SCALES = KB * (W + X);  // a stage: KB blocks' rows, then their scales
  static constexpr int XS = BM * KB / 64, STAGE = SCALES + 256 * (XS + 1);
  static constexpr int WL = KB * BN / 8 / WAVES, XL = KB * BM / 8 / WAVES;  // row loads of a wave
  static constexpr int LOADS = WL + XL + 1;                                 // and one of scales
  static_assert(BN % (8 * WAVES) == 0 && BM % (8 * WAVES) == 0 && BM * KB % 64 == 0 && XS < WAVES && BN * KB <= 64 * BLOCK && 128 % (16 * TN) == 0);
  static_assert(STAGES * STAGE <= 160 * 1024 && LOADS * (STAGES - 1) <= 63);
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
  constexpr int WR = T::WL / T::KB, XR = T::XL / T::KB;  // row loads of a block
  uint32_t woff[WR], xoff[XR];
#pragma unroll
  for (int i = 0; i < WR; ++i)
    woff[i] = (uint32_t)(min(n0 + 8 * (wave + T::WAVES * i) + lrow, a.n - 1) - n0) * (uint32_t)a.k + 16u * piece;
#pragma unroll
  for (int i = 0; i < XR; ++i)
    xoff[i] = (uint32_t)(min(t0 + 8 * (wave + T::WAVES * i) + lrow, a.tokens - 1) - t0) * (uint32_t)a.k + 16u * piece;
  // a load of scales: KB blocks side by side of 64 / KB tokens (the waves below XS) or weight rows of blocks
  const bool tokens_scales = wave < T::XS;
  const float* sbase = tokens_scales ? a.xs + (int64_t)t0 * a.blocks : a.ws + (int64_t)(n0 / BLOCK) * a.blocks;
  const uint32_t sdst = T::SCALES + 256u * (tokens_scales ? wave : T::XS);
  const uint32_t srow = (uint32_t)(tokens_scales ? min(t0 + (64 * wave + lane) / T::KB, a.tokens - 1) - t0
                                                 : min(lane / T::KB, (a.n - 1) / BLOCK - n0 / BLOCK)) * (uint32_t)a.blocks;
  // Load i of the LOADS of the blocks KB step .. of a step. Blocks behind the last read that one again, and are not used.
  auto issue = [&](int step, int i) {
    const uint32_t slot = lds_addr(lds + step % T::STAGES * T::STAGE);
    if (i == T::WL + T::XL) return dma4(sbase, 4u * (srow + (uint32_t)min(T::KB * step + lane % T::KB, a.blocks - 1)), slot + sdst);
    const int kb = i < T::WL ? i / WR : (i - T::WL) / XR;
    const int b = min(T::KB * step + kb, a.blocks - 1);
    // pieces behind the rows' end read the block's first one
    const uint32_t off = (uint32_t)BLOCK * b - (TAIL && BLOCK * b + 16 * piece >= a.k ? 16u * piece : 0u);
    const uint32_t to = slot + kb * (T::W + T::X);
    if (i < T::WL) dma16<T::ONCE>(wbase, woff[i % WR] + off, to + 1024 * (wave + T::WAVES * (i % WR)));
    else dma16(xbase, xoff[(i - T::WL) % XR] + off, to + T::W + 1024 * (wave + T::WAVES * ((i - T::WL) % XR)));
  };

  f32x4 acc[T::TN][T::TM];
#pragma unroll
  for (int i = 0; i < T::TN; ++i)
#pragma unroll
    for (int m = 0; m < T::TM; ++m) acc[i][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const int c = lane % 16, g = lane / 16;
  const uint32_t pos = 16u * (uint32_t)(g ^ (c % 8));
  const uint32_t wrow = (uint32_t)(16 * T::TN * wn + c) * BLOCK + pos, xrow = T::W + (uint32_t)(16 * T::TM * wm + c) * BLOCK + pos;
  const uint32_t xscale = T::SCALES + 4u * T::KB * (16 * T::TM * wm + c);
  const uint32_t wscale = T::SCALES + 256u * T::XS + 4u * T::KB * (16 * T::TN * wn / BLOCK);

  // A step's sums. The multiply-adds of a matrix instruction's results stand beside the instruction TM later, so that
  // none waits for them (the last ones of a block beside the next block's first). With AHEAD the loads of the step STAGES - 1
  // behind it go out between the instructions of the step's first two thirds.
  f32x4 d[T::TM];
  float f[T::TM];
#pragma unroll
  for (int m = 0; m < T::TM; ++m) d[m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f[m] = 0.0f;
  auto step = [&](int p, auto ahead, auto last) {
    constexpr bool AHEAD = decltype(ahead)::value, LAST = decltype(last)::value;
    const uint8_t* s = lds + p % T::STAGES * T::STAGE;
#pragma unroll
    for (int kb = 0; kb < T::KB; ++kb) {
      const int b = T::KB * p + kb;
      if (LAST && kb > 0 && b >= a.blocks) break;
      auto frag = [&](uint32_t at) {
        at += kb * (T::W + T::X);
        Frag f = {*reinterpret_cast<const uint4*>(s + at), *reinterpret_cast<const uint4*>(s + (at ^ 64u))};
        if (TAIL && LAST && b == a.blocks - 1) zero_behind(f, g, (a.k - b * BLOCK) / 16);
        return Operand<F32>(f);
      };
      Operand<F32> x[T::TM], w[2];
      w[0] = frag(wrow);
#pragma unroll
      for (int m = 0; m < T::TM; ++m) x[m] = frag(xrow + 16 * BLOCK * m);
      const float ws = *reinterpret_cast<const float*>(s + wscale + 4 * kb);
      float xs[T::TM];
#pragma unroll
      for (int m = 0; m < T::TM; ++m) xs[m] = *reinterpret_cast<const float*>(s + xscale + 64 * T::KB * m + 4 * kb);
#pragma unroll
      for (int i = 0; i < T::TN; ++i) {
        if (i + 1 < T::TN) w[(i + 1) % 2] = frag(wrow + 16 * BLOCK * (i + 1));
        if (AHEAD) {
          constexpr int PER = (3 * T::LOADS + 2 * T::TN * T::KB - 1) / (2 * T::TN * T::KB);
          const int at = kb * T::TN + i;
#pragma unroll
          for (int q = at * PER; q < (at + 1) * PER && q < T::LOADS; ++q) issue(p + T::STAGES - 1, q);
        }
#pragma unroll
        for (int m = 0; m < T::TM; ++m) {
          const f32x4 r = Operand<F32>::product(w[i % 2], x[m]);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[(i + T::TN - 1) % T::TN][m][e] = fmaf(d[m][e], f[m], acc[(i + T::TN - 1) % T::TN][m][e]);
          if (i == 0) f[m] = ws * xs[m];
          d[m] = r;
          __builtin_amdgcn_sched_barrier(0);  // the order as it is written
        }
      }
    }
  };
  const std::true_type yes;
  const std::false_type no;
  const int steps = (a.blocks + T::KB - 1) / T::KB;
  int p = 0;
  for (; p < T::STAGES - 1 && p < steps; ++p)
#pragma unroll
    for (int i = 0; i < T::LOADS; ++i) issue(p, i);
  // at the top of a step its loads have landed in every wave, and every wave is done with the slot that the next
  // loads overwrite
  for (p = 0; p + T::STAGES - 1 < steps; ++p) {
    wait_loads<T::LOADS * (T::STAGES - 2)>();
    step(p, yes, no);
  }
  for (; p + 1 < steps; ++p) {
    wait_step<T::LOADS, T::STAGES - 2>(steps - 1 - p);
    step(p, no, no);
  }
  wait_loads<0>();
  step(p, no, yes);
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

template <typename T, bool F32>
static void launch_stream(const Args& a, hipStream_t s) {
  const int64_t n_tiles = (a.n + T::BN - 1) / T::BN, t_tiles = (a.tokens + T::BM - 1) / T::BM;
  const dim3 grid(grid_of("wm_linear_fp8", n_tiles * t_tiles, 64 * T::W));
  if (a.k % BLOCK) hipLaunchKernelGGL((stream_kernel<T, F32, true>), grid, dim3(64 * T::W), 0, s, a, (int)n_tiles);
  else hipLaunchKernelGGL((stream_kernel<T, F32, false>), grid, dim3(64 * T::W), 0, s, a, (int)n_tiles);
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

// The kernel of a shape. All times here but those of the last paragraph are of calls in a row on one to three matrices, which
// the 256 MB cache holds where they are small; from memory the shapes of 1 to 256 tokens take 1.2 to 1.5 times as
// long (captured, 32, 96 and 256 tokens of 5120 to 4608: 7.6, 11.7 and 18.6 us warm, 11.1, 14.8 and 25.1 cold). Up to 16 tokens the weights' way from memory is all: 16 weight rows a block with 8 waves while
// that gives two blocks a CU at most, 32 with 4 waves beyond (one token of 7168 to 4096 5.8 us and 7.3, to 24576 31.7 and
// 26.8). Their rows pass once, so their loads are non-temporal (1 token of 7168 to 24576 30.2 us without, 26.8 with, six to
// 129,280 154 and 134; for 64 tokens, where two blocks take a row, 12.3 with and 9.7 without).
// Otherwise the shape with the lowest cost, rounds of 256 blocks times what a block of K takes in a round. Larger tiles move fewer
// bytes and take more matrix instructions a barrier, smaller ones fill the chip sooner; the rounds decide. Costs are
// in units of 10 ns, measured at one round and more of K = 7168 to bf16; fp32 takes 1.6 times of each. The sizes' times in
// us, the cheapest first and the next ones by cost:
//   64 x 4096 x 7168   32 x 32 10.1, 64 x 32 13.4        256 x 4096 x 7168  64 x 64 19.1, 64 x 128 23, 64 x 32 27.5
//   128 x 4096 x 7168  64 x 32 14.5, 64 x 64 16.4        512 x 4096 x 7168  64 x 128 28, 128 x 128 34, 64 x 64 35
//   96 x 4608 x 5120   64 x 32 11.7, 64 x 64 12.8        1024 x 4096 x 7168  128 x 128 41.5, 64 x 128 53, 128 x 256 55
//   300 x 7168 x 2048  128 x 128 12.9, 64 x 64 18.4      2048 x 4096 x 7168  128 x 256 82, 128 x 128 91, 256 x 256 92
//   1501 x 1283 x 2560  64 x 128 12.9, 64 x 64 16        4096 x 4096 x 7168  256 x 256 112, 128 x 256 147
//
// Where the choice falls on the 64 x 64 or the 128 x 128 tile, one token tile and weights that no cache holds from call to
// call pass once, with twice the blocks of K a step, so longer runs of a row, two steps deep, and non-temporal loads (in turn
// without and with; 64 x 24576 x 7168 58.4 and 49.4, 128 x 129280 x 7168 287 and 254, to fp32 313 and 292, 64 x 20480 x 5120 (105 MB)
// 43.4 and 36.1; 64 x 16384 x 5120 (84 MB, held by the 256 MB cache) 17.1 and 22.9, 128 x 32768 x 2048 (67 MB) 22.4 and 22.6).
// The other shapes have no such form. The streams of 32 tokens read large weights at 5.1 to 5.4 TB/s as they are (17, 24 and 32 x
// 129280 x 7168 172, 177 and 183 us, to fp32 179, 182 and 191; 32 x 24576 x 7168 39); 64 x 128 tiles, which 65 to 128 tokens
// of 16384 x 7168 (117 MB) take, at 3.1 to 3.3 (37 to 40 us cold).
constexpr int64_t ONCE_BYTES = 100000000;
template <bool F32>
static void launch(const Args& a, hipStream_t s) {
  if (a.tokens <= 16) {
    const bool few = a.n <= 8192;
    if (a.tokens <= 8) return few ? launch_stream<Stream<1, 1, 8, 8, 4>, F32>(a, s) : launch_stream<Stream<2, 1, 8, 4, 3>, F32>(a, s);
    return few ? launch_stream<Stream<1, 1, 16, 8, 4>, F32>(a, s) : launch_stream<Stream<2, 1, 16, 4, 3>, F32>(a, s);
  }
  constexpr int SHAPES = F32 ? 7 : 8;  // bf16 operands are twice the registers: no 256 x 256
  constexpr struct { int n, t, cost; } shape[8] = {{16, 32, 8}, {32, 32, 13}, {64, 32, 21}, {64, 64, 28},
                                                   {64, 128, 45}, {128, 128, 70}, {128, 256, 135}, {256, 256, 175}};
  int best = 0;
  int64_t least = INT64_MAX;
  for (int i = 0; i < SHAPES; ++i) {
    const int64_t blocks = ((int64_t)(a.n + shape[i].n - 1) / shape[i].n) * ((a.tokens + shape[i].t - 1) / shape[i].t);
    const int64_t cost = (blocks + 255) / 256 * shape[i].cost;
    if (cost < least) least = cost, best = i;
  }
  const bool once = a.tokens <= shape[best].t && (int64_t)a.n * a.k >= ONCE_BYTES;
  switch (best) {
    case 0: return launch_stream<Stream<1, 2, 32, 4, 3>, F32>(a, s);
    case 1: return launch_stream<Stream<2, 2, 32, 4, 2>, F32>(a, s);
    case 2: return launch_stream<Stream<4, 2, 32, 4, 2>, F32>(a, s);
    case 3:
      if (once) return launch_tiled<Tile<2, 1, 2, 4, 4, 2, true>, F32>(a, s);
      return launch_tiled<Tile<2, 1, 2, 4, 2, 4>, F32>(a, s);
    case 4: return launch_tiled<Tile<2, 2, 2, 4, 2, 3>, F32>(a, s);
    case 5:
      if (once) return launch_tiled<Tile<4, 2, 2, 4, 2, 2, true>, F32>(a, s);
      return launch_tiled<Tile<4, 2, 2, 4, 1, 4>, F32>(a, s);
    case 6: return launch_tiled<Tile<4, 4, 2, 4, 1, 3>, F32>(a, s);
    default:
      if constexpr (!F32) launch_tiled<Tile<8, 4, 2, 4, 1, 2>, F32>(a, s);
  }
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
