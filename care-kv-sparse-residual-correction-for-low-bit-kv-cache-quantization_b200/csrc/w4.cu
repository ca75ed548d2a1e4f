// Products of a few activation rows with a 4-bit weight:
//   y[m][n] = sum_G s[n][G] sum_{k in group G} c[n][k] x[m][k],
// codes c in -8..7, one scale per (row, group of channels).
//
// Codes are small integers, exact in fp16 and bf16, so the inner sums run on
// the tensor cores (m16n8k16, fp32 accumulators) with the weight rows on the
// M side and up to 8 activation rows on the N side of one instruction; the
// scale multiplies the group's fp32 sum, so no weight is ever rounded.  fp32
// activations are split into three bf16 terms whose sum is the value itself.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "internal.h"
#include "launch.h"
#include "ptx.cuh"
#include "tcgen05.cuh"

namespace cg = cooperative_groups;

namespace carekv {
namespace {

// ── layout ──────────────────────────────────────────────────────────────
// A tile is 16 weight rows x 128 channels, 1 KB of codes: lane l = 4 g + t
// of a warp holds, for row g and then for row g + 8 of the tile, 16 bytes =
// four words, word j with the codes of channels 32 j + 8 t .. + 7.  These are
// the lane's fragments of two m16n8k16 products per word, so a warp reads a
// tile with two coalesced 16-byte loads per lane and no exchange; the
// channels of the product's k index are permuted alike on the activation
// side, whose 8 channels of word j are 16 consecutive bytes.
// Nibble i of a word holds code + 8 of channel 2 i (i < 4) or 2 (i - 4) + 1,
// so one mask picks the pair (2p, 2p + 1) into the two halves of a register.
// Scales of a tile: [16 rows][ns], ns = 128 / group below 128, else 1.
// The 8 tiles (panels) of 128 rows at the same channels lie together, blocks
// of 128 rows one after another: one 8 KB copy brings a block's tile (8
// copies of 1 KB, a panel's tiles in a row, took 0.9 us a tile).
constexpr int kTileRows = 16, kTileK = 128, kTileBytes = 1024, kBlockPanels = 8;

__host__ __device__ inline int64_t tile_at(int64_t panel, int kt, int kt_n) {
  return (panel / kBlockPanels * kt_n + kt) * kBlockPanels + panel % kBlockPanels;
}

__host__ __device__ inline int tile_scales(int group) { return group >= kTileK ? 1 : kTileK / group; }

__global__ void __launch_bounds__(256) w4_pack_kernel(const uint8_t* __restrict__ packed, const void* __restrict__ scale,
                                                      int N, int K, int group, int dt, uint32_t* __restrict__ codes,
                                                      void* __restrict__ scales, int64_t words, int kt_n) {
  const int64_t w = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (w >= words) return;
  const int64_t tile = w >> 8;
  const int in = static_cast<int>(w & 255), hi = in >> 7, lane = (in >> 2) & 31, j = in & 3;
  const int64_t panel = tile / kBlockPanels / kt_n * kBlockPanels + tile % kBlockPanels;
  const int kt = static_cast<int>(tile / kBlockPanels % kt_n);
  const int64_t n = panel * kTileRows + hi * 8 + (lane >> 2);
  const int k0 = kt * kTileK + 32 * j + 8 * (lane & 3);
  uint32_t v = 0x88888888u;   // code 0
  if (n < N && k0 < K) {
    // reference row format: low nibble = even channel, two's complement
    const uint8_t* p = packed + n * (K / 2) + k0 / 2;
    v = 0;
    for (int b = 0; b < 4; ++b) {
      const uint32_t x = p[b] ^ 0x88u;
      v |= (x & 15u) << (4 * b) | (x >> 4) << (4 * b + 16);
    }
  }
  codes[w] = v;
  const int ns = tile_scales(group);
  if (in < kTileRows * ns) {
    const int64_t row = panel * kTileRows + in / ns;
    const int k = kt * kTileK + (in % ns) * group;
    const float s = row < N && k < K ? load_act(scale, row * (K / group) + k / group, dt) : 0.f;
    store_act(scales, tile * (kTileRows * ns) + in, s, dt);
  }
}

// dense row-major weight, c * s rounded to the scale's type
__global__ void __launch_bounds__(256) w4_dequant_kernel(const uint32_t* __restrict__ codes,
                                                         const void* __restrict__ scales, int N, int K, int group,
                                                         int dt, void* __restrict__ out, int64_t words, int kt_n) {
  const int64_t w = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (w >= words) return;
  const int64_t tile = w >> 8;
  const int in = static_cast<int>(w & 255), hi = in >> 7, lane = (in >> 2) & 31, j = in & 3;
  const int row = hi * 8 + (lane >> 2);
  const int64_t n = (tile / kBlockPanels / kt_n * kBlockPanels + tile % kBlockPanels) * kTileRows + row;
  const int kk = 32 * j + 8 * (lane & 3);
  const int64_t k0 = tile / kBlockPanels % kt_n * kTileK + kk;
  if (n >= N || k0 >= K) return;
  const int ns = tile_scales(group);
  const float s = load_act(scales, tile * (kTileRows * ns) + row * ns + (ns > 1 ? kk / group : 0), dt);
  const uint32_t v = codes[w];
  for (int p = 0; p < 4; ++p) {
    store_act(out, n * K + k0 + 2 * p, static_cast<float>(static_cast<int>((v >> (4 * p)) & 15u) - 8) * s, dt);
    store_act(out, n * K + k0 + 2 * p + 1, static_cast<float>(static_cast<int>((v >> (4 * p + 16)) & 15u) - 8) * s, dt);
  }
}

// ── products ────────────────────────────────────────────────────────────
__device__ __forceinline__ uint32_t bsub(uint32_t a, uint32_t b) {
  __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<uint32_t*>(&r);
}
// D = A . B + C, m16n8k16.  Not volatile: the compiler may put independent
// products between two that share a sum.
template <bool F16>
__device__ __forceinline__ void mma_add(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  if constexpr (F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same with C = 0
template <bool F16>
__device__ __forceinline__ void mma_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  if constexpr (F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%10,%10,%10,%10};\n"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// The 8 codes of a word as four exact pairs: a nibble put at mantissa bit b
// of a float whose exponent makes that bit worth 1 reads as 2^e + u, and one
// subtraction of 2^e + 8 leaves the code.  fp16 has room for nibbles at bits
// 0 and 4 (one shift per word), bf16 at bit 0 only (three).  Mask and
// exponent are one three-input operation if one of the two constants is in a
// register: they are kernel arguments, which the compiler cannot fold (as
// literals they took two operations per pair, 32 of 189 per tile).
struct Keys {
  uint32_t e0, e4;   // exponents of nibbles at bit 0 and (fp16) bit 4, in both halves
};
template <bool F16>
constexpr Keys kKeys = F16 ? Keys{0x64006400u, 0x54005400u} : Keys{0x43004300u, 0u};

template <bool F16>
__device__ __forceinline__ void codes8(uint32_t w, const Keys& k, uint32_t (&r)[4]) {
  if constexpr (F16) {
    const uint32_t v = w >> 8;
    r[0] = h2sub((w & 0x000F000Fu) | k.e0, 0x64086408u);
    r[1] = h2sub((w & 0x00F000F0u) | k.e4, 0x54805480u);
    r[2] = h2sub((v & 0x000F000Fu) | k.e0, 0x64086408u);
    r[3] = h2sub((v & 0x00F000F0u) | k.e4, 0x54805480u);
  } else {
#pragma unroll
    for (int p = 0; p < 4; ++p) r[p] = bsub(((w >> (4 * p)) & 0x000F000Fu) | k.e0, 0x43084308u);
  }
}

template <int DT>
struct Act;   // activation fragments: 8 channels as TERMS x 4 pairs
template <>
struct Act<CAREKV_F16> {
  static constexpr int kTerms = 1;
  static constexpr bool kF16 = true;
  using T = __half;
  using S = __half;
  static __device__ __forceinline__ void load(const T* p, uint32_t (&b)[1][4]) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
    b[0][0] = v.x, b[0][1] = v.y, b[0][2] = v.z, b[0][3] = v.w;
  }
  static __device__ __forceinline__ float scale(S s) { return __half2float(s); }
  static __device__ __forceinline__ T out(float v) { return __float2half_rn(v); }
};
template <>
struct Act<CAREKV_BF16> {
  static constexpr int kTerms = 1;
  static constexpr bool kF16 = false;
  using T = __nv_bfloat16;
  using S = __nv_bfloat16;
  static __device__ __forceinline__ void load(const T* p, uint32_t (&b)[1][4]) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
    b[0][0] = v.x, b[0][1] = v.y, b[0][2] = v.z, b[0][3] = v.w;
  }
  static __device__ __forceinline__ float scale(S s) { return __bfloat162float(s); }
  static __device__ __forceinline__ T out(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Act<CAREKV_F32> {
  static constexpr int kTerms = 3;
  static constexpr bool kF16 = false;
  using T = float;
  using S = float;
  // x = hi + mid + lo: each term the upper 16 bits of what is left, 8
  // significand bits of the 24, so the split is exact (down to bf16's
  // smallest numbers); infinities and NaN stay in the first term, a NaN by its
  // quiet bit (its payload may lie in the lower 16 bits alone)
  static __device__ __forceinline__ void load(const T* p, uint32_t (&b)[3][4]) {
    float x[8];
    *reinterpret_cast<float4*>(x) = __ldg(reinterpret_cast<const float4*>(p));
    *reinterpret_cast<float4*>(x + 4) = __ldg(reinterpret_cast<const float4*>(p) + 1);
#pragma unroll
    for (int i = 0; i < 3; ++i) {
#pragma unroll
      for (int k = 0; k < 8; k += 2) {
        uint32_t lo = __float_as_uint(x[k]), hi = __float_as_uint(x[k + 1]);
        if (i == 0) {
          if ((lo & 0x7fffffffu) > 0x7f800000u) lo |= 0x00400000u;
          if ((hi & 0x7fffffffu) > 0x7f800000u) hi |= 0x00400000u;
        }
        b[i][k / 2] = prmt(lo, hi, 0x7632);
        x[k] = (lo & 0x7f800000u) == 0x7f800000u ? 0.f : x[k] - __uint_as_float(lo & 0xffff0000u);
        x[k + 1] = (hi & 0x7f800000u) == 0x7f800000u ? 0.f : x[k + 1] - __uint_as_float(hi & 0xffff0000u);
      }
    }
  }
  static __device__ __forceinline__ float scale(S s) { return s; }
  static __device__ __forceinline__ T out(float v) { return v; }
};

// Half a word of the tile (16 of its 32 channels): codes of rows g / g + 8
// times the activations of one column tile, added to a fp32 sum.
template <typename A>
__device__ __forceinline__ void mma_half(float (&sum)[4], const uint32_t (&a)[4], const uint32_t (&b)[4],
                                         const uint32_t (&x)[A::kTerms][4], int h, bool first) {
#pragma unroll
  for (int i = 0; i < A::kTerms; ++i) {
    if (first && i == 0) mma_first<A::kF16>(sum, a[2 * h], b[2 * h], a[2 * h + 1], b[2 * h + 1], x[i][2 * h], x[i][2 * h + 1]);
    else mma_add<A::kF16>(sum, a[2 * h], b[2 * h], a[2 * h + 1], b[2 * h + 1], x[i][2 * h], x[i][2 * h + 1]);
  }
}
__device__ __forceinline__ void add_scaled(float (&acc)[4], const float (&sum)[4], float s0, float s1) {
  acc[0] = fmaf(s0, sum[0], acc[0]);
  acc[1] = fmaf(s0, sum[1], acc[1]);
  acc[2] = fmaf(s1, sum[2], acc[2]);
  acc[3] = fmaf(s1, sum[3], acc[3]);
}

// A tile's codes and scales (rows g and g + 8) as one lane holds them.
template <typename S, int NS>
struct alignas(sizeof(S) * NS) ScaleVec {
  S v[NS];
};
template <typename S, int NS>
struct Tile {
  uint4 c0, c1;
  ScaleVec<S, NS> s0, s1;
};
__device__ __forceinline__ uint32_t word(const uint4& v, int j) { return j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w; }

// Few rows (up to 8 MT): one CTA per RT x 16 weight rows, its WK warps take
// the tiles of the rows in turn and add their sums in shared memory.  The
// next tile's loads are issued before the present tile's products;
// activations come through L1.  Column lanes past the last row repeat row 0
// (their sums are not stored).  Bound by the latency of the loads at as many
// warps as the registers leave room for: with all inputs out of the L2, 1 row
// x 13824 x 5120 11.6 us, 3.2 TB/s (issue active 49% of the time, 28 warps an
// SM at most); 1 x 4096 x 4096 4.6 us; 16 rows x 14336 x 4096 22.5 us (issue
// active 40%, 12 warps an SM at 153 registers).
template <int DT, int NS, int MT, int RT, int WK>
__global__ void __launch_bounds__(WK * 32) w4_kernel(const typename Act<DT>::T* __restrict__ x, int64_t ldx, int M,
                                                     const uint4* __restrict__ codes,
                                                     const typename Act<DT>::S* __restrict__ scales, int N, int K,
                                                     int kt_n, int panels, const Keys keys,
                                                     typename Act<DT>::T* __restrict__ out) {
  using A = Act<DT>;
  using Scale = ScaleVec<typename A::S, NS>;
  constexpr int kPer = 4 / NS;   // 32-channel words under one scale
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int panel = blockIdx.x * RT;
  const int m0 = blockIdx.y * 8 * MT;
  // weight rows past the last panel repeat it
  const uint4* cp[RT];
  const Scale* sp[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int64_t tile = tile_at(min(panel + r, panels - 1), warp, kt_n);
    cp[r] = codes + tile * 64 + lane;
    sp[r] = reinterpret_cast<const Scale*>(scales) + tile * kTileRows + g;
  }
  const typename A::T* xp[MT];
#pragma unroll
  for (int n = 0; n < MT; ++n) {
    const int m = m0 + 8 * n + g;
    xp[n] = x + (m < M ? m : 0) * ldx + warp * kTileK + 8 * t;
  }
  float acc[RT][MT][4] = {};
  Tile<typename A::S, NS> buf[2][RT];
  auto fetch = [&](Tile<typename A::S, NS> (&d)[RT]) {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      d[r].c0 = __ldg(cp[r]);
      d[r].c1 = __ldg(cp[r] + 32);
      d[r].s0 = sp[r][0];
      d[r].s1 = sp[r][8];
      cp[r] += WK * kBlockPanels * 64;
      sp[r] += WK * kBlockPanels * kTileRows;
    }
  };
  auto multiply = [&](const Tile<typename A::S, NS> (&d)[RT], int words) {
    // the two halves of a word have sums of their own: a product waits for
    // the one before it on the same sum
    float sum[2][RT][MT][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t xb[MT][A::kTerms][4];
#pragma unroll
      for (int n = 0; n < MT; ++n) {
        if (j < words) {
          A::load(xp[n] + 32 * j, xb[n]);
        } else {   // channels past the last: code 0 times 0
#pragma unroll
          for (int i = 0; i < A::kTerms; ++i) xb[n][i][0] = xb[n][i][1] = xb[n][i][2] = xb[n][i][3] = 0u;
        }
      }
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        uint32_t a[4], b[4];
        codes8<A::kF16>(word(d[r].c0, j), keys, a);
        codes8<A::kF16>(word(d[r].c1, j), keys, b);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int n = 0; n < MT; ++n) mma_half<A>(sum[h][r][n], a, b, xb[n], h, j % kPer == 0);
        if (j % kPer == kPer - 1) {
          const float s0 = A::scale(d[r].s0.v[j / kPer]), s1 = A::scale(d[r].s1.v[j / kPer]);
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int n = 0; n < MT; ++n) add_scaled(acc[r][n], sum[h][r][n], s0, s1);
        }
      }
    }
#pragma unroll
    for (int n = 0; n < MT; ++n) xp[n] += WK * kTileK;
  };
  // words of the tile that hold channels: 4 but in the last tile of a K that
  // is no multiple of 128
  auto words = [&](int kt) { return min(4, (K - kt * kTileK) >> 5); };
  int kt = warp;
  if (kt < kt_n) fetch(buf[0]);
  for (; kt + WK < kt_n; kt += 2 * WK) {
    fetch(buf[1]);
    multiply(buf[0], 4);
    if (kt + 2 * WK < kt_n) fetch(buf[0]);
    const int w = words(kt + WK);
    if (w == 4) multiply(buf[1], 4);
    else multiply(buf[1], w);
  }
  if (kt < kt_n) {
    const int w = words(kt);
    if (w == 4) multiply(buf[0], 4);
    else multiply(buf[0], w);
  }
  __shared__ float red[WK][8 * MT][RT * kTileRows + 1];
#pragma unroll
  for (int n = 0; n < MT; ++n) {
    if (m0 + 8 * n + 2 * t >= M) continue;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      red[warp][8 * n + 2 * t][16 * r + g] = acc[r][n][0];
      red[warp][8 * n + 2 * t + 1][16 * r + g] = acc[r][n][1];
      red[warp][8 * n + 2 * t][16 * r + g + 8] = acc[r][n][2];
      red[warp][8 * n + 2 * t + 1][16 * r + g + 8] = acc[r][n][3];
    }
  }
  __syncthreads();
  const int mn = min(8 * MT, M - m0);
  for (int i = threadIdx.x; i < mn * RT * kTileRows; i += WK * 32) {
    const int m = i / (RT * kTileRows), r = i % (RT * kTileRows);
    const int n = panel * kTileRows + r;
    if (n >= N) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < WK; ++w) v += red[w][m][r];
    out[static_cast<int64_t>(m0 + m) * N + n] = A::out(v);
  }
}

// More rows (up to NT = 32 or 64, 16-bit) on tcgen05: a CTA takes 128 weight
// rows, the M side of the instruction, against the NT activation rows of its N
// side.  A thread owns a weight row: it turns the row's 128 codes of a tile
// into 16-bit numbers in 64 columns of its TMEM lane, from where the
// instruction reads them as operand A, so the dequantized weight never passes
// through shared memory (2 bytes per code written and read back there would
// bound the kernel below HBM speed); the activations' tile is operand B, by
// TMA.  Each scale group has a product sum of its own in TMEM, which the row's
// thread multiplies by its scale and adds in fp32 registers: weights stay
// exact.  Groups of four warps take the tiles in turn, each converting, issuing
// its products (one warp issuing for all took 0.5 us a tile), waiting for them
// and adding by itself; what hides the waits is the other groups' work, so
// there are as many as the registers allow (the NT sums of a row are held by
// each).  Codes and scales come through shared memory too, by bulk copies
// several tiles ahead: with the two tiles a thread could hold in registers the
// loads in flight bounded the kernel (5120 rows of 13824 channels, 64
// activation rows: 35.5 us instead of 28.6; 29.9 with all inputs out of the
// L2, 1.3 TB/s or 303 TFLOP/s).  Bound by the chain of a group's tile,
// conversion -> products -> scaled sums, which has one buffer of codes: the
// tensor pipe is active 19% of the time and issue 32%.  The channels are split
// over the CTAs of a cluster, which add their sums through distributed shared
// memory in a fixed order.
template <int NS, int NT>
struct TcLayout {
  static constexpr int kStages = NT == 64 ? 6 : 8;
  static constexpr int kGroups = NT == 32 ? 3 : 2;                  // of four warps, 128 or 168 registers a thread
  static constexpr int kSums = NT == 64 ? 2 : 1;                    // 64-column buffers of sums per group
  static constexpr int kThreads = kGroups * 128 + 32;
  static constexpr int kX = NT * kTileK * 2;                        // one tile of activations
  static constexpr int kCodes = kX, kScales = kCodes + kBlockPanels * kTileBytes;   // of the tile's 8 panels
  static constexpr int kBytesIn = kScales + 128 * NS * 2;
  static constexpr int kStage = (kBytesIn + 1023) / 1024 * 1024;
  static constexpr int kPart = kStages * kStage;                    // float [kGroups - 1][NT][128]
  static constexpr int kBar = kPart + (kGroups - 1) * NT * 128 * 4;
  static constexpr int kBars = 2 * kStages + kGroups * kSums + 1;
  static constexpr int kBytes = kBar + kBars * 8 + 16;
  static_assert(kGroups * (64 + 64 * kSums) <= 512, "TMEM columns");
};

template <int DT, int NS, int NT>
__global__ void __launch_bounds__(TcLayout<NS, NT>::kThreads, 1)
    w4_tc_kernel(const __grid_constant__ CUtensorMap xmap, int M, const uint4* __restrict__ codes,
                 const typename Act<DT>::S* __restrict__ scales, int N, int kt_n, const Keys keys, typename Act<DT>::T* __restrict__ out) {
  using A = Act<DT>;
  using Ly = TcLayout<NS, NT>;
  using Scale = ScaleVec<typename A::S, NS>;
  constexpr int W = Ly::kGroups, kLoad = 4 * W, kCols = 64 + 64 * Ly::kSums;
  constexpr int kSteps = kTileK / 16 / NS;   // instructions per scale group
  // scale groups handed over at once: as many as 64 columns of sums hold
  constexpr int kBatch = NS < 64 / NT ? NS : 64 / NT, kBatches = NS / kBatch;
  extern __shared__ __align__(1024) unsigned char sm[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + Ly::kBar);
  // a stage has come / been read; per group of warps and buffer: sums ready
  uint64_t *x_full = bars, *x_empty = bars + Ly::kStages, *d_full = bars + 2 * Ly::kStages,
           *done = d_full + W * Ly::kSums;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Ly::kBars);
  volatile int* dead = reinterpret_cast<volatile int*>(tmem_slot + 1);
  cg::cluster_group cluster = cg::this_cluster();
  const int splits = cluster.num_blocks(), split = cluster.block_rank();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row0 = (blockIdx.x / splits) * 128, m0 = blockIdx.y * NT;
  const int kt0 = static_cast<int>(static_cast<int64_t>(kt_n) * split / splits);
  const int tiles = static_cast<int>(static_cast<int64_t>(kt_n) * (split + 1) / splits) - kt0;
  float* part = reinterpret_cast<float*>(sm + Ly::kPart);
  bool ok = true;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    ok = ok && __all_sync(0xffffffffu, wait_or(bar, parity, dead));
  };
  if (warp == kLoad) tmem_alloc(tmem_slot, 512);
  if (threadIdx.x == 0) {
    for (int i = 0; i < Ly::kStages; ++i) {
      mbar_init(x_full + i, 1);
      mbar_init(x_empty + i, 1);
    }
    for (int i = 0; i < W * Ly::kSums; ++i) mbar_init(d_full + i, 1);
    mbar_init(done, W);
    *dead = 0;
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;   // group w: A at kCols w, sums at kCols w + 64 + 64 buffer
  if (warp == kLoad) {
    int i = 0;
    const int64_t tile0 = tile_at(row0 / kTileRows, kt0, kt_n);
    for (; i < tiles && ok; ++i) {
      const int s = i % Ly::kStages;
      wait(x_empty + s, ((i / Ly::kStages) & 1) ^ 1);
      if (!ok) break;
      unsigned char* st = sm + s * Ly::kStage;
      if (lane == 0) {
        mbar_expect_tx(x_full + s, Ly::kBytesIn);
        tma_load_2d(st, &xmap, (kt0 + i) * kTileK, m0, x_full + s);
        tma_load_2d(st + NT * 128, &xmap, (kt0 + i) * kTileK + 64, m0, x_full + s);
        const int64_t tile = tile0 + static_cast<int64_t>(i) * kBlockPanels;
        bulk_g2s(st + Ly::kCodes, codes + tile * 64, kBlockPanels * kTileBytes, x_full + s);
        bulk_g2s(st + Ly::kScales, scales + tile * (kTileRows * NS), 128 * NS * 2, x_full + s);
      }
    }
    // a copy in flight must land before the CTA ends (all have when ok)
    if (!ok)
      for (int j = max(0, i - Ly::kStages); j < i; ++j) mbar_wait(x_full + j % Ly::kStages, (j / Ly::kStages) & 1);
  } else {
    const int w = warp >> 2, row = threadIdx.x & 127;
    const uint32_t base = tmem + kCols * w + (static_cast<uint32_t>(warp & 3) << 21);
    // the group's first warp issues its products
    constexpr uint32_t kId = mma_idesc(128, NT, !A::kF16, false);
    const bool issuer = (warp & 3) == 0;
    const uint32_t lead = elect_one();
    const uint64_t xd = smem_desc(smem_addr(sm), 16, 1024);
    auto products = [&](int s, int batch, int c) {
#pragma unroll
      for (int g = 0; g < kBatch; ++g)
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          const int step = (batch * kBatch + g) * kSteps + k;
          mma_ts(tmem + kCols * w + 64 + 64 * (c % Ly::kSums) + g * NT, tmem + kCols * w + 8 * step,
                 xd + s * (Ly::kStage / 16) + (step / 4) * (NT * 128 / 16) + (step % 4) * 2, kId, k > 0, lead);
        }
      mma_commit(d_full + w * Ly::kSums + c % Ly::kSums, lead);
    };
    float2 acc[NT / 2];
#pragma unroll
    for (int i = 0; i < NT / 2; ++i) acc[i] = make_float2(0.f, 0.f);
    // one tile: its products follow its codes, so A is free when the last
    // sums of the tile before it have come
    for (int i = w, n = 0; i < tiles; i += W, ++n) {
      const int s = i % Ly::kStages;
      wait(x_full + s, (i / Ly::kStages) & 1);
      Scale sc;
      if (ok) {
        // the row's 64 bytes: word j of channels 32 j + 8 t .. in c[t]
        const unsigned char* st = sm + s * Ly::kStage;
        const uint4* cp = reinterpret_cast<const uint4*>(st + Ly::kCodes) + row * 4;
        const uint4 c[4] = {cp[0], cp[1], cp[2], cp[3]};
        sc = reinterpret_cast<const Scale*>(st + Ly::kScales)[row];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t v[16];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            uint32_t q[4];
            codes8<A::kF16>(word(c[t], j), keys, q);
#pragma unroll
            for (int p = 0; p < 4; ++p) v[4 * t + p] = q[p];
          }
          tmem_st16(base + 16 * j, v);
        }
        tmem_wait_st();
      }
      tc_fence_before();
      named_sync(2 + w, 128);   // the whole tile is converted, the sums before it are taken
      tc_fence_after();
      constexpr int kAhead = kBatches < Ly::kSums ? kBatches : Ly::kSums;
      if (ok && issuer) {
#pragma unroll
        for (int b = 0; b < kAhead; ++b) products(s, b, n * kBatches + b);
        if (kAhead == kBatches) mma_commit(x_empty + s, lead);
      }
#pragma unroll
      for (int b = 0; b < kBatches; ++b) {
        const int c = n * kBatches + b;
        wait(d_full + w * Ly::kSums + c % Ly::kSums, (c / Ly::kSums) & 1);
        tc_fence_after();
        if (ok) {
          constexpr int kLd = 32;
#pragma unroll
          for (int h = 0; h < kBatch * NT; h += kLd) {
            const float f = A::scale(sc.v[b * kBatch + h / NT]);
            uint32_t x[kLd];
            tmem_ld32(base + 64 + 64 * (c % Ly::kSums) + h, x);
#pragma unroll
            for (int i = 0; i < kLd / 2; ++i) {
              float2& y = acc[(h % NT) / 2 + i];
              y = fma2(make_float2(f, f), make_float2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), y);
            }
          }
        }
        if (b + kAhead < kBatches) {   // the buffer's next sums, when all four warps have taken these
          tc_fence_before();
          named_sync(2 + w, 128);
          tc_fence_after();
          if (ok && issuer) {
            products(s, b + kAhead, c + kAhead);
            if (b + kAhead + 1 == kBatches) mma_commit(x_empty + s, lead);
          }
        }
      }
    }
    if (issuer) {   // nothing of ours may still run or arrive when the CTA ends
      mma_commit(done, lead);
      if (!mbar_wait(done, 0)) {
        *dead = 1;
        ok = false;
      }
    }
    __syncwarp();
    if (!ok) {   // a wait ran out: the rows say so
#pragma unroll
      for (int i = 0; i < NT / 2; ++i) acc[i] = make_float2(__int_as_float(0x7fc00000), __int_as_float(0x7fc00000));
    }
    if (w > 0) {
#pragma unroll
      for (int i = 0; i < NT; ++i) part[((w - 1) * NT + i) * 128 + row] = (i & 1) ? acc[i / 2].y : acc[i / 2].x;
    }
    named_sync(1, W * 128);
    if (w == 0) {
      const int n0 = row0 + row;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        float v = (i & 1) ? acc[i / 2].y : acc[i / 2].x;
#pragma unroll
        for (int g = 0; g < W - 1; ++g) v += part[(g * NT + i) * 128 + row];
        if (splits > 1) part[i * 128 + row] = v;
        else if (m0 + i < M && n0 < N) out[static_cast<int64_t>(m0 + i) * N + n0] = A::out(v);
      }
    }
  }
  tc_fence_before();
  if (splits > 1) {
    cluster.sync();
    // every CTA finishes its share of the activation rows
    if (warp < 4 * W) {
      const int mn = min(NT, M - m0), r = threadIdx.x & 127;
      for (int m = split + splits * (threadIdx.x >> 7); m < mn; m += W * splits) {
        float v = 0.f, p[8];   // all reads on their way before the first sum
#pragma unroll
        for (int s = 0; s < 8; ++s) p[s] = s < splits ? cluster.map_shared_rank(part, s)[m * 128 + r] : 0.f;
#pragma unroll
        for (int s = 0; s < 8; ++s) v += p[s];
        if (row0 + r < N) out[static_cast<int64_t>(m0 + m) * N + row0 + r] = A::out(v);
      }
    }
    cluster.sync();   // no CTA leaves while another reads its sums
  } else {
    __syncthreads();
  }
  report_wait(dead);
  if (warp == kLoad) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int DT, int NS, int MT, int RT, int WK>
cudaError_t launch_few(const carekv_w4_t& w, const void* x, int64_t ldx, int M, void* out, cudaStream_t st) {
  using A = Act<DT>;
  const int kt_n = (w.k + kTileK - 1) / kTileK, panels = (w.n + kTileRows - 1) / kTileRows;
  const dim3 grid((panels + RT - 1) / RT, (M + 8 * MT - 1) / (8 * MT));
  w4_kernel<DT, NS, MT, RT, WK><<<grid, WK * 32, 0, st>>>(static_cast<const typename A::T*>(x), ldx, M,
                                                          static_cast<const uint4*>(w.codes),
                                                          static_cast<const typename A::S*>(w.scales), w.n, w.k, kt_n,
                                                          panels, kKeys<A::kF16>, static_cast<typename A::T*>(out));
  return cudaGetLastError();
}
// Clusters of `size` (1 .. 8) CTAs of `kernel` that the current device holds at
// once; asked once per host thread, device and kernel.
template <typename K>
int max_clusters(K* kernel, int size, int threads, int smem) {
  static thread_local const void* known[64][9] = {};
  static thread_local int count[64][9] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  const bool keep = dev >= 0 && dev < 64;
  if (keep && known[dev][size] == reinterpret_cast<const void*>(kernel)) return count[dev][size];
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(size);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim = {static_cast<unsigned>(size), 1, 1};
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
    (void)cudaGetLastError();
    return 0;
  }
  if (keep) {
    known[dev][size] = reinterpret_cast<const void*>(kernel);
    count[dev][size] = n;
  }
  return n;
}

template <int DT, int NS, int NT>
cudaError_t launch_tc(const carekv_w4_t& w, const void* x, int64_t ldx, int M, void* out, cudaStream_t st) {
  using A = Act<DT>;
  using Ly = TcLayout<NS, NT>;
  const int kt_n = (w.k + kTileK - 1) / kTileK;
  const int blocks = (w.n + 127) / 128, cols = (M + NT - 1) / NT;
  const TensorMapEncode encode = tensor_map_encode();
  if (!encode) return cudaErrorNotSupported;
  // activations [M][k] in boxes of NT rows x 64 channels; rows and channels
  // past the end read as zero
  CUtensorMap map;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(w.k), static_cast<cuuint64_t>(M)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ldx) * 2};
  const cuuint32_t box[2] = {64, NT}, step[2] = {1, 1};
  if (encode(&map, DT == CAREKV_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
             const_cast<void*>(x), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return cudaErrorInvalidValue;
  auto kernel = w4_tc_kernel<DT, NS, NT>;
  const cudaError_t e = allow_smem<Ly::kBytes>(kernel);
  if (e != cudaSuccess) return e;
  // CTAs of a cluster: the most that still run all at once, at least 4 tiles each
  int splits = 1;
  for (int s = 2; s <= 8 && blocks * cols * s <= sm_count() && kt_n >= 4 * s; ++s)
    if (blocks * cols <= max_clusters(kernel, s, Ly::kThreads, Ly::kBytes)) splits = s;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks * splits, cols);
  cfg.blockDim = dim3(Ly::kThreads);
  cfg.dynamicSmemBytes = Ly::kBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim = {static_cast<unsigned>(splits), 1, 1};
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, map, M, static_cast<const uint4*>(w.codes),
                            static_cast<const typename A::S*>(w.scales), w.n, kt_n, kKeys<A::kF16>,
                            static_cast<typename A::T*>(out));
}
// Which form.  Up to 16 rows (any number in fp32) the few-row kernel, with as
// many warps per 16 weight rows as the number of such panels leaves room for.
// Measured with 4 / 8 / 16 warps, us on the device, weights out of the L2:
//   1 row:   864 panels of 5120 channels 11.1 / 11.9 / 13.2, 320 of 13824
//            18.7 / 13.1 / 13.9, 256 of 4096 7.6 / 5.4 / 4.7
//   16 rows: 864 panels of 5120 (two panels a CTA with 4 warps) 14.9 / 17.9 /
//            25.2, 320 of 13824 27.5 / 19.5 / 27.5, 64 of 4096 9.5 / 6.6 / 4.4
// Beyond 16 rows that kernel reads the weight again for every 16, and the
// tcgen05 kernel takes over where the weight is large: 32 rows x 14336 x 4096
// 28.2 against 21.2 us, and the same 10.8 at 32 x 4096 x 4096; 64 x 5120 x
// 13824 52.3 against 29.6, 64 x 4096 x 4096 19.3 against 15.2, 40 x 5632 x 2048
// 11.2 against 11.8, 48 x 700 x 512 2.4 against 10.3.
template <int DT, int NS>
cudaError_t launch_ns(const carekv_w4_t& w, const void* x, int64_t ldx, int M, void* out, cudaStream_t st) {
  const int panels = (w.n + kTileRows - 1) / kTileRows, sms = sm_count();
  if (M <= 8 || DT == CAREKV_F32) {
    if (panels >= 4 * sms) return launch_few<DT, NS, 1, 1, 4>(w, x, ldx, M, out, st);
    if (panels >= 2 * sms) return launch_few<DT, NS, 1, 1, 8>(w, x, ldx, M, out, st);
    return launch_few<DT, NS, 1, 1, 16>(w, x, ldx, M, out, st);
  }
  if constexpr (DT != CAREKV_F32) {
    const int64_t codes = static_cast<int64_t>(w.n) * w.k;
    if (M > 32 && codes >= (8 << 20)) return launch_tc<DT, NS, 64>(w, x, ldx, M, out, st);
    if (M > 16 && M <= 32 && codes >= (32 << 20)) return launch_tc<DT, NS, 32>(w, x, ldx, M, out, st);
    if (panels >= (M > 16 ? sms : 4 * sms)) return launch_few<DT, NS, 2, 2, 4>(w, x, ldx, M, out, st);
    if (panels >= sms) return launch_few<DT, NS, 2, 1, 8>(w, x, ldx, M, out, st);
    return launch_few<DT, NS, 2, 1, 16>(w, x, ldx, M, out, st);
  }
  return cudaErrorInvalidValue;
}
template <int DT>
cudaError_t launch_dt(const carekv_w4_t& w, const void* x, int64_t ldx, int M, void* out, cudaStream_t st) {
  switch (tile_scales(w.group_size)) {
    case 4: return launch_ns<DT, 4>(w, x, ldx, M, out, st);
    case 2: return launch_ns<DT, 2>(w, x, ldx, M, out, st);
    default: return launch_ns<DT, 1>(w, x, ldx, M, out, st);
  }
}

int64_t tiles(int n, int k) {
  return static_cast<int64_t>((n + 127) / 128) * kBlockPanels * ((k + kTileK - 1) / kTileK);
}

}  // namespace

cudaError_t w4_wait_errors(int32_t* set, cudaStream_t st) { return take_wait_errors(set, st); }

void w4_layout(int n, int k, int group, int dt, size_t sizes[2]) {
  const int64_t t = tiles(n, k);
  sizes[0] = static_cast<size_t>(t) * kTileBytes;
  sizes[1] = static_cast<size_t>(t) * kTileRows * tile_scales(group) * (dt == CAREKV_F32 ? 4 : 2);
}

cudaError_t launch_w4_pack(const void* packed, const void* scale, const carekv_w4_t& w, void* codes, void* scales,
                           cudaStream_t st) {
  const int64_t words = tiles(w.n, w.k) * (kTileBytes / 4);
  w4_pack_kernel<<<static_cast<unsigned>((words + 255) / 256), 256, 0, st>>>(
      static_cast<const uint8_t*>(packed), scale, w.n, w.k, w.group_size, w.dtype, static_cast<uint32_t*>(codes),
      scales, words, (w.k + kTileK - 1) / kTileK);
  return cudaGetLastError();
}

cudaError_t launch_w4_dequant(const carekv_w4_t& w, void* out, cudaStream_t st) {
  const int64_t words = tiles(w.n, w.k) * (kTileBytes / 4);
  w4_dequant_kernel<<<static_cast<unsigned>((words + 255) / 256), 256, 0, st>>>(
      static_cast<const uint32_t*>(w.codes), w.scales, w.n, w.k, w.group_size, w.dtype, out, words,
      (w.k + kTileK - 1) / kTileK);
  return cudaGetLastError();
}

cudaError_t launch_w4(const carekv_w4_t& w, const void* x, int64_t ldx, int M, void* out, cudaStream_t st) {
  // rows lie along grid.y, 8 at least to a CTA: 65535 of them in one launch
  constexpr int kMost = 8 * 65535;
  const int es = w.dtype == CAREKV_F32 ? 4 : 2;
  for (int m = 0; m < M;) {
    const int n = std::min(M - m, kMost);
    const void* xm = static_cast<const char*>(x) + m * ldx * es;
    void* om = static_cast<char*>(out) + static_cast<int64_t>(m) * w.n * es;
    const cudaError_t e = w.dtype == CAREKV_F16    ? launch_dt<CAREKV_F16>(w, xm, ldx, n, om, st)
                          : w.dtype == CAREKV_BF16 ? launch_dt<CAREKV_BF16>(w, xm, ldx, n, om, st)
                                                   : launch_dt<CAREKV_F32>(w, xm, ldx, n, om, st);
    if (e != cudaSuccess) return e;
    m += n;
  }
  return cudaSuccess;
}

}  // namespace carekv
