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
constexpr int kTileRows = 16, kTileK = 128, kTileBytes = 1024;

__host__ __device__ inline int tile_scales(int group) { return group >= kTileK ? 1 : kTileK / group; }

__global__ void __launch_bounds__(256) w4_pack_kernel(const uint8_t* __restrict__ packed, const void* __restrict__ scale,
                                                      int N, int K, int group, int dt, uint32_t* __restrict__ codes,
                                                      void* __restrict__ scales, int64_t words, int kt_n) {
  const int64_t w = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (w >= words) return;
  const int64_t tile = w >> 8;
  const int in = static_cast<int>(w & 255), hi = in >> 7, lane = (in >> 2) & 31, j = in & 3;
  const int64_t panel = tile / kt_n;
  const int kt = static_cast<int>(tile % kt_n);
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
  const int64_t n = tile / kt_n * kTileRows + row;
  const int kk = 32 * j + 8 * (lane & 3);
  const int64_t k0 = tile % kt_n * kTileK + kk;
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
  // smallest numbers); infinities and NaN stay in the first term
  static __device__ __forceinline__ void load(const T* p, uint32_t (&b)[3][4]) {
    float x[8];
    *reinterpret_cast<float4*>(x) = __ldg(reinterpret_cast<const float4*>(p));
    *reinterpret_cast<float4*>(x + 4) = __ldg(reinterpret_cast<const float4*>(p) + 1);
#pragma unroll
    for (int i = 0; i < 3; ++i) {
#pragma unroll
      for (int k = 0; k < 8; k += 2) {
        const uint32_t lo = __float_as_uint(x[k]), hi = __float_as_uint(x[k + 1]);
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
// (their sums are not stored).
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
    const int64_t tile = static_cast<int64_t>(min(panel + r, panels - 1)) * kt_n + warp;
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
      cp[r] += WK * 64;
      sp[r] += WK * kTileRows;
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

// More rows (up to 8 MT, 16-bit): the CTA's 8 warps take RT x 16 weight rows
// each and share the activations; codes, scales and activations of the next
// kWideStages - 1 tiles are on their way in shared memory.  The channels are
// split over the CTAs of a cluster, which add their sums through distributed
// shared memory in a fixed order.
constexpr int kWideWarps = 8, kWideStages = 4;

template <int NS, int MT, int RT>
struct WideLayout {
  static constexpr int kRows = kWideWarps * RT * kTileRows;
  static constexpr int kX = 8 * MT * kTileK * 2;
  static constexpr int kCodes = kWideWarps * RT * kTileBytes;
  static constexpr int kScales = kRows * NS * 2;
  static constexpr int kStage = kX + kCodes + kScales;
  static constexpr int kSum = 8 * MT * (kRows + 1) * 4;   // [m][row], reuses the stages
  static constexpr int kBytes = kSum > kWideStages * kStage ? kSum : kWideStages * kStage;
};

__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(in ? 16 : 0)
               : "memory");
}

template <int DT, int NS, int MT, int RT>
__global__ void __launch_bounds__(kWideWarps * 32) w4_wide_kernel(const typename Act<DT>::T* __restrict__ x, int64_t ldx,
                                                                  int M, const uint4* __restrict__ codes,
                                                                  const typename Act<DT>::S* __restrict__ scales, int N,
                                                                  int K, int kt_n, int panels, const Keys keys,
                                                                  typename Act<DT>::T* __restrict__ out) {
  using A = Act<DT>;
  using Ly = WideLayout<NS, MT, RT>;
  using Scale = ScaleVec<typename A::S, NS>;
  constexpr int kPer = 4 / NS, kThreads = kWideWarps * 32;
  extern __shared__ __align__(16) unsigned char sm[];
  cg::cluster_group cluster = cg::this_cluster();
  const int splits = cluster.num_blocks(), split = cluster.block_rank();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int row0 = (blockIdx.x / splits) * Ly::kRows;
  const int m0 = blockIdx.y * 8 * MT;
  const int kt0 = static_cast<int>(static_cast<int64_t>(kt_n) * split / splits);
  const int kt1 = static_cast<int>(static_cast<int64_t>(kt_n) * (split + 1) / splits);

  // this thread's 16-byte pieces of a stage; weight rows past the last panel
  // repeat it (their sums are not stored), activation rows past the last and
  // channels past K are zero.  Chunk c of activation row m lies at
  // c ^ 4 (m & 1), so that the 2 rows x 4 chunks a quarter warp reads fall on
  // different banks.
  constexpr int kCodePieces = kWideWarps * RT * 64 / kThreads, kXPieces = 8 * MT * 16 / kThreads;
  const uint4* code_src[kCodePieces];
#pragma unroll
  for (int i = 0; i < kCodePieces; ++i) {
    const int at = threadIdx.x + i * kThreads;
    const int64_t panel = min(row0 / kTileRows + (at >> 6), panels - 1);
    code_src[i] = codes + (panel * kt_n + kt0) * 64 + (at & 63);
  }
  constexpr int kScalePieces = Ly::kScales / 16;   // at most 512 bytes x RT x ...: one or two per thread
  constexpr int kPanelPieces = kTileRows * NS * 2 / 16;
  auto stage = [&](int kt) {
    if (kt < kt1) {
      unsigned char* d = sm + (kt % kWideStages) * Ly::kStage;
#pragma unroll
      for (int i = 0; i < kXPieces; ++i) {
        const int at = threadIdx.x + i * kThreads, m = at >> 4, c = at & 15, k = kt * kTileK + 8 * c;
        const bool in = m0 + m < M && k < K;
        cp_async16(d + m * 256 + ((c ^ ((m & 1) << 2)) << 4), in ? x + (m0 + m) * ldx + k : x, in);
      }
      d += Ly::kX;
#pragma unroll
      for (int i = 0; i < kCodePieces; ++i) {
        cp_async16(d + (threadIdx.x + i * kThreads) * 16, code_src[i], true);
        code_src[i] += 64;
      }
      d += Ly::kCodes;
      for (int i = threadIdx.x; i < kScalePieces; i += kThreads) {
        const int64_t panel = min(row0 / kTileRows + i / kPanelPieces, panels - 1);
        cp_async16(d + i * 16, scales + (panel * kt_n + kt) * (kTileRows * NS) + i % kPanelPieces * 8, true);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kWideStages - 1; ++i) stage(kt0 + i);
  float acc[RT][MT][4] = {};
  for (int kt = kt0; kt < kt1; ++kt) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kWideStages - 2) : "memory");
    __syncthreads();   // tile kt has landed for all; the stage of tile kt - 1 is free
    stage(kt + kWideStages - 1);
    const unsigned char* d = sm + (kt % kWideStages) * Ly::kStage;
    Tile<typename A::S, NS> cur[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const uint4* c = reinterpret_cast<const uint4*>(d + Ly::kX + (warp * RT + r) * kTileBytes);
      cur[r].c0 = c[lane];
      cur[r].c1 = c[lane + 32];
      const Scale* s = reinterpret_cast<const Scale*>(d + Ly::kX + Ly::kCodes) + (warp * RT + r) * kTileRows;
      cur[r].s0 = s[g];
      cur[r].s1 = s[g + 8];
    }
    const unsigned char* xs = d + g * 256;
    float sum[RT][MT][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t a[RT][4], b[RT][4];
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        codes8<A::kF16>(word(cur[r].c0, j), keys, a[r]);
        codes8<A::kF16>(word(cur[r].c1, j), keys, b[r]);
      }
uint32_t xb[MT][1][4];
#pragma unroll
      for (int n = 0; n < MT; ++n) {
        const uint4 v = *reinterpret_cast<const uint4*>(xs + n * (8 * 256) + (((4 * j + t) ^ ((g & 1) << 2)) << 4));
        xb[n][0][0] = v.x, xb[n][0][1] = v.y, xb[n][0][2] = v.z, xb[n][0][3] = v.w;
      }
      // products that share a sum are MT RT apart
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int n = 0; n < MT; ++n) mma_half<A>(sum[r][n], a[r], b[r], xb[n], h, j % kPer == 0 && h == 0);
      if (j % kPer == kPer - 1) {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const float s0 = A::scale(cur[r].s0.v[j / kPer]), s1 = A::scale(cur[r].s1.v[j / kPer]);
#pragma unroll
          for (int n = 0; n < MT; ++n) add_scaled(acc[r][n], sum[r][n], s0, s1);
        }
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  float* part = reinterpret_cast<float*>(sm);
  constexpr int kLd = Ly::kRows + 1;
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int n = 0; n < MT; ++n) {
      float* p = part + (8 * n + 2 * t) * kLd + (warp * RT + r) * kTileRows + g;
      p[0] = acc[r][n][0];
      p[kLd] = acc[r][n][1];
      p[8] = acc[r][n][2];
      p[kLd + 8] = acc[r][n][3];
    }
  cluster.sync();
  // every CTA finishes its share of the activation rows
  const int mn = min(8 * MT, M - m0);
  for (int m = split; m < mn; m += splits)
    for (int r = threadIdx.x; r < Ly::kRows && row0 + r < N; r += kThreads) {
      float v = 0.f, p[8];   // all reads on their way before the first sum
#pragma unroll
      for (int s = 0; s < 8; ++s) p[s] = s < splits ? cluster.map_shared_rank(part, s)[m * kLd + r] : 0.f;
#pragma unroll
      for (int s = 0; s < 8; ++s) v += p[s];
      out[static_cast<int64_t>(m0 + m) * N + row0 + r] = A::out(v);
    }
  cluster.sync();   // no CTA leaves while another reads its sums
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
template <int DT, int NS, int MT, int RT>
cudaError_t launch_wide(const carekv_w4_t& w, const void* x, int64_t ldx, int M, void* out, cudaStream_t st) {
  using A = Act<DT>;
  using Ly = WideLayout<NS, MT, RT>;
  const int kt_n = (w.k + kTileK - 1) / kTileK, panels = (w.n + kTileRows - 1) / kTileRows;
  const int blocks = (w.n + Ly::kRows - 1) / Ly::kRows, cols = (M + 8 * MT - 1) / (8 * MT);
  // CTAs of a cluster: as many as fill the GPU, at least 4 tiles of channels each
  constexpr int kPerSm = MT == 2 ? 2 : 1;
  const int splits = std::max(1, std::min({8, kPerSm * 148 / (blocks * cols), kt_n / 4}));
  auto kernel = w4_wide_kernel<DT, NS, MT, RT>;
  const cudaError_t e = allow_smem<Ly::kBytes>(kernel);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks * splits, cols);
  cfg.blockDim = dim3(kWideWarps * 32);
  cfg.dynamicSmemBytes = Ly::kBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim = {static_cast<unsigned>(splits), 1, 1};
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<const typename A::T*>(x), ldx, M,
                            static_cast<const uint4*>(w.codes), static_cast<const typename A::S*>(w.scales), w.n, w.k,
                            kt_n, panels, kKeys<A::kF16>, static_cast<typename A::T*>(out));
}
// Which form: up to 8 rows the few-row kernel, with as many warps per 16
// weight rows as the number of such panels leaves room for (1 row, us per
// call with 4 / 8 / 16 warps: 864 panels of 5120 channels 11.1 / 11.9 / 13.3,
// 320 panels of 13824 18.8 / 13.0 / 15.1, 256 panels of 4096 5.5 / 4.4 / 4.2);
// above that the wide kernel.
template <int DT, int NS>
cudaError_t launch_ns(const carekv_w4_t& w, const void* x, int64_t ldx, int M, void* out, cudaStream_t st) {
  const int panels = (w.n + kTileRows - 1) / kTileRows;
  if (M <= 8 || DT == CAREKV_F32) {
    if (panels >= 4 * 148) return launch_few<DT, NS, 1, 1, 4>(w, x, ldx, M, out, st);
    if (panels >= 2 * 148) return launch_few<DT, NS, 1, 1, 8>(w, x, ldx, M, out, st);
    return launch_few<DT, NS, 1, 1, 16>(w, x, ldx, M, out, st);
  }
  if constexpr (DT != CAREKV_F32) {
    if (M <= 16) return launch_wide<DT, NS, 2, 2>(w, x, ldx, M, out, st);
    return launch_wide<DT, NS, 4, 2>(w, x, ldx, M, out, st);
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
  return static_cast<int64_t>((n + kTileRows - 1) / kTileRows) * ((k + kTileK - 1) / kTileK);
}

}  // namespace

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
  if (M == 0) return cudaSuccess;
  if (w.dtype == CAREKV_F16) return launch_dt<CAREKV_F16>(w, x, ldx, M, out, st);
  if (w.dtype == CAREKV_BF16) return launch_dt<CAREKV_BF16>(w, x, ldx, M, out, st);
  return launch_dt<CAREKV_F32>(w, x, ldx, M, out, st);
}

}  // namespace carekv
