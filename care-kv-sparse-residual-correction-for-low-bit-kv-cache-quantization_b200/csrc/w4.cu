// Products of a few activation rows with a 4-bit weight:
//   y[m][n] = sum_G s[n][G] sum_{k in group G} c[n][k] x[m][k],
// codes c in -8..7, one scale per (row, group of channels).
//
// Codes are small integers, exact in fp16 and bf16, so the inner sums run on
// the tensor cores (m16n8k16, fp32 accumulators) with the weight rows on the
// M side and up to 8 activation rows on the N side of one instruction; the
// scale multiplies the group's fp32 sum, so no weight is ever rounded.  fp32
// activations are split into three bf16 terms whose sum is the value itself.
#include <algorithm>

#include "common.cuh"
#include "internal.h"
#include "ptx.cuh"

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
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The 8 codes of a word as four exact pairs: a nibble put at mantissa bit b
// of a float whose exponent makes that bit worth 1 reads as 2^e + u, and one
// subtraction of 2^e + 8 leaves the code.  fp16 has room for nibbles at bits
// 0 and 4 (one shift per word), bf16 at bit 0 only (three).
template <bool F16>
__device__ __forceinline__ void codes8(uint32_t w, uint32_t (&r)[4]) {
  if constexpr (F16) {
    const uint32_t v = w >> 8;
    r[0] = h2sub((w & 0x000F000Fu) | 0x64006400u, 0x64086408u);
    r[1] = h2sub((w & 0x00F000F0u) | 0x54005400u, 0x54805480u);
    r[2] = h2sub((v & 0x000F000Fu) | 0x64006400u, 0x64086408u);
    r[3] = h2sub((v & 0x00F000F0u) | 0x54005400u, 0x54805480u);
  } else {
#pragma unroll
    for (int p = 0; p < 4; ++p) r[p] = bsub(((w >> (4 * p)) & 0x000F000Fu) | 0x43004300u, 0x43084308u);
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

// One CTA per 16 weight rows: its WK warps take the row's tiles in turn and
// add their sums in shared memory.
template <int DT, int NS, int MT, int WK>
__global__ void __launch_bounds__(WK * 32) w4_kernel(const typename Act<DT>::T* __restrict__ x, int64_t ldx, int M,
                                                     const uint4* __restrict__ codes,
                                                     const typename Act<DT>::S* __restrict__ scales, int N, int K,
                                                     int kt_n, typename Act<DT>::T* __restrict__ out) {
  using A = Act<DT>;
  constexpr int kPer = 4 / NS;   // 32-channel words under one scale
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int64_t panel = blockIdx.x;
  const int m0 = blockIdx.y * 8 * MT;
  float acc[MT][4] = {};
  for (int kt = warp; kt < kt_n; kt += WK) {
    const int64_t tile = panel * kt_n + kt;
    const uint4 c0 = __ldg(codes + tile * 64 + lane), c1 = __ldg(codes + tile * 64 + 32 + lane);
    const uint32_t w0[4] = {c0.x, c0.y, c0.z, c0.w}, w1[4] = {c1.x, c1.y, c1.z, c1.w};
    float sum[MT][4] = {};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t a[4], b[4];
      codes8<A::kF16>(w0[j], a);
      codes8<A::kF16>(w1[j], b);
      const int k = kt * kTileK + 32 * j + 8 * t;
#pragma unroll
      for (int n = 0; n < MT; ++n) {
        const int m = m0 + 8 * n + g;
        uint32_t xb[A::kTerms][4] = {};
        if (m < M && k < K) A::load(x + m * ldx + k, xb);
#pragma unroll
        for (int i = 0; i < A::kTerms; ++i) {
          if constexpr (A::kF16) {
            mma_f16(sum[n], a[0], b[0], a[1], b[1], xb[i][0], xb[i][1]);
            mma_f16(sum[n], a[2], b[2], a[3], b[3], xb[i][2], xb[i][3]);
          } else {
            mma_bf16(sum[n], a[0], b[0], a[1], b[1], xb[i][0], xb[i][1]);
            mma_bf16(sum[n], a[2], b[2], a[3], b[3], xb[i][2], xb[i][3]);
          }
        }
      }
      if (j % kPer == kPer - 1) {
        const auto* sp = scales + tile * (kTileRows * NS) + j / kPer;
        const float s0 = A::scale(sp[g * NS]), s1 = A::scale(sp[(g + 8) * NS]);
#pragma unroll
        for (int n = 0; n < MT; ++n) {
          acc[n][0] = fmaf(s0, sum[n][0], acc[n][0]);
          acc[n][1] = fmaf(s0, sum[n][1], acc[n][1]);
          acc[n][2] = fmaf(s1, sum[n][2], acc[n][2]);
          acc[n][3] = fmaf(s1, sum[n][3], acc[n][3]);
          sum[n][0] = sum[n][1] = sum[n][2] = sum[n][3] = 0.f;
        }
      }
    }
  }
  __shared__ float red[WK][8 * MT][kTileRows + 1];
#pragma unroll
  for (int n = 0; n < MT; ++n) {
    red[warp][8 * n + 2 * t][g] = acc[n][0];
    red[warp][8 * n + 2 * t + 1][g] = acc[n][1];
    red[warp][8 * n + 2 * t][g + 8] = acc[n][2];
    red[warp][8 * n + 2 * t + 1][g + 8] = acc[n][3];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 8 * MT * kTileRows; i += WK * 32) {
    const int m = i / kTileRows, r = i % kTileRows;
    const int64_t n = panel * kTileRows + r;
    if (m0 + m >= M || n >= N) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < WK; ++w) v += red[w][m][r];
    out[static_cast<int64_t>(m0 + m) * N + n] = A::out(v);
  }
}

template <int DT, int NS, int MT>
cudaError_t launch_mt(const carekv_w4_t& w, const void* x, int64_t ldx, int M, void* out, cudaStream_t st) {
  using A = Act<DT>;
  constexpr int WK = 8;
  const int kt_n = (w.k + kTileK - 1) / kTileK;
  const dim3 grid((w.n + kTileRows - 1) / kTileRows, (M + 8 * MT - 1) / (8 * MT));
  w4_kernel<DT, NS, MT, WK><<<grid, WK * 32, 0, st>>>(static_cast<const typename A::T*>(x), ldx, M,
                                                      static_cast<const uint4*>(w.codes),
                                                      static_cast<const typename A::S*>(w.scales), w.n, w.k, kt_n,
                                                      static_cast<typename A::T*>(out));
  return cudaGetLastError();
}
template <int DT, int NS>
cudaError_t launch_ns(const carekv_w4_t& w, const void* x, int64_t ldx, int M, void* out, cudaStream_t st) {
  if (M <= 8) return launch_mt<DT, NS, 1>(w, x, ldx, M, out, st);
  if (M <= 16) return launch_mt<DT, NS, 2>(w, x, ldx, M, out, st);
  return launch_mt<DT, NS, 4>(w, x, ldx, M, out, st);
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
