// Rotary positions: pair i of a row at position p turns by p * theta_i,
//   (a, b) -> f (a cos - b sin, b cos + a sin),
// pairs (i, i + rd/2) ("half" layout) or (2i, 2i + 1) (interleaved) of the
// first rd channels; the other channels are copied.
//
// The angle is kept in turns: freq[i] = theta_i / 2 pi as a 64-bit fraction,
// so p * freq[i] mod 2^64 is the exact phase of any position (negative ones
// too) and one integer product replaces the range reduction that an fp32
// angle of 1e5 radians has already lost its digits to.  No cos / sin table
// is read: the kernel's only traffic is the rows themselves (read once,
// written once) and the positions, so prompts are bound by HBM and single
// tokens by the launch.
//
// Measured: 4 x 4096 tokens of 32 + 8 heads of 128 in bf16 58.2 us, 5.77 TB/s
// (88% of a plain copy's rate), 3 x 1021 tokens of 40 + 40 heads in fp32 with
// 96 of 128 channels turned 50.4 us, 4.98 TB/s (issue active 68% of the time,
// 84% of the warps resident: what keeps it from a copy's rate is not known);
// one token 2.5 us.  Twice to four times the tokens per CTA, streaming stores
// and several rows in flight per thread changed neither by more than 1%.
//
// A CTA takes ktok tokens: its threads first put the tokens' cos / sin in
// shared memory (one pair each), then walk the tokens' heads with 16-byte
// accesses, so a pair's angle is computed once for all heads.
#include <algorithm>

#include "common.cuh"
#include "internal.h"

namespace carekv {
namespace {

constexpr int kThreads = 256;

// How a thread's vector finds the partner of its elements.
enum Mode {
  kHalfPair,   // half layout, both vectors of V pairs aligned: one thread turns both
  kInter,      // interleaved: the pairs lie inside the vector (V even)
  kAny         // own vector, partners by single loads: half layout at any rd, and V = 1
};

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T e[V];
};

template <typename T, int V, int MODE>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const carekv_rotary_t a, const int n_tok, const int ktok,
                                                          const int chunks) {
  extern __shared__ float2 cs[];   // [ktok][rd / 2] (f cos, f sin)
  const int half = a.rotary_dim >> 1, rd = a.rotary_dim, D = a.head_dim;
  const int tok0 = blockIdx.x * ktok;
  const int nt = min(ktok, n_tok - tok0);
  for (int i = threadIdx.x; i < nt * half; i += kThreads) {
    const int t = tok0 + i / half, p = i % half;
    const int64_t at = (t / a.tokens) * a.position_stride[0] + (t % a.tokens) * a.position_stride[1];
    const int64_t pos = a.position_bytes == 8 ? static_cast<const int64_t*>(a.positions)[at]
                                              : static_cast<const int32_t*>(a.positions)[at];
    const uint64_t turn = static_cast<uint64_t>(pos) * static_cast<uint64_t>(a.freq[p]);
    float s, c;
    // the phase's top 32 bits as a signed fraction of half a turn
    sincospif(static_cast<float>(static_cast<int32_t>(turn >> 32)) * 0x1p-31f, &s, &c);
    cs[i] = make_float2(c * a.factor, (a.inverse ? -s : s) * a.factor);
  }
  __syncthreads();
  const int rows_step = kThreads / chunks;
  const int c = threadIdx.x % chunks, r0 = threadIdx.x / chunks;
  if (r0 >= rows_step) return;
  const int H = a.q.heads + a.k.heads;
  for (int r = r0; r < nt * H; r += rows_step) {
    const int ti = r / H, h0 = r - ti * H;
    const bool is_k = h0 >= a.q.heads;
    const carekv_rows_t& x = is_k ? a.k : a.q;
    const int h = is_k ? h0 - a.q.heads : h0;
    const int t = tok0 + ti;
    const int64_t b = t / a.tokens, tt = t % a.tokens;
    const T* in = static_cast<const T*>(x.in) + b * x.in_stride[0] + tt * x.in_stride[1] + h * x.in_stride[2];
    T* out = static_cast<T*>(x.out) + b * x.out_stride[0] + tt * x.out_stride[1] + h * x.out_stride[2];
    const float2* cst = cs + ti * half;
    if constexpr (MODE == kHalfPair) {
      // chunks: rd / 2V pairs of vectors, then (D - rd) / V copied vectors
      if (c * V < half) {
        const Vec<T, V> u = *reinterpret_cast<const Vec<T, V>*>(in + c * V);
        const Vec<T, V> w = *reinterpret_cast<const Vec<T, V>*>(in + half + c * V);
        Vec<T, V> y, z;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float2 k = cst[c * V + i];
          const float p = to_f(u.e[i]), q = to_f(w.e[i]);
          y.e[i] = from_f<T>(p * k.x - q * k.y);
          z.e[i] = from_f<T>(q * k.x + p * k.y);
        }
        *reinterpret_cast<Vec<T, V>*>(out + c * V) = y;
        *reinterpret_cast<Vec<T, V>*>(out + half + c * V) = z;
      } else {
        const int j = rd + (c - half / V) * V;
        *reinterpret_cast<Vec<T, V>*>(out + j) = *reinterpret_cast<const Vec<T, V>*>(in + j);
      }
    } else {
      const int j0 = c * V;
      const Vec<T, V> u = *reinterpret_cast<const Vec<T, V>*>(in + j0);
      Vec<T, V> y = u;
      if constexpr (MODE == kInter) {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
          if (j0 + i < rd) {
            const float2 k = cst[(j0 + i) >> 1];
            const float p = to_f(u.e[i]), q = to_f(u.e[i + 1]);
            y.e[i] = from_f<T>(p * k.x - q * k.y);
            y.e[i + 1] = from_f<T>(q * k.x + p * k.y);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int j = j0 + i;
          if (j < rd) {
            const bool second = a.interleaved ? (j & 1) : j >= half;
            const int p = a.interleaved ? j >> 1 : (second ? j - half : j);
            const float o = to_f(in[a.interleaved ? (j ^ 1) : (second ? p : p + half)]);
            const float2 k = cst[p];
            y.e[i] = from_f<T>(second ? to_f(u.e[i]) * k.x + o * k.y : to_f(u.e[i]) * k.x - o * k.y);
          }
        }
      }
      *reinterpret_cast<Vec<T, V>*>(out + j0) = y;
    }
  }
}

template <typename T, int V, int MODE>
cudaError_t launch(const carekv_rotary_t& a, int chunks, cudaStream_t st) {
  const int n_tok = a.batch * a.tokens;
  const int half = a.rotary_dim / 2;
  // tokens per CTA: enough rows for a few vectors per thread, so the angles
  // (one per thread and round) stay small beside the rows
  const int rows_step = kThreads / chunks;
  int ktok = (4 * rows_step + a.q.heads + a.k.heads - 1) / (a.q.heads + a.k.heads);
  ktok = std::max(1, std::min(ktok, std::min(n_tok, 4096 / half)));
  rotary_kernel<T, V, MODE><<<(n_tok + ktok - 1) / ktok, kThreads, ktok * half * sizeof(float2), st>>>(a, n_tok, ktok,
                                                                                                     chunks);
  return cudaGetLastError();
}

bool rows_aligned(const carekv_rows_t& r, int64_t elem) {
  if (r.heads == 0) return true;
  uint64_t m = reinterpret_cast<uintptr_t>(r.in) | reinterpret_cast<uintptr_t>(r.out);
  for (int i = 0; i < 3; ++i) m |= static_cast<uint64_t>(r.in_stride[i] * elem) | static_cast<uint64_t>(r.out_stride[i] * elem);
  return (m & 15) == 0;
}

template <typename T>
cudaError_t launch_t(const carekv_rotary_t& a, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const int D = a.head_dim, half = a.rotary_dim / 2;
  // 16-byte accesses where every row starts on a 16-byte boundary and the
  // row is a whole number of vectors; single elements otherwise
  if (rows_aligned(a.q, sizeof(T)) && rows_aligned(a.k, sizeof(T)) && D % V == 0 && D / V <= kThreads) {
    if (a.interleaved) return launch<T, V, kInter>(a, D / V, st);
    if (half % V == 0) return launch<T, V, kHalfPair>(a, half / V + (D - a.rotary_dim) / V, st);
    return launch<T, V, kAny>(a, D / V, st);
  }
  return launch<T, 1, kAny>(a, D, st);
}

}  // namespace

cudaError_t launch_rotary(const carekv_rotary_t& a, cudaStream_t st) {
  if (static_cast<int64_t>(a.batch) * a.tokens == 0 || a.q.heads + a.k.heads == 0) return cudaSuccess;
  if (a.dtype == CAREKV_F16) return launch_t<__half>(a, st);
  if (a.dtype == CAREKV_BF16) return launch_t<__nv_bfloat16>(a, st);
  return launch_t<float>(a, st);
}

}  // namespace carekv
