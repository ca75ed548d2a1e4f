// Attention of a batch over one shared prefix, computed once for all rows.
//
// For row r and head h, with s_t = scale q . k_t over the prefix tokens the
// row sees: o = sum_t e^{s_t} v_t / sum_t e^{s_t} and lse = log sum_t e^{s_t}.
// The state (o', lse') of the row's own tokens joins as one more term:
//   L = e^{lse} + e^{lse'},  out = (e^{lse} o + e^{lse'} o') / L,  log L.
// Rows of all sequences and the query heads of one kv head form one matrix,
// so every K / V tile is read once for all of them.  The prefix is split over
// CTAs; each writes its unnormalised sum, running maximum and weight sum in
// fp32 and combine_kernel joins them with the rows' own state.
#include <algorithm>

#include "common.cuh"
#include "internal.h"

namespace carekv {
namespace {

constexpr float kL2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct PrefixArgs {
  carekv_prefix_t p;
  const void* q;
  int64_t q_row, q_head;   // strides in elements
  int rows, heads, group;  // group: query heads per kv head
  float scale2;            // scale log2 e: scores in base 2
  const int32_t* lengths;
  int splits, split_tokens;
  float* po;               // [splits][rows * heads][D] unnormalised sums
  float2* ml;              // [splits][rows * heads] base-2 maximum, weight sum
};

// tokens of the prefix that row r sees
__device__ __forceinline__ int visible(const PrefixArgs& a, int r) {
  return a.lengths ? min(max(a.lengths[r], 0), a.p.tokens) : a.p.tokens;
}

// ── fp32 FMA form ───────────────────────────────────────────────────────
// A warp per row; the CTA's 8 rows share 32-token tiles of K and V.
constexpr int kFmaRows = 8, kFmaTok = 32, kFmaMaxD = 256;

__global__ void __launch_bounds__(kFmaRows * 32) prefix_fma_kernel(const PrefixArgs a) {
  extern __shared__ float sm[];
  const int D = a.p.head_dim, dt = a.p.dtype;
  float* sq = sm;                          // [8][D]
  float* sk = sq + kFmaRows * D;           // [32][D + 1]
  float* sv = sk + kFmaTok * (D + 1);      // [32][D]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = blockIdx.y, split = blockIdx.z;
  const int rho = blockIdx.x * kFmaRows + warp;
  const bool live = rho < a.rows * a.group;
  const int r = live ? rho / a.group : 0, h = kvh * a.group + (live ? rho % a.group : 0);
  const int t_begin = split * a.split_tokens;
  const int t_end = min(t_begin + a.split_tokens, a.p.tokens);
  const int see = live ? min(visible(a, r), t_end) : 0;
  for (int c = lane; c < D; c += 32) sq[warp * D + c] = live ? load_act(a.q, r * a.q_row + h * a.q_head + c, dt) * a.scale2 : 0.f;
  float m = -INFINITY, l = 0.f, o[kFmaMaxD / 32] = {};
  for (int t0 = t_begin; t0 < t_end; t0 += kFmaTok) {
    __syncthreads();
    const int n = min(kFmaTok, t_end - t0);
    for (int i = threadIdx.x; i < n * D; i += kFmaRows * 32) {
      const int t = i / D, c = i % D;
      sk[t * (D + 1) + c] = load_act(a.p.k, kvh * a.p.k_stride[0] + (t0 + t) * a.p.k_stride[1] + c, dt);
      sv[i] = load_act(a.p.v, kvh * a.p.v_stride[0] + (t0 + t) * a.p.v_stride[1] + c, dt);
    }
    __syncthreads();
    if (t0 >= see) continue;
    const int nv = min(n, see - t0);
    float s = -INFINITY;
    if (lane < nv) {
      s = 0.f;
      for (int c = 0; c < D; ++c) s = fmaf(sq[warp * D + c], sk[lane * (D + 1) + c], s);
    }
    const float mn = fmaxf(m, warp_max(s));
    const float base = mn == -INFINITY ? 0.f : mn;   // nothing seen yet: all weights 0
    const float w = exp2f(s - base), corr = exp2f(m - base);
    l = fmaf(l, corr, warp_sum(w));
    m = mn;
#pragma unroll
    for (int i = 0; i < kFmaMaxD / 32; ++i) o[i] *= corr;
    for (int t = 0; t < nv; ++t) {
      const float wt = __shfl_sync(0xffffffffu, w, t);
#pragma unroll
      for (int i = 0; i < kFmaMaxD / 32; ++i)
        if (lane + 32 * i < D) o[i] = fmaf(wt, sv[t * D + lane + 32 * i], o[i]);
    }
  }
  if (!live) return;
  const int64_t at = static_cast<int64_t>(split) * a.rows * a.heads + static_cast<int64_t>(r) * a.heads + h;
  if (lane == 0) a.ml[at] = make_float2(m, l);
#pragma unroll
  for (int i = 0; i < kFmaMaxD / 32; ++i)
    if (lane + 32 * i < D) a.po[at * D + lane + 32 * i] = o[i];
}

// ── join ────────────────────────────────────────────────────────────────
// One warp per (row, head): the splits' sums and the row's own state.
__global__ void __launch_bounds__(256) prefix_combine_kernel(const float* __restrict__ po, const float2* __restrict__ ml,
                                                             int splits, int64_t n, int D, int dt,
                                                             const void* __restrict__ tail,
                                                             const float* __restrict__ tail_lse,
                                                             void* __restrict__ out, float* __restrict__ lse) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (i >= n) return;
  const float lt = tail_lse ? tail_lse[i] * kL2e : -INFINITY;
  float m = -INFINITY;
  for (int s = lane; s < splits; s += 32) m = fmaxf(m, ml[s * n + i].x);
  m = fmaxf(warp_max(m), lt);
  if (m == -INFINITY) m = 0.f;
  // a state of no tokens (lse -inf) takes no part, whatever its values hold
  const bool own = lt != -INFINITY;
  const float wt = own ? exp2f(lt - m) : 0.f;
  float L = wt;
  for (int s = 0; s < splits; ++s) {
    const float2 x = ml[s * n + i];
    L = fmaf(exp2f(x.x - m), x.y, L);
  }
  const float inv = L > 0.f || L != L ? 1.f / L : 0.f;
  for (int c = lane; c < D; c += 32) {
    float o = own ? wt * load_act(tail, i * D + c, dt) : 0.f;
    for (int s = 0; s < splits; ++s) o = fmaf(exp2f(ml[s * n + i].x - m), po[(s * n + i) * D + c], o);
    store_act(out, i * D + c, o * inv, dt);
  }
  if (lse && lane == 0) lse[i] = L > 0.f || L != L ? (m + log2f(L)) * kLn2 : -INFINITY;
}

// splits of the prefix: enough CTAs for the GPU, at least 128 tokens each
int plan_splits(const carekv_prefix_t& p, int rows, int heads) {
  const int64_t ctas = static_cast<int64_t>(p.num_kv_heads) *
                       ((static_cast<int64_t>(rows) * (heads / p.num_kv_heads) + kFmaRows - 1) / kFmaRows);
  const int want = static_cast<int>(std::min<int64_t>(64, (2 * 148 + ctas - 1) / std::max<int64_t>(1, ctas)));
  return std::max(1, std::min(want, (p.tokens + 127) / 128));
}

}  // namespace

size_t prefix_workspace_bytes(const carekv_prefix_t& p, int rows, int heads) {
  return static_cast<size_t>(plan_splits(p, rows, heads)) * rows * heads * (p.head_dim + 2) * sizeof(float);
}

cudaError_t launch_prefix(const carekv_prefix_t& p, const void* q, int64_t q_row, int64_t q_head, int rows, int heads,
                          float scale, const int32_t* lengths, const void* tail, const float* tail_lse, void* out,
                          float* lse, void* ws, cudaStream_t st) {
  const int64_t n = static_cast<int64_t>(rows) * heads;
  if (n == 0) return cudaSuccess;
  PrefixArgs a;
  a.p = p;
  a.q = q;
  a.q_row = q_row;
  a.q_head = q_head;
  a.rows = rows;
  a.heads = heads;
  a.group = heads / p.num_kv_heads;
  a.scale2 = scale * kL2e;
  a.lengths = lengths;
  a.splits = p.tokens > 0 ? plan_splits(p, rows, heads) : 0;
  a.split_tokens = a.splits ? ((p.tokens + a.splits - 1) / a.splits + kFmaTok - 1) / kFmaTok * kFmaTok : 0;
  a.ml = static_cast<float2*>(ws);
  a.po = reinterpret_cast<float*>(a.ml + a.splits * n);
  if (a.splits) {
    const size_t smem = (kFmaRows * p.head_dim + kFmaTok * (2 * p.head_dim + 1)) * sizeof(float);
    cudaError_t e = cudaFuncSetAttribute(prefix_fma_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 96 * 1024);
    if (e != cudaSuccess) return e;
    const dim3 grid((rows * a.group + kFmaRows - 1) / kFmaRows, p.num_kv_heads, a.splits);
    prefix_fma_kernel<<<grid, kFmaRows * 32, smem, st>>>(a);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  prefix_combine_kernel<<<static_cast<unsigned>((n + 7) / 8), 256, 0, st>>>(a.po, a.ml, a.splits, n, p.head_dim,
                                                                           p.dtype, tail, tail_lse, out, lse);
  return cudaGetLastError();
}

}  // namespace carekv
