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
#include "tcgen05.cuh"

namespace carekv {
namespace {

constexpr float kL2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// How the prefix is cut: a unit is one block of tokens for one tile of rows,
// units are numbered tile by tile (tiles of kv head 0 first) and CTA c takes
// units [start(c), start(c + 1)).  What a CTA has of a tile it does not hold
// whole is a partial, in slot 2c if the CTA starts inside the tile (or at its
// first unit), in slot 2c + 1 if the tile starts inside the CTA.
struct Split {
  int tile_rows;    // rows of a kv head per tile
  int block;        // tokens per unit
  int tiles;        // tiles per kv head
  int blocks;       // units per tile
  int64_t units;
  int ctas;
  __host__ __device__ int64_t start(int64_t c) const { return c * units / ctas; }
  __host__ __device__ int cta_of(int64_t u) const { return static_cast<int>(((u + 1) * ctas - 1) / units); }
};

struct PrefixArgs {
  carekv_prefix_t p;
  const void* q;
  int64_t q_row, q_head;   // strides in elements
  int rows, heads, group;  // group: query heads per kv head
  float scale2;            // scale log2 e: scores in base 2
  const int32_t* lengths;
  const void* tail;        // own state of the rows, or null
  const float* tail_lse;
  void* out;
  float* lse;
  float* po;               // unnormalised partial sums [slot][tile row][D]
  float2* ml;              // [slot][tile row]: base-2 maximum, weight sum
  Split sp;
};

// tokens of the prefix that row r sees
__device__ __forceinline__ int visible(const PrefixArgs& a, int r) {
  return a.lengths ? min(max(a.lengths[r], 0), a.p.tokens) : a.p.tokens;
}

// ── fp32 FMA form ───────────────────────────────────────────────────────
// What the tensor-core form does not take: fp32, head sizes other than 64
// and 128, rows that do not start on 16-byte boundaries.  A warp per row; the
// CTA's 8 rows share 32-token tiles of K and V; grid.z splits the prefix.
constexpr int kFmaRows = 8, kFmaTok = 32, kFmaMaxD = 256;

__global__ void __launch_bounds__(kFmaRows * 32) prefix_fma_kernel(const PrefixArgs a, const int split_tokens) {
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
  const int t_begin = split * split_tokens;
  const int t_end = min(t_begin + split_tokens, a.p.tokens);
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

// ── tensor-core form ────────────────────────────────────────────────────
// One CTA per SM, 10 warps: two groups of four softmax warps (a thread per
// row), one warp that loads K / V tiles by TMA, one that issues the products.
// A group owns a stream: 128 TMEM columns of scores S (overwritten in place
// by the 16-bit weights P) and D columns of output sums O.
//  * PAIR = false (at most 128 rows per kv head: bound by the K / V bytes):
//    both streams share the tile of rows and take alternate token blocks, so
//    one group's exponentials run beside the other's products; their two
//    states are joined when the CTA is done with the tile.
//  * PAIR = true (more rows: bound by products and exponentials): the streams
//    are two tiles of 128 rows that take the same blocks, so a K / V tile in
//    shared memory serves 256 rows.
// A block: S = Q K^T (shared x shared), P = 2^(S scale2 - m) from the
// registers of the row's thread back to TMEM, O += P V (TMEM x shared, V
// read MN-major from its [token][channel] tile).  The running maximum m is
// only raised when a block exceeds it by 2^8, so O is rescaled a few times
// per row and not at every block; the weights stay below 2^8 (2^15 in fp16,
// where m is kept 2^7 low so that small weights stay normal numbers) and the
// weight sum is kept in fp32 from the unrounded weights.  Rounding P to the
// 16-bit type of V is what the matrix instruction takes: an error of half an
// ulp per weight, independent between tokens, like the result's own rounding.
constexpr int kTcThreads = 320, kTcRows = 128, kTcBlock = 128;
constexpr float kRaise = 8.f;

template <int D, bool PAIR>
struct TcLayout {
  static constexpr int kQ = kTcRows * D * 2 * (PAIR ? 2 : 1);
  static constexpr int kSlot = kTcBlock * D * 2;                 // one K or V tile
  static constexpr int kSlots = (224 * 1024 - kQ) / kSlot;       // 224 KB with Q
  static constexpr int kMl = kQ + kSlots * kSlot;                // float2 [2][128]
  static constexpr int kBar = kMl + 2 * kTcRows * 8;
  static constexpr int kBars = 2 * kSlots + 8;
  static constexpr int kBytes = kBar + kBars * 8 + 16;
};

// A wait that gives up after about a second, or as soon as another wait of
// the CTA has.
__device__ __forceinline__ bool wait_or(uint64_t* bar, uint32_t parity, volatile int* dead) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity)) {
    if (*dead || clock64() - t0 > (1ll << 31)) {
      *dead = 1;
      return false;
    }
  }
  return true;
}

struct Segment {
  int kvh, rho0;      // first row of the tile within the kv head
  int b0, nb;         // token blocks that some row of the tile sees
  int top;            // tokens that some row of the tile sees
  int slot;           // partial slot, -1: the CTA holds the whole tile
};

// The part of a tile in [u, u_end); the whole warp calls it.
__device__ __forceinline__ Segment segment_at(const PrefixArgs& a, int64_t u, int64_t u_begin, int64_t u_end,
                                              int64_t* next) {
  Segment s;
  const int64_t tile = u / a.sp.blocks, tile0 = tile * a.sp.blocks;
  const int64_t end = min(u_end, tile0 + a.sp.blocks);
  *next = end;
  s.kvh = static_cast<int>(tile / a.sp.tiles);
  s.rho0 = static_cast<int>(tile - static_cast<int64_t>(s.kvh) * a.sp.tiles) * a.sp.tile_rows;
  s.b0 = static_cast<int>(u - tile0);
  s.nb = static_cast<int>(end - u);
  s.slot = end - u == a.sp.blocks ? -1 : 2 * static_cast<int>(blockIdx.x) + (u == u_begin ? 0 : 1);
  s.top = a.p.tokens;
  if (a.lengths) {
    const int last = min(s.rho0 + a.sp.tile_rows, a.rows * a.group) - 1;
    int top = 0;
    for (int r = s.rho0 / a.group + (threadIdx.x & 31); r <= last / a.group; r += 32) top = max(top, visible(a, r));
    s.top = __reduce_max_sync(0xffffffffu, top);
    s.nb = max(0, min(s.nb, (s.top + kTcBlock - 1) / kTcBlock - s.b0));
  }
  return s;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool BF>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if constexpr (BF) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    return pack_h2(lo, hi);
  }
}

// The state of one row -- maximum m, weight sum l, C channels of the sums
// from channel c0 on -- as a partial or, for a whole tile, the row's result.
template <int D, int C, bool BF>
__device__ __forceinline__ void store_row(const PrefixArgs& a, const Segment& s, int rho, int tile_row, float m, float l,
                                          int c0, const float (&o)[C], bool first) {
  if (s.slot >= 0) {
    const int64_t at = static_cast<int64_t>(s.slot) * a.sp.tile_rows + tile_row;
    if (first) a.ml[at] = make_float2(m, l);
    float4* d = reinterpret_cast<float4*>(a.po + at * D + c0);
#pragma unroll
    for (int i = 0; i < C / 4; ++i) d[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
    return;
  }
  const int64_t i = static_cast<int64_t>(rho / a.group) * a.heads + s.kvh * a.group + rho % a.group;
  const float lt = a.tail ? a.tail_lse[i] * kL2e : -INFINITY;
  float top = fmaxf(m, lt);
  if (top == -INFINITY) top = 0.f;
  const bool own = lt != -INFINITY;
  const float wo = exp2f(m - top), wt = own ? exp2f(lt - top) : 0.f;
  const float L = fmaf(wo, l, wt);
  const float inv = L > 0.f || L != L ? 1.f / L : 0.f;
  if (first && a.lse) a.lse[i] = L > 0.f || L != L ? (top + log2f(L)) * kLn2 : -INFINITY;
  uint4* d = reinterpret_cast<uint4*>(static_cast<char*>(a.out) + (i * D + c0) * 2);
  const uint4* t = reinterpret_cast<const uint4*>(static_cast<const char*>(a.tail) + (i * D + c0) * 2);
#pragma unroll
  for (int k = 0; k < C / 8; ++k) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = wo * o[8 * k + j];
    if (own) {
      const uint4 x = t[k];
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float2 f;
        if constexpr (BF) f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[j]));
        else f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
        v[2 * j] = fmaf(wt, f.x, v[2 * j]);
        v[2 * j + 1] = fmaf(wt, f.y, v[2 * j + 1]);
      }
    }
    d[k] = make_uint4(pack16<BF>(v[0] * inv, v[1] * inv), pack16<BF>(v[2] * inv, v[3] * inv),
                      pack16<BF>(v[4] * inv, v[5] * inv), pack16<BF>(v[6] * inv, v[7] * inv));
  }
}

template <int D, bool BF, bool PAIR>
__global__ void __launch_bounds__(kTcThreads, 1) prefix_tc_kernel(const PrefixArgs a,
                                                                  const __grid_constant__ CUtensorMap kmap,
                                                                  const __grid_constant__ CUtensorMap vmap,
                                                                  const int k_heads, const int v_heads) {
  using Ly = TcLayout<D, PAIR>;
  extern __shared__ __align__(1024) unsigned char smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Ly::kBar);
  uint64_t *full = bars, *empty = bars + Ly::kSlots, *s_full = bars + 2 * Ly::kSlots, *p_full = s_full + 2,
           *o_full = s_full + 4, *q_full = s_full + 6, *done = s_full + 7;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Ly::kBars);
  volatile int* dead = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 9) tmem_alloc(tmem_slot, 512);
  if (threadIdx.x == 0) {
    for (int i = 0; i < Ly::kSlots; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(p_full + i, 4);
      mbar_init(o_full + i, 1);
    }
    mbar_init(q_full, 256);
    mbar_init(done, 1);
    *dead = 0;
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // columns: S (and P) of stream s at 128 s, O at 256 + 128 s
  const int64_t u_begin = a.sp.start(blockIdx.x), u_end = a.sp.start(blockIdx.x + 1);
  bool ok = true;

  if (warp == 8) {
    // ── loads, in the order in which the products use them ──
    int cnt = 0;
    auto load = [&](const CUtensorMap* map, int z, int block) {
      const int slot = cnt % Ly::kSlots;
      ok = ok && __all_sync(0xffffffffu, wait_or(empty + slot, ((cnt / Ly::kSlots) & 1) ^ 1, dead));
      if (!ok) return;
      if (lane == 0) {
        unsigned char* dst = smem + Ly::kQ + slot * Ly::kSlot;
        mbar_expect_tx(full + slot, Ly::kSlot);
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          tma_load_3d(dst + c * (kTcBlock * 128), map, 64 * c, block * kTcBlock, z, full + slot);
      }
      ++cnt;
    };
    for (int64_t u = u_begin; u < u_end && ok;) {
      const Segment s = segment_at(a, u, u_begin, u_end, &u);
      const int zk = s.kvh * k_heads, zv = s.kvh * v_heads;
      if (s.nb > 0) load(&kmap, zk, s.b0);
      if (!PAIR && s.nb > 1) load(&kmap, zk, s.b0 + 1);
      for (int b = 0; b < s.nb && ok; ++b) {
        load(&vmap, zv, s.b0 + b);
        const int n = b + (PAIR ? 1 : 2);
        if (n < s.nb) load(&kmap, zk, s.b0 + n);
      }
    }
    // a copy in flight must land before the CTA ends (all have when ok)
    if (!ok && lane == 0)
      for (int i = max(0, cnt - Ly::kSlots); i < cnt; ++i) mbar_wait(full + i % Ly::kSlots, (i / Ly::kSlots) & 1);
  } else if (warp == 9) {
    // ── products ──
    constexpr uint32_t kIdS = mma_idesc(kTcRows, kTcBlock, BF, false), kIdO = mma_idesc(kTcRows, D, BF, true);
    const uint32_t base = smem_addr(smem);
    int cnt = 0, seg = 0;
    uint32_t ph[2] = {0, 0};
    // next tile in load order
    auto take = [&]() {
      const int slot = cnt % Ly::kSlots;
      ok = ok && __all_sync(0xffffffffu, wait_or(full + slot, (cnt / Ly::kSlots) & 1, dead));
      ++cnt;
      return slot;
    };
    auto scores = [&](int stream, int slot) {
      if (!ok || lane != 0) return;
      const uint32_t qa = base + (PAIR ? stream * (kTcRows * D * 2) : 0), ka = base + Ly::kQ + slot * Ly::kSlot;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint32_t off = (k / 4) * (kTcRows * 128) + (k % 4) * 32;
        mma_ss(tmem + 128 * stream, smem_desc(qa + off, 16, 1024), smem_desc(ka + off, 16, 1024), kIdS, k > 0);
      }
      mma_commit(s_full + stream);
    };
    auto sums = [&](int stream, int slot, int steps, bool acc) {
      if (!ok || lane != 0) return;
      const uint32_t va = base + Ly::kQ + slot * Ly::kSlot;
      for (int k = 0; k < steps; ++k)
        mma_ts(tmem + 256 + 128 * stream, tmem + 128 * stream + 8 * k,
               smem_desc(va + k * (16 * 128), kTcBlock * 128, 1024), kIdO, acc || k > 0);
    };
    auto release = [&](int slot) {
      if (ok && lane == 0) mma_commit(empty + slot);
    };
    auto weights_ready = [&](int stream) {
      ok = ok && __all_sync(0xffffffffu, wait_or(p_full + stream, ph[stream], dead));
      ph[stream] ^= 1;
      tc_fence_after();
    };
    for (int64_t u = u_begin; u < u_end && ok;) {
      const Segment s = segment_at(a, u, u_begin, u_end, &u);
      if (s.nb == 0) continue;
      ok = ok && __all_sync(0xffffffffu, wait_or(q_full, seg & 1, dead));
      ++seg;
      int ks = take();
      scores(0, ks);
      if (PAIR) {
        scores(1, ks);
        release(ks);
      } else {
        release(ks);
        if (s.nb > 1) {
          ks = take();
          scores(1, ks);
          release(ks);
        }
      }
      for (int b = 0; b < s.nb && ok; ++b) {
        const int seen = min(kTcBlock, s.top - (s.b0 + b) * kTcBlock), steps = (seen + 15) / 16;
        const int first = PAIR ? 0 : b & 1;
        weights_ready(first);
        const int vs = take();
        if (ok && lane == 0 && seen < 16 * steps && s.top < a.p.tokens) {
          // tokens of the last step that no row sees: their weights are 0,
          // and 0 times whatever they hold must be 0
          unsigned char* v = smem + Ly::kQ + vs * Ly::kSlot;
          for (int t = seen; t < 16 * steps; ++t)
            for (int c = 0; c < D / 64; ++c)
              for (int i = 0; i < 8; ++i)
                *reinterpret_cast<uint4*>(v + c * (kTcBlock * 128) + t * 128 + 16 * i) = make_uint4(0, 0, 0, 0);
          fence_proxy_async();
        }
        sums(first, vs, steps, PAIR ? b > 0 : b > 1);
        if constexpr (PAIR) {
          const bool more = b + 1 < s.nb;
          if (more) {
            ks = take();
            scores(0, ks);
          } else if (ok && lane == 0) {
            mma_commit(o_full);
          }
          weights_ready(1);
          sums(1, vs, steps, b > 0);
          release(vs);
          if (more) {
            scores(1, ks);
            release(ks);
          } else if (ok && lane == 0) {
            mma_commit(o_full + 1);
          }
        } else {
          release(vs);
          if (b + 2 < s.nb) {
            ks = take();
            scores(first, ks);
            release(ks);
          } else if (ok && lane == 0) {
            mma_commit(o_full + first);
          }
        }
      }
    }
    if (!ok && lane == 0) {   // nothing of ours may still run when TMEM is freed
      mma_commit(done);
      mbar_wait(done, 0);
    }
    __syncwarp();
  } else {
    // ── softmax: stream `st`, row `t` of its tile ──
    const int st = warp >> 2, t = threadIdx.x & 127;
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;   // TMEM lane 32 (warp % 4)
    const uint32_t ts = tmem + 128 * st + lanes, to = tmem + 256 + 128 * st + lanes;
    const float bias = BF ? 0.f : 7.f;
    const int total = a.rows * a.group;
    uint32_t ph = 0, oph = 0;
    float2* ml = reinterpret_cast<float2*>(smem + Ly::kMl);
    for (int64_t u = u_begin; u < u_end;) {
      const Segment s = segment_at(a, u, u_begin, u_end, &u);
      const int tile_row = PAIR ? st * kTcRows + t : t;
      const int rho = s.rho0 + tile_row;
      const bool live = rho < total;
      const bool warp_live = rho - lane < total;
      const int r = live ? rho / a.group : 0, h = s.kvh * a.group + (live ? rho - r * a.group : 0);
      const int vis = live ? visible(a, r) : 0;
      const int n_own = s.nb == 0 ? 0 : PAIR ? s.nb : (s.nb + 1 - st) >> 1;   // blocks of this stream
      if (s.nb > 0) {
        // the tile's query rows, in the swizzled layout of the products
        constexpr int kCols = PAIR ? D : D / 2;
        const int c0 = PAIR ? 0 : st * kCols;
        unsigned char* q = smem + (PAIR ? st * (kTcRows * D * 2) : 0);
        const char* src = static_cast<const char*>(a.q) + (r * a.q_row + h * a.q_head + c0) * 2;
#pragma unroll
        for (int i = 0; i < kCols / 8; ++i) {
          const int c = c0 + 8 * i;
          const uint4 v = live ? __ldg(reinterpret_cast<const uint4*>(src) + i) : make_uint4(0, 0, 0, 0);
          *reinterpret_cast<uint4*>(q + (c >> 6) * (kTcRows * 128) + t * 128 + ((((c & 63) >> 3) ^ (t & 7)) << 4)) = v;
        }
        fence_proxy_async();
        mbar_arrive(q_full);
      }
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < n_own; ++j) {
        ok = ok && __all_sync(0xffffffffu, wait_or(s_full + st, ph, dead));
        ph ^= 1;
        tc_fence_after();
        if (ok && warp_live) {
          const int t0 = (s.b0 + (PAIR ? j : 2 * j + st)) * kTcBlock;
          uint32_t x[128];
          tmem_ld128(ts, x);
          if (__any_sync(0xffffffffu, t0 + kTcBlock > vis)) {
#pragma unroll
            for (int i = 0; i < 128; ++i)
              if (t0 + i >= vis) x[i] = 0xff800000u;
          }
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 128; ++i) mx[i & 3] = fmaxf(mx[i & 3], __uint_as_float(x[i]));
          const float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale2 - bias;
          const bool raise = mt > m + kRaise;
          if (__any_sync(0xffffffffu, raise)) {
            const float mn = raise ? mt : m;
            const float f = raise ? ex2(m - mn) : 1.f;
            m = mn;
            l *= f;
            if (j > 0) {
#pragma unroll 1
              for (int c = 0; c < D; c += 32) {
                uint32_t o[32];
                tmem_ld32(to + c, o);
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                tmem_st32(to + c, o);
              }
            }
          }
          const float mb = m == -INFINITY ? 0.f : -m;
          float sum[4] = {};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float p0 = ex2(fmaf(__uint_as_float(x[32 * c + 2 * i]), a.scale2, mb));
              const float p1 = ex2(fmaf(__uint_as_float(x[32 * c + 2 * i + 1]), a.scale2, mb));
              sum[i & 1] += p0;
              sum[2 + (i & 1)] += p1;
              w[i] = pack16<BF>(p0, p1);
            }
            tmem_st16(ts + 16 * c, w);
          }
          l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + st);
      }
      if (n_own > 0) {
        ok = ok && __all_sync(0xffffffffu, wait_or(o_full + st, oph, dead));
        oph ^= 1;
        tc_fence_after();
      }
      if (!ok) {   // a wait ran out: the rows say so
        m = 0.f;
        l = __int_as_float(0x7fc00000);
      }
      if constexpr (PAIR) {
        if (warp_live) {
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t x[32];
            float o[32];
            if (ok && n_own > 0) tmem_ld32(to + c, x);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = ok && n_own > 0 ? __uint_as_float(x[i]) : 0.f;
            if (live) store_row<D, 32, BF>(a, s, rho, tile_row, m, l, c, o, c == 0);
          }
        }
        tc_fence_before();
      } else {
        // join the streams: this thread takes half of the row's channels
        ml[st * kTcRows + t] = make_float2(m, l);
        named_sync(1, 256);
        if (warp_live) {
          const float2 y = ml[(st ^ 1) * kTcRows + t];
          float top = fmaxf(m, y.x);
          const float base = top == -INFINITY ? 0.f : top;
          const float fo = ex2(m - base), fy = ex2(y.x - base);
          const float f0 = st == 0 ? fo : fy, f1 = st == 0 ? fy : fo;
          const float ls = fo * l + fy * y.y;
          const bool h0 = ok && s.nb > 0, h1 = ok && s.nb > 1;
#pragma unroll 1
          for (int c = st * (D / 2); c < (st + 1) * (D / 2); c += 32) {
            uint32_t x[32];
            float o[32];
            if (h0) tmem_ld32(tmem + 256 + lanes + c, x);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = h0 ? f0 * __uint_as_float(x[i]) : 0.f;
            if (h1) {
              tmem_ld32(tmem + 384 + lanes + c, x);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = fmaf(f1, __uint_as_float(x[i]), o[i]);
            }
            if (live) store_row<D, 32, BF>(a, s, rho, tile_row, top, ls, c, o, c == 0);
          }
        }
        tc_fence_before();
        named_sync(1, 256);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ── join ────────────────────────────────────────────────────────────────
// One warp per (row, head): the partials and the row's own state.  TC: the
// partials of the tensor-core form, rows of whole tiles are done already;
// else those of the FMA form, [split][row].
template <bool TC>
__global__ void __launch_bounds__(256) prefix_combine_kernel(const PrefixArgs a, const int splits) {
  const int64_t n = static_cast<int64_t>(a.rows) * a.heads;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, D = a.p.head_dim, dt = a.p.dtype;
  if (i >= n) return;
  int parts = splits, c0 = 0, tile_row = 0;
  int64_t u0 = 0;
  if constexpr (TC) {
    const int r = static_cast<int>(i / a.heads), h = static_cast<int>(i - static_cast<int64_t>(r) * a.heads);
    const int kvh = h / a.group, rho = r * a.group + h % a.group;
    tile_row = rho % a.sp.tile_rows;
    u0 = (static_cast<int64_t>(kvh) * a.sp.tiles + rho / a.sp.tile_rows) * a.sp.blocks;
    c0 = a.sp.cta_of(u0);
    parts = a.sp.cta_of(u0 + a.sp.blocks - 1) - c0 + 1;
    if (parts == 1) return;
  }
  auto at = [&](int s) -> int64_t {
    if constexpr (TC) {
      const int64_t slot = 2 * (c0 + s) + (a.sp.start(c0 + s) >= u0 ? 0 : 1);
      return slot * a.sp.tile_rows + tile_row;
    } else {
      return s * n + i;
    }
  };
  const float lt = a.tail ? a.tail_lse[i] * kL2e : -INFINITY;
  float m = -INFINITY;
  for (int s = lane; s < parts; s += 32) m = fmaxf(m, a.ml[at(s)].x);
  m = fmaxf(warp_max(m), lt);
  if (m == -INFINITY) m = 0.f;
  // a state of no tokens (lse -inf) takes no part, whatever its values hold
  const bool own = lt != -INFINITY;
  const float wt = own ? exp2f(lt - m) : 0.f;
  float L = wt, o[kFmaMaxD / 32];
#pragma unroll
  for (int k = 0; k < kFmaMaxD / 32; ++k)
    o[k] = own && lane + 32 * k < D ? wt * load_act(a.tail, i * D + lane + 32 * k, dt) : 0.f;
  for (int s = 0; s < parts; ++s) {
    const int64_t p = at(s);
    const float2 x = a.ml[p];
    const float w = exp2f(x.x - m);
    L = fmaf(w, x.y, L);
    if (w != 0.f) {
#pragma unroll
      for (int k = 0; k < kFmaMaxD / 32; ++k)
        if (lane + 32 * k < D) o[k] = fmaf(w, a.po[p * D + lane + 32 * k], o[k]);
    }
  }
  const bool any = L > 0.f || L != L;
  const float inv = any ? 1.f / L : 0.f;
#pragma unroll
  for (int k = 0; k < kFmaMaxD / 32; ++k)
    if (lane + 32 * k < D) store_act(a.out, i * D + lane + 32 * k, o[k] * inv, dt);
  if (a.lse && lane == 0) a.lse[i] = any ? (m + log2f(L)) * kLn2 : -INFINITY;
}

// ── host ────────────────────────────────────────────────────────────────
int sm_count() {
  static thread_local int count[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (count[dev] == 0 &&
      cudaDeviceGetAttribute(&count[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 148;
  return count[dev];
}

// FMA form: splits of the prefix, enough CTAs for the GPU, at least 128 tokens each
int fma_splits(const carekv_prefix_t& p, int rows, int heads) {
  const int64_t ctas = static_cast<int64_t>(p.num_kv_heads) *
                       ((static_cast<int64_t>(rows) * (heads / p.num_kv_heads) + kFmaRows - 1) / kFmaRows);
  const int want = static_cast<int>(std::min<int64_t>(64, (2 * 148 + ctas - 1) / std::max<int64_t>(1, ctas)));
  return std::max(1, std::min(want, (p.tokens + 127) / 128));
}

Split tc_split(const carekv_prefix_t& p, int rows, int heads) {
  Split s;
  const int64_t per_head = static_cast<int64_t>(rows) * (heads / p.num_kv_heads);
  s.tile_rows = per_head <= kTcRows ? kTcRows : 2 * kTcRows;
  s.tiles = static_cast<int>((per_head + s.tile_rows - 1) / s.tile_rows);
  s.blocks = (p.tokens + kTcBlock - 1) / kTcBlock;
  s.units = static_cast<int64_t>(s.tiles) * p.num_kv_heads * s.blocks;
  s.ctas = static_cast<int>(std::min<int64_t>(sm_count(), s.units));
  return s;
}

bool tc_shape(const carekv_prefix_t& p) {
  return p.dtype != CAREKV_F32 && (p.head_dim == 64 || p.head_dim == 128) && p.tokens > 0;
}

// [heads][tokens][D] with 64-channel x 128-token boxes.  A stride of an axis
// of one element is never used; heads on one another (stride 0) are one head.
bool tensor_map(CUtensorMap* map, const void* base, const carekv_prefix_t& p, const int64_t stride[2], int* head_step) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static Encode encode = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<Encode>(f);
  }();
  if (!encode) return false;
  const int64_t row = static_cast<int64_t>(p.head_dim) * 2;
  const int64_t tok = p.tokens > 1 ? stride[1] * 2 : row;
  const bool one = p.num_kv_heads == 1 || stride[0] == 0;
  const int64_t head = one ? tok * p.tokens : stride[0] * 2;
  *head_step = one ? 0 : 1;
  if (tok <= 0 || head <= 0 || tok % 16 || head % 16 || (reinterpret_cast<uintptr_t>(base) & 15)) return false;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(p.head_dim), static_cast<cuuint64_t>(p.tokens),
                              static_cast<cuuint64_t>(one ? 1 : p.num_kv_heads)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(tok), static_cast<cuuint64_t>(head)};
  const cuuint32_t box[3] = {64, kTcBlock, 1}, step[3] = {1, 1, 1};
  return encode(map, p.dtype == CAREKV_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool BF, bool PAIR>
cudaError_t launch_tc(const PrefixArgs& a, const CUtensorMap& km, const CUtensorMap& vm, int kh, int vh,
                      cudaStream_t st) {
  constexpr int smem = TcLayout<D, PAIR>::kBytes;
  static_assert(smem <= 232448, "shared memory of one CTA");
  const cudaError_t e =
      cudaFuncSetAttribute(prefix_tc_kernel<D, BF, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  prefix_tc_kernel<D, BF, PAIR><<<a.sp.ctas, kTcThreads, smem, st>>>(a, km, vm, kh, vh);
  return cudaGetLastError();
}
template <int D, bool BF>
cudaError_t launch_tc(const PrefixArgs& a, const CUtensorMap& km, const CUtensorMap& vm, int kh, int vh,
                      cudaStream_t st) {
  return a.sp.tile_rows == kTcRows ? launch_tc<D, BF, false>(a, km, vm, kh, vh, st)
                                   : launch_tc<D, BF, true>(a, km, vm, kh, vh, st);
}

template <bool TC>
cudaError_t launch_combine(const PrefixArgs& a, int splits, cudaStream_t st) {
  const int64_t n = static_cast<int64_t>(a.rows) * a.heads;
  prefix_combine_kernel<TC><<<static_cast<unsigned>((n + 7) / 8), 256, 0, st>>>(a, splits);
  return cudaGetLastError();
}

}  // namespace

// room for either form
size_t prefix_workspace_bytes(const carekv_prefix_t& p, int rows, int heads) {
  const size_t row = static_cast<size_t>(p.head_dim + 2) * sizeof(float);
  size_t n = static_cast<size_t>(fma_splits(p, rows, heads)) * rows * heads;
  if (tc_shape(p) && rows > 0) {
    const Split s = tc_split(p, rows, heads);
    n = std::max(n, static_cast<size_t>(2) * s.ctas * s.tile_rows);
  }
  return n * row;
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
  a.tail = tail;
  a.tail_lse = tail_lse;
  a.out = out;
  a.lse = lse;
  const uintptr_t m = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) |
                      reinterpret_cast<uintptr_t>(tail) | static_cast<uintptr_t>(q_row * 2) |
                      static_cast<uintptr_t>(q_head * 2);
  CUtensorMap km, vm;
  int kh, vh;
  if (tc_shape(p) && (m & 15) == 0 && tensor_map(&km, p.k, p, p.k_stride, &kh) &&
      tensor_map(&vm, p.v, p, p.v_stride, &vh)) {
    a.sp = tc_split(p, rows, heads);
    a.po = static_cast<float*>(ws);
    a.ml = reinterpret_cast<float2*>(a.po + static_cast<size_t>(2) * a.sp.ctas * a.sp.tile_rows * p.head_dim);
    const bool bf = p.dtype == CAREKV_BF16;
    const cudaError_t e = p.head_dim == 128 ? (bf ? launch_tc<128, true>(a, km, vm, kh, vh, st)
                                                  : launch_tc<128, false>(a, km, vm, kh, vh, st))
                                            : (bf ? launch_tc<64, true>(a, km, vm, kh, vh, st)
                                                  : launch_tc<64, false>(a, km, vm, kh, vh, st));
    if (e != cudaSuccess) return e;
    // no tile is cut when every CTA starts on a tile
    bool cut = false;
    for (int c = 1; c < a.sp.ctas && !cut; ++c) cut = a.sp.start(c) % a.sp.blocks != 0;
    return cut ? launch_combine<true>(a, 0, st) : cudaSuccess;
  }
  const int splits = p.tokens > 0 ? fma_splits(p, rows, heads) : 0;
  a.po = static_cast<float*>(ws);
  a.ml = reinterpret_cast<float2*>(a.po + static_cast<size_t>(splits) * n * p.head_dim);
  if (splits) {
    const int split_tokens = ((p.tokens + splits - 1) / splits + kFmaTok - 1) / kFmaTok * kFmaTok;
    const size_t smem = (kFmaRows * p.head_dim + kFmaTok * (2 * p.head_dim + 1)) * sizeof(float);
    cudaError_t e = cudaFuncSetAttribute(prefix_fma_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 96 * 1024);
    if (e != cudaSuccess) return e;
    const dim3 grid((rows * a.group + kFmaRows - 1) / kFmaRows, p.num_kv_heads, splits);
    prefix_fma_kernel<<<grid, kFmaRows * 32, smem, st>>>(a, split_tokens);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  return launch_combine<false>(a, splits, st);
}

}  // namespace carekv
