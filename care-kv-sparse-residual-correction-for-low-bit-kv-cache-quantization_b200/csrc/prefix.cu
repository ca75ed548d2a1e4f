// Attention of a batch over one shared prefix, computed once for all rows.
//
// For row r and head h, with s_t = scale q . k_t over the prefix tokens the
// row sees: o = sum_t e^{s_t} v_t / sum_t e^{s_t} and lse = log sum_t e^{s_t}.
// The state (o', lse') of the row's own tokens joins as one more term:
//   L = e^{lse} + e^{lse'},  out = (e^{lse} o + e^{lse'} o') / L,  log L.
// Rows of all sequences and the query heads of one kv head form one matrix,
// so every K / V tile is read once for all of them.  The prefix is split over
// CTAs; each writes its unnormalised sum, running maximum and weight sum in
// fp32 and a second kernel joins them with the rows' own state.
#include <algorithm>

#include "common.cuh"
#include "internal.h"
#include "launch.h"
#include "tcgen05.cuh"

namespace carekv {
namespace {

constexpr float kL2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// How the prefix is cut: a unit is one block of tokens for one tile of rows,
// units are numbered tile by tile (tiles of kv head 0 first).  CTA c takes
// `whole` whole tiles, from tile c * whole on, and a share of the units of the
// tiles after those: every group of `group` consecutive units is shared
// evenly by `per` CTAs, a group being one tile or all that is left.  What a
// CTA has of a tile it does not hold whole is a partial, in slot 2c if it
// begins the CTA's share, else in slot 2c + 1.
struct Split {
  int tile_rows;    // rows of a kv head per tile
  int tiles;        // tiles per kv head
  int blocks;       // units per tile
  int ctas;
  int whole, first;            // first: first shared unit, ctas * whole * blocks
  int group, per, base, rem;   // base, rem = group / per, group % per
  __host__ __device__ int start(int c) const {   // first unit of CTA c's share
    const int g = c / per, i = c - g * per;
    return first + g * group + i * base + (i < rem ? i : rem);
  }
  __host__ __device__ int cta_of(int u) const {   // of a shared unit
    const int g = (u - first) / group, v = u - first - g * group, cut = rem * (base + 1);
    return g * per + (v < cut ? v / (base + 1) : rem + (v - cut) / base);
  }
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
  bool out32;              // out starts on a 32-byte boundary
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
// Bound by shared-memory reads, about one word per multiply-add: 16 rows x 32
// heads of 128 on 32768 tokens of 8 kv heads 4.1 ms, 2.1 TFLOP/s, where the
// tensor-core form takes 27 us.
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
// registers of the row's thread back to TMEM, O += P V (TMEM x shared, V read
// MN-major from its [token][channel] tile).  The running maximum m is only
// raised when a block exceeds it by 2^8, so O is rescaled a few times per row
// and not at every block; the weights stay below 2^8 (2^15 in fp16, where m is
// kept 2^7 low so that small weights stay normal numbers) and the weight sum
// is kept in fp32 from the unrounded weights.  Rounding P to the 16-bit type of
// V is what the matrix instruction takes: an error of half an ulp per weight,
// independent between tokens, like the result's own rounding (root mean square
// against 64 bits, relative, where fp32 weights give 1.66e-3 in bf16 and
// 2.06e-4 in fp16: up to 2.05e-3 and 2.6e-4).  The lazy maximum and the
// exponentials on the FMA pipe are published techniques.  Measured: 64 rows x
// 40 heads of 128 on 8191 tokens of 40 kv heads 40.8 us a call with the join,
// 4.1 TB/s of K / V (about 4 us until the first bytes arrive, and the join,
// are what a copy does not have); 2048 rows x 32 heads of 128 on 8192 tokens
// of 8 kv heads 305 us a call, 900 TFLOP/s (the kernel alone 256 us when the
// GPU pauses between calls and its clock stays high), bound by the chain S ->
// maximum -> weights -> P V of a stream (the tensor pipe is active 51% of the
// time, issue 38%).  Two threads per row, and registers moved to the softmax
// warps, lost more to spills than they gained.
constexpr int kTcThreads = 320, kTcRows = 128, kTcBlock = 128;
constexpr float kRaise = 8.f;
// One of so many pairs of weights is computed on the FMA pipe: the 16
// special-function lanes of an SM take 2048 cycles for a block's 256 rows x
// 128 weights, half of what the block takes (2048 rows x 32 heads of 128 on
// 8192 tokens of 8 kv heads, calls back to back: 288 us without, 278 with
// every eighth, 284 with every fourth, 299 with every second).
constexpr int kFmaEvery = 8;

template <int D, bool PAIR>
struct TcLayout {
  static constexpr int kQ = kTcRows * D * 2 * (PAIR ? 2 : 1);
  static constexpr int kSlot = kTcBlock * D * 2;                 // one K or V tile
  static constexpr int kSlots = (224 * 1024 - kQ) / kSlot;       // 224 KB with Q
  static constexpr int kMl = kQ + kSlots * kSlot;                // float2 [2][128]
  static constexpr int kBar = kMl + 2 * kTcRows * 8;
  static constexpr int kBars = 2 * kSlots + 10;
  static constexpr int kBytes = kBar + kBars * 8 + 16;
};

struct Segment {
  int kvh, rho0;      // first row of the tile within the kv head
  int b0, nb;         // token blocks that some row of the tile sees
  int top;            // tokens that some row of the tile sees
  int slot;           // partial slot, -1: the CTA holds the whole tile
};

// A CTA's units: its whole tiles, then its share.
struct Units {
  int whole_end, share, end;
  __device__ __forceinline__ int begin(const Split& sp) {
    const int c = blockIdx.x;
    whole_end = (c + 1) * sp.whole * sp.blocks;
    share = sp.start(c);
    end = sp.start(c + 1);
    return sp.whole ? c * sp.whole * sp.blocks : share;
  }
};

// The part of a tile from unit u on (u < un.end); the whole warp calls it.
__device__ __forceinline__ Segment segment_at(const PrefixArgs& a, const Units& un, int u, int* next) {
  Segment s;
  const int tile = u / a.sp.blocks, tile0 = tile * a.sp.blocks;
  const bool whole = u < un.share;
  const int end = whole ? tile0 + a.sp.blocks : min(un.end, tile0 + a.sp.blocks);
  *next = whole && end == un.whole_end ? un.share : end;
  s.kvh = tile / a.sp.tiles;
  s.rho0 = (tile - s.kvh * a.sp.tiles) * a.sp.tile_rows;
  s.b0 = u - tile0;
  s.nb = end - u;
  s.slot = end - u == a.sp.blocks ? -1 : 2 * static_cast<int>(blockIdx.x) + (u == un.share ? 0 : 1);
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
// 2^y of two values on the FMA pipe, 0 below y = -126 (as ex2 has it; hidden
// tokens come as -inf): y = n + f with n the nearest integer (by adding
// 1.5 2^23), |f| <= 1/2, a degree-4 polynomial for 2^f (fitted for the least
// relative error, 2.6e-6) and n added to its exponent (Cody and Waite's
// scheme).
__device__ __forceinline__ float2 ex2_fma(float2 y) {
  const float2 big = make_float2(12582912.f, 12582912.f), nbig = make_float2(-12582912.f, -12582912.f);
  const float2 r = add2(y, big), n = add2(r, nbig);
  const float2 f = fma2(n, make_float2(-1.f, -1.f), y);
  float2 p = fma2(f, make_float2(0x1.3997d4p-7f, 0x1.3997d4p-7f), make_float2(0x1.ca1440p-5f, 0x1.ca1440p-5f));
  p = fma2(p, f, make_float2(0x1.ec06dap-3f, 0x1.ec06dap-3f));
  p = fma2(p, f, make_float2(0x1.62e0dcp-1f, 0x1.62e0dcp-1f));
  p = fma2(p, f, make_float2(0x1.ffffe8p-1f, 0x1.ffffe8p-1f));
  return make_float2(y.x < -126.f ? 0.f : __uint_as_float(__float_as_uint(p.x) + (__float_as_uint(r.x) << 23)),
                     y.y < -126.f ? 0.f : __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(r.y) << 23)));
}
__device__ __forceinline__ float max_nan(float x, float y) {   // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
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

// A whole 32-byte sector per lane: the rows of a warp lie apart, and two
// 16-byte stores would each write half a sector.  The store wants p on a
// 32-byte boundary (`aligned`); elsewhere it is two stores of 16 bytes.
__device__ __forceinline__ void store32(void* p, const uint32_t (&w)[8], bool aligned) {
  if (!aligned) {
    reinterpret_cast<uint4*>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    reinterpret_cast<uint4*>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
    return;
  }
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// The state of one row -- maximum m, weight sum l, C channels of the sums
// from channel c0 on -- as a partial or, for a whole tile, the row's result.
template <int D, int C, bool BF>
__device__ __forceinline__ void store_row(const PrefixArgs& a, const Segment& s, int rho, int tile_row, float m, float l,
                                          int c0, const float (&o)[C], bool first) {
  if (s.slot >= 0) {
    const int64_t at = static_cast<int64_t>(s.slot) * a.sp.tile_rows + tile_row;
    if (first) a.ml[at] = make_float2(m, l);
#pragma unroll
    for (int i = 0; i < C; i += 8) {
      uint32_t w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = __float_as_uint(o[i + j]);
      store32(a.po + at * D + c0 + i, w, true);
    }
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
  char* d = static_cast<char*>(a.out) + (i * D + c0) * 2;
  const uint4* t = reinterpret_cast<const uint4*>(static_cast<const char*>(a.tail) + (i * D + c0) * 2);
#pragma unroll
  for (int k = 0; k < C; k += 16) {
    uint32_t w[8];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const uint4 x = own ? t[k / 8 + g] : make_uint4(0, 0, 0, 0);
      const uint32_t y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = k + 8 * g + 2 * j;
        float2 f;
        if constexpr (BF) f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&y[j]));
        else f = __half22float2(*reinterpret_cast<const __half2*>(&y[j]));
        w[4 * g + j] = pack16<BF>(fmaf(wt, f.x, wo * o[c]) * inv, fmaf(wt, f.y, wo * o[c + 1]) * inv);
      }
    }
    store32(d + 2 * k, w, a.out32);
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
  // p_half / p_full: weights of the first / last 64 tokens of a block
  uint64_t *full = bars, *empty = bars + Ly::kSlots, *s_full = bars + 2 * Ly::kSlots, *p_half = s_full + 2,
           *p_full = s_full + 4, *o_full = s_full + 6, *q_full = s_full + 8, *done = s_full + 9;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Ly::kBars);
  volatile int* dead = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Units un;
  const int u_begin = un.begin(a.sp);
  bool ok = true;

  if (warp == 8) {
    // ── loads, in the order in which the products use them; the first ones
    // are on their way before the CTA has set up the rest ──
    if (lane == 0) {
      for (int i = 0; i < Ly::kSlots; ++i) {
        mbar_init(full + i, 1);
        mbar_init(empty + i, 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(s_full + i, 1);
        mbar_init(p_half + i, 4);
        mbar_init(p_full + i, 4);
        mbar_init(o_full + i, 1);
      }
      mbar_init(q_full, 256);
      mbar_init(done, 1);
      *dead = 0;
      fence_mbar_init();
    }
    __syncwarp();
    // With one tile per kv head every K / V byte is read once: it leaves the
    // L2 first (16 rows on 32768 tokens 39.6 -> 37.5 us a call).  With several,
    // the other tiles' CTAs find it there; the policy makes no difference then
    // (2048 rows on 8192: 283 us with and without).
    const uint64_t policy = l2_evict_first();
    int cnt = 0;
    bool synced = false;
    auto sync_once = [&]() {
      if (!synced) {
        tc_fence_before();
        __syncthreads();
        synced = true;
      }
    };
    auto load = [&](const CUtensorMap* map, int z, int block) {
      const int slot = cnt % Ly::kSlots;
      if (cnt >= Ly::kSlots) {
        sync_once();
        ok = ok && __all_sync(0xffffffffu, wait_or(empty + slot, ((cnt / Ly::kSlots) & 1) ^ 1, dead));
        if (!ok) return;
      }
      if (lane == 0) {
        unsigned char* dst = smem + Ly::kQ + slot * Ly::kSlot;
        mbar_expect_tx(full + slot, Ly::kSlot);
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          if constexpr (PAIR) tma_load_3d(dst + c * (kTcBlock * 128), map, 64 * c, block * kTcBlock, z, full + slot);
          else tma_load_3d_pol(dst + c * (kTcBlock * 128), map, 64 * c, block * kTcBlock, z, full + slot, policy);
      }
      ++cnt;
    };
    for (int u = u_begin; u < un.end && ok;) {
      const Segment s = segment_at(a, un, u, &u);
      const int zk = s.kvh * k_heads, zv = s.kvh * v_heads;
      if (s.nb > 0) load(&kmap, zk, s.b0);
      if (!PAIR && s.nb > 1) load(&kmap, zk, s.b0 + 1);
      for (int b = 0; b < s.nb && ok; ++b) {
        load(&vmap, zv, s.b0 + b);
        const int n = b + (PAIR ? 1 : 2);
        if (n < s.nb) load(&kmap, zk, s.b0 + n);
      }
    }
    sync_once();
    // a copy in flight must land before the CTA ends (all have when ok)
    if (!ok && lane == 0)
      for (int i = max(0, cnt - Ly::kSlots); i < cnt; ++i) mbar_wait(full + i % Ly::kSlots, (i / Ly::kSlots) & 1);
  } else if (warp == 9) {
    // ── products ──
    tmem_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t tmem = *tmem_slot;   // columns: S (and P) of stream s at 128 s, O at 256 + 128 s
    constexpr uint32_t kIdS = mma_idesc(kTcRows, kTcBlock, BF, false), kIdO = mma_idesc(kTcRows, D, BF, true);
    const uint32_t base = smem_addr(smem), lead = elect_one();
    // descriptors of the first Q and tile; others differ in the address field
    // (16-byte units) alone
    const uint64_t qd = smem_desc(base, 16, 1024), kd = smem_desc(base + Ly::kQ, 16, 1024),
                   vd = smem_desc(base + Ly::kQ, kTcBlock * 128, 1024);
    int cnt = 0, seg = 0;
    uint32_t ph[2] = {0, 0};
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      ok = ok && __all_sync(0xffffffffu, wait_or(bar, parity, dead));
    };
    // next tile in load order
    auto take = [&]() {
      const int slot = cnt % Ly::kSlots;
      wait(full + slot, (cnt / Ly::kSlots) & 1);
      ++cnt;
      return slot;
    };
    auto scores = [&](int stream, int slot) {
      if (!ok) return;
      const uint64_t qa = qd + (PAIR ? stream * (kTcRows * D * 2 / 16) : 0), ka = kd + slot * (Ly::kSlot / 16);
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const int off = ((k / 4) * (kTcRows * 128) + (k % 4) * 32) / 16;
        mma_ss(tmem + 128 * stream, qa + off, ka + off, kIdS, k > 0, lead);
      }
      mma_commit(s_full + stream, lead);
    };
    // O += P V for the tokens of half h, 16 a step
    auto sums = [&](int stream, int slot, int h, int steps, bool acc) {
      if (!ok) return;
      const uint32_t o = tmem + 256 + 128 * stream, p = tmem + 128 * stream + 32 * h;
      const uint64_t va = vd + slot * (Ly::kSlot / 16) + h * (64 * 128 / 16);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (4 * h + k < steps) mma_ts(o, p + 8 * k, va + k * (16 * 128 / 16), kIdO, acc || h > 0 || k > 0, lead);
    };
    auto release = [&](int slot) {
      if (ok) mma_commit(empty + slot, lead);
    };
    auto finish = [&](int stream) {
      if (ok) mma_commit(o_full + stream, lead);
    };
    for (int u = u_begin; u < un.end && ok;) {
      const Segment s = segment_at(a, un, u, &u);
      if (s.nb == 0) continue;
      wait(q_full, seg & 1);
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
        int vs = 0;
#pragma unroll
        for (int i = 0; i < (PAIR ? 2 : 1); ++i) {
          const int stream = PAIR ? i : b & 1;
          const bool acc = b > (PAIR ? 0 : 1);
          wait(p_half + stream, ph[stream]);
          if (i == 0) {
            vs = take();
            if (ok && seen < 16 * steps && s.top < a.p.tokens) {
              // tokens of the last step that no row sees: their weights are
              // 0, and 0 times whatever they hold must be 0
              unsigned char* v = smem + Ly::kQ + vs * Ly::kSlot;
              for (int j = lane; j < (16 * steps - seen) * (D / 8); j += 32) {
                const int t = seen + j / (D / 8), c = j % (D / 8);
                *reinterpret_cast<uint4*>(v + (c >> 3) * (kTcBlock * 128) + t * 128 + 16 * (c & 7)) = make_uint4(0, 0, 0, 0);
              }
              fence_proxy_async();
              __syncwarp();
            }
          }
          tc_fence_after();
          sums(stream, vs, 0, steps, acc);
          wait(p_full + stream, ph[stream]);
          ph[stream] ^= 1;
          tc_fence_after();
          sums(stream, vs, 1, steps, acc);
          const int n = b + (PAIR ? 1 : 2);
          if (!PAIR || i == 1) release(vs);
          if (n < s.nb) {
            if (!PAIR || i == 0) ks = take();
            scores(stream, ks);
            if (!PAIR || i == 1) release(ks);
          } else {
            finish(stream);
          }
        }
      }
    }
    if (!ok) {   // nothing of ours may still run when TMEM is freed
      mma_commit(done, lead);
      mbar_wait(done, 0);
    }
    __syncwarp();
  } else {
    // ── softmax: stream `st`, row `t` of its tile ──
    const int st = warp >> 2, t = threadIdx.x & 127;
    const int tile_row = PAIR ? st * kTcRows + t : t;
    const float bias = BF ? 0.f : 7.f;
    const int total = a.rows * a.group;
    // a row's place: query row r, kv head group member h
    int rho, r, h;
    auto place = [&](const Segment& s) {
      rho = s.rho0 + tile_row;
      r = rho < total ? rho / a.group : 0;
      h = s.kvh * a.group + (rho < total ? rho - r * a.group : 0);
    };
    // The tile's query rows to shared memory, in the swizzled layout of the
    // products: the warp copies its 32 rows (PAIR: all channels, else its
    // half), kRow lanes a row; rows past the last are zero.
    auto q_fetch = [&]() {
      constexpr int kCols = PAIR ? D : D / 2, kRow = kCols / 8;
      const int64_t off = rho < total ? (r * a.q_row + h * a.q_head) * 2 : -1;
      unsigned char* q = smem + (PAIR ? st * (kTcRows * D * 2) : 0);
      const int c = (PAIR ? 0 : st * kCols) + 8 * (lane % kRow);
#pragma unroll 4
      for (int i = 0; i < 32; i += 32 / kRow) {
        const int row = i + lane / kRow, tr = (warp & 3) * 32 + row;
        const int64_t at = __shfl_sync(0xffffffffu, off, row);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(
                         q + (c >> 6) * (kTcRows * 128) + tr * 128 + ((((c & 63) >> 3) ^ (tr & 7)) << 4))),
                     "l"(static_cast<const char*>(a.q) + (at < 0 ? 0 : at + 2 * c)), "r"(at < 0 ? 0 : 16)
                     : "memory");
      }
    };
    auto q_ready = [&]() {
      asm volatile("cp.async.wait_all;" ::: "memory");
      fence_proxy_async();
      mbar_arrive(q_full);
    };
    int u_next;
    Segment s = segment_at(a, un, u_begin, &u_next);
    place(s);
    if (s.nb > 0) q_fetch();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot, lanes = static_cast<uint32_t>(warp & 3) << 21;   // TMEM lane 32 (warp % 4)
    const uint32_t ts = tmem + 128 * st + lanes, to = tmem + 256 + 128 * st + lanes;
    uint32_t ph = 0, oph = 0;
    float2* ml = reinterpret_cast<float2*>(smem + Ly::kMl);
    if (s.nb > 0) q_ready();
    for (;;) {
      const bool live = rho < total, warp_live = rho - lane < total;
      const int vis = live ? visible(a, r) : a.p.tokens;   // rows past the last: whatever
      const int n_own = s.nb == 0 ? 0 : PAIR ? s.nb : (s.nb + 1 - st) >> 1;   // blocks of this stream
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < n_own; ++j) {
        ok = ok && __all_sync(0xffffffffu, wait_or(s_full + st, ph, dead));
        ph ^= 1;
        tc_fence_after();
        const bool work = ok && warp_live;
        // 32 columns at a time (128 scores would not fit the registers), the
        // next 32 on their way: once for the maximum, once for the weights.
        // The loops stay loops: the code is fetched anew by every launch, and
        // its size shows in the first block's time.
        uint32_t xa[32], xb[32];
        float2 sum[2] = {{0.f, 0.f}, {0.f, 0.f}};
        float mb = 0.f;
        const int t0 = (s.b0 + (PAIR ? j : 2 * j + st)) * kTcBlock;
        const bool edge = work && __any_sync(0xffffffffu, t0 + kTcBlock > vis);
        auto hide = [&](uint32_t (&x)[32], int c) {
          if (edge) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (t0 + c + i >= vis) x[i] = 0xff800000u;
          }
        };
        if (work) {
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          auto maxima = [&](uint32_t (&x)[32], int c) {
            hide(x, c);
#pragma unroll
            for (int i = 0; i < 32; ++i) mx[i & 3] = max_nan(mx[i & 3], __uint_as_float(x[i]));
          };
          tmem_ld32_start(ts, xa);
#pragma unroll 1
          for (int c = 0; c < kTcBlock; c += 64) {
            tmem_landed(xa);
            tmem_ld32_start(ts + c + 32, xb);
            maxima(xa, c);
            tmem_landed(xb);
            tmem_ld32_start(ts + (c + 64) % kTcBlock, xa);   // at the end: the first columns again
            maxima(xb, c + 32);
          }
          float mt = max_nan(max_nan(mx[0], mx[1]), max_nan(mx[2], mx[3])) * a.scale2 - bias;
          if (mt == INFINITY) mt = __int_as_float(0x7fc00000);   // the row's weights are inf - inf
          const bool raise = !(mt <= m + kRaise);                // NaN raises too and makes all weights NaN
          if (__any_sync(0xffffffffu, raise)) {
            const float mn = raise ? mt : m;
            const float f = raise ? ex2(m - mn) : 1.f;
            m = mn;
            l *= f;
            if (j > 0) {
              tmem_landed(xa);
#pragma unroll 1
              for (int c = 0; c < D; c += 32) {
                tmem_ld32(to + c, xb);
#pragma unroll
                for (int i = 0; i < 32; ++i) xb[i] = __float_as_uint(__uint_as_float(xb[i]) * f);
                tmem_st32(to + c, xb);
              }
            }
          }
          mb = m == -INFINITY ? 0.f : -m;
        }
        // weights of tokens c .. c + 31 to columns c / 2 .. of P, which lie
        // over scores that are in registers or done by then
        auto weights = [&](uint32_t (&x)[32], int c) {
          hide(x, c);
          const float2 sc = make_float2(a.scale2, a.scale2), mb2 = make_float2(mb, mb);
          float2 p[16];
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i)
            p[i] = fma2(make_float2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), sc, mb2);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (i % kFmaEvery != 0) p[i] = make_float2(ex2(p[i].x), ex2(p[i].y));
#pragma unroll
          for (int i = 0; i < 16; i += kFmaEvery) p[i] = ex2_fma(p[i]);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            sum[i & 1] = add2(sum[i & 1], p[i]);
            w[i] = pack16<BF>(p[i].x, p[i].y);
          }
          tmem_st16(ts + c / 2, w);
        };
#pragma unroll 1
        for (int c = 0; c < kTcBlock; c += 64) {
          if (work) {
            tmem_landed(xa);
            tmem_ld32_start(ts + c + 32, xb);
            weights(xa, c);
            tmem_landed(xb);
            if (c == 0) tmem_ld32_start(ts + 64, xa);
            weights(xb, c + 32);
            tmem_wait_st();
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive((c == 0 ? p_half : p_full) + st);
        }
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      }
      const Segment done_s = s;
      const int done_rho = rho;
      const bool more = u_next < un.end;
      if (more) {
        s = segment_at(a, un, u_next, &u_next);
        place(s);
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
        if (more && s.nb > 0) {   // this stream's products with the old rows are done
          q_fetch();
          q_ready();
        }
        if (warp_live) {
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t x[32];
            float o[32];
            if (ok && n_own > 0) tmem_ld32(to + c, x);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = ok && n_own > 0 ? __uint_as_float(x[i]) : 0.f;
            if (live) store_row<D, 32, BF>(a, done_s, done_rho, tile_row, m, l, c, o, c == 0);
          }
        }
        tc_fence_before();
      } else {
        // join the streams: this thread takes half of the row's channels
        ml[st * kTcRows + t] = make_float2(m, l);
        named_sync(1, 256);
        if (more && s.nb > 0) {   // both streams' products are done
          q_fetch();
          q_ready();
        }
        if (warp_live) {
          const float2 y = ml[(st ^ 1) * kTcRows + t];
          const float top = fmaxf(m, y.x);
          const float base = top == -INFINITY ? 0.f : top;
          const float fo = ex2(m - base), fy = ex2(y.x - base);
          const float f0 = st == 0 ? fo : fy, f1 = st == 0 ? fy : fo;
          const float ls = fo * l + fy * y.y;
          const bool h0 = ok && done_s.nb > 0, h1 = ok && done_s.nb > 1;
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
            if (live) store_row<D, 32, BF>(a, done_s, done_rho, tile_row, top, ls, c, o, c == 0);
          }
        }
        tc_fence_before();
        if (more) named_sync(1, 256);   // the sums may be overwritten
      }
      if (!more) break;
    }
  }
  tc_fence_before();
  __syncthreads();
  report_wait(dead);
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(*tmem_slot, 512);
  }
}

// ── join ────────────────────────────────────────────────────────────────
// A CTA per 8 rows of a shared tile, a warp per (row, head): the partials and
// the row's own state.  Lane s finds partial s (of up to 32 at a time) and its
// weight; then the partials are read eight at a time, a row of D floats per
// warp load.
template <int D, bool BF>
__global__ void __launch_bounds__(256) prefix_combine_kernel(const PrefixArgs a) {
  constexpr int V = D / 32;
  struct alignas(4 * V) Vec {
    float v[V];
  };
  struct alignas(2 * V) Vec16 {
    uint32_t v[V / 2];
  };
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int ctas = a.sp.tile_rows / 8;
  const int tile = a.sp.ctas * a.sp.whole + static_cast<int>(blockIdx.x) / ctas;
  const int u0 = tile * a.sp.blocks;
  const int c0 = a.sp.cta_of(u0), parts = a.sp.cta_of(u0 + a.sp.blocks - 1) - c0 + 1;
  const int kvh = tile / a.sp.tiles;
  const int tile_row = (static_cast<int>(blockIdx.x) % ctas) * 8 + (threadIdx.x >> 5);
  const int rho = (tile - kvh * a.sp.tiles) * a.sp.tile_rows + tile_row;
  if (parts == 1 || rho >= a.rows * a.group) return;
  const int r = rho / a.group;
  const int64_t i = static_cast<int64_t>(r) * a.heads + kvh * a.group + (rho - r * a.group);
  auto at = [&](int s) { return (2 * (c0 + s) + (a.sp.start(c0 + s) >= u0 ? 0 : 1)) * a.sp.tile_rows + tile_row; };
  const float lt = a.tail ? a.tail_lse[i] * kL2e : -INFINITY;
  // a state of no tokens (lse -inf) takes no part, whatever its values hold
  const bool own = lt != -INFINITY;
  Vec16 tv = {};
  if (own) tv = reinterpret_cast<const Vec16*>(static_cast<const char*>(a.tail) + i * D * 2)[lane];
  // the first 32 partials' states stay in registers for the second pass
  int p0 = 0;
  float2 x0 = make_float2(-INFINITY, 0.f);
  if (lane < parts) {
    p0 = at(lane);
    x0 = a.ml[p0];
  }
  float m = x0.x;
  for (int s = 32 + lane; s < parts; s += 32) m = fmaxf(m, a.ml[at(s)].x);
  m = fmaxf(warp_max(m), lt);
  if (m == -INFINITY) m = 0.f;
  const float wt = own ? exp2f(lt - m) : 0.f;
  float L = 0.f, o[V];
#pragma unroll
  for (int k = 0; k < V; k += 2) {
    float2 f;
    if constexpr (BF) f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&tv.v[k / 2]));
    else f = __half22float2(*reinterpret_cast<const __half2*>(&tv.v[k / 2]));
    o[k] = own ? wt * f.x : 0.f;
    o[k + 1] = own ? wt * f.y : 0.f;
  }
  for (int s0 = 0; s0 < parts; s0 += 32) {
    int p = p0;
    float2 x = x0;
    if (s0 > 0) {
      x = make_float2(-INFINITY, 0.f);
      if (s0 + lane < parts) {
        p = at(s0 + lane);
        x = a.ml[p];
      }
    }
    const float w = exp2f(x.x - m);
    L = fmaf(w, x.y, L);
    const int cnt = min(32, parts - s0);
    for (int s = 0; s < cnt; s += 8) {
      Vec v[8];
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        f[j] = __shfl_sync(0xffffffffu, w, (s + j) & 31);
        const int64_t q = __shfl_sync(0xffffffffu, p, (s + j) & 31);
        if (s + j < cnt && f[j] != 0.f) v[j] = reinterpret_cast<const Vec*>(a.po + q * D)[lane];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (s + j < cnt && f[j] != 0.f) {
#pragma unroll
          for (int k = 0; k < V; ++k) o[k] = fmaf(f[j], v[j].v[k], o[k]);
        }
    }
  }
  L = warp_sum(L) + wt;
  const bool any = L > 0.f || L != L;
  const float inv = any ? 1.f / L : 0.f;
  Vec16 y;
#pragma unroll
  for (int k = 0; k < V; k += 2) y.v[k / 2] = pack16<BF>(o[k] * inv, o[k + 1] * inv);
  reinterpret_cast<Vec16*>(static_cast<char*>(a.out) + i * D * 2)[lane] = y;
  if (a.lse && lane == 0) a.lse[i] = any ? (m + log2f(L)) * kLn2 : -INFINITY;
}

// The same for the FMA form's partials, [split][row].
__global__ void __launch_bounds__(256) prefix_fma_combine_kernel(const PrefixArgs a, const int splits) {
  const int64_t n = static_cast<int64_t>(a.rows) * a.heads;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, D = a.p.head_dim, dt = a.p.dtype;
  if (i >= n) return;
  const float lt = a.tail ? a.tail_lse[i] * kL2e : -INFINITY;
  float m = -INFINITY;
  for (int s = lane; s < splits; s += 32) m = fmaxf(m, a.ml[s * n + i].x);
  m = fmaxf(warp_max(m), lt);
  if (m == -INFINITY) m = 0.f;
  const bool own = lt != -INFINITY;
  const float wt = own ? exp2f(lt - m) : 0.f;
  float L = wt, o[kFmaMaxD / 32];
#pragma unroll
  for (int k = 0; k < kFmaMaxD / 32; ++k)
    o[k] = own && lane + 32 * k < D ? wt * load_act(a.tail, i * D + lane + 32 * k, dt) : 0.f;
  for (int s = 0; s < splits; ++s) {
    const int64_t p = s * n + i;
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
// FMA form: splits of the prefix, enough CTAs for the GPU, at least 128 tokens each
int fma_splits(const carekv_prefix_t& p, int rows, int heads) {
  const int64_t ctas = static_cast<int64_t>(p.num_kv_heads) *
                       ((static_cast<int64_t>(rows) * (heads / p.num_kv_heads) + kFmaRows - 1) / kFmaRows);
  const int want = static_cast<int>(std::min<int64_t>(64, (2 * sm_count() + ctas - 1) / std::max<int64_t>(1, ctas)));
  return std::max(1, std::min(want, (p.tokens + 127) / 128));
}

// Every CTA works on one SM for the whole launch.  With no more tiles than
// SMs, either the CTAs of a tile share it evenly, or all CTAs share all units
// evenly and most of them cross a tile's end, which costs about kCross units
// (the state of one tile written out, the pipeline filled for the next).  A
// tile of few units stays whole: the join is a launch of its own, as long as
// about kJoin units.  With more tiles than SMs, each CTA takes as many whole
// ones as all can have and a share of the rest.
constexpr int kCross = 4, kJoin = 4;

bool tc_split(const carekv_prefix_t& p, int rows, int heads, Split* s) {
  const int64_t per_head = static_cast<int64_t>(rows) * (heads / p.num_kv_heads);
  s->tile_rows = per_head <= kTcRows ? kTcRows : 2 * kTcRows;
  s->tiles = static_cast<int>((per_head + s->tile_rows - 1) / s->tile_rows);
  s->blocks = static_cast<int>((static_cast<int64_t>(p.tokens) + kTcBlock - 1) / kTcBlock);
  const int64_t tiles = static_cast<int64_t>(s->tiles) * p.num_kv_heads, units = tiles * s->blocks;
  if (units > (1 << 30)) return false;
  const int sms = sm_count();
  s->whole = 0;
  s->ctas = sms;
  if (tiles <= sms) {
    const int per = s->blocks <= kJoin ? 1 : static_cast<int>(std::min<int64_t>(sms / tiles, s->blocks));
    const int64_t even = (units + sms - 1) / sms;
    if (s->blocks <= kJoin || (s->blocks + per - 1) / per <= even + kCross) {
      s->group = s->blocks;
      s->per = per;
      s->ctas = static_cast<int>(tiles) * per;
    } else {
      s->group = static_cast<int>(units);
      s->per = s->ctas = static_cast<int>(std::min<int64_t>(sms, units));
    }
  } else {
    s->whole = static_cast<int>(tiles / sms);
    s->group = static_cast<int>(tiles % sms) * s->blocks;   // may be 0: nothing is shared
    s->per = sms;
  }
  s->first = s->ctas * s->whole * s->blocks;
  s->base = s->group / s->per;
  s->rem = s->group % s->per;
  return true;
}

bool tc_shape(const carekv_prefix_t& p) {
  return p.dtype != CAREKV_F32 && (p.head_dim == 64 || p.head_dim == 128) && p.tokens > 0;
}

// [heads][tokens][D] with 64-channel x 128-token boxes.  A stride of an axis
// of one element is never used; heads on one another (stride 0) are one head.
bool tensor_map(CUtensorMap* map, const void* base, const carekv_prefix_t& p, const int64_t stride[2], int* head_step) {
  const TensorMapEncode encode = tensor_map_encode();
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
  const cudaError_t e = allow_smem<smem>(prefix_tc_kernel<D, BF, PAIR>);
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

// The join of the shared tiles; it starts while the products' last CTAs run
// and waits for them itself.
cudaError_t launch_combine(const PrefixArgs& a, cudaStream_t st) {
  const int tiles = a.sp.tiles * a.p.num_kv_heads - a.sp.ctas * a.sp.whole;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * (a.sp.tile_rows / 8)));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const bool bf = a.p.dtype == CAREKV_BF16;
  if (a.p.head_dim == 128)
    return bf ? cudaLaunchKernelEx(&cfg, prefix_combine_kernel<128, true>, a)
              : cudaLaunchKernelEx(&cfg, prefix_combine_kernel<128, false>, a);
  return bf ? cudaLaunchKernelEx(&cfg, prefix_combine_kernel<64, true>, a)
            : cudaLaunchKernelEx(&cfg, prefix_combine_kernel<64, false>, a);
}

}  // namespace

cudaError_t prefix_wait_errors(int32_t* set, cudaStream_t st) { return take_wait_errors(set, st); }

// room for either form, and for the partial sums to start on a 32-byte
// boundary (store32) in a buffer that starts on one of 16
size_t prefix_workspace_bytes(const carekv_prefix_t& p, int rows, int heads) {
  const size_t row = static_cast<size_t>(p.head_dim + 2) * sizeof(float);
  size_t n = static_cast<size_t>(fma_splits(p, rows, heads)) * rows * heads;
  Split s;
  if (tc_shape(p) && rows > 0 && tc_split(p, rows, heads, &s))
    n = std::max(n, static_cast<size_t>(2) * s.ctas * s.tile_rows);
  return n ? n * row + 16 : 0;
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
  a.out32 = (reinterpret_cast<uintptr_t>(out) & 31) == 0;
  a.po = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(ws) + 31) & ~uintptr_t{31});
  const uintptr_t m = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) |
                      reinterpret_cast<uintptr_t>(tail) | static_cast<uintptr_t>(q_row * 2) |
                      static_cast<uintptr_t>(q_head * 2);
  CUtensorMap km, vm;
  int kh, vh;
  if (tc_shape(p) && (m & 15) == 0 && tc_split(p, rows, heads, &a.sp) && tensor_map(&km, p.k, p, p.k_stride, &kh) &&
      tensor_map(&vm, p.v, p, p.v_stride, &vh)) {
    a.ml = reinterpret_cast<float2*>(a.po + static_cast<size_t>(2) * a.sp.ctas * a.sp.tile_rows * p.head_dim);
    const bool bf = p.dtype == CAREKV_BF16;
    const cudaError_t e = p.head_dim == 128 ? (bf ? launch_tc<128, true>(a, km, vm, kh, vh, st)
                                                  : launch_tc<128, false>(a, km, vm, kh, vh, st))
                                            : (bf ? launch_tc<64, true>(a, km, vm, kh, vh, st)
                                                  : launch_tc<64, false>(a, km, vm, kh, vh, st));
    if (e != cudaSuccess) return e;
    // no tile is cut when every share starts on one
    const bool cut = a.sp.group == a.sp.blocks ? a.sp.per > 1 : a.sp.rem != 0 || a.sp.base % a.sp.blocks != 0;
    return cut ? launch_combine(a, st) : cudaSuccess;
  }
  const int splits = p.tokens > 0 ? fma_splits(p, rows, heads) : 0;
  a.ml = reinterpret_cast<float2*>(a.po + static_cast<size_t>(splits) * n * p.head_dim);
  if (splits) {
    const int split_tokens = ((p.tokens + splits - 1) / splits + kFmaTok - 1) / kFmaTok * kFmaTok;
    const size_t smem = (kFmaRows * p.head_dim + kFmaTok * (2 * p.head_dim + 1)) * sizeof(float);
    cudaError_t e = allow_smem<96 * 1024>(prefix_fma_kernel);
    if (e != cudaSuccess) return e;
    const dim3 grid((rows * a.group + kFmaRows - 1) / kFmaRows, p.num_kv_heads, splits);
    prefix_fma_kernel<<<grid, kFmaRows * 32, smem, st>>>(a, split_tokens);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  prefix_fma_combine_kernel<<<static_cast<unsigned>((n + 7) / 8), 256, 0, st>>>(a, splits);
  return cudaGetLastError();
}

}  // namespace carekv
