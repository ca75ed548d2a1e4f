// Inline-PTX helpers for the 5th-generation tensor cores (sm_100a): TMEM
// allocation and access, descriptors, tcgen05.mma, and tiled TMA loads.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <cstdint>

#include "ptx.cuh"

namespace carekv {

// ── TMEM ────────────────────────────────────────────────────────────────
// Whole-warp calls; the address of the allocation is written to shared memory.
__device__ __forceinline__ void tmem_alloc(uint32_t* smem_slot, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(smem_slot)),
               "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t addr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

#define CAREKV_R8(a, i) "=r"(a[i]), "=r"(a[i + 1]), "=r"(a[i + 2]), "=r"(a[i + 3]), "=r"(a[i + 4]), "=r"(a[i + 5]), "=r"(a[i + 6]), "=r"(a[i + 7])
#define CAREKV_W8(a, i) "r"(a[i]), "r"(a[i + 1]), "r"(a[i + 2]), "r"(a[i + 3]), "r"(a[i + 4]), "r"(a[i + 5]), "r"(a[i + 6]), "r"(a[i + 7])

// 32 consecutive columns of the lane's TMEM row; the load has completed on return
// (the wait is part of the same statement, so no use can move before it).
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : CAREKV_R8(r, 0), CAREKV_R8(r, 8), CAREKV_R8(r, 16), CAREKV_R8(r, 24)
      : "r"(addr)
      : "memory");
}
// The same in two steps: the load starts, and tmem_landed waits for all loads
// of the thread; the registers pass through the wait, so no use of them can
// be moved before it.
__device__ __forceinline__ void tmem_ld32_start(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : CAREKV_R8(r, 0), CAREKV_R8(r, 8), CAREKV_R8(r, 16), CAREKV_R8(r, 24)
      : "r"(addr)
      : "memory");
}
#define CAREKV_P8(a, i) "+r"(a[i]), "+r"(a[i + 1]), "+r"(a[i + 2]), "+r"(a[i + 3]), "+r"(a[i + 4]), "+r"(a[i + 5]), "+r"(a[i + 6]), "+r"(a[i + 7])
__device__ __forceinline__ void tmem_landed(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : CAREKV_P8(r, 0), CAREKV_P8(r, 8), CAREKV_P8(r, 16), CAREKV_P8(r, 24)::"memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          addr),
      CAREKV_W8(r, 0), CAREKV_W8(r, 8)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      CAREKV_W8(r, 0), CAREKV_W8(r, 8), CAREKV_W8(r, 16), CAREKV_W8(r, 24)
      : "memory");
}

// ── descriptors ─────────────────────────────────────────────────────────
// Shared-memory operand in 128-byte swizzled atoms (8 rows of 128 bytes,
// 1024-byte aligned).  K-major: `stride` is the distance of 8-row groups
// (lead unused).  MN-major: `lead` is the distance of 64-element blocks along
// MN, `stride` that of 8-row groups along K.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead, uint32_t stride) {
  return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(lead >> 4) << 16) |
         (static_cast<uint64_t>(stride >> 4) << 32) | (uint64_t{1} << 46) | (uint64_t{2} << 61);
}
// kind::f16 instruction: fp32 accumulators, A and B both fp16 or both bf16,
// A K-major, B K-major or (mn_b) MN-major.
__host__ __device__ constexpr uint32_t mma_idesc(int m, int n, bool bf16, bool mn_b) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (mn_b ? 1u << 16 : 0u) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
// One lane of a converged warp, the same one every time (its products and
// commits are then ordered).
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t is;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(is));
  return is;
}
// The products are predicated on `lead` instead of standing in a branch of
// one lane: all operands but the predicate are the same in the whole warp,
// so they can stay in uniform registers, where the instruction wants them
// (a single lane's branch took 0.6 us to issue eight products).
// D (TMEM) = A (shared) . B (shared) [+ D]
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc, uint32_t lead) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %4, 0;\n setp.ne.u32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(acc)), "r"(lead)
      : "memory");
}
// D (TMEM) = A (TMEM, pairs of 16-bit values per column) . B (shared) [+ D]
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc, uint32_t lead) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %4, 0;\n setp.ne.u32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(acc)), "r"(lead)
      : "memory");
}
// One arrival on `bar` when every product the lead lane issued has completed.
__device__ __forceinline__ void mma_commit(uint64_t* bar, uint32_t lead) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.u32 q, %1, 0;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(smem_addr(bar)),
      "r"(lead)
      : "memory");
}

// ── tiled loads ─────────────────────────────────────────────────────────
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_addr(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
      : "memory");
}
// ... with an L2 eviction policy
__device__ __forceinline__ void tma_load_3d_pol(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar,
                                                uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], "
      "[%1, {%2, %3, %4}], [%5], %6;" ::"r"(smem_addr(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar)), "l"(policy)
      : "memory");
}
// A wait that gives up after about a second, or as soon as another wait of
// the CTA has (`dead`, in shared memory).
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
// Set by a CTA one of whose waits gave up; its results are NaN.  One per
// source file; the host takes it with take_wait_errors.
static __device__ int wait_errors;
__device__ __forceinline__ void report_wait(volatile int* dead) {   // once per CTA, after its last barrier
  if (threadIdx.x == 0 && *dead) atomicOr(&wait_errors, 1);
}
// Reads and clears the flag (synchronizes the stream).
static inline cudaError_t take_wait_errors(int32_t* set, cudaStream_t st) {
  void* p = nullptr;
  cudaError_t e = cudaGetSymbolAddress(&p, wait_errors);
  if (e == cudaSuccess) e = cudaMemcpyAsync(set, p, sizeof(int), cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && *set) e = cudaMemsetAsync(p, 0, sizeof(int), st);
  return e;
}
// two fp32 operations per instruction
__device__ __forceinline__ float2 fma2(float2 x, float2 y, float2 z) {
  float2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(*reinterpret_cast<uint64_t*>(&r))
      : "l"(*reinterpret_cast<uint64_t*>(&x)), "l"(*reinterpret_cast<uint64_t*>(&y)), "l"(*reinterpret_cast<uint64_t*>(&z)));
  return r;
}
__device__ __forceinline__ float2 add2(float2 x, float2 y) {
  float2 r;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(*reinterpret_cast<uint64_t*>(&r))
      : "l"(*reinterpret_cast<uint64_t*>(&x)), "l"(*reinterpret_cast<uint64_t*>(&y)));
  return r;
}
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_addr(dst)),
      "l"(map), "r"(x), "r"(y), "r"(smem_addr(bar))
      : "memory");
}
__device__ __forceinline__ void named_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

}  // namespace carekv
