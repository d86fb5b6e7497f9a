// Blackwell primitives shared by the tensor-core kernels: mbarriers with
// bounded waits, TMA loads, tcgen05 MMA / TMEM access, packed fp32 math, and
// the host's tensor-map encoder.
#pragma once

#include <cuda.h>

#include "common.cuh"

namespace h3 {

constexpr int kTileBytes = 128 * 128 * 2;   // one 128x128 bf16 tile
constexpr int kHalfBytes = kTileBytes / 2;  // one 128x64 swizzle box
constexpr uint64_t kWaitLimitNs = 4000000000ull;  // 4 s
constexpr uint64_t kDrainNs = 10000000ull;  // 10 ms, of a wait for the waiter's own copies (they take microseconds)

// ------------------------------------------------------------- primitives
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ uint64_t globaltimer() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}

// Bytes that never come: the barrier's phase does not complete (a test hook).
__device__ __forceinline__ void mbar_stall(uint32_t bar) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], 16;" ::"r"(bar) : "memory");
}

__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}

// Bounded wait; false on abort/timeout.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int32_t* abort_flag,
                                          int32_t* status, uint64_t limit_ns = kWaitLimitNs) {
  for (int i = 0; i < 64; ++i)
    if (mbar_try(bar, parity)) return true;
  const uint64_t t0 = globaltimer();
  while (true) {
    if (mbar_try(bar, parity)) return true;
    if (*abort_flag) return false;
    // another CTA's wait already gave up: stop instead of timing out again
    // (one status word per launch, so a systematic stall ends in one limit)
    if (status && *(volatile int32_t*)status != 0) {
      *abort_flag = 1;
      return false;
    }
    if (globaltimer() - t0 > limit_ns) {
      *abort_flag = 1;
      if (status) atomicExch(status, (int32_t)H3C_ERR_TIMEOUT);
      return false;
    }
  }
}

// The same for calls whose status word is only written, so that those beside
// or behind a failed one are not drawn in (a grid of at most a CTA an SM ends in
// one limit all the same).  PACED: from the 65th try on a try every 200 ns, as
// polls without a pause take issue slots from the warps that are waited for
// (dense rows against 16,384 keys, 4,096 x 40: 1,180 us; 1,325 without, 1,310
// and 1,370 with nanosleep and with the suspension that try_wait can be given).
// Folded rows wait for HBM or for few warps, and are faster without (32 members
// over 65,536 keys and 512 of their own: 102.5 us, 106.5 with).
template <bool PACED = true>
__device__ __forceinline__ bool mbar_wait_alone(uint32_t bar, uint32_t parity, volatile int32_t* abort_flag,
                                                int32_t* status, uint64_t limit_ns) {
  for (int i = 0; i < 64; ++i)
    if (mbar_try(bar, parity)) return true;
  const uint64_t t0 = globaltimer();
  while (true) {
    if (mbar_try(bar, parity)) return true;
    if (*abort_flag) return false;
    uint64_t now = globaltimer();
    if (now - t0 > limit_ns) {
      *abort_flag = 1;
      atomicExch(status, (int32_t)H3C_ERR_TIMEOUT);
      return false;
    }
    if constexpr (PACED) {
      const uint64_t next = now + 200;
      while (now < next) now = globaltimer();
    }
  }
}

// After an abort, behind every role's end: a copy that one role had just issued
// when another gave up lands before the block's shared memory is given back.
__device__ __forceinline__ void settle() {
  const uint64_t t0 = globaltimer();
  for (int i = 0; i < 100000 && globaltimer() - t0 < 1000000; ++i) __nanosleep(1000);
}

__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

// 3D tiled TMA load (no multicast): coordinates (d, token, head).
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1,
                                            int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], "
      "[%2];" ::"r"(dst),
      "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// MMA and commit are issued by a whole converged warp, one lane elected by
// elect.sync: the MMA warp runs its loop with all 32 lanes (no divergent
// single-lane branch around the issue), which measured 3% faster than a
// lane-0-only issuer (block-sparse at S = 124,992 and dense).
// D[tmem] (+)= A[smem desc] * B[smem desc]
__device__ __forceinline__ void mma_ss_w(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}

// D[tmem] (+)= A[tmem] * B[smem desc]
__device__ __forceinline__ void mma_ts_w(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}

__device__ __forceinline__ void tc_commit_w(uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
      : "memory");
}

#define H3_TMEM_LD16(addr, r)                                                                                 \
  asm volatile(                                                                                               \
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];" \
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),       \
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])  \
      : "r"(addr))

#define H3_TMEM_ST16(addr, r)                                                                                  \
  asm volatile(                                                                                                \
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" \
      ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),       \
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])              \
      : "memory")

__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// (x0, x1) = (s0, s1) * k + b on the packed f32x2 pipe; k, b hold a scalar
// in both halves.
__device__ __forceinline__ void fma2(float& x0, float& x1, uint32_t s0, uint32_t s1, uint64_t k, uint64_t b) {
  asm("{\n\t.reg .b64 a, d;\n\tmov.b64 a, {%2, %3};\n\t"
      "fma.rn.ftz.f32x2 d, a, %4, %5;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(x0), "=f"(x1)
      : "r"(s0), "r"(s1), "l"(k), "l"(b));
}

__device__ __forceinline__ uint64_t add2(uint64_t acc, float a, float b) {
  uint64_t r;
  asm("{\n\t.reg .b64 t;\n\tmov.b64 t, {%2, %3};\n\tadd.rn.ftz.f32x2 %0, %1, t;\n\t}"
      : "=l"(r)
      : "l"(acc), "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ uint64_t dup2(float v) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %1};" : "=l"(r) : "f"(v));
  return r;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// Shared-memory matrix descriptor, 128-byte swizzle (layout type 2),
// descriptor version 1; lbo/sbo in bytes.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  uint64_t d = 0;
  d |= (uint64_t)((addr >> 4) & 0x3FFF);
  d |= (uint64_t)((lbo >> 4) & 0x3FFF) << 16;
  d |= (uint64_t)((sbo >> 4) & 0x3FFF) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

// Instruction descriptor, kind::f16: bf16 x bf16 -> f32, M = 128, N = 128.
constexpr uint32_t idesc_bf16(bool b_mn_major) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((128u >> 3) << 17) |
         ((128u >> 4) << 24);
}

// The low word of a shared-memory matrix descriptor; the high word (128-byte
// swizzle, version 1, 1024 bytes between groups of eight rows) is the same for
// every tile here: 0x40004040.
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) {
  return ((addr >> 4) & 0x3FFF) | ((lbo >> 4) << 16);
}

// Products of 128 x 128 x 128 as one group, one lane elected for all of it and
// the descriptors stepped in 32 bits: a lean issuer, since one that spills to
// local memory (shared memory leaves next to no L1) reads it back from L2
// between products.
// D (+)= A B^T, both tiles K-major in shared memory (desc_lo(tile, 16)).
__device__ __forceinline__ void mma_tile_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, t, e;\n\t.reg .b32 ra, rb;\n\t.reg .b64 da, db;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.eq.u32 t, 0, 0;\n\t"
      "add.u32 ra, %1, 0;\n\t"
      "add.u32 rb, %2, 0;\n\t"
      "mov.b64 da, {ra, 0x40004040};\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t"
      "add.u32 ra, %1, 2;\n\t"
      "add.u32 rb, %2, 2;\n\t"
      "mov.b64 da, {ra, 0x40004040};\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, t;\n\t"
      "add.u32 ra, %1, 4;\n\t"
      "add.u32 rb, %2, 4;\n\t"
      "mov.b64 da, {ra, 0x40004040};\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, t;\n\t"
      "add.u32 ra, %1, 6;\n\t"
      "add.u32 rb, %2, 6;\n\t"
      "mov.b64 da, {ra, 0x40004040};\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, t;\n\t"
      "add.u32 ra, %1, 1024;\n\t"
      "add.u32 rb, %2, 1024;\n\t"
      "mov.b64 da, {ra, 0x40004040};\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, t;\n\t"
      "add.u32 ra, %1, 1026;\n\t"
      "add.u32 rb, %2, 1026;\n\t"
      "mov.b64 da, {ra, 0x40004040};\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, t;\n\t"
      "add.u32 ra, %1, 1028;\n\t"
      "add.u32 rb, %2, 1028;\n\t"
      "mov.b64 da, {ra, 0x40004040};\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, t;\n\t"
      "add.u32 ra, %1, 1030;\n\t"
      "add.u32 rb, %2, 1030;\n\t"
      "mov.b64 da, {ra, 0x40004040};\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, t;\n\t"
      "}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc)
      : "memory");
}

// D (+)= A B, A packed bf16 at 64 TMEM columns, B a tile with the summed axis
// along its rows (desc_lo(tile, kHalfBytes)).
__device__ __forceinline__ void mma_tile_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, t, e;\n\t.reg .b32 ra, rb;\n\t.reg .b64 db;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.eq.u32 t, 0, 0;\n\t"
      "add.u32 ra, %1, 0;\n\t"
      "add.u32 rb, %2, 0;\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [ra], db, %3, p;\n\t"
      "add.u32 ra, %1, 8;\n\t"
      "add.u32 rb, %2, 128;\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [ra], db, %3, t;\n\t"
      "add.u32 ra, %1, 16;\n\t"
      "add.u32 rb, %2, 256;\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [ra], db, %3, t;\n\t"
      "add.u32 ra, %1, 24;\n\t"
      "add.u32 rb, %2, 384;\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [ra], db, %3, t;\n\t"
      "add.u32 ra, %1, 32;\n\t"
      "add.u32 rb, %2, 512;\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [ra], db, %3, t;\n\t"
      "add.u32 ra, %1, 40;\n\t"
      "add.u32 rb, %2, 640;\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [ra], db, %3, t;\n\t"
      "add.u32 ra, %1, 48;\n\t"
      "add.u32 rb, %2, 768;\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [ra], db, %3, t;\n\t"
      "add.u32 ra, %1, 56;\n\t"
      "add.u32 rb, %2, 896;\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [ra], db, %3, t;\n\t"
      "}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc)
      : "memory");
}

// Steps 0-5 and 6-7 of mma_tile_ts (a and b as for all of it).
__device__ __forceinline__ void mma_tile_ts_0_6(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, t, e;\n\t.reg .b32 ra, rb;\n\t.reg .b64 db;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.eq.u32 t, 0, 0;\n\t"
      "add.u32 ra, %1, 0;\n\t"
      "add.u32 rb, %2, 0;\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [ra], db, %3, p;\n\t"
      "add.u32 ra, %1, 8;\n\t"
      "add.u32 rb, %2, 128;\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [ra], db, %3, t;\n\t"
      "add.u32 ra, %1, 16;\n\t"
      "add.u32 rb, %2, 256;\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [ra], db, %3, t;\n\t"
      "add.u32 ra, %1, 24;\n\t"
      "add.u32 rb, %2, 384;\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [ra], db, %3, t;\n\t"
      "add.u32 ra, %1, 32;\n\t"
      "add.u32 rb, %2, 512;\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [ra], db, %3, t;\n\t"
      "add.u32 ra, %1, 40;\n\t"
      "add.u32 rb, %2, 640;\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [ra], db, %3, t;\n\t"
      "}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc)
      : "memory");
}

__device__ __forceinline__ void mma_tile_ts_6_8(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, t, e;\n\t.reg .b32 ra, rb;\n\t.reg .b64 db;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.eq.u32 t, 0, 0;\n\t"
      "add.u32 ra, %1, 48;\n\t"
      "add.u32 rb, %2, 768;\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [ra], db, %3, p;\n\t"
      "add.u32 ra, %1, 56;\n\t"
      "add.u32 rb, %2, 896;\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [ra], db, %3, t;\n\t"
      "}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc)
      : "memory");
}

// Steps 0-3 and 4-7, for an A in two places (b as for all of it; a of the
// second is that of step 4).
__device__ __forceinline__ void mma_tile_ts_0_4(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, t, e;\n\t.reg .b32 ra, rb;\n\t.reg .b64 db;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.eq.u32 t, 0, 0;\n\t"
      "add.u32 ra, %1, 0;\n\t"
      "add.u32 rb, %2, 0;\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [ra], db, %3, p;\n\t"
      "add.u32 ra, %1, 8;\n\t"
      "add.u32 rb, %2, 128;\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [ra], db, %3, t;\n\t"
      "add.u32 ra, %1, 16;\n\t"
      "add.u32 rb, %2, 256;\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [ra], db, %3, t;\n\t"
      "add.u32 ra, %1, 24;\n\t"
      "add.u32 rb, %2, 384;\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [ra], db, %3, t;\n\t"
      "}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc)
      : "memory");
}

__device__ __forceinline__ void mma_tile_ts_4_8(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, t, e;\n\t.reg .b32 ra, rb;\n\t.reg .b64 db;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.eq.u32 t, 0, 0;\n\t"
      "add.u32 ra, %1, 0;\n\t"
      "add.u32 rb, %2, 512;\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [ra], db, %3, p;\n\t"
      "add.u32 ra, %1, 8;\n\t"
      "add.u32 rb, %2, 640;\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [ra], db, %3, t;\n\t"
      "add.u32 ra, %1, 16;\n\t"
      "add.u32 rb, %2, 768;\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [ra], db, %3, t;\n\t"
      "add.u32 ra, %1, 24;\n\t"
      "add.u32 rb, %2, 896;\n\t"
      "mov.b64 db, {rb, 0x40004040};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [ra], db, %3, t;\n\t"
      "}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc)
      : "memory");
}

// Four-dimensional form: coordinates (d, token, head, batch).
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2,
                                            int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
      "[%2];" ::"r"(dst),
      "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

// The same for what is read once: the first to leave L2, so that a long stream
// does not push out what is used again (the kernel's own code, for one).
__device__ __forceinline__ uint64_t evict_first() {
  uint64_t policy;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  return policy;
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2,
                                            int c3, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], "
      "[%1, {%3, %4, %5, %6}], [%2], %7;" ::"r"(dst),
      "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "l"(policy)
      : "memory");
}

// 4D tiled TMA store from shared memory, the end of a bulk group of this
// thread's stores, and the wait until at most N of its groups still read shared
// memory.
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(map),
               "r"(src), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}
__device__ __forceinline__ void tma_store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void tma_store_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}

// 16 bytes from global to shared memory, asynchronously.
__device__ __forceinline__ void copy16(uint32_t dst, const uint16_t* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// Zeros where not `in` (src is then only an address).
__device__ __forceinline__ void copy16_or_zero(uint32_t dst, const uint16_t* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// 32 bytes to global memory, a whole sector in one store; p needs 16-byte
// alignment only (rows are no further aligned), so it is two stores where p is
// not on a sector.
__device__ __forceinline__ void store32(uint16_t* p, const uint32_t* w) {
  if (!((uintptr_t)p & 31)) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else {
    reinterpret_cast<uint4*>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    reinterpret_cast<uint4*>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

// Brings a 4D box into L2.
__device__ __forceinline__ void tma_prefetch_4d(const CUtensorMap* map, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global.tile [%0, {%1, %2, %3, %4}];" ::"l"(map), "r"(c0), "r"(c1),
               "r"(c2), "r"(c3)
               : "memory");
}

// Columns [from, to) of the warp's lanes, to a multiple of 16; waits for it.
__device__ __forceinline__ void fill_columns(uint32_t addr, int from, int to, uint32_t value) {
  int c = from;
#pragma unroll 1
  for (; c & 15; ++c)
    asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(addr + c), "r"(value) : "memory");
#pragma unroll 1
  for (; c < to; c += 16)
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%1,%1,%1,%1,%1,%1,%1,%1,%1,%1,%1,%1,%1,%1,%1};" ::"r"(
                     addr + c),
                 "r"(value)
                 : "memory");
  tmem_wait_st();
}

// Orders this thread's shared-memory writes before later reads by TMA or MMA.
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// --------------------------------------------------------------- host side
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Looked up once per process (thread-safe static initialisation).
inline EncodeTiledFn get_encode() {
  static const EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      return (EncodeTiledFn)p;
    return (EncodeTiledFn) nullptr;
  }();
  return fn;
}

}  // namespace h3
