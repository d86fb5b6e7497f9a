// Gradient of cross attention on the Blackwell tensor cores.
//
//   P = 2^(scale log2(e) q.k - lse2);  delta_i = do_i.o_i;  dS = P (do v^T - delta)
//   dq = scale dS k;  dk = scale dS^T q;  dv = P^T do   (sums over the heads of a group)
//
// (delta_i = sum_j P_ij dP_ij / sum_j P_ij too, and is taken so of members with
// up to 128 keys).  delta_kernel goes over do and out once, unless kv_len <= 128; then
// two passes, so that every sum has one owner and a fixed order (no atomics):
//   dq_kernel    a CTA holds 128 queries and walks the keys: S, dP, dq += dS K
//   dkv_kernel   a CTA holds 128 keys and walks the queries of all heads of
//                the group: S^T, dP^T, dv += P^T do, dk += dS^T Q
// Seven products of 128x128x128 a tile pair instead of the five that a single
// pass with atomics on dq would make.  P and dS enter their products in bf16
// from TMEM (they never touch shared memory); sums are fp32.
//
// Roles of a CTA's 12 warps: 0 TMA producer, 1 MMA issuer, 2 TMEM owner (and
// a second issuer in dq_kernel), 4-7 and 8-11 elementwise: each warpgroup takes
// 64 of a tile's 128 columns of every row (thread = row = TMEM lane).  Every
// wait is bounded (attn_tc.cu; a CTA that gives up does so alone).
//
// dkv_kernel's work, all (key tile, query block) pairs in a row, is cut into
// equal runs, one a CTA; a key tile that is cut leaves fp32 partial sums that
// dkv_join_kernel adds in the order of the queries.
#include <climits>
#include <mutex>

#include "conditioning.cuh"

namespace h3 {
namespace {

constexpr int kThreads = 384;
constexpr int kSms = 148;
constexpr float kLog2e = 1.4426950408889634f;
constexpr uint32_t kIdKK = idesc_bf16(false), kIdKM = idesc_bf16(true);

struct BwdArgs {
  CrossShape n;
  Rows out, dout, dq, dk, dv;
  const int32_t* kv_lens;
  const float* lse;
  float scale;
  float* nl2;                 // [batch * heads, query blocks * 128]: -lse log2(e)
  float* delta;
  float* part;                // [ctas, 2 (head, tail), 2 (dk, dv), 128 * 128]
  int32_t q_blocks;
  int32_t* status;
  uint64_t wait_limit_ns;
  int32_t stall;              // test hook: barrier (from q_full, kv_full on) that never completes
  int32_t q_b, q_h, k_b, k_h, v_b, v_h, g_b, g_h;
  Div by_blocks, by_heads, by_group;
};

__device__ __forceinline__ uint64_t pair2(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}

// (s0, s1) * k + b, two fp32 at a time
__device__ __forceinline__ uint64_t fma_2(uint64_t a, uint64_t k, uint64_t b) {
  uint64_t r;
  asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(k), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add_2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.ftz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul_2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.ftz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float lo2(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi2(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }

// What dq and dk are scaled by.  The softmax over one key is 1 whatever its
// logit: what rounding left of dS there (a few rows in a million) is taken out.
__device__ __forceinline__ float ds_scale(const BwdArgs& a, int len) { return len == 1 ? 0.f : a.scale; }

__device__ __forceinline__ void tma_tile(uint32_t dst, const CUtensorMap* m, uint32_t bar, int tok, int h, int b) {
  tma_load_4d(dst, m, bar, 0, tok, h, b);
  tma_load_4d(dst + kHalfBytes, m, bar, 64, tok, h, b);
}

// 512 bytes of a float array into shared memory
__device__ __forceinline__ void bulk_512(uint32_t dst, const float* src, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], 512, [%2];" ::"r"(dst), "l"(src),
      "r"(bar)
      : "memory");
}

__device__ __forceinline__ void load64(uint32_t addr, uint32_t* v) {
#pragma unroll
  for (int c = 0; c < 4; ++c) H3_TMEM_LD16(addr + 16 * c, (&v[16 * c]));
  tmem_wait_ld();
}

enum { kFirst = 1, kLast = 2, kEnd = 4, kZeroShift = 8 };

__device__ __forceinline__ uint32_t alloc_tmem(int warp, uint32_t* slot) {
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(slot)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  return *slot;
}

// Common exit: no MMA may still write TMEM when it is released.
__device__ __forceinline__ void release_tmem(int warp, uint32_t tmem, volatile int32_t* abort_flag, uint64_t* done) {
  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    if (*abort_flag) {
      volatile int32_t zero = 0;
      mbar_wait(smem_u32(done), 0, &zero, nullptr);
      settle();
      __syncwarp();
    }
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// ------------------------------------------------------------------ delta
__device__ __forceinline__ float dot8(const uint4& x, const uint4& y) {
  const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s = fmaf(__uint_as_float(xw[i] << 16), __uint_as_float(yw[i] << 16), s);
    s = fmaf(__uint_as_float(xw[i] & 0xffff0000u), __uint_as_float(yw[i] & 0xffff0000u), s);
  }
  return s;
}

// delta = do.out and -lse log2(e) of every row, padded to whole blocks of
// queries (0 and -inf there, so that P is 0).  HBM-bound: 512 bytes a row.
// 16 lanes take a row; a CTA has 16 tokens of kHeads heads, a group its
// token's heads one after the other (neighbours in memory), all in flight.
// 1.3 million rows of 512 bytes: 109 us, 6.2 TB/s (8 heads a CTA, at half the
// occupancy: 134).
constexpr int kHeads = 4;

__global__ void __launch_bounds__(256) delta_kernel(const __grid_constant__ BwdArgs a) {
  asm volatile("griddepcontrol.launch_dependents;");
  const int c = threadIdx.x & 15, tok = blockIdx.x * 16 + (threadIdx.x >> 4);
  const bool live = tok < a.n.q_len;
  const int per_b = (a.n.heads + kHeads - 1) / kHeads;
  for (int y = blockIdx.y; y < per_b * a.n.batch; y += gridDim.y) {
    const int b = y / per_b, h0 = (y - b * per_b) * kHeads;
    uint4 o[kHeads], g[kHeads];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      o[i] = g[i] = make_uint4(0, 0, 0, 0);
      if (live && h0 + i < a.n.heads) {
        o[i] = __ldcs(reinterpret_cast<const uint4*>(a.out.at(b, tok, h0 + i)) + c);
        g[i] = *(reinterpret_cast<const uint4*>(a.dout.at(b, tok, h0 + i)) + c);
      }
    }
    const int64_t bh = (int64_t)b * a.n.heads + h0 + c;  // lane c < kHeads: its head's
    const bool mine = c < kHeads && h0 + c < a.n.heads;
    const float lse = mine && live ? a.lse[bh * a.n.q_len + tok] : INFINITY;
    float delta = 0.f;
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      float v = dot8(o[i], g[i]);
#pragma unroll
      for (int m = 8; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
      if (c == i) delta = v;
    }
    if (mine) {
      const int64_t pad = bh * a.q_blocks * 128 + tok;
      a.nl2[pad] = lse * -kLog2e;
      a.delta[pad] = delta;
    }
  }
}

// --------------------------------------------------------------------- dq
// Shared memory: q and do of the unit, three K and two V tiles (224 KB).
// TMEM columns: dq 0, S 128, dP 256, dS (two buffers) 384 and 448.  Of block
// e+1, S and dP run while block e is in the elementwise warps; dq of e
// follows, so a K tile is held for two blocks and needs the third buffer to
// be loaded ahead.  Four more warps (12-15) take dq out and write it, so that
// the elementwise warps only go from block to block.  Working delta out in here, by either kind of warp, took 5,000 to
// 12,000 cycles a unit of three to eight blocks of 2,200: code that runs once
// a unit waits for its instructions, constants and rows each time.  15,731 x
// 56 rows and 332 keys: 265-285 us; 2 x 16,384 x 40 and 1,024 ragged keys:
// 705, 2,200 cycles a block (its products 1,536, the exponentials of a tile
// 1,024 of the MUFU units between two TMEM round trips).
struct __align__(16) DqBarriers {
  float nl2[2][128], delta[2][128];  // by unit parity
  float weights[128];                // half 1's share of a row's sum of P
  uint64_t q_full, q_empty, g_full, g_empty;
  uint64_t k_full[3], k_empty[3], v_full[2], v_empty[2];
  uint64_t n_full[2];                // -lse2 and delta of unit u on [u & 1]
  uint64_t s_full, s_empty, dp_full, dp_empty, dq_full, dq_empty, sum_full[2], done;
  // block e on [e & 1]: S and dP of e + 1 are issued before the issuer waits
  // for dS of e, so one barrier could complete twice before that wait
  uint64_t ds_full[2];
  uint32_t tmem_base;
  int32_t abort;
  int32_t info[8];
  int32_t lens[kLens];
};
constexpr int kDqThreads = 512;
constexpr int kDqTiles = 7 * kTileBytes;
constexpr int kDqSmem = kDqTiles + (int)sizeof(DqBarriers);
static_assert(kDqSmem <= 227 * 1024, "shared memory");

struct DqUnit {
  int b, h, t0, len, n;
  __device__ DqUnit(const BwdArgs& a, const int32_t* lens, int u) {
    const int x = a.by_blocks(u);
    t0 = (u - x * a.q_blocks) * 128;
    b = a.by_heads(x);
    h = x - b * a.n.heads;
    len = b < kLens ? lens[b] : kv_len_of(a.kv_lens, a.n.kv_len, b);
    n = (len + 127) >> 7;
  }
};

// ONE: no member has more than one block of keys.  delta_kernel is then not
// needed: -lse2 is taken from lse (the next unit's a unit ahead) and left for
// dkv_kernel together with delta.  Forward and gradient of 15,731 x 56 rows
// and 77 keys: 451 us; 479 with masks of registers, and 80 more with
// delta_kernel before it.
template <bool ONE>
__global__ void __launch_bounds__(kDqThreads, 1)
    dq_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
              const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_g,
              const __grid_constant__ BwdArgs a, int units) {
  extern __shared__ __align__(1024) uint8_t smem[];
  if (!tiles_aligned(smem, a.status)) return;
  uint8_t *sQ = smem, *sG = smem + kTileBytes, *sK = smem + 2 * kTileBytes, *sV = smem + 5 * kTileBytes;
  DqBarriers* bars = (DqBarriers*)(smem + kDqTiles);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int32_t* abort_flag = &bars->abort;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 3; ++i) {
      mbar_init(smem_u32(&bars->k_full[i]), 1);
      mbar_init(smem_u32(&bars->k_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bars->v_full[i]), 1);
      mbar_init(smem_u32(&bars->v_empty[i]), 1);
      mbar_init(smem_u32(&bars->ds_full[i]), 256);
      mbar_init(smem_u32(&bars->n_full[i]), 1);
      mbar_init(smem_u32(&bars->sum_full[i]), 128);
    }
    mbar_init(smem_u32(&bars->q_full), 1);
    mbar_init(smem_u32(&bars->q_empty), 1);
    mbar_init(smem_u32(&bars->g_full), 1);
    mbar_init(smem_u32(&bars->g_empty), 1);
    mbar_init(smem_u32(&bars->s_full), 1);
    mbar_init(smem_u32(&bars->s_empty), 256);
    mbar_init(smem_u32(&bars->dp_full), 1);
    mbar_init(smem_u32(&bars->dp_empty), 256);
    mbar_init(smem_u32(&bars->dq_full), 1);
    mbar_init(smem_u32(&bars->dq_empty), 128);
    mbar_init(smem_u32(&bars->done), 2);
    if (a.stall >= 0 && &bars->q_full + a.stall <= &bars->ds_full[1]) mbar_stall(smem_u32(&bars->q_full + a.stall));
    bars->abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x >= 128 && threadIdx.x < 128 + kLens && threadIdx.x - 128 < a.n.batch)
    bars->lens[threadIdx.x - 128] = kv_len_of(a.kv_lens, a.n.kv_len, threadIdx.x - 128);
  const uint32_t tmem = alloc_tmem(warp, &bars->tmem_base);
  asm volatile("griddepcontrol.launch_dependents;");
  // placed while the kernel before runs; nothing is read or written before its end
  asm volatile("griddepcontrol.wait;" ::: "memory");
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    return mbar_wait_alone(smem_u32(bar), parity, abort_flag, a.status, a.wait_limit_ns);
  };
  // Register split of the launch's 512 x 128: 128 x 48 + 256 x 176 + 128 x 112.
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    if (warp == 0 && lane == 0) {
      // in the order in which the buffers free.  q and do have one each, so
      // what is not hidden of their latency is paid every unit: those of the
      // next unit are brought into L2 meanwhile (4,000 cycles from HBM under
      // load, 1,200 from there).
      int e = 0, qn = 0, nv = 0, ng = 0;  // K tiles, q tiles, V tiles, do tiles loaded
      int kr = 0;
      uint32_t kp = 0;
      bool ok = true;
      for (int u = blockIdx.x; ok && u < units; u += gridDim.x) {
        const DqUnit x(a, bars->lens, u);
        if (x.n == 0) continue;
        const int hk = a.by_group(x.h);
        if (!(ok = wait(&bars->q_empty, (qn & 1) ^ 1))) break;
        uint32_t bar = smem_u32(&bars->q_full);
        mbar_expect_tx(bar, kTileBytes);
        tma_tile(smem_u32(sQ), &tm_q, bar, x.t0, x.h * a.q_h, x.b * a.q_b);
        ++qn;
        if (u + (int)gridDim.x < units) {
          const DqUnit y(a, bars->lens, u + gridDim.x);
#pragma unroll
          for (int c = 0; c < 128; c += 64) {
            tma_prefetch_4d(&tm_q, c, y.t0, y.h * a.q_h, y.b * a.q_b);
            tma_prefetch_4d(&tm_g, c, y.t0, y.h * a.g_h, y.b * a.g_b);
          }
        }
        for (int j = 0; j < x.n; ++j) {
          if (!(ok = wait(&bars->k_empty[kr], kp ^ 1))) break;
          const int valid = x.len - 128 * j;
          // key rows past the member's length hold whatever the caller left
          // there: the issuer clears them (0 x NaN would reach dq)
          bars->info[e & 7] = (j == 0 ? kFirst : 0) | (j == x.n - 1 ? kLast : 0) |
                              (valid < 128 && x.len < a.n.kv_len ? valid << kZeroShift : 0);
          bar = smem_u32(&bars->k_full[kr]);
          mbar_expect_tx(bar, kTileBytes);
          tma_tile(smem_u32(sK + kr * kTileBytes), &tm_k, bar, 128 * j, hk * a.k_h, x.b * a.k_b);
          ++e;
          if (++kr == 3) {
            kr = 0;
            kp ^= 1;
          }
          if (!(ok = wait(&bars->v_empty[nv & 1], ((nv >> 1) & 1) ^ 1))) break;
          bar = smem_u32(&bars->v_full[nv & 1]);
          mbar_expect_tx(bar, kTileBytes);
          tma_tile(smem_u32(sV + (nv & 1) * kTileBytes), &tm_v, bar, 128 * j, hk * a.v_h, x.b * a.v_b);
          ++nv;
          if (j == 0) {
            // (g_empty: dP of the last unit, whose last block follows on the
            // elementwise warps' reading -lse2 and delta of the unit before)
            if (!(ok = wait(&bars->g_empty, (ng & 1) ^ 1))) break;
            bar = smem_u32(&bars->g_full);
            mbar_expect_tx(bar, kTileBytes);
            tma_tile(smem_u32(sG), &tm_g, bar, x.t0, x.h * a.g_h, x.b * a.g_b);
            if constexpr (!ONE) {
              bar = smem_u32(&bars->n_full[ng & 1]);
              mbar_expect_tx(bar, 1024);
              const int64_t pad = ((int64_t)x.b * a.n.heads + x.h) * a.q_blocks * 128 + x.t0;
              bulk_512(smem_u32(bars->nl2[ng & 1]), a.nl2 + pad, bar);
              bulk_512(smem_u32(bars->delta[ng & 1]), a.delta + pad, bar);
            }
            ++ng;
          }
        }
      }
      if (ok && wait(&bars->k_empty[kr], kp ^ 1) && wait(&bars->v_empty[nv & 1], ((nv >> 1) & 1) ^ 1)) {
        bars->info[e & 7] = kEnd;
        mbar_arrive(smem_u32(&bars->k_full[kr]));
        mbar_arrive(smem_u32(&bars->v_full[nv & 1]));
      } else {  // abort: every load in flight lands before anyone may exit
        volatile int32_t zero = 0;
        for (int x = max(0, e - 3); x < e; ++x)
          mbar_wait(smem_u32(&bars->k_full[x % 3]), (x / 3) & 1, &zero, nullptr, kDrainNs);
        for (int x = max(0, nv - 2); x < nv; ++x)
          mbar_wait(smem_u32(&bars->v_full[x & 1]), (x >> 1) & 1, &zero, nullptr, kDrainNs);
        if (qn) mbar_wait(smem_u32(&bars->q_full), (qn - 1) & 1, &zero, nullptr, kDrainNs);
        if (ng) mbar_wait(smem_u32(&bars->g_full), (ng - 1) & 1, &zero, nullptr, kDrainNs);
        for (int x = ONE ? ng : max(0, ng - 2); x < ng; ++x)
          mbar_wait(smem_u32(&bars->n_full[x & 1]), (x >> 1) & 1, &zero, nullptr, kDrainNs);
      }
    } else if (warp == 1 || warp == 2) {
      // Two issuers, one of S and one of dP and dq, so that the waits of one
      // (100-200 cycles each) pass while the products of the other run.
      auto iwait = [&](uint64_t* bar, uint32_t par) -> bool {
        int got = 0;
        if (lane == 0) got = wait(bar, par) ? 1 : 0;
        return __shfl_sync(0xffffffff, got, 0) != 0;
      };
      int e = 0, un = 0, kr = 0;
      if (warp == 1) {
        uint32_t kp = 0;
        while (iwait(&bars->k_full[kr], kp)) {
          tc_fence_after();
          const int info = ((volatile int32_t*)bars->info)[e & 7];
          if (info & kEnd) break;
          if (info >> kZeroShift) {
            uint4* k = reinterpret_cast<uint4*>(sK + kr * kTileBytes);
            for (int x = (info >> kZeroShift) * 8 + lane; x < 1024; x += 32) k[x] = k[1024 + x] = make_uint4(0, 0, 0, 0);
            fence_async_shared();
            __syncwarp();
          }
          if (info & kFirst) {
            if (!iwait(&bars->q_full, un & 1)) break;
            ++un;
          }
          if (e > 0 && !iwait(&bars->s_empty, (e - 1) & 1)) break;
          tc_fence_after();
          mma_tile_ss(tmem + 128, desc_lo(smem_u32(sQ), 16), desc_lo(smem_u32(sK + kr * kTileBytes), 16), kIdKK, 0);
          tc_commit_w(smem_u32(&bars->s_full));
          if (info & kLast) tc_commit_w(smem_u32(&bars->q_empty));
          ++e;
          if (++kr == 3) {
            kr = 0;
            kp ^= 1;
          }
        }
      } else {
        int dn = 0, pk = 0;
        auto issue_dq = [&](int p, int info, int k) -> bool {  // dq += dS_p K_p
          if (info & kFirst) {
            if (dn > 0 && !iwait(&bars->dq_empty, (dn - 1) & 1)) return false;
            ++dn;
          }
          if (!iwait(&bars->ds_full[p & 1], (p >> 1) & 1)) return false;
          tc_fence_after();
          const uint32_t ds = tmem + 384 + 64 * (p & 1);
          mma_tile_ts(tmem, ds, desc_lo(smem_u32(sK + k * kTileBytes), kHalfBytes), kIdKM, !(info & kFirst));
          tc_commit_w(smem_u32(&bars->k_empty[k]));
          if (info & kLast) tc_commit_w(smem_u32(&bars->dq_full));
          return true;
        };
        int pinfo = kLast;  // no product of the block before is due
        while (iwait(&bars->v_full[e & 1], (e >> 1) & 1)) {
          const int info = ((volatile int32_t*)bars->info)[e & 7];
          if (info & kEnd) break;
          if (info & kFirst) {
            if (!iwait(&bars->g_full, un & 1)) break;
            ++un;
          }
          if (e > 0 && !iwait(&bars->dp_empty, (e - 1) & 1)) break;
          tc_fence_after();
          mma_tile_ss(tmem + 256, desc_lo(smem_u32(sG), 16), desc_lo(smem_u32(sV + (e & 1) * kTileBytes), 16), kIdKK, 0);
          tc_commit_w(smem_u32(&bars->dp_full));
          tc_commit_w(smem_u32(&bars->v_empty[e & 1]));
          if (info & kLast) tc_commit_w(smem_u32(&bars->g_empty));
          // dq of the block before; of a unit's last block at once, as the next
          // dP waits for the next unit's do
          if (!(pinfo & kLast) && !issue_dq(e - 1, pinfo, pk)) break;
          if ((info & kLast) && !issue_dq(e, info, kr)) break;
          pinfo = info;
          pk = kr;
          ++e;
          if (++kr == 3) kr = 0;
        }
      }
      tc_commit_w(smem_u32(&bars->done));
    }
  } else if (warp < 12) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
    // one outcome a warp: the TMEM accesses need its lanes together
    auto wait_w = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
    const int w = (warp - 4) >> 2, q = warp & 3, r = 32 * q + lane;
    const uint32_t lane_base = tmem + ((uint32_t)(32 * q) << 16);
    const uint64_t sl2 = dup2(a.scale * kLog2e);
    int e = 0, un = 0, n1 = 0;  // blocks, units, units of one block
    bool ok = true;
    auto row_of = [&](const DqUnit& x) { return ((int64_t)x.b * a.n.heads + x.h) * a.q_blocks * 128 + x.t0 + r; };
    auto lse_of = [&](int u) {  // rows past the queries: P is 0
      if (u >= units) return 0.f;
      const DqUnit x(a, bars->lens, u);
      return x.t0 + r < a.n.q_len ? a.lse[((int64_t)x.b * a.n.heads + x.h) * a.n.q_len + x.t0 + r] : INFINITY;
    };
    [[maybe_unused]] float ahead = 0.f;
    if constexpr (ONE) ahead = lse_of(blockIdx.x);
    for (int u = blockIdx.x; ok && u < units; u += gridDim.x) {
      const DqUnit x(a, bars->lens, u);
      float nl2;
      if constexpr (ONE) {
        nl2 = ahead * -kLog2e;
        ahead = lse_of(u + gridDim.x);
      }
      if (x.n == 0) continue;
      uint64_t ndelta = 0;
      if constexpr (!ONE) {
        if (!(ok = wait_w(&bars->n_full[un & 1], (un >> 1) & 1))) break;
        nl2 = bars->nl2[un & 1][r];
        if (x.n > 1) ndelta = dup2(-bars->delta[un & 1][r]);
      }
      const uint64_t nl2x2 = dup2(nl2);
      ++un;
      for (int j = 0; j < x.n; ++j, ++e) {
        if (!(ok = wait_w(&bars->s_full, e & 1))) break;
        tc_fence_after();
        const int valid = x.len - 128 * j - 64 * w;  // this half's
        // (ONE: keys past the length weigh 0, in TMEM: each unit comes to the
        // mask, and masks of registers are four times the code; where units have
        // more blocks either takes the same time)
        if (ONE && valid < 64) fill_columns(lane_base + 128 + 64 * w, max(valid, 0), 64, __float_as_uint(-INFINITY));
        uint32_t s[64];
        load64(lane_base + 128 + 64 * w, s);
        tc_fence_before();
        mbar_arrive(smem_u32(&bars->s_empty));
        float p[64];
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const uint64_t v = fma_2(pair2(s[2 * c], s[2 * c + 1]), sl2, nl2x2);
          p[2 * c] = ex2(lo2(v));
          p[2 * c + 1] = ex2(hi2(v));
        }
        if (!(ok = wait_w(&bars->dp_full, e & 1))) break;
        tc_fence_after();
        if (ONE && valid < 64) fill_columns(lane_base + 256 + 64 * w, max(valid, 0), 64, 0u);
        uint32_t d[64];
        load64(lane_base + 256 + 64 * w, d);
        if (ONE || x.n == 1) {
          // All keys are here, so delta is sum(P dP) / sum(P) in fp32 and not
          // do.out: the rounding of out shows in dS where keys are few, and
          // that of lse in a weight near 1.  Half 1 hands its sum of P dP over
          // in the place of delta, half 0 delta in that of -lse2, which both
          // have read; the places are the unit's until dp_empty.
          float own = 0.f, ps = 0.f;
#pragma unroll
          for (int c = 0; c < 64; ++c)
            if (ONE || c < valid) {
              own = fmaf(p[c], __uint_as_float(d[c]), own);
              ps += p[c];
            }
          float *other = &bars->delta[(un - 1) & 1][r], *all = &bars->nl2[(un - 1) & 1][r];
          if (w == 1) {
            *other = own;
            bars->weights[r] = ps;
            fence_async_shared();
            mbar_arrive(smem_u32(&bars->sum_full[1]));
            if (!(ok = wait_w(&bars->sum_full[0], n1 & 1))) break;
            own = *all;
          } else {
            if (!(ok = wait_w(&bars->sum_full[1], n1 & 1))) break;
            ps += bars->weights[r];
            own = ps > 0.f ? (own + *other) / ps : 0.f;
            *all = own;
            fence_async_shared();
            mbar_arrive(smem_u32(&bars->sum_full[0]));
            a.delta[row_of(x)] = own;  // for dkv_kernel
            if (ONE) a.nl2[row_of(x)] = nl2;
          }
          ++n1;
          ndelta = dup2(-own);
        }
        tc_fence_before();
        mbar_arrive(smem_u32(&bars->dp_empty));
        uint32_t pk[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const uint64_t v = mul_2(add_2(pair2(d[2 * c], d[2 * c + 1]), ndelta),
                                   pair2(__float_as_uint(p[2 * c]), __float_as_uint(p[2 * c + 1])));
          pk[c] = pack_bf16(lo2(v), hi2(v));
        }
        if (!ONE && valid < 64) {  // keys past the length, whatever their values gave
#pragma unroll
          for (int c = 0; c < 32; ++c) pk[c] = 2 * c + 1 < valid ? pk[c] : 2 * c < valid ? pk[c] & 0xffffu : 0u;
        }
        const uint32_t ds = lane_base + 384 + 64 * (e & 1) + 32 * w;
        H3_TMEM_ST16(ds, (&pk[0]));
        H3_TMEM_ST16(ds + 16, (&pk[16]));
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(smem_u32(&bars->ds_full[e & 1]));
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 112;");
    auto wait_w = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
    const int q = warp & 3;
    int un = 0;
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
      const DqUnit x(a, bars->lens, u);
      const int t = x.t0 + 32 * q + lane;
      uint16_t* go = a.dq.at(x.b, t, x.h);
      // all of dq comes out before anything else is done with it: the next
      // unit's first product into it waits, and behind that product its dP
      // (out by halves: 348 us at 15,731 x 56 rows and 332 keys against 280)
      uint32_t k[64];
      if (x.n > 0) {
        if (!wait_w(&bars->dq_full, un & 1)) break;
        ++un;
        tc_fence_after();
        const float f = ds_scale(a, x.len);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t v[32];
          H3_TMEM_LD16(tmem + ((uint32_t)(32 * q) << 16) + 32 * c, (&v[0]));
          H3_TMEM_LD16(tmem + ((uint32_t)(32 * q) << 16) + 32 * c + 16, (&v[16]));
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i)
            k[16 * c + i] = pack_bf16(__uint_as_float(v[2 * i]) * f, __uint_as_float(v[2 * i + 1]) * f);
        }
        tc_fence_before();
        mbar_arrive(smem_u32(&bars->dq_empty));
      } else {
#pragma unroll
        for (int i = 0; i < 64; ++i) k[i] = 0u;
      }
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (t < a.n.q_len) store32(go + 16 * c, &k[8 * c]);
    }
  }
  release_tmem(warp, tmem, abort_flag, &bars->done);
}

// ------------------------------------------------------------------ dk, dv
// Shared memory: K and V of the unit, three q and two do tiles (224 KB), -lse2
// and delta of two query blocks.  TMEM columns: dk 0, dv 128, S^T 256, dP^T
// 384; a warpgroup writes its half of P^T (dS^T) over its own half of S^T
// (dP^T), so neither waits for the other's loads.  A q tile is held from S(e)
// to dk(e), over one block's time and a half, so it needs the third buffer to
// be loaded ahead.  15,731 x 56 rows and 332 keys: 292 us, 3,500 cycles a
// block, 2,048 of them in its four products (58% of the tensor pipe's time).
struct __align__(16) DkvBarriers {
  float nl2[2][128], delta[2][128];
  uint64_t kv_full, kv_empty;
  uint64_t q_full[3], q_empty[3], g_full[2], g_empty[2];
  uint64_t s_full, dp_full, p_full, ds_full, acc_full, acc_empty, done;
  uint32_t tmem_base;
  int32_t abort;
  int32_t info[8];
};
constexpr int kDkvTiles = 7 * kTileBytes;
constexpr int kDkvSmem = kDkvTiles + (int)sizeof(DkvBarriers);
static_assert(kDkvSmem <= 227 * 1024, "shared memory");

// The run of (key tile, query block) pairs of one CTA, over key tiles that
// hold valid keys: tile order member, key head, tile.
struct DkvWalk {
  int64_t pos, end;
  int b, len, tiles;          // current member
  int64_t base;               // its first position
  int steps;                  // query blocks of a key tile: those of all heads of the group
  // current segment
  int hk, tile, it0, it1;
  __device__ DkvWalk(const BwdArgs& a, int cta, int ctas) {
    steps = a.n.group * a.q_blocks;
    int64_t all = 0;
    for (int i = 0; i < a.n.batch; ++i) all += (kv_len_of(a.kv_lens, a.n.kv_len, i) + 127) >> 7;
    all *= (int64_t)a.n.kv_heads * steps;
    const int64_t share = (all + ctas - 1) / ctas;
    pos = min(all, share * cta);
    end = min(all, pos + share);
    b = -1;
    base = 0;
    len = tiles = 0;
  }
  __device__ bool next(const BwdArgs& a) {
    if (pos >= end) return false;
    while (b < 0 || pos >= base + (int64_t)tiles * a.n.kv_heads * steps) {
      if (b >= 0) base += (int64_t)tiles * a.n.kv_heads * steps;
      ++b;
      len = kv_len_of(a.kv_lens, a.n.kv_len, b);
      tiles = (len + 127) >> 7;
    }
    const int64_t off = pos - base;
    const int u = (int)(off / steps);
    hk = u / tiles;
    tile = u - hk * tiles;
    it0 = (int)(off - (int64_t)u * steps);
    it1 = (int)min((int64_t)steps, it0 + (end - pos));
    pos += it1 - it0;
    return true;
  }
};

__global__ void __launch_bounds__(kThreads, 1)
    dkv_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
               const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_g,
               const __grid_constant__ BwdArgs a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  if (!tiles_aligned(smem, a.status)) return;
  uint8_t *sK = smem, *sV = smem + kTileBytes, *sQ = smem + 2 * kTileBytes, *sG = smem + 5 * kTileBytes;
  DkvBarriers* bars = (DkvBarriers*)(smem + kDkvTiles);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int32_t* abort_flag = &bars->abort;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 3; ++i) {
      mbar_init(smem_u32(&bars->q_full[i]), 1);
      mbar_init(smem_u32(&bars->q_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bars->g_full[i]), 1);
      mbar_init(smem_u32(&bars->g_empty[i]), 1);
    }
    mbar_init(smem_u32(&bars->kv_full), 1);
    mbar_init(smem_u32(&bars->kv_empty), 1);
    mbar_init(smem_u32(&bars->s_full), 1);
    mbar_init(smem_u32(&bars->dp_full), 1);
    mbar_init(smem_u32(&bars->p_full), 256);
    mbar_init(smem_u32(&bars->ds_full), 256);
    mbar_init(smem_u32(&bars->acc_full), 1);
    mbar_init(smem_u32(&bars->acc_empty), 256);
    mbar_init(smem_u32(&bars->done), 1);
    if (a.stall >= 0 && &bars->kv_full + a.stall <= &bars->done) mbar_stall(smem_u32(&bars->kv_full + a.stall));
    bars->abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  const uint32_t tmem = alloc_tmem(warp, &bars->tmem_base);
  asm volatile("griddepcontrol.launch_dependents;");
  // Placed while the kernel before runs.  What that one writes (-lse2, delta)
  // is read, and anything written, after its end: the producer waits for it
  // behind the first loads of inputs, the others here (38.6 us for 41.3 in a
  // step of 3 x 257 x 8 rows; the same in dq_kernel cost the clip 2%).
  if (warp >= 2) asm volatile("griddepcontrol.wait;" ::: "memory");
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    return mbar_wait_alone(smem_u32(bar), parity, abort_flag, a.status, a.wait_limit_ns);
  };
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 0 && lane == 0) {
      DkvWalk seg(a, blockIdx.x, gridDim.x);
      int e = 0, ng = 0, sn = 0, qr = 0;  // q tiles, do tiles and segments loaded
      uint32_t qp = 0;
      bool ok = true;
      while (ok && seg.next(a)) {
        if (!(ok = wait(&bars->kv_empty, (sn & 1) ^ 1))) break;
        uint32_t bar = smem_u32(&bars->kv_full);
        mbar_expect_tx(bar, 2 * kTileBytes);
        tma_tile(smem_u32(sK), &tm_k, bar, 128 * seg.tile, seg.hk * a.k_h, seg.b * a.k_b);
        tma_tile(smem_u32(sV), &tm_v, bar, 128 * seg.tile, seg.hk * a.v_h, seg.b * a.v_b);
        ++sn;
        int g = seg.it0 / a.q_blocks, qb = seg.it0 - g * a.q_blocks;
        for (int it = seg.it0; it < seg.it1; ++it) {
          const int h = seg.hk * a.n.group + g;
          if (!(ok = wait(&bars->q_empty[qr], qp ^ 1))) break;
          bars->info[e & 7] = (it == seg.it0 ? kFirst : 0) | (it == seg.it1 - 1 ? kLast : 0);
          bar = smem_u32(&bars->q_full[qr]);
          mbar_expect_tx(bar, kTileBytes);
          tma_tile(smem_u32(sQ + qr * kTileBytes), &tm_q, bar, 128 * qb, h * a.q_h, seg.b * a.q_b);
          ++e;
          if (++qr == 3) {
            qr = 0;
            qp ^= 1;
          }
          const int i = ng & 1;
          if (!(ok = wait(&bars->g_empty[i], ((ng >> 1) & 1) ^ 1))) break;
          bar = smem_u32(&bars->g_full[i]);
          mbar_expect_tx(bar, kTileBytes + 1024);
          tma_tile(smem_u32(sG + i * kTileBytes), &tm_g, bar, 128 * qb, h * a.g_h, seg.b * a.g_b);
          const int64_t pad = (((int64_t)seg.b * a.n.heads + h) * a.q_blocks + qb) * 128;
          if (ng == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
          bulk_512(smem_u32(bars->nl2[i]), a.nl2 + pad, bar);
          bulk_512(smem_u32(bars->delta[i]), a.delta + pad, bar);
          ++ng;
          if (++qb == a.q_blocks) {
            qb = 0;
            ++g;
          }
        }
      }
      if (ok && wait(&bars->q_empty[qr], qp ^ 1)) {
        bars->info[e & 7] = kEnd;
        mbar_arrive(smem_u32(&bars->q_full[qr]));
      } else {  // abort: every load in flight lands before anyone may exit
        volatile int32_t zero = 0;
        for (int x = max(0, e - 3); x < e; ++x)
          mbar_wait(smem_u32(&bars->q_full[x % 3]), (x / 3) & 1, &zero, nullptr, kDrainNs);
        for (int x = max(0, ng - 2); x < ng; ++x)
          mbar_wait(smem_u32(&bars->g_full[x & 1]), (x >> 1) & 1, &zero, nullptr, kDrainNs);
        if (sn) mbar_wait(smem_u32(&bars->kv_full), (sn - 1) & 1, &zero, nullptr, kDrainNs);
      }
    } else if (warp == 1) {
      // dv(e-1) S(e) dk(e-1) dP(e): the order keeps P^T (dS^T) in place until
      // its product has read it.  The elementwise warps wait for dv(e-1) and
      // S(e) in turn, 1,300 of a block's 3,500 cycles, yet what was tried
      // against that is slower: P^T through shared memory with S a block ahead
      // leaves q two buffers (397 us against 292 at 15,731 x 56 rows and 332
      // keys), a product of N = 64 for either warpgroup reads K and V twice
      // (341), and a second issuer for dk and dP takes 7% more.
      auto iwait = [&](uint64_t* bar, uint32_t par) -> bool {
        int got = 0;
        if (lane == 0) got = wait(bar, par) ? 1 : 0;
        return __shfl_sync(0xffffffff, got, 0) != 0;
      };
      int e = 0, pinfo = 0, segs = 0, accs = 0, qr = 0, pq = 0;
      uint32_t qp = 0;
      bool ok = true;
      auto issue_dv = [&](int p) -> bool {  // dv += P^T do
        if (pinfo & kFirst) {  // the epilogue of the last segment has read dk and dv
          if (accs > 0 && !iwait(&bars->acc_empty, (accs - 1) & 1)) return false;
          ++accs;
        }
        if (!iwait(&bars->p_full, p & 1)) return false;
        tc_fence_after();
        const uint32_t g = desc_lo(smem_u32(sG + (p & 1) * kTileBytes), kHalfBytes);
        mma_tile_ts_0_4(tmem + 128, tmem + 256, g, kIdKM, !(pinfo & kFirst));
        mma_tile_ts_4_8(tmem + 128, tmem + 320, g, kIdKM, 1);
        return true;
      };
      auto issue_dk = [&](int p) -> bool {  // dk += dS^T q
        if (!iwait(&bars->ds_full, p & 1)) return false;
        tc_fence_after();
        const uint32_t x = desc_lo(smem_u32(sQ + pq * kTileBytes), kHalfBytes);
        mma_tile_ts_0_4(tmem, tmem + 384, x, kIdKM, !(pinfo & kFirst));
        mma_tile_ts_4_8(tmem, tmem + 448, x, kIdKM, 1);
        tc_commit_w(smem_u32(&bars->q_empty[pq]));
        // do, and -lse2 and delta, which the elementwise warps have read
        // before they handed dS over
        tc_commit_w(smem_u32(&bars->g_empty[p & 1]));
        if (pinfo & kLast) tc_commit_w(smem_u32(&bars->acc_full));
        return true;
      };
      while (true) {
        ok = (e == 0 || issue_dv(e - 1)) && iwait(&bars->q_full[qr], qp);
        if (!ok) break;
        const int info = ((volatile int32_t*)bars->info)[e & 7];
        if (info & kEnd) break;
        if (info & kFirst) {
          if (!(ok = iwait(&bars->kv_full, segs & 1))) break;
          ++segs;
        }
        tc_fence_after();
        mma_tile_ss(tmem + 256, desc_lo(smem_u32(sK), 16), desc_lo(smem_u32(sQ + qr * kTileBytes), 16), kIdKK, 0);
        tc_commit_w(smem_u32(&bars->s_full));
        ok = (e == 0 || issue_dk(e - 1)) && iwait(&bars->g_full[e & 1], (e >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        mma_tile_ss(tmem + 384, desc_lo(smem_u32(sV), 16), desc_lo(smem_u32(sG + (e & 1) * kTileBytes), 16), kIdKK, 0);
        tc_commit_w(smem_u32(&bars->dp_full));
        if (info & kLast) tc_commit_w(smem_u32(&bars->kv_empty));
        pinfo = info;
        pq = qr;
        ++e;
        if (++qr == 3) {
          qr = 0;
          qp ^= 1;
        }
      }
      if (ok && e > 0) issue_dk(e - 1);
      tc_commit_w(smem_u32(&bars->done));
    } else if (warp >= 2) {
      // gradients of key tiles without a valid key: 0
      const int64_t first = (int64_t)blockIdx.x * 2 + (warp - 2), step = (int64_t)gridDim.x * 2;
      for (int b = 0; b < a.n.batch; ++b) {
        const int t0 = (kv_len_of(a.kv_lens, a.n.kv_len, b) + 127) & ~127;
        for (int64_t x = first; x < (int64_t)max(0, a.n.kv_len - t0) * a.n.kv_heads; x += step) {
          const int64_t t = t0 + x / a.n.kv_heads, h = x % a.n.kv_heads;
          uint16_t* row = lane < 16 ? a.dk.at(b, t, h) : a.dv.at(b, t, h);
          reinterpret_cast<uint4*>(row)[lane & 15] = make_uint4(0, 0, 0, 0);
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // one outcome a warp: the TMEM accesses need its lanes together
    auto wait_w = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
    const int w = (warp - 4) >> 2, q = warp & 3, r = 32 * q + lane;
    const uint32_t lane_base = tmem + ((uint32_t)(32 * q) << 16);
    const uint64_t sl2 = dup2(a.scale * kLog2e);
    DkvWalk seg(a, blockIdx.x, gridDim.x);
    int e = 0, sn = 0;
    bool ok = true;
    while (ok && seg.next(a)) {
      for (int it = seg.it0; it < seg.it1; ++it, ++e) {
        if (!wait_w(&bars->g_full[e & 1], (e >> 1) & 1) || !wait_w(&bars->s_full, e & 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t s[64];
        load64(lane_base + 256 + 64 * w, s);
        const uint64_t* nl2 = reinterpret_cast<const uint64_t*>(bars->nl2[e & 1] + 64 * w);
        float p[64];
        uint32_t pk[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const uint64_t v = fma_2(pair2(s[2 * c], s[2 * c + 1]), sl2, nl2[c]);
          p[2 * c] = ex2(lo2(v));
          p[2 * c + 1] = ex2(hi2(v));
          pk[c] = pack_bf16(p[2 * c], p[2 * c + 1]);
        }
        H3_TMEM_ST16(lane_base + 256 + 64 * w, (&pk[0]));
        H3_TMEM_ST16(lane_base + 256 + 64 * w + 16, (&pk[16]));
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(smem_u32(&bars->p_full));
        if (!wait_w(&bars->dp_full, e & 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
        load64(lane_base + 384 + 64 * w, s);
        const uint64_t* delta = reinterpret_cast<const uint64_t*>(bars->delta[e & 1] + 64 * w);
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const uint64_t v = mul_2(add_2(pair2(s[2 * c], s[2 * c + 1]), delta[c] ^ 0x8000000080000000ull),
                                   pair2(__float_as_uint(p[2 * c]), __float_as_uint(p[2 * c + 1])));
          pk[c] = pack_bf16(lo2(v), hi2(v));
        }
        H3_TMEM_ST16(lane_base + 384 + 64 * w, (&pk[0]));
        H3_TMEM_ST16(lane_base + 384 + 64 * w + 16, (&pk[16]));
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(smem_u32(&bars->ds_full));
      }
      if (!ok || !wait_w(&bars->acc_full, sn & 1)) break;
      ++sn;
      tc_fence_after();
      // warpgroup 0 writes dk, 1 dv
      const bool head = seg.it0 > 0, tail = seg.it1 < seg.steps;
      const int key = seg.tile * 128 + r;
      const bool valid = key < seg.len, live = key < a.n.kv_len;
      const float f = w ? 1.0f : ds_scale(a, seg.len);
      const Rows& out = w ? a.dv : a.dk;
      uint16_t* go = live ? out.at(seg.b, key, seg.hk) : nullptr;
      float4* po = reinterpret_cast<float4*>(a.part + (((int64_t)blockIdx.x * 2 + (head ? 0 : 1)) * 2 + w) * 16384);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        uint32_t v[16];
        H3_TMEM_LD16(lane_base + 128 * w + 16 * c, v);
        tmem_wait_ld();
        if (head || tail) {
          // column-major in groups of four, so that a warp's stores are contiguous
#pragma unroll
          for (int i = 0; i < 4; ++i)
            po[(4 * c + i) * 128 + r] = make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]),
                                                    __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3]));
        } else if (live) {
          uint32_t k[8];
#pragma unroll
          for (int i = 0; i < 8; ++i)
            k[i] = valid ? pack_bf16(__uint_as_float(v[2 * i]) * f, __uint_as_float(v[2 * i + 1]) * f) : 0u;
          store32(go + 16 * c, k);
        }
      }
      tc_fence_before();
      mbar_arrive(smem_u32(&bars->acc_empty));
    }
  }
  release_tmem(warp, tmem, abort_flag, &bars->done);
}

// Adds the partial sums of the key tiles that were cut.  Block (x, y): the
// tile that the start of CTA x + 1's run cuts (if it is the first such start
// inside the tile), rows 16 (y % 8).. and column groups 16 (y / 8).. of the 64
// that dk and dv have.  What it costs is latency, so eight sums are in flight
// (one after the other in a quarter of the threads: 13 us for 20 tiles).
__global__ void __launch_bounds__(256) dkv_join_kernel(const __grid_constant__ BwdArgs a, int ctas) {
  const int c = blockIdx.x + 1;
  DkvWalk own(a, c, ctas);
  const int64_t start = own.pos, share = DkvWalk(a, 1, ctas).pos;  // share: CTA 1 starts there
  const bool cut = start < own.end && own.next(a) && own.it0 > 0;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!cut) return;
  const int64_t first = start - own.it0, last = first + own.steps - 1;
  const int c0 = (int)(first / share), c1 = (int)(last / share);
  if (c0 != c - 1) return;  // an earlier start cuts the tile too
  const int r = (blockIdx.y & 7) * 16 + (threadIdx.x & 15), key = own.tile * 128 + r;
  if (key >= a.n.kv_len) return;
  const int k = (blockIdx.y >> 3) * 16 + (threadIdx.x >> 4), which = k >> 5, cg = k & 31;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int i = c0; i <= c1; ++i) {
    const float4 v = reinterpret_cast<const float4*>(
        a.part + (((int64_t)i * 2 + (i == c0 ? 1 : 0)) * 2 + which) * 16384)[cg * 128 + r];
    sum.x += v.x;
    sum.y += v.y;
    sum.z += v.z;
    sum.w += v.w;
  }
  const float f = which ? 1.0f : ds_scale(a, own.len);
  uint2 o = make_uint2(pack_bf16(sum.x * f, sum.y * f), pack_bf16(sum.z * f, sum.w * f));
  if (key >= own.len) o = make_uint2(0, 0);
  *reinterpret_cast<uint2*>((which ? a.dv : a.dk).at(own.b, key, own.hk) + 4 * cg) = o;
}

__global__ void __launch_bounds__(256) zero_kv_kernel(CrossShape n, Rows dk, Rows dv) {
  const int64_t rows = (int64_t)n.batch * n.kv_len * n.kv_heads;
  const int lane = threadIdx.x & 31;
  for (int64_t x = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5; x < rows;
       x += ((int64_t)gridDim.x * blockDim.x) >> 5) {
    const int64_t h = x % n.kv_heads, bt = x / n.kv_heads;
    uint16_t* row = (lane < 16 ? dk : dv).at(bt / n.kv_len, bt % n.kv_len, h);
    reinterpret_cast<uint4*>(row)[lane & 15] = make_uint4(0, 0, 0, 0);
  }
}

unsigned warps_grid(int64_t rows) { return (unsigned)((rows + 7) / 8 < kSms * 8 ? (rows + 7) / 8 : kSms * 8); }

int dkv_ctas(const CrossShape& n) {
  const int64_t steps = (int64_t)n.group * ((n.q_len + 127) / 128);
  const int64_t all = (int64_t)n.batch * n.kv_heads * ((n.kv_len + 127) / 128) * steps;
  return (int)(all < kSms ? all : kSms);
}

// Attributes of a kernel, set once a device; its register split needs exactly
// `regs` registers a thread at launch.
template <typename K>
cudaError_t prepare(K* kernel, int smem, int regs, std::once_flag* once, cudaError_t* result) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  std::call_once(once[dev], [&] {
    cudaError_t r = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    cudaFuncAttributes fa;
    if (r == cudaSuccess) r = cudaFuncGetAttributes(&fa, kernel);
    if (r == cudaSuccess && fa.numRegs != regs) r = cudaErrorInvalidConfiguration;
    result[dev] = r;
  });
  return result[dev];
}

// A launch that may be placed before the kernel before it ends; the kernel
// waits for that itself (griddepcontrol.wait) before it reads its results.
template <typename... P, typename... A>
cudaError_t launch_after(void (*kernel)(P...), dim3 grid, int threads, int smem, cudaStream_t s, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace

size_t cross_bwd_workspace(const CrossShape& n) {
  if (!n.batch || !n.q_len || !n.kv_len) return 0;
  const size_t rows = (size_t)n.batch * n.heads * ((n.q_len + 127) / 128) * 128;
  return 2 * rows * sizeof(float) + (size_t)dkv_ctas(n) * 4 * 16384 * sizeof(float);
}

cudaError_t launch_cross_bwd(const CrossLaunch& L, cudaStream_t s, std::string* err) {
  const CrossShape& n = L.n;
  if (n.q_len == 0) {
    const int64_t rows = (int64_t)n.batch * n.kv_len * n.kv_heads;
    if (rows) zero_kv_kernel<<<warps_grid(rows), 256, 0, s>>>(n, L.dk, L.dv);
    return cudaGetLastError();
  }
  BwdArgs a{};
  a.n = n;
  a.out = L.out, a.dout = L.dout, a.dq = L.dq, a.dk = L.dk, a.dv = L.dv;
  a.kv_lens = L.kv_lens;
  a.lse = L.lse;
  a.scale = L.scale;
  a.q_blocks = (n.q_len + 127) / 128;
  a.by_blocks = make_div(a.q_blocks), a.by_heads = make_div(n.heads), a.by_group = make_div(n.group);
  const int64_t rows = (int64_t)n.batch * n.heads * a.q_blocks * 128;
  a.nl2 = (float*)L.ws;
  a.delta = a.nl2 + rows;
  a.part = a.delta + rows;
  a.status = L.status;
  a.wait_limit_ns = L.wait_limit_ns;
  a.stall = L.stall;
  a.q_b = L.q.b != 0, a.q_h = L.q.h != 0;
  a.k_b = L.k.b != 0, a.k_h = L.k.h != 0;
  a.v_b = L.v.b != 0, a.v_h = L.v.h != 0;
  a.g_b = L.dout.b != 0, a.g_h = L.dout.h != 0;
  CUtensorMap mq, mk{}, mv{}, mg;
  if (!make_map4(&mq, L.q, n.q_len, n.heads, n.batch, err) || !make_map4(&mg, L.dout, n.q_len, n.heads, n.batch, err))
    return cudaErrorInvalidValue;
  if (n.kv_len && (!make_map4(&mk, L.k, n.kv_len, n.kv_heads, n.batch, err) ||
                   !make_map4(&mv, L.v, n.kv_len, n.kv_heads, n.batch, err)))
    return cudaErrorInvalidValue;
  const bool one = n.kv_len > 0 && n.kv_len <= 128;
  static std::once_flag once_q[2][64], once_kv[64];
  static cudaError_t res_q[2][64], res_kv[64];
  cudaError_t e = one ? prepare(dq_kernel<true>, kDqSmem, 128, once_q[1], res_q[1])
                      : prepare(dq_kernel<false>, kDqSmem, 128, once_q[0], res_q[0]);
  if (e == cudaSuccess) e = prepare(dkv_kernel, kDkvSmem, 168, once_kv, res_kv);
  if (e != cudaSuccess) return e;
  const int units = n.batch * n.heads * a.q_blocks, dq_ctas = units < kSms ? units : kSms;
  const int ctas = n.kv_len ? dkv_ctas(n) : 0;
  const int groups = (n.heads + kHeads - 1) / kHeads * n.batch;
  if (one) {
    dq_kernel<true><<<dq_ctas, kDqThreads, kDqSmem, s>>>(mq, mk, mv, mg, a, units);
    e = cudaGetLastError();
  } else if (!ctas) {
    dq_kernel<false><<<dq_ctas, kDqThreads, kDqSmem, s>>>(mq, mk, mv, mg, a, units);
    e = cudaGetLastError();
  } else {
    delta_kernel<<<dim3(a.q_blocks * 8, groups < 65535 ? groups : 65535), 256, 0, s>>>(a);
    e = cudaGetLastError();
    if (e == cudaSuccess) e = launch_after(dq_kernel<false>, dq_ctas, kDqThreads, kDqSmem, s, mq, mk, mv, mg, a, units);
  }
  if (ctas && e == cudaSuccess) e = launch_after(dkv_kernel, ctas, kThreads, kDkvSmem, s, mq, mk, mv, mg, a);
  if (ctas > 1 && e == cudaSuccess) e = launch_after(dkv_join_kernel, dim3(ctas - 1, 32), 256, 0, s, a, ctas);
  return e;
}

}  // namespace h3
