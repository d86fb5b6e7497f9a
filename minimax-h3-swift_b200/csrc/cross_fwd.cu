// Cross attention and attention over a shared prefix on the Blackwell tensor
// cores: tcgen05.mma with TMEM accumulators, TMA-staged K/V tiles, a
// persistent CTA an SM.
//
//   o_i = sum_j 2^(s_ij - m_i) v_j / l_i,  s_ij = scale log2(e) q_i.k_j
//
// one pass over the keys with a running maximum m and sum l (fp32); weights
// enter the second product in bf16, everything else is fp32 until the output.
//
// Work is cut into units: a block of query rows against all keys of one
// source.  A CTA takes whole units in turn, or, where there are too few units
// for the SMs, an equal share of all (unit, key tile) pairs in a row; a unit
// that is cut, or whose rows have two sources, leaves fp32 partial results
// (o, m, l) that a second kernel joins in a fixed order.  Row blocks:
//   dense   q_len >= 128: 2 x 128 tokens of one head, Q tiles by TMA; keys are
//           the prefix's and then the member's own (compiled twice: kShort)
//   folded  q_len < 128: a row is (member, token, head of the group), so one
//           K/V tile serves all query heads of its key head and, for the
//           prefix, the whole batch; rows are gathered.  The
//           prefix and each member's own keys are units of their own.
//           More than 128 rows: two row tiles share each K/V tile (dual).
//           Up to 128: the two halves of the CTA take alternate K/V tiles of
//           the same rows (single) and their results are joined through TMEM;
//           one half alone would reach 5.3 of the 6.5 TB/s that HBM gives.
//
// Roles of a CTA's 16 warps: 0 K/V producer (TMA); 1 MMA issuer; 2 owns TMEM;
// 3 query tiles of dense rows (TMA); 4-7 and 8-11 softmax of half 0 and 1,
// thread = row = TMEM lane; 12-15 epilogue of both halves and, for folded
// rows, the gather of the next queries.  TMEM: half t has S (then P, packed
// bf16, over its first 64 columns) at 256t and O at 256t + 128.  K/V entries
// run through a ring of 2 (3 in single mode, where each entry is needed for
// two steps); the producer hands each entry's flags to the issuer through
// shared memory.  The next unit's Q and K/V loads, its first S and softmax
// overlap the epilogue of this one, which with 3-4 key tiles a unit is a third
// of a unit's time.
//
// What bounds it: dense, the alternation of each half's products (1,024
// cycles a key tile) and softmax (2,200, of them 1,024 of the MUFU units), and
// from 1,024 keys on the power cap (1.4-1.6 GHz): 32,768 x 40 rows against 512
// keys 340 us (1.0 PFLOP/s), against 4,096 2.4-2.5 ms (1.1).
// Below 256 keys the units' turn-over: 128 keys 165 us, 4.1 TB/s.  Single: HBM
// (64 members of 4,096 keys and 8 key heads: 184 us, 5.8 TB/s; one token over
// 65,536 keys: 59 us for 41 at the copy rate, the rest the start, whose code
// and queries come from HBM behind the first keys, and the join).  Dual: as
// dense (32 members of 5 rows over 65,536 keys and 512 of their own: 103 us).
// Every wait is bounded (see attn_tc.cu; a CTA that gives up does so alone).
#include <algorithm>
#include <climits>
#include <mutex>
#include <type_traits>

#include "conditioning.cuh"

namespace h3 {
namespace {

constexpr int kThreads = 512;
constexpr int kSms = 148;
// What a unit of folded rows costs beside its key tiles, in key tiles: its
// queries and its results pass through one buffer each.  24 members with 64
// keys of their own over 65,536 shared ones: 149 us without it, 75 with 2; 16
// members of 4 x 14 rows with 300 over 4,000: 40 and 34; 32 members with 512
// over 65,536: 107 and 111.
constexpr int kUnitCost = 2;

// kShort: dense rows against few key tiles, see the mask of the last tile
enum { kDense = 0, kSingle = 1, kDual = 2, kShort = 3 };
constexpr int kShortTiles = 3;
constexpr bool is_dense(int mode) { return mode == kDense || mode == kShort; }

// The units of one source of keys: the prefix (folded rows only), or the
// members' own keys (dense rows: the prefix's and their own).
struct Source {
  int32_t per;                // row blocks of a key head (prefix), of a member's (key) head (own)
  int32_t units;
  int32_t tiles;              // key tiles of a unit
  int32_t pitch;              // its places in the linear split: its tiles and its own cost
  int32_t rows;               // rows of a block: 128 or 256
  int32_t tpc;                // key tiles a CTA in the linear split; 0: whole units in turn
  int32_t start;              // first position of its units in that split
  // partial results: slots of a unit at most, rows of a slot; o as
  // [units, slots, 32, stride] groups of four channels, ml as [units, slots,
  // stride], so that a warp's 32 rows are contiguous
  int32_t slots, stride;
  Div by_per, by_pitch, by_tpc;
};

struct FwdArgs {
  CrossShape n;
  Source src[2];              // prefix, own
  int32_t units_p, units_o;   // units of either
  int32_t tpc;
  int32_t mode;
  int32_t np;                 // key tiles of the prefix
  int32_t fold_rows;          // folded: rows of a key head over the batch
  int32_t two_sources;        // every row has results of both
  Div by_heads, by_kv_heads, by_group, by_q_len;
  Rows q, out;
  const int32_t* kv_lens;
  float* lse;
  float scale_log2;
  float4* part_o[2];
  float2* part_ml[2];
  int32_t* status;
  uint64_t wait_limit_ns;
  int32_t stall;              // test hook: barrier (from Barriers::q_full on) that never completes
  // 1 where an operand's tensor map has the axis, 0 where it is broadcast
  int32_t q_b, q_h, k_b, k_h, v_b, v_h, pk_h, pv_h;
};

// One run of key tiles of one unit.
struct Seg {
  int own, unit;              // source and unit of it
  int b, hk, h;               // h: dense only
  int row0, row_end;          // tokens (dense) or folded rows
  int npre, len;              // tiles of the unit that are the prefix's; valid own keys
  int j0, n;                  // first tile, tiles with valid keys (0: nothing to do)
  int slot;                   // partial slot
  bool direct;                // the whole result of its rows
};

// (dense rows have no units of the prefix)
template <int MODE>
struct SegIter {
  uint32_t pos, end;          // key tiles of the linear split, or units
  __device__ explicit SegIter(const FwdArgs& a) {
    if (a.tpc) {
      const uint32_t total = (uint32_t)(a.units_p * a.src[0].pitch + a.units_o * a.src[1].pitch);
      pos = blockIdx.x * a.tpc;
      end = min(total, pos + a.tpc);
    } else {
      pos = blockIdx.x;
      end = a.units_p + a.units_o;
    }
  }
  __device__ bool next(const FwdArgs& a, const int32_t* lens, Seg& s) {
    int j1, tiles;
    s.slot = 0;
    if (a.tpc) {
      do {
        if (pos >= end) return false;
        const uint32_t pre = is_dense(MODE) ? 0 : a.units_p * a.src[0].pitch;
        s.own = is_dense(MODE) || pos >= pre;
        const Source& c = a.src[s.own];
        const uint32_t off = s.own ? pos - pre : pos;
        tiles = c.tiles;
        s.unit = c.by_pitch(off);
        s.j0 = (int)off - s.unit * c.pitch;
        j1 = min(c.pitch, s.j0 + (int)(end - pos));
        s.slot = blockIdx.x - c.by_tpc(pos - s.j0);
        pos += j1 - s.j0;
      } while (!is_dense(MODE) && s.j0 >= tiles);
      if (!is_dense(MODE)) j1 = min(j1, tiles);
    } else {
      if (pos >= end) return false;
      s.own = is_dense(MODE) || (int)pos >= a.units_p;
      s.unit = (int)pos - (!is_dense(MODE) && s.own ? a.units_p : 0);
      tiles = a.src[s.own].tiles;
      s.j0 = 0;
      j1 = tiles;
      pos += gridDim.x;
    }
    const Source& c = a.src[s.own];
    const int x = c.by_per(s.unit), rt = s.unit - x * c.per;
    int limit;
    if (!s.own) {
      s.hk = x;
      s.row0 = rt * c.rows;
      s.row_end = min(a.fold_rows, s.row0 + c.rows);
      s.b = 0;
      s.len = 0;
      s.npre = limit = a.np;
    } else {
      if (is_dense(MODE)) {
        s.b = a.by_heads(x);
        s.h = x - s.b * a.n.heads;
        s.hk = a.by_group(s.h);
        s.row0 = rt * c.rows;
        s.row_end = min(a.n.q_len, s.row0 + c.rows);
        s.npre = a.np;
      } else {
        s.b = a.by_kv_heads(x);
        s.hk = x - s.b * a.n.kv_heads;
        const int rows = a.n.q_len * a.n.group;
        s.row0 = s.b * rows + rt * c.rows;
        s.row_end = min((s.b + 1) * rows, s.row0 + c.rows);
        s.npre = 0;
      }
      s.len = s.b < kLens ? lens[s.b] : kv_len_of(a.kv_lens, a.n.kv_len, s.b);
      limit = s.npre + ((s.len + 127) >> 7);
    }
    s.n = max(0, min(j1, limit) - s.j0);
    s.direct = s.j0 == 0 && j1 == tiles && (is_dense(MODE) || !a.two_sources);
    return true;
  }
  // valid keys of tile j of the segment's unit
  static __device__ int valid(const FwdArgs& a, const Seg& s, int j) {
    return min(128, j < s.npre ? a.n.prefix_len - 128 * j : s.len - 128 * (j - s.npre));
  }
};

template <int MODE>
struct Layout {
  static constexpr int kRing = MODE == kSingle ? 3 : 2;  // K/V entries
  static constexpr int kQTiles = MODE == kSingle ? 1 : 2;
  // the rest of 224 KB in dense mode: two 4 KB output buffers an epilogue warp
  static constexpr int kTiles = 7 * kTileBytes;
};

struct __align__(8) Barriers {
  uint64_t q_full[2], q_empty[2];
  uint64_t kv_full[3], k_empty[3], v_empty[3];
  uint64_t s_full[2], p_half[2], p_full[2], o_full[2], o_empty[2], ml_full[2];
  uint64_t done;              // every MMA has retired
  uint32_t tmem_base;
  int32_t abort;
  int32_t info[16];           // flags of entry e at [e & 15]
  int32_t lens[kLens];
  float2 ml[2][128];          // maximum and sum of a half's rows
};

// flags of an entry: bit t: half t takes it; 2 + t / 4 + t: first / last of the segment for half t
enum { kFirst = 2, kLast = 4, kSegFirst = 1 << 6, kSegLast = 1 << 7, kEnd = 1 << 8, kApart = 1 << 9, kZeroShift = 16 };

constexpr int kSmemBytes = 7 * kTileBytes + (int)sizeof(Barriers);
static_assert(kSmemBytes <= 227 * 1024, "shared memory");

constexpr int kApartTiles = 8;  // key tiles from which a segment's halves start apart

// Instruction descriptor, kind::f16: bf16 x bf16 -> f32, M = N = 128.
constexpr uint32_t kIdS = idesc_bf16(false), kIdPV = idesc_bf16(true);

template <int MODE>
__global__ void __launch_bounds__(kThreads, 1)
    cross_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_pk,
                     const __grid_constant__ CUtensorMap tm_pv, const __grid_constant__ CUtensorMap tm_o,
                     const __grid_constant__ FwdArgs a) {
  using L = Layout<MODE>;
  constexpr bool SINGLE = MODE == kSingle, dense = is_dense(MODE);
  extern __shared__ __align__(1024) uint8_t smem[];
  if (!tiles_aligned(smem, a.status)) return;
  uint8_t* sQ = smem;
  uint8_t* sKV = smem + L::kQTiles * kTileBytes;  // entry r: K at 2r, V at 2r + 1
  Barriers* bars = (Barriers*)(smem + L::kTiles);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int32_t* abort_flag = &bars->abort;

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(smem_u32(&bars->q_full[t]), 128);  // folded only
      mbar_init(smem_u32(&bars->q_empty[t]), 1);
      mbar_init(smem_u32(&bars->s_full[t]), 1);
      mbar_init(smem_u32(&bars->p_half[t]), 128);
      mbar_init(smem_u32(&bars->p_full[t]), 128);
      mbar_init(smem_u32(&bars->o_full[t]), 1);
      mbar_init(smem_u32(&bars->o_empty[t]), 128);
      mbar_init(smem_u32(&bars->ml_full[t]), 128);
    }
    for (int r = 0; r < 3; ++r) {
      // dense: the K/V producer, and of a segment's first entry the Q loader
      // (one wait of the issuer for all of it; of others the producer again)
      mbar_init(smem_u32(&bars->kv_full[r]), dense ? 2 : 1);
      mbar_init(smem_u32(&bars->k_empty[r]), 1);
      mbar_init(smem_u32(&bars->v_empty[r]), 1);
    }
    mbar_init(smem_u32(&bars->done), 1);
    if (a.stall >= 0 && bars->q_full + a.stall <= &bars->done) mbar_stall(smem_u32(bars->q_full + a.stall));
    bars->abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x >= 128 && threadIdx.x < 128 + kLens && threadIdx.x - 128 < a.n.batch)
    bars->lens[threadIdx.x - 128] = kv_len_of(a.kv_lens, a.n.kv_len, threadIdx.x - 128);
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                     smem_u32(&bars->tmem_base)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  asm volatile("griddepcontrol.launch_dependents;");
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    return mbar_wait_alone<dense>(smem_u32(bar), parity, abort_flag, a.status, a.wait_limit_ns);
  };

  // Register split of the launch's 512 x 128: 128 x 48 + 256 x 192 + 128 x 80.
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    if (warp == 0) {
      // ------------------------------------------------------- TMA producer
      if (lane == 0) {
        SegIter<MODE> it(a);
        Seg s{};
        [[maybe_unused]] const uint64_t once = evict_first();
        int ec = 0, r = 0, issued = 0;
        uint32_t ph = 0;
        bool ok = true;
        while (ok && it.next(a, bars->lens, s)) {
          if (s.n == 0) continue;
          const bool act1 = !SINGLE && s.row0 + 128 < s.row_end;
          for (int i = 0; ok && i < s.n; ++i) {
            const int j = s.j0 + i;
            int info;
            if (SINGLE) {
              const int t = ec & 1;
              info = (1 << t) | (i < 2 ? 1 << (kFirst + t) : 0) | (i >= s.n - 2 ? 1 << (kLast + t) : 0) |
                     (i == 0 ? kSegFirst : 0) | (i == s.n - 1 ? kSegLast : 0);
            } else {
              const int act = act1 ? 3 : 1;
              info = act | (i == 0 ? act << kFirst : 0) | (i == s.n - 1 ? act << kLast : 0) |
                     (i == 0 && act1 && s.n >= kApartTiles ? kApart : 0);
            }
            const bool pre = j < s.npre;
            // value rows past the member's length hold whatever the caller
            // left there, and 0 x NaN would reach the result: the issuer
            // clears them (TMA itself clears rows past the operand's end)
            const int valid = SegIter<MODE>::valid(a, s, j);
            if (!pre && valid < 128 && s.len < a.n.kv_len) info |= valid << kZeroShift;
            if (!wait(&bars->k_empty[r], ph ^ 1) || !wait(&bars->v_empty[r], ph ^ 1)) {
              ok = false;
              break;
            }
            const uint32_t bar = smem_u32(&bars->kv_full[r]);
            bars->info[ec & 15] = info;
            if (!SINGLE && dense && i > 0) mbar_arrive(bar);
            mbar_expect_tx(bar, 2 * kTileBytes);
            const uint32_t dk = smem_u32(sKV + 2 * r * kTileBytes), dv = dk + kTileBytes;
            // both half tiles; of folded rows each key tile is read once (a prefix
            // of 65,536 keys, 1 row: 56 us, 61 with the tiles kept in L2 like
            // any other load)
            auto load = [&](uint32_t dst, const CUtensorMap* map, int tok, int h, int b) {
#pragma unroll
              for (int x = 0; x < 2; ++x)
                if constexpr (dense) tma_load_4d(dst + x * kHalfBytes, map, bar, 64 * x, tok, h, b);
                else tma_load_4d(dst + x * kHalfBytes, map, bar, 64 * x, tok, h, b, once);
            };
            if (pre) {
              load(dk, &tm_pk, 128 * j, s.hk * a.pk_h, 0);
              load(dv, &tm_pv, 128 * j, s.hk * a.pv_h, 0);
            } else {
              const int tok = 128 * (j - s.npre);
              load(dk, &tm_k, tok, s.hk * a.k_h, s.b * a.k_b);
              load(dv, &tm_v, tok, s.hk * a.v_h, s.b * a.v_b);
            }
            ++issued;
            ++ec;
            if (++r == L::kRing) {
              r = 0;
              ph ^= 1;
            }
          }
        }
        if (ok && wait(&bars->k_empty[r], ph ^ 1) && wait(&bars->v_empty[r], ph ^ 1)) {
          bars->info[ec & 15] = kEnd;
          mbar_arrive(smem_u32(&bars->kv_full[r]));
          if (!SINGLE && dense) mbar_arrive(smem_u32(&bars->kv_full[r]));
        } else {
          // abort: every load in flight lands before anyone may exit (an entry
          // that the Q loader did not join never completes: a short limit)
          volatile int32_t zero = 0;
          for (int e = max(0, issued - L::kRing); e < issued; ++e, zero = 0)
            mbar_wait(smem_u32(&bars->kv_full[e % L::kRing]), (e / L::kRing) & 1, &zero, nullptr, kDrainNs);
        }
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------ MMA issuer
      // Per entry and half: the PV of the half's previous entry (its P is
      // ready once its softmax arrives), then its S of this entry, so that
      // the halves alternate between tensor pipe and softmax.
      auto iwait = [&](uint64_t* bar, uint32_t par) -> bool {
        int got = 0;
        if (lane == 0) got = wait(bar, par & 1) ? 1 : 0;
        return __shfl_sync(0xffffffff, got, 0) != 0;
      };
      // phase bits: 0 K/V ring, 1 + t Q, 3 + t P
      uint32_t ph = 0;
      // entry whose PV is due: ring slot, its first / last flags as bits 4, 5; or -1
      int pend0 = -1, pend1 = -1;
      const uint32_t q_lo = desc_lo(smem_u32(sQ), 16), k_lo = desc_lo(smem_u32(sKV), 16);
      const uint32_t v_lo = desc_lo(smem_u32(sKV) + kTileBytes, kHalfBytes);
      constexpr uint32_t kTileLo = kTileBytes >> 4;
      int ec = 0, r = 0;
      using T0 = std::integral_constant<int, 0>;
      using T1 = std::integral_constant<int, 1>;
      auto issue_pv = [&](auto tile) -> bool {
        constexpr int t = decltype(tile)::value;
        int& pend = t == 0 ? pend0 : pend1;
        const int slot = pend & 15, other = t == 0 ? pend1 : pend0;
        if (!iwait(&bars->p_half[t], ph >> (3 + t))) return false;
        tc_fence_after();
        const uint32_t b = v_lo + 2 * slot * kTileLo;
        mma_tile_ts_0_6(tmem + 256 * t + 128, tmem + 256 * t, b, kIdPV, !(pend & 16));
        if (!iwait(&bars->p_full[t], ph >> (3 + t))) return false;
        tc_fence_after();
        ph ^= 1u << (3 + t);
        mma_tile_ts_6_8(tmem + 256 * t + 128, tmem + 256 * t, b, kIdPV, 1);
        if (pend & 32) tc_commit_w(smem_u32(&bars->o_full[t]));
        if (other < 0 || (other & 15) != slot) tc_commit_w(smem_u32(&bars->v_empty[slot]));
        pend = -1;
        return true;
      };
      auto issue_s = [&](auto tile, int info) -> bool {
        constexpr int t = decltype(tile)::value;
        if (!SINGLE && !dense && (info & (1 << (kFirst + t)))) {
          if (!iwait(&bars->q_full[t], ph >> (1 + t))) return false;
          tc_fence_after();
          ph ^= 1u << (1 + t);
        }
        mma_tile_ss(tmem + 256 * t, q_lo + (SINGLE ? 0 : t) * kTileLo, k_lo + 2 * r * kTileLo, kIdS, 0);
        tc_commit_w(smem_u32(&bars->s_full[t]));
        if (!SINGLE && (info & (1 << (kLast + t)))) tc_commit_w(smem_u32(&bars->q_empty[t]));
        (t == 0 ? pend0 : pend1) = r | (((info >> (kFirst + t)) & 1) << 4) | (((info >> (kLast + t)) & 1) << 5);
        return true;
      };
      bool ok;
      while (true) {
        if (SINGLE) {
          if (ec & 1) ok = pend1 < 0 || issue_pv(T1{});
          else ok = pend0 < 0 || issue_pv(T0{});
        } else {
          ok = pend0 < 0 || issue_pv(T0{});
        }
        if (!ok || !iwait(&bars->kv_full[r], ph)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const int info = ((volatile int32_t*)bars->info)[ec & 15];
        if (info & kEnd) break;
        if (info >> kZeroShift) {
          // rows [valid, 128) of V; a row is 128 bytes of either half tile
          uint4* v = reinterpret_cast<uint4*>(sKV + (2 * r + 1) * kTileBytes);
          for (int x = (info >> kZeroShift) * 8 + lane; x < 1024; x += 32) v[x] = v[1024 + x] = make_uint4(0, 0, 0, 0);
          fence_async_shared();
          __syncwarp();
        }
        if (SINGLE && (info & kSegFirst)) {
          if (!iwait(&bars->q_full[0], ph >> 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          ph ^= 2;
        }
        if (info & 1) ok = issue_s(T0{}, info);
        if (!SINGLE && ok && pend1 >= 0) ok = issue_pv(T1{});
        // Any distance between the halves of 1,024 cycles up (that of their
        // products) lasts.  At half a period their exponentials do not meet on
        // the MUFU units, so half 1 begins a long segment when half 0's first
        // weights are out (4,096 keys: 2.48 ms against 2.56; below 8 tiles the
        // wait costs what it gains).
        if (dense && ok && (info & kApart)) ok = iwait(&bars->p_half[0], ph >> 3);
        if (ok && (info & 2)) ok = issue_s(T1{}, info);
        if (!ok) break;
        tc_commit_w(smem_u32(&bars->k_empty[r]));
        if (SINGLE && (info & kSegLast)) tc_commit_w(smem_u32(&bars->q_empty[0]));
        ++ec;
        if (++r == L::kRing) {
          r = 0;
          ph ^= 1;
        }
      }
      if (ok && pend0 >= 0) ok = issue_pv(T0{});
      if (ok && pend1 >= 0) issue_pv(T1{});
      // aborted or not: MMAs retire in order, so this covers all of them
      tc_commit_w(smem_u32(&bars->done));
    } else if constexpr (dense) {
      // -------------------------------------------------- Q tiles (TMA)
      if (warp == 3 && lane == 0) {
        // A segment's Q tiles complete its first entry's barrier.  That the
        // last segment's S has read Q (q_empty) says that every barrier of
        // its entries has completed, so this arrival falls in the right phase.
        // The segment after it goes to L2 meanwhile: one buffer covers L2's
        // latency, not HBM's.
        SegIter<MODE> it(a);
        Seg s{}, following{};
        const uint64_t once = evict_first();  // (4% at 128-332 keys)
        int qn0 = 0, qn1 = 0, ec = 0;
        bool more = it.next(a, bars->lens, following);
        while (more) {
          s = following;
          more = it.next(a, bars->lens, following);
          if (more && following.n > 0 && following.j0 == 0)
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (c < 2 || following.row0 + 128 < following.row_end)
                tma_prefetch_4d(&tm_q, 64 * (c & 1), following.row0 + 64 * (c & 2), following.h * a.q_h,
                                following.b * a.q_b);
          if (s.n == 0) continue;
          const bool act1 = s.row0 + 128 < s.row_end;
          const uint32_t bar = smem_u32(&bars->kv_full[ec % L::kRing]);
          auto load = [&](int t) {
            const uint32_t dst = smem_u32(sQ + t * kTileBytes);
            tma_load_4d(dst, &tm_q, bar, 0, s.row0 + 128 * t, s.h * a.q_h, s.b * a.q_b, once);
            tma_load_4d(dst + kHalfBytes, &tm_q, bar, 64, s.row0 + 128 * t, s.h * a.q_h, s.b * a.q_b, once);
          };
          if (!wait(&bars->q_empty[0], (qn0++ & 1) ^ 1)) break;
          mbar_expect_tx(bar, act1 ? 2 * kTileBytes : kTileBytes);
          load(0);
          if (act1) {
            if (!wait(&bars->q_empty[1], (qn1++ & 1) ^ 1)) break;
            load(1);
          }
          ec += s.n;
        }
      }
    }
  } else if (warp < 12) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    // one outcome a warp: the TMEM accesses need its lanes together
    auto wait_w = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
    // ---------------------------------------------------------------- softmax
    const int t = (warp - 4) >> 2, q = warp & 3;
    const int r = 32 * q + lane;  // row of the tile = TMEM lane
    const uint32_t lane_base = tmem + ((uint32_t)(32 * q) << 16);
    const uint32_t tS = lane_base + 256 * t, tO = tS + 128;
    const float sl2 = a.scale_log2;
    const uint64_t sl2x2 = dup2(sl2);
    SegIter<MODE> it(a);
    Seg s{};
    int ec = 0, ns = 0, nseg = 0;
    bool ok = true;
    while (ok && it.next(a, bars->lens, s)) {
      const int i0 = SINGLE ? ((ec ^ t) & 1) : 0;
      const int step = SINGLE ? 2 : 1;
      const int nt = SINGLE ? (s.n - i0 + 1) / 2 : (s.row0 + 128 * t < s.row_end ? s.n : 0);
      ec += s.n;
      if (nt == 0) continue;
      float m = -1e30f, l = 0.f;
      for (int x = 0; ok && x < nt; ++x) {
        const int valid = SegIter<MODE>::valid(a, s, s.j0 + i0 + x * step);
        if (!wait_w(&bars->s_full[t], ns & 1)) {
          ok = false;
          break;
        }
        ++ns;
        tc_fence_after();
        uint32_t v[128];
#pragma unroll
        for (int c = 0; c < 8; ++c) H3_TMEM_LD16(tS + 16 * c, (&v[16 * c]));
        tmem_wait_ld();
        // Keys past the end.  128 selects are 4 KB of code, with which a unit's
        // code no longer stays in the instruction cache where each unit comes to
        // them soon: there -inf is written to TMEM instead, in a loop, and the
        // row loaded again.  15,731 x 56 rows against 77 keys 137 us (selects:
        // 168), 332 keys 255 (275), 32 members with 512 keys over 65,536 shared
        // 104 (115).  From four tiles on the selects are faster, since the code
        // around them comes out faster: 16,384 keys 1,285 us (1,324 with the loop).
        if (valid < 128) {
          if constexpr (MODE == kDense) {
#pragma unroll
            for (int c = 0; c < 128; ++c)
              if (c >= valid) v[c] = __float_as_uint(-INFINITY);
          } else {
            fill_columns(tS, valid, 128, __float_as_uint(-INFINITY));
#pragma unroll
            for (int c = 0; c < 8; ++c) H3_TMEM_LD16(tS + 16 * c, (&v[16 * c]));
            tmem_wait_ld();
          }
        }
        float mxa[8];
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          float w = __uint_as_float(v[16 * g]);
#pragma unroll
          for (int c = 1; c < 15; c += 2)
            w = max3(w, __uint_as_float(v[16 * g + c]), __uint_as_float(v[16 * g + c + 1]));
          mxa[g] = fmaxf(w, __uint_as_float(v[16 * g + 15]));
        }
        const float mx = max3(max3(mxa[0], mxa[1], mxa[2]), max3(mxa[3], mxa[4], mxa[5]), fmaxf(mxa[6], mxa[7]));
        // finite even where every logit so far is -inf (its weights are then 0)
        const float mxs = fmaxf(mx * sl2, -1e30f);
        // the running maximum moves only when the new one is over 8 above it
        // (a factor 256 in the weights), so O is rarely rescaled
        const bool need = x > 0 && mxs > m + 8.0f;
        if (x == 0) m = mxs;
        if (__any_sync(0xffffffff, need)) {
          const float f = need ? ex2(m - mxs) : 1.0f;
          if (need) {
            l *= f;
            m = mxs;
          }
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            uint32_t o[16];
            H3_TMEM_LD16(tO + 16 * c, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            H3_TMEM_ST16(tO + 16 * c, o);
          }
        }
        const uint64_t negm = dup2(-m);
        uint64_t sum2 = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float x0, x1;
            fma2(x0, x1, v[32 * c + 2 * e], v[32 * c + 2 * e + 1], sl2x2, negm);
            const float p0 = ex2(x0), p1 = ex2(x1);
            sum2 = add2(sum2, p0, p1);
            pk[e] = pack_bf16(p0, p1);
          }
          H3_TMEM_ST16(tS + 16 * c, pk);
          if (c == 2) {  // keys 0-95 of P are in TMEM: the first six PV steps may start
            // (once the epilogue has read O and (m, l) of the last segment: waited
            // for here, not by the issuer, whose waits delay both halves)
            if (x == 0 && nseg > 0) ok = wait_w(&bars->o_empty[t], (nseg - 1) & 1);
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(smem_u32(&bars->p_half[t]));
          }
        }
        l += __uint_as_float((uint32_t)sum2) + __uint_as_float((uint32_t)(sum2 >> 32));
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(smem_u32(&bars->p_full[t]));
      }
      if (!ok) break;
      bars->ml[t][r] = make_float2(m, l);
      ++nseg;
      mbar_arrive(smem_u32(&bars->ml_full[t]));
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    // --------------------------------------------------------------- epilogue
    auto wait_w = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
    const int q = warp & 3, r = 32 * q + lane;
    const uint32_t tO = tmem + ((uint32_t)(32 * q) << 16) + 128;
    uint8_t* stage = smem + 6 * kTileBytes + q * 8192;  // dense: two boxes of 32 rows x 64 columns
    SegIter<MODE> it(a);
    Seg s{};
    int ec = 0, n0 = 0, n1 = 0;  // segments of either half
    // half t's (m, l) and O are there
    auto arrived = [&](int t, int& n, float2& ml) {
      if (!wait_w(&bars->ml_full[t], n & 1)) return false;
      ml = bars->ml[t][r];
      if (!wait_w(&bars->o_full[t], n & 1)) return false;
      ++n;
      return true;
    };
    // dense rows of tile t, whole: boxes of 32 rows x 64 columns by TMA
    auto finish_box = [&](int t, bool has, float2 ml) {
      tc_fence_after();
      const int row0 = s.row0 + 128 * t + 32 * q;
      const float f = 1.0f / fmaxf(ml.y, 1e-30f);
      if (a.lse && row0 + lane < s.row_end)
        a.lse[((int64_t)s.b * a.n.heads + s.h) * a.n.q_len + row0 + lane] =
            ml.y == 0.f ? -INFINITY : (ml.x + lg2(ml.y)) * 0.69314718055994531f;
#pragma unroll 1
      for (int p = 0; p < 2; ++p) {
        uint8_t* box = stage + p * 4096;
        if (lane == 0) tma_store_wait_read<1>();  // the box two groups ago has been read
        __syncwarp();
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          // a load's latency is 200-400 cycles beside the other warps' TMEM
          // traffic, so as many columns as the registers hold
          uint32_t x[32];
          if (has) {
            H3_TMEM_LD16(tO + 256 * t + 64 * p + 32 * c, (&x[0]));
            H3_TMEM_LD16(tO + 256 * t + 64 * p + 32 * c + 16, (&x[16]));
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) x[e] = 0u;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const auto two = [&](int k) {
              return pack_bf16(__uint_as_float(x[8 * e + k]) * f, __uint_as_float(x[8 * e + k + 1]) * f);
            };
            *reinterpret_cast<uint4*>(box + lane * 128 + (((4 * c + e) ^ (lane & 7)) << 4)) =
                make_uint4(two(0), two(2), two(4), two(6));
          }
        }
        fence_async_shared();
        __syncwarp();
        if (lane == 0) {
          if (row0 < s.row_end)
            tma_store_4d(&tm_o, smem_u32(box), 64 * p, row0, s.h * (a.out.h != 0), s.b * (a.out.b != 0));
          tma_store_commit();  // a group for every box that was filled, empty or not: the waits count them
        }
      }
    };
    // any other rows of tile t: O of half t (f0) and, where has1, of half 1
    // (f1), to the output or to the partial results
    auto finish_rows = [&](int t, bool has0, bool has1, float2 ml, float f0, float f1) {
      tc_fence_after();
      const int row = s.row0 + 128 * t + r;
      const bool live = row < s.row_end;
      int tok = row, b = s.b, h = s.h;
      if (!dense) {
        const int bt = a.by_group(row);
        b = a.by_q_len(bt);
        tok = bt - b * a.n.q_len;
        h = s.hk * a.n.group + (row - bt * a.n.group);
      }
      const int64_t out_row = ((int64_t)b * a.n.heads + h) * a.n.q_len + tok;
      const Source& c1 = a.src[s.own];
      const int64_t part = (int64_t)s.unit * c1.slots + s.slot;
      if (s.direct) {
        const float inv = 1.0f / fmaxf(ml.y, 1e-30f);
        f0 *= inv;
        f1 *= inv;
        if (live && a.lse) a.lse[out_row] = ml.y == 0.f ? -INFINITY : (ml.x + lg2(ml.y)) * 0.69314718055994531f;
      } else if (live) {
        a.part_ml[s.own][part * c1.stride + 128 * t + r] = ml;
      }
      if (!has0 && !has1 && !s.direct) return;
      uint16_t* go = a.out.p + (live ? b * a.out.b + tok * a.out.t + h * a.out.h : 0);
      float4* po = a.part_o[s.own] + part * 32 * c1.stride + 128 * t + r;
#pragma unroll 1
      for (int c = 0; c < 128; c += 16) {
        uint32_t x[16], y[16];
        if (has0) H3_TMEM_LD16(tO + 256 * t + c, x);
        if (has1) H3_TMEM_LD16(tO + 256 + c, y);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float o = has0 ? __uint_as_float(x[e]) * f0 : 0.f;
          if (has1) o = fmaf(__uint_as_float(y[e]), f1, o);
          x[e] = __float_as_uint(o);
        }
        if (!live) continue;
        if (s.direct) {
          uint32_t k[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) k[e] = pack_bf16(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1]));
          store32(go + c, k);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            po[(c / 4 + e) * c1.stride] = make_float4(__uint_as_float(x[4 * e]), __uint_as_float(x[4 * e + 1]),
                                                      __uint_as_float(x[4 * e + 2]), __uint_as_float(x[4 * e + 3]));
        }
      }
    };
    // Folded: the next segment's Q rows, once the last S has read this one's.
    // 16 lanes take a row, 8 rows a pass of the 128 threads; rows past the
    // block are zero.  All passes of both tiles are in flight together, by
    // asynchronous copies: at the start every SM's first K/V loads queue at HBM,
    // and four rounds of loads through registers took 13,000 cycles there.
    // Swizzle: 16-byte chunk c of row r sits at c ^ (r & 7).
    auto gather = [&](const Seg& g, int t, int& qn) {
      if (!wait_w(&bars->q_empty[t], (qn & 1) ^ 1)) return false;
      ++qn;
      const int c = lane & 15, first = 2 * q + (lane >> 4);
      const uint32_t dst = smem_u32(sQ + t * kTileBytes + (c >> 3) * kHalfBytes) + (((c & 7) ^ (first & 7)) << 4);
#pragma unroll 4
      for (int r0 = first; r0 < 128; r0 += 8) {
        const int row = g.row0 + 128 * t + r0;
        const bool in = row < g.row_end;
        const int tok = a.by_group(in ? row : g.row0), b = a.by_q_len(tok);
        copy16_or_zero(dst + r0 * 128,
                       a.q.at(b, tok - b * a.n.q_len, g.hk * a.n.group + ((in ? row : g.row0) - tok * a.n.group)) + 8 * c,
                       in);
      }
      copies_commit();
      return true;
    };
    int qn0 = 0, qn1 = 0;
    auto gather_next = [&](SegIter<MODE> ahead) {
      Seg g{};
      while (ahead.next(a, bars->lens, g)) {
        if (g.n == 0) continue;
        const bool two = !SINGLE && g.row0 + 128 < g.row_end;
        if (!gather(g, 0, qn0)) return false;
        if (two && !gather(g, 1, qn1)) return false;
        if (two) copies_wait<1>();
        else copies_wait<0>();
        fence_async_shared();
        mbar_arrive(smem_u32(&bars->q_full[0]));
        if (two) {
          copies_wait<0>();
          fence_async_shared();
          mbar_arrive(smem_u32(&bars->q_full[1]));
        }
        return true;
      }
      return true;
    };
    if (!dense && !gather_next(it)) it.pos = it.end;
    while (it.next(a, bars->lens, s)) {
      if (!dense && s.n > 0 && !gather_next(it)) break;
      float2 ml0 = make_float2(-1e30f, 0.f);
      if (SINGLE) {
        float2 ml1 = ml0;
        const bool has0 = s.n > (ec & 1), has1 = s.n > ((ec ^ 1) & 1);
        ec += s.n;
        if ((has0 && !arrived(0, n0, ml0)) || (has1 && !arrived(1, n1, ml1))) break;
        const float top = fmaxf(ml0.x, ml1.x), f0 = ex2(ml0.x - top), f1 = ex2(ml1.x - top);
        finish_rows(0, has0, has1, make_float2(top, ml0.y * f0 + ml1.y * f1), f0, f1);
        tc_fence_before();
        if (has0) mbar_arrive(smem_u32(&bars->o_empty[0]));
        if (has1) mbar_arrive(smem_u32(&bars->o_empty[1]));
      } else {
#pragma unroll 1
        for (int t = 0; t < 2; ++t) {
          if (t && s.row0 + 128 >= s.row_end) continue;
          if (s.n > 0 && !arrived(t, t ? n1 : n0, ml0)) goto out;
          if (dense && s.direct) finish_box(t, s.n > 0, ml0);
          else finish_rows(t, s.n > 0, false, ml0, 1.f, 0.f);
          tc_fence_before();
          if (s.n > 0) mbar_arrive(smem_u32(&bars->o_empty[t]));
        }
      }
    }
  out:
    copies_wait<0>();
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  }

  // ------------------------------------------------------------------ exit
  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    if (bars->abort) {  // no MMA may still write TMEM when it is released
      volatile int32_t zero = 0;
      mbar_wait(smem_u32(&bars->done), 0, &zero, nullptr);
      settle();
      __syncwarp();
    }
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// The partial results of a row from one source: n slots of a unit.
struct Runs {
  const float4* o;
  const float2* ml;
  int n, stride;
  __device__ Runs(const FwdArgs& a, int own, int unit, int row) {
    const Source& c = a.src[own];
    const uint32_t first = c.start + (uint32_t)unit * c.pitch;
    n = c.tpc ? (int)(c.by_tpc(first + c.tiles - 1) - c.by_tpc(first)) + 1 : 1;
    stride = c.stride;
    o = a.part_o[own] + (int64_t)unit * c.slots * 32 * stride + row;
    ml = a.part_ml[own] + (int64_t)unit * c.slots * stride + row;
  }
};

// A softmax over some of the keys: maximum, sum and 16 channels of o.
struct Some {
  float m, l, o[16];
  __device__ void add(float m2, float l2, const float* o2) {
    const float top = fmaxf(m, m2), f = ex2(m - top), g = l2 == 0.f ? 0.f : ex2(m2 - top);
    m = top;
    l = l * f + l2 * g;
#pragma unroll
    for (int c = 0; c < 16; ++c) o[c] = o[c] * f + (l2 == 0.f ? 0.f : o2[c] * g);  // l2 = 0: o2 was not written
  }
};

// Joins the slots of 32 rows, in a fixed order.  A lane has a row, the 32 warps
// of the block 16 channels of every fourth slot each; a slot's o is read along
// with its (m, l), four slots at a time, since what this costs is latency
// (with 8 warps, the maximum first and the slots one after the other: 10 us
// behind the kernel whose results it joins, against 4).
constexpr int kJoinThreads = 1024;

__device__ __forceinline__ void join_rows(const Runs* runs, int sources, bool live, uint16_t* out, float* lse) {
  __shared__ float box[2][18][256];
  const int w = (threadIdx.x >> 5) & 7, part = threadIdx.x >> 8, at = threadIdx.x & 255;
  Some a;
  a.m = -1e30f;
  a.l = 0.f;
#pragma unroll
  for (int c = 0; c < 16; ++c) a.o[c] = 0.f;
  if (live)
    for (int k = 0; k < sources; ++k) {
      const Runs& r = runs[k];
#pragma unroll 2
      for (int i = part; i < r.n; i += 4) {
        const float2 e = r.ml[i * r.stride];
        float4 v[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = r.o[((int64_t)i * 32 + 4 * w + c) * r.stride];
        a.add(e.x, e.y, reinterpret_cast<const float*>(v));
      }
    }
  auto put = [&](int b) {
    box[b][0][at] = a.m;
    box[b][1][at] = a.l;
#pragma unroll
    for (int c = 0; c < 16; ++c) box[b][2 + c][at] = a.o[c];
  };
  auto take = [&](int b) {
    float o[16];
#pragma unroll
    for (int c = 0; c < 16; ++c) o[c] = box[b][2 + c][at];
    a.add(box[b][0][at], box[b][1][at], o);
  };
  if (part >= 2) put(part - 2);
  __syncthreads();
  if (part < 2) take(part);
  __syncthreads();
  if (part == 1) put(0);
  __syncthreads();
  if (part == 0 && live) {
    take(0);
    const float inv = 1.0f / fmaxf(a.l, 1e-30f);
    uint32_t k[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) k[e] = pack_bf16(a.o[2 * e] * inv, a.o[2 * e + 1] * inv);
    store32(out + 16 * w, k);
    if (lse && w == 0) *lse = a.l == 0.f ? -INFINITY : (a.m + lg2(a.l)) * 0.69314718055994531f;
  }
}

// Dense units: block (x, y) joins rows 32y..32y+31 of the unit that the start
// of CTA x + 1's run cuts (if it is the first such start inside the unit).
__global__ void __launch_bounds__(kJoinThreads) join_dense_kernel(const __grid_constant__ FwdArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Source& c = a.src[1];
  const uint32_t start = (blockIdx.x + 1) * c.tpc;
  const int u = c.by_pitch(start), j0 = start - u * c.pitch;
  if (u >= c.units || j0 == 0 || c.by_tpc(start - j0) != blockIdx.x) return;
  const int bh = c.by_per(u), b = a.by_heads(bh), h = bh - b * a.n.heads;
  const int r = blockIdx.y * 32 + (threadIdx.x & 31), t = (u - bh * c.per) * c.rows + r;
  const Runs runs(a, 1, u, r);
  join_rows(&runs, 1, t < a.n.q_len, a.out.at(b, t, h), a.lse ? a.lse + (int64_t)bh * a.n.q_len + t : nullptr);
}

// Folded rows: block (x, y) joins rows 32x..32x+31 of key head y.
__global__ void __launch_bounds__(kJoinThreads) join_folded_kernel(const __grid_constant__ FwdArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int fr0 = blockIdx.x * 32 + (threadIdx.x & 31);
  const bool live = fr0 < a.fold_rows;
  const int fr = live ? fr0 : 0;
  const int bt = a.by_group(fr), b = a.by_q_len(bt), tok = bt - b * a.n.q_len;
  const Source &p = a.src[0], &o = a.src[1];
  const int in_b = fr - b * a.n.q_len * a.n.group;
  for (int hk = blockIdx.y; hk < a.n.kv_heads; hk += gridDim.y) {
    const int h = hk * a.n.group + (fr - bt * a.n.group);
    const int up = hk * p.per + fr / p.rows, uo = (b * a.n.kv_heads + hk) * o.per + in_b / o.rows;
    const int64_t row = ((int64_t)b * a.n.heads + h) * a.n.q_len + tok;
    float* lse = a.lse ? a.lse + row : nullptr;
    uint16_t* out = a.out.at(b, tok, h);
    if (a.two_sources) {
      const Runs runs[2] = {Runs(a, 0, up, fr % p.rows), Runs(a, 1, uo, in_b % o.rows)};
      join_rows(runs, 2, live, out, lse);
    } else {
      const Runs runs = p.units ? Runs(a, 0, up, fr % p.rows) : Runs(a, 1, uo, in_b % o.rows);
      join_rows(&runs, 1, live && runs.n > 1, out, lse);  // else written by its unit
    }
    __syncthreads();
  }
}

// No keys at all: zeros and -inf.
__global__ void __launch_bounds__(256) no_keys_kernel(CrossShape n, Rows out, float* lse) {
  const int64_t rows = (int64_t)n.batch * n.heads * n.q_len;
  for (int64_t row = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5; row < rows;
       row += ((int64_t)gridDim.x * blockDim.x) >> 5) {
    const int64_t bh = row / n.q_len;
    *reinterpret_cast<uint2*>(out.at(bh / n.heads, row % n.q_len, bh % n.heads) + 4 * (threadIdx.x & 31)) =
        make_uint2(0, 0);
    if (lse && (threadIdx.x & 31) == 0) lse[row] = -INFINITY;
  }
}

// Everything about a call that its sizes decide.
struct FwdPlan {
  FwdArgs a;                  // sizes and split only
  int ctas;                   // 0: no keys at all
  bool join;
  size_t part_bytes[2];       // partial results of either source
};

FwdPlan plan_fwd(const CrossShape& n) {
  auto div = [](int64_t d) { return make_div((uint32_t)(d > 0 ? d : 1)); };
  FwdPlan p{};
  FwdArgs& a = p.a;
  a.n = n;
  a.np = (n.prefix_len + 127) / 128;
  const int nb = (n.kv_len + 127) / 128;
  Source* src = a.src;
  if (n.q_len >= 128) {
    a.mode = kDense;
    src[1].rows = src[1].stride = 256;
    src[1].per = (n.q_len + 255) / 256;
    src[1].tiles = a.np + nb;
    src[1].units = src[1].tiles ? n.batch * n.heads * src[1].per : 0;
  } else {
    // (a member's rows alone rarely fill two tiles where the batch's do, but a
    // launch of their own in single mode measured 129 us against 112 for 32
    // members over a 64k prefix)
    const int rows[2] = {n.batch * n.q_len * n.group, n.q_len * n.group};
    a.fold_rows = rows[0];
    a.mode = rows[a.np ? 0 : 1] <= 128 ? kSingle : kDual;
    for (int k = 0; k < 2; ++k) {
      src[k].rows = a.mode == kSingle ? 128 : 256;
      src[k].per = (rows[k] + src[k].rows - 1) / src[k].rows;
      src[k].tiles = k ? nb : a.np;
      src[k].units = src[k].tiles ? n.kv_heads * src[k].per * (k ? n.batch : 1) : 0;
      src[k].stride = src[k].per == 1 ? rows[k] : src[k].rows;
    }
  }
  a.units_p = src[0].units, a.units_o = src[1].units;
  a.two_sources = a.units_p && a.units_o;
  for (int k = 0; k < 2; ++k)
    if (src[k].units) src[k].pitch = src[k].tiles + (a.mode == kDense ? 0 : kUnitCost);
  const int64_t units = (int64_t)a.units_p + a.units_o;
  const int64_t pre = (int64_t)a.units_p * src[0].pitch, total = pre + (int64_t)a.units_o * src[1].pitch;
  const int64_t longest = std::max(src[0].pitch, src[1].pitch);
  const int64_t share = (total + kSms - 1) / kSms;
  // whole units in turn cost up to one unit more than the even share; the
  // linear split costs the partial results' traffic and the join, about the
  // time of 4 tiles
  if ((units + kSms - 1) / kSms * longest > share + share / 10 + 4 && total < INT_MAX) a.tpc = (int32_t)share;
  p.ctas = (int)(a.tpc ? (total + a.tpc - 1) / a.tpc : (units < kSms ? units : kSms));
  p.join = a.two_sources || (a.tpc && a.tpc % (int32_t)longest != 0);
  for (int k = 0; k < 2; ++k) {
    if (src[k].units) {
      src[k].tpc = a.tpc;
      src[k].start = k && a.tpc ? (int32_t)pre : 0;
      src[k].slots = a.tpc ? (src[k].tiles - 1) / a.tpc + 2 : 1;
    }
    src[k].by_per = div(src[k].per), src[k].by_pitch = div(src[k].pitch), src[k].by_tpc = div(src[k].tpc);
    if (p.join) p.part_bytes[k] = ((size_t)src[k].units * src[k].slots * src[k].stride * (512 + 8) + 255) / 256 * 256;
  }
  a.by_heads = div(n.heads), a.by_kv_heads = div(n.kv_heads), a.by_group = div(n.group), a.by_q_len = div(n.q_len);
  return p;
}

template <int MODE>
cudaError_t launch_fwd(const FwdArgs& a, int ctas, const CUtensorMap* m, cudaStream_t s) {
  static std::once_flag once[64];
  static cudaError_t set_result[64];
  int dev = 0;
  cudaError_t de = cudaGetDevice(&dev);
  if (de != cudaSuccess) return de;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  std::call_once(once[dev], [dev] {
    cudaError_t e =
        cudaFuncSetAttribute(cross_fwd_kernel<MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
    // the register split needs exactly 128 a thread at launch
    cudaFuncAttributes fa;
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&fa, cross_fwd_kernel<MODE>);
    if (e == cudaSuccess && fa.numRegs != 128) e = cudaErrorInvalidConfiguration;
    set_result[dev] = e;
  });
  if (set_result[dev] != cudaSuccess) return set_result[dev];
  cross_fwd_kernel<MODE><<<ctas, kThreads, kSmemBytes, s>>>(m[0], m[1], m[2], m[3], m[4], m[5], a);
  return cudaGetLastError();
}

unsigned warps_grid(int64_t rows) { return (unsigned)((rows + 7) / 8 < kSms * 8 ? (rows + 7) / 8 : kSms * 8); }

}  // namespace

size_t cross_fwd_workspace(const CrossShape& n) {
  if (!n.batch || !n.q_len) return 0;
  const FwdPlan p = plan_fwd(n);
  return p.part_bytes[0] + p.part_bytes[1];
}

cudaError_t launch_cross_fwd(const CrossLaunch& L, cudaStream_t s, std::string* err) {
  const CrossShape& n = L.n;
  const int64_t rows = (int64_t)n.batch * n.heads * n.q_len;
  if (rows == 0) return cudaSuccess;
  FwdPlan p = plan_fwd(n);
  if (!p.ctas) {
    no_keys_kernel<<<warps_grid(rows), 256, 0, s>>>(n, L.out, L.lse);
    return cudaGetLastError();
  }
  FwdArgs& a = p.a;
  a.q = L.q;
  a.out = L.out;
  a.kv_lens = L.kv_lens;
  a.lse = L.lse;
  a.scale_log2 = L.scale * 1.4426950408889634f;
  for (int k = 0; k < 2; ++k) {
    a.part_o[k] = (float4*)(L.ws + (k ? p.part_bytes[0] : 0));
    a.part_ml[k] = (float2*)(a.part_o[k] + (size_t)a.src[k].units * a.src[k].slots * a.src[k].stride * 32);
  }
  a.status = L.status;
  a.wait_limit_ns = L.wait_limit_ns;
  a.stall = L.stall;
  a.q_b = L.q.b != 0, a.q_h = L.q.h != 0;
  a.k_b = L.k.b != 0, a.k_h = L.k.h != 0;
  a.v_b = L.v.b != 0, a.v_h = L.v.h != 0;
  a.pk_h = L.pk.h != 0, a.pv_h = L.pv.h != 0;
  CUtensorMap m[6] = {};
  const bool dense = a.mode == kDense;
  if (dense && (!make_map4(&m[0], L.q, n.q_len, n.heads, n.batch, err) ||
                !make_map4(&m[5], L.out, n.q_len, n.heads, n.batch, err, 32)))
    return cudaErrorInvalidValue;
  if (n.kv_len && (!make_map4(&m[1], L.k, n.kv_len, n.kv_heads, n.batch, err) ||
                   !make_map4(&m[2], L.v, n.kv_len, n.kv_heads, n.batch, err)))
    return cudaErrorInvalidValue;
  if (n.prefix_len && (!make_map4(&m[3], L.pk, n.prefix_len, n.kv_heads, 1, err) ||
                       !make_map4(&m[4], L.pv, n.prefix_len, n.kv_heads, 1, err)))
    return cudaErrorInvalidValue;
  cudaError_t e = dense && a.src[1].tiles <= kShortTiles ? launch_fwd<kShort>(a, p.ctas, m, s)
                  : dense             ? launch_fwd<kDense>(a, p.ctas, m, s)
                  : a.mode == kSingle ? launch_fwd<kSingle>(a, p.ctas, m, s)
                                      : launch_fwd<kDual>(a, p.ctas, m, s);
  if (e != cudaSuccess || !p.join) return e;
  // placed while the attention kernel runs; waits for its end before it reads
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dense ? dim3(p.ctas - 1, 8)
                      : dim3((a.fold_rows + 31) / 32, n.kv_heads < 65535 ? n.kv_heads : 65535);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, dense ? join_dense_kernel : join_folded_kernel, a);
}

}  // namespace h3
