// Per-head RMSNorm of queries and keys with their rotation, and its gradient.
//
//   y = R n,  n = x r w,  r = 1 / sqrt(mean(x^2) + eps)
//   g = R^T dy;  dw = sum g x r;  dx = r (g w - x r mean(g w x r))
//
// All in fp32, one rounding to bf16 at the end.  Memory-bound: 512 bytes a
// row forward (read and written once), 768 backward.  Eight threads hold a
// row of 128 channels as 64 pairs, thread t the pairs 8t..8t+7: pair p is
// (p, half + p) where p < half and two plain channels above, so a rotation
// never leaves its thread.
#include "conditioning.cuh"

namespace h3 {
namespace {

constexpr int kThreads = 256;
constexpr int kCtas = 2;                // an SM
constexpr int kGroups = kThreads / 8;   // rows a CTA works on at a time

struct Operand {
  QkNormOperand o;
  Div heads, tokens;
  uint32_t rows;
  uint32_t runs;              // of 4 << shift rows, one warp's
  int shift;
};

struct NormArgs {
  Operand op[2];
  float eps;
  float* ws;                  // backward: [gridDim.x][2][128] partial sums of dw
};

struct Place {
  uint32_t b, s, h;
};

__device__ __forceinline__ Place place(uint32_t row, const Operand& p) {
  const uint32_t tok = p.heads(row), b = p.tokens(tok);
  return {b, tok - b * (uint32_t)p.o.tokens, row - tok * (uint32_t)p.o.heads};
}

// Channels of a thread's pairs 8t..8t+7: the first ones at a, the second ones
// at b.  VEC: both are eight contiguous channels (half a multiple of 8; the
// plain pairs are then 16 contiguous channels, taken as two runs of eight,
// which is another pairing of them but pairs do not matter there).
template <bool VEC>
struct Channels {
  int t, half;
  __device__ Channels(int thread, int half_) : t(thread), half(half_) {}
  __device__ int first(int i) const {
    const int p = 8 * t + i;
    if (VEC) return 8 * t < half ? p : 16 * t + i;
    return p < half ? p : 2 * p;
  }
  __device__ int second(int i) const {
    const int p = 8 * t + i;
    if (VEC) return 8 * t < half ? half + p : 16 * t + 8 + i;
    return p < half ? half + p : 2 * p + 1;
  }
  // raw bf16 words of the 16 channels
  __device__ void load(const uint16_t* p, uint4 (&v)[2]) const {
    if (VEC) {
      v[0] = __ldcs(reinterpret_cast<const uint4*>(p + first(0)));
      v[1] = __ldcs(reinterpret_cast<const uint4*>(p + second(0)));
    } else {
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = p[first(2 * i)] | ((uint32_t)p[first(2 * i + 1)] << 16);
        w[4 + i] = p[second(2 * i)] | ((uint32_t)p[second(2 * i + 1)] << 16);
      }
      v[0] = make_uint4(w[0], w[1], w[2], w[3]);
      v[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
  }
  // a, b: eight values each, two a word
  __device__ void store(uint16_t* p, const uint64_t* a, const uint64_t* b) const {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = pack_bf16(__uint_as_float((uint32_t)a[i]), __uint_as_float((uint32_t)(a[i] >> 32)));
      w[4 + i] = pack_bf16(__uint_as_float((uint32_t)b[i]), __uint_as_float((uint32_t)(b[i] >> 32)));
    }
    if (VEC) {
      *reinterpret_cast<uint4*>(p + first(0)) = make_uint4(w[0], w[1], w[2], w[3]);
      *reinterpret_cast<uint4*>(p + second(0)) = make_uint4(w[4], w[5], w[6], w[7]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[first(i)] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
        p[second(i)] = (uint16_t)(w[4 + (i >> 1)] >> (16 * (i & 1)));
      }
    }
  }
};

// Two fp32 values side by side, two operations an instruction.
using f2 = uint64_t;
__device__ __forceinline__ f2 two(uint32_t lo, uint32_t hi) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ f2 mul(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 fma(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float lo_of(f2 v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi_of(f2 v) { return __uint_as_float((uint32_t)(v >> 32)); }

__device__ __forceinline__ void unpack(const uint4& u, f2* f) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = two(w[i] << 16, w[i] & 0xffff0000u);
}

__device__ __forceinline__ float sum8(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 4);
  v += __shfl_xor_sync(0xffffffffu, v, 2);
  return v + __shfl_xor_sync(0xffffffffu, v, 1);
}

// The rotation of the thread's eight pairs at one token: table entries
// (t0, t1; t2, t3) as bf16, kept from row to row while the token stays.
template <bool VEC>
struct Rotation {
  uint4 e[4];
  bool on;                    // the thread's pairs are turned
  uint32_t b = 0xffffffffu, s = 0;
  __device__ Rotation(const QkNormOperand& o, int t) : on(o.table && 8 * t < o.half) {}
  static __device__ const uint16_t* entries(const QkNormOperand& o, uint32_t b, uint32_t s, int t) {
    return o.table + b * o.table_batch + (int64_t)s * o.half * 4 + 32 * t;
  }
  __device__ __forceinline__ void at(const QkNormOperand& o, uint32_t tb, uint32_t ts, int t) {
    if (!on || (tb == b && ts == s)) return;
    b = tb, s = ts;
    const uint16_t* row = entries(o, b, s, t);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (VEC) {
        e[i] = *reinterpret_cast<const uint4*>(row + 8 * i);
      } else {  // 8-byte aligned entries; those past half are not there
        const uint2 id = make_uint2(0x3f80u, 0x3f800000u);
        const uint2* q = reinterpret_cast<const uint2*>(row) + 2 * i;
        const uint2 e0 = 8 * t + 2 * i < o.half ? q[0] : id, e1 = 8 * t + 2 * i + 1 < o.half ? q[1] : id;
        e[i] = make_uint4(e0.x, e0.y, e1.x, e1.y);
      }
    }
  }
  // by the table's matrices, or by their transposes
  template <bool BACK>
  __device__ __forceinline__ void turn(f2* a, f2* c) const {
    if (!on) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f2 t0 = two(e[i].x << 16, e[i].z << 16), t1 = two(e[i].x & 0xffff0000u, e[i].z & 0xffff0000u);
      const f2 t2 = two(e[i].y << 16, e[i].w << 16), t3 = two(e[i].y & 0xffff0000u, e[i].w & 0xffff0000u);
      const f2 u = a[i];
      a[i] = fma(t0, u, mul(BACK ? t2 : t1, c[i]));
      c[i] = fma(BACK ? t1 : t2, u, mul(t3, c[i]));
    }
  }
};

// Rows of a group of eight threads, in order: a warp takes runs of 4 << shift
// consecutive rows (its four groups one row each at a time), so that the rows
// of a token, and with them a table entry, mostly follow one another.  N
// operands' offsets go along; only the start of a run divides.
template <int N>
struct Cursor {
  const Operand& p;
  uint32_t run, row, left;    // the warp's run, the group's row, rows until the next run
  uint32_t b, s, h;
  int64_t off[N];
  const Rows* of[N];
  __device__ Cursor(const Operand& p_, const Rows& r0) : p(p_) {
    of[0] = &r0;
    seek((blockIdx.x * kThreads + threadIdx.x) >> 5);
  }
  __device__ Cursor(const Operand& p_, const Rows& r0, const Rows& r1) : p(p_) {
    of[0] = &r0;
    of[N - 1] = &r1;
    seek((blockIdx.x * kThreads + threadIdx.x) >> 5);
  }
  __device__ void seek(uint32_t to) {
    run = to;
    row = (run << (2 + p.shift)) + ((threadIdx.x >> 3) & 3);
    left = 1u << p.shift;
    const Place at = place(row, p);
    b = at.b, s = at.s, h = at.h;
#pragma unroll
    for (int i = 0; i < N; ++i) off[i] = b * of[i]->b + s * of[i]->t + h * of[i]->h;
  }
  __device__ __forceinline__ bool more() const { return run < p.runs; }  // the same for the whole warp
  __device__ __forceinline__ bool live() const { return row < p.rows; }
  __device__ __forceinline__ void next() {
    if (--left == 0) {
      seek(run + gridDim.x * (kThreads / 32));
      return;
    }
    row += 4;
    h += 4;
#pragma unroll
    for (int i = 0; i < N; ++i) off[i] += 4 * of[i]->h;
    while (h >= (uint32_t)p.o.heads) {
      h -= p.o.heads;
      ++s;
#pragma unroll
      for (int i = 0; i < N; ++i) off[i] += of[i]->t - p.o.heads * of[i]->h;
      if (s == (uint32_t)p.o.tokens) {
        s = 0;
        ++b;
#pragma unroll
        for (int i = 0; i < N; ++i) off[i] += of[i]->b - p.o.tokens * of[i]->t;
      }
    }
  }
};

// HBM-bound, with bytes in flight and instructions not far behind.  A thread's
// own 32 bytes a row run through a ring of six rows in shared memory that only
// it reads (no barrier), 96 KB an SM; the table's entries stay in registers
// from row to row, positions advance without divisions, and the arithmetic
// takes two values an instruction.  5 million rows of 40 heads: 427 us, 6.0
// TB/s (two rows in flight in registers, all else each row: 545).  Where heads
// are few the table is read nearly each row: 262,144 tokens of 2 x 3 heads
// take 237 us, 4.5 TB/s with the tables' bytes.
template <bool VEC>
__global__ void __launch_bounds__(kThreads, kCtas) qk_norm_fwd_kernel(const __grid_constant__ NormArgs a) {
  constexpr int kStages = 6;
  __shared__ uint4 ring[VEC ? kStages : 1][2][kThreads];
  const int t = threadIdx.x & 7;
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
    const Operand& p = a.op[k];
    if (p.rows == 0) continue;
    const Channels<VEC> ch(t, p.o.half);
    const int c0 = ch.first(0), c1 = ch.second(0);
    Cursor<1> in(p, p.o.x), at(p, p.o.y);
    auto fetch = [&](int slot) {
      if (in.more()) {
        if (in.live()) {
          const uint16_t* x = p.o.x.p + in.off[0];
          copy16(smem_u32(&ring[slot][0][threadIdx.x]), x + c0);
          copy16(smem_u32(&ring[slot][1][threadIdx.x]), x + c1);
        }
        in.next();
      }
      copies_commit();
    };
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < kStages; ++i) fetch(i);
    }
    uint4 raw[2];
    f2 wx[4], wy[4];
    ch.load(p.o.w, raw);
    unpack(raw[0], wx);
    unpack(raw[1], wy);
    Rotation<VEC> rot(p.o, t);
    int slot = 0;
#pragma unroll 1
    for (; at.more(); at.next()) {
      const bool live = at.live();
      if (live) rot.at(p.o, at.b, at.s, t);
      if constexpr (VEC) {
        copies_wait<kStages - 1>();
        raw[0] = ring[slot][0][threadIdx.x];
        raw[1] = ring[slot][1][threadIdx.x];
      } else {
        if (live) ch.load(p.o.x.p + in.off[0], raw);
        in.next();
      }
      f2 x[4], y[4];
      unpack(raw[0], x);
      unpack(raw[1], y);
      f2 ss = mul(x[0], x[0]);
#pragma unroll
      for (int i = 1; i < 4; ++i) ss = fma(x[i], x[i], ss);
#pragma unroll
      for (int i = 0; i < 4; ++i) ss = fma(y[i], y[i], ss);
      const float r = rsqrtf(sum8(lo_of(ss) + hi_of(ss)) * (1.0f / 128.0f) + a.eps);
      const f2 r2 = dup2(r);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = mul(x[i], mul(r2, wx[i]));
        y[i] = mul(y[i], mul(r2, wy[i]));
      }
      rot.template turn<false>(x, y);
      if (live) ch.store(p.o.y.p + at.off[0], x, y);
      if constexpr (VEC) {
        fetch(slot);
        if (++slot == kStages) slot = 0;
      }
    }
    if constexpr (VEC) copies_wait<0>();
  }
}

// The same walk over x and the gradient, 64 bytes a row in a ring of three;
// each thread sums dw of its 16 channels in registers, the CTA joins its
// groups in shared memory and leaves one partial sum an operand.  5 million
// rows: 598 us, 6.45 TB/s (831 without the ring).
template <bool VEC>
__global__ void __launch_bounds__(kThreads, kCtas) qk_norm_bwd_kernel(const __grid_constant__ NormArgs a) {
  constexpr int kStages = 3;
  __shared__ union {
    uint4 ring[VEC ? kStages : 1][4][kThreads];
    float part[kGroups][128];
  } sm;
  const int t = threadIdx.x & 7, g = threadIdx.x >> 3;
  asm volatile("griddepcontrol.launch_dependents;");
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
    const Operand& p = a.op[k];
    const Channels<VEC> ch(t, p.o.half);
    f2 da[4] = {}, db[4] = {};
    if (p.rows) {
      const int c0 = ch.first(0), c1 = ch.second(0);
      Cursor<2> in(p, p.o.x, p.o.g);
      Cursor<1> at(p, p.o.y);
      auto fetch = [&](int slot) {
        if (in.more()) {
          if (in.live()) {
            const uint16_t *x = p.o.x.p + in.off[0], *go = p.o.g.p + in.off[1];
            copy16(smem_u32(&sm.ring[slot][0][threadIdx.x]), x + c0);
            copy16(smem_u32(&sm.ring[slot][1][threadIdx.x]), x + c1);
            copy16(smem_u32(&sm.ring[slot][2][threadIdx.x]), go + c0);
            copy16(smem_u32(&sm.ring[slot][3][threadIdx.x]), go + c1);
          }
          in.next();
        }
        copies_commit();
      };
      if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < kStages; ++i) fetch(i);
      }
      uint4 w[2], raw[2], rawg[2];
      ch.load(p.o.w, w);
      Rotation<VEC> rot(p.o, t);
      int slot = 0;
#pragma unroll 1
      for (; at.more(); at.next()) {
        const bool live = at.live();
        if (live) rot.at(p.o, at.b, at.s, t);
        if constexpr (VEC) {
          copies_wait<kStages - 1>();
          raw[0] = sm.ring[slot][0][threadIdx.x];
          raw[1] = sm.ring[slot][1][threadIdx.x];
          rawg[0] = sm.ring[slot][2][threadIdx.x];
          rawg[1] = sm.ring[slot][3][threadIdx.x];
        } else {
          if (live) {
            ch.load(p.o.x.p + in.off[0], raw);
            ch.load(p.o.g.p + in.off[1], rawg);
          }
          in.next();
        }
        f2 x[4], y[4], gx[4], gy[4], wx[4], wy[4];
        unpack(raw[0], x);
        unpack(raw[1], y);
        unpack(rawg[0], gx);
        unpack(rawg[1], gy);
        unpack(w[0], wx);
        unpack(w[1], wy);
        rot.template turn<true>(gx, gy);
        f2 ss = mul(x[0], x[0]), c2 = mul(mul(gx[0], wx[0]), x[0]);
#pragma unroll
        for (int i = 1; i < 4; ++i) {
          ss = fma(x[i], x[i], ss);
          c2 = fma(mul(gx[i], wx[i]), x[i], c2);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          ss = fma(y[i], y[i], ss);
          c2 = fma(mul(gy[i], wy[i]), y[i], c2);
        }
        const float r = rsqrtf(sum8(lo_of(ss) + hi_of(ss)) * (1.0f / 128.0f) + a.eps);
        const float c = sum8(lo_of(c2) + hi_of(c2)) * r * r * (1.0f / 128.0f);
        if (live) {
          const f2 r2 = dup2(r), mc = dup2(-c);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            da[i] = fma(gx[i], mul(x[i], r2), da[i]);
            db[i] = fma(gy[i], mul(y[i], r2), db[i]);
            x[i] = mul(r2, fma(x[i], mc, mul(gx[i], wx[i])));
            y[i] = mul(r2, fma(y[i], mc, mul(gy[i], wy[i])));
          }
          ch.store(p.o.y.p + at.off[0], x, y);
        }
        if constexpr (VEC) {
          fetch(slot);
          if (++slot == kStages) slot = 0;
        }
      }
      if constexpr (VEC) copies_wait<0>();
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sm.part[g][ch.first(i)] = i & 1 ? hi_of(da[i >> 1]) : lo_of(da[i >> 1]);
      sm.part[g][ch.second(i)] = i & 1 ? hi_of(db[i >> 1]) : lo_of(db[i >> 1]);
    }
    __syncthreads();
    if (threadIdx.x < 128) {
      float s = 0.f;
#pragma unroll 8
      for (int i = 0; i < kGroups; ++i) s += sm.part[i][threadIdx.x];
      a.ws[((int64_t)blockIdx.x * 2 + k) * 128 + threadIdx.x] = s;
    }
    __syncthreads();
  }
}

// Sums the partial results of all CTAs in their order: thread (c, j) every
// eighth one, then the eight in shared memory.
__global__ void __launch_bounds__(1024) qk_norm_dw_kernel(const __grid_constant__ NormArgs a, int parts) {
  __shared__ float sum[8][128];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int c = threadIdx.x & 127, j = threadIdx.x >> 7;
  float s = 0.f;
#pragma unroll 8
  for (int i = j; i < parts; i += 8) s += a.ws[((int64_t)i * 2 + blockIdx.x) * 128 + c];
  sum[j][c] = s;
  __syncthreads();
  if (j == 0) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += sum[i][c];
    a.op[blockIdx.x].o.dw[c] = s;
  }
}

constexpr int kGrid = 148 * kCtas;
// Sixteen-byte accesses need a rotation of whole vectors and a table aligned to them.
bool vectors(const QkNormOperand& o) {
  return o.half % 8 == 0 && !((uintptr_t)o.table & 15) && !(o.table_batch & 7);
}

NormArgs args_of(const QkNormLaunch& l, uint32_t* most) {
  NormArgs a{};
  *most = 0;
  for (int k = 0; k < 2; ++k) {
    Operand& p = a.op[k];
    p.o = l.op[k];
    p.rows = (uint32_t)((int64_t)l.batch * p.o.tokens * p.o.heads);
    p.heads = make_div((uint32_t)p.o.heads);
    p.tokens = make_div((uint32_t)(p.o.tokens > 0 ? p.o.tokens : 1));
    // runs of up to 32 rows where every warp of the full grid has one
    while (p.shift < 3 && p.rows / (8u << p.shift) >= (uint32_t)kGrid * (kThreads / 32)) ++p.shift;
    p.runs = (p.rows + (4u << p.shift) - 1) >> (2 + p.shift);
    *most = p.rows > *most ? p.rows : *most;
  }
  a.eps = l.eps;
  a.ws = l.ws;
  return a;
}

unsigned grid_of(uint32_t rows) {
  const uint32_t want = (rows + kGroups - 1) / kGroups;
  return want < 1 ? 1 : want < kGrid ? want : kGrid;
}

}  // namespace

size_t qk_norm_bwd_workspace() { return (size_t)kGrid * 2 * 128 * sizeof(float); }

cudaError_t launch_qk_norm_fwd(const QkNormLaunch& l, cudaStream_t s) {
  const bool vec = vectors(l.op[0]) && vectors(l.op[1]);
  uint32_t rows;
  const NormArgs a = args_of(l, &rows);
  if (rows == 0) return cudaSuccess;
  const unsigned grid = grid_of(rows);
  if (vec) qk_norm_fwd_kernel<true><<<grid, kThreads, 0, s>>>(a);
  else qk_norm_fwd_kernel<false><<<grid, kThreads, 0, s>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_qk_norm_bwd(const QkNormLaunch& l, cudaStream_t s) {
  const bool vec = vectors(l.op[0]) && vectors(l.op[1]);
  uint32_t rows;
  const NormArgs a = args_of(l, &rows);
  const unsigned grid = grid_of(rows);
  if (vec) qk_norm_bwd_kernel<true><<<grid, kThreads, 0, s>>>(a);
  else qk_norm_bwd_kernel<false><<<grid, kThreads, 0, s>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  // placed while the gradient kernel runs; waits for its end before it reads
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2);
  cfg.blockDim = dim3(1024);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, qk_norm_dw_kernel, a, (int)grid);
}

}  // namespace h3
