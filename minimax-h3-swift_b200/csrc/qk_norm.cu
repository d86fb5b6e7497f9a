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
constexpr int kGroups = kThreads / 8;   // rows a CTA has in hand at a time

struct Operand {
  QkNormOperand o;
  Div heads, tokens;
  uint32_t rows;
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
  __device__ void store(uint16_t* p, const float* a, const float* b) const {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = pack_bf16(a[2 * i], a[2 * i + 1]);
      w[4 + i] = pack_bf16(b[2 * i], b[2 * i + 1]);
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

__device__ __forceinline__ void unpack(const uint4& u, float* f) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

__device__ __forceinline__ float sum8(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 4);
  v += __shfl_xor_sync(0xffffffffu, v, 2);
  return v + __shfl_xor_sync(0xffffffffu, v, 1);
}

// Turns the thread's pairs by the token's table entries (t0, t1; t2, t3), or
// by their transpose.
template <bool VEC, bool BACK>
__device__ __forceinline__ void rotate(const QkNormOperand& o, const Place& at, int t, float* a, float* b) {
  if (!o.table || 8 * t >= o.half) return;
  const uint16_t* row = o.table + at.b * o.table_batch + (int64_t)at.s * o.half * 4 + 32 * t;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint4 e;
    if (VEC) {
      e = *reinterpret_cast<const uint4*>(row + 8 * i);
    } else {  // 8-byte aligned entries; those past half are not there
      const uint2 id = make_uint2(0x3f80u, 0x3f800000u);
      const uint2* p = reinterpret_cast<const uint2*>(row) + 2 * i;
      const uint2 e0 = 8 * t + 2 * i < o.half ? p[0] : id, e1 = 8 * t + 2 * i + 1 < o.half ? p[1] : id;
      e = make_uint4(e0.x, e0.y, e1.x, e1.y);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t lo = k ? e.z : e.x, hi = k ? e.w : e.y;
      const float t0 = __uint_as_float(lo << 16), t1 = __uint_as_float(lo & 0xffff0000u);
      const float t2 = __uint_as_float(hi << 16), t3 = __uint_as_float(hi & 0xffff0000u);
      float &x = a[2 * i + k], &y = b[2 * i + k];
      const float u = x;
      x = t0 * u + (BACK ? t2 : t1) * y;
      y = (BACK ? t1 : t2) * u + t3 * y;
    }
  }
}

// Two rows a group of eight threads in flight; 3 CTAs of 256 threads an SM.
template <bool VEC>
__global__ void __launch_bounds__(kThreads, 3) qk_norm_fwd_kernel(const __grid_constant__ NormArgs a) {
  constexpr int U = 2;
  const int t = threadIdx.x & 7, g = threadIdx.x >> 3;
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
    const Operand& p = a.op[k];
    if (p.rows == 0) continue;
    const Channels<VEC> ch(t, p.o.half);
    uint4 w[2];
    ch.load(p.o.w, w);
    for (uint32_t r0 = blockIdx.x * (U * kGroups); r0 < p.rows; r0 += gridDim.x * (U * kGroups)) {
      uint4 raw[U][2];
      Place at[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t row = r0 + u * kGroups + g;
        at[u] = place(row < p.rows ? row : r0, p);
        ch.load(p.o.x.at(at[u].b, at[u].s, at[u].h), raw[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float x[8], y[8], wx[8], wy[8];
        unpack(raw[u][0], x);
        unpack(raw[u][1], y);
        unpack(w[0], wx);
        unpack(w[1], wy);
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += x[i] * x[i] + y[i] * y[i];
        const float r = 1.0f / sqrtf(sum8(ss) * (1.0f / 128.0f) + a.eps);
        if (r0 + u * kGroups + g >= p.rows) continue;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] *= r * wx[i];
          y[i] *= r * wy[i];
        }
        rotate<VEC, false>(p.o, at[u], t, x, y);
        ch.store(p.o.y.at(at[u].b, at[u].s, at[u].h), x, y);
      }
    }
  }
}

// The same walk; each thread sums dw of its 16 channels in registers, the CTA
// joins its groups in shared memory and leaves one partial sum an operand.
template <bool VEC>
__global__ void __launch_bounds__(kThreads, 2) qk_norm_bwd_kernel(const __grid_constant__ NormArgs a) {
  constexpr int U = 2;
  __shared__ float part[kGroups][128];
  const int t = threadIdx.x & 7, g = threadIdx.x >> 3;
  asm volatile("griddepcontrol.launch_dependents;");
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
    const Operand& p = a.op[k];
    const Channels<VEC> ch(t, p.o.half);
    float da[8] = {}, db[8] = {};
    uint4 w[2];
    ch.load(p.o.w, w);
    for (uint32_t r0 = blockIdx.x * (U * kGroups); r0 < p.rows; r0 += gridDim.x * (U * kGroups)) {
      uint4 raw[U][2], rawg[U][2];
      Place at[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t row = r0 + u * kGroups + g;
        at[u] = place(row < p.rows ? row : r0, p);
        ch.load(p.o.x.at(at[u].b, at[u].s, at[u].h), raw[u]);
        ch.load(p.o.g.at(at[u].b, at[u].s, at[u].h), rawg[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float x[8], y[8], gx[8], gy[8], wx[8], wy[8];
        unpack(raw[u][0], x);
        unpack(raw[u][1], y);
        unpack(rawg[u][0], gx);
        unpack(rawg[u][1], gy);
        unpack(w[0], wx);
        unpack(w[1], wy);
        rotate<VEC, true>(p.o, at[u], t, gx, gy);
        float ss = 0.f, c = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          ss += x[i] * x[i] + y[i] * y[i];
          c += gx[i] * wx[i] * x[i] + gy[i] * wy[i] * y[i];
        }
        const float r = 1.0f / sqrtf(sum8(ss) * (1.0f / 128.0f) + a.eps);
        c = sum8(c) * r * r * (1.0f / 128.0f);
        if (r0 + u * kGroups + g >= p.rows) continue;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          da[i] += gx[i] * (x[i] * r);
          db[i] += gy[i] * (y[i] * r);
          x[i] = r * (gx[i] * wx[i] - x[i] * c);
          y[i] = r * (gy[i] * wy[i] - y[i] * c);
        }
        ch.store(p.o.y.at(at[u].b, at[u].s, at[u].h), x, y);
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      part[g][ch.first(i)] = da[i];
      part[g][ch.second(i)] = db[i];
    }
    __syncthreads();
    if (threadIdx.x < 128) {
      float s = 0.f;
#pragma unroll 8
      for (int i = 0; i < kGroups; ++i) s += part[i][threadIdx.x];
      a.ws[((int64_t)blockIdx.x * 2 + k) * 128 + threadIdx.x] = s;
    }
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

constexpr int kSms = 148;
constexpr int kFwdCtas = kSms * 3, kBwdCtas = kSms * 2;

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
    *most = p.rows > *most ? p.rows : *most;
  }
  a.eps = l.eps;
  a.ws = l.ws;
  return a;
}

unsigned grid_of(uint32_t rows, int most) {
  const uint32_t want = (rows + 2 * kGroups - 1) / (2 * kGroups);
  return want < 1 ? 1 : want < (uint32_t)most ? want : (unsigned)most;
}

}  // namespace

size_t qk_norm_bwd_workspace() { return (size_t)kBwdCtas * 2 * 128 * sizeof(float); }

cudaError_t launch_qk_norm_fwd(const QkNormLaunch& l, cudaStream_t s) {
  uint32_t rows;
  const NormArgs a = args_of(l, &rows);
  if (rows == 0) return cudaSuccess;
  const unsigned grid = grid_of(rows, kFwdCtas);
  if (vectors(l.op[0]) && vectors(l.op[1])) qk_norm_fwd_kernel<true><<<grid, kThreads, 0, s>>>(a);
  else qk_norm_fwd_kernel<false><<<grid, kThreads, 0, s>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_qk_norm_bwd(const QkNormLaunch& l, cudaStream_t s) {
  uint32_t rows;
  const NormArgs a = args_of(l, &rows);
  const unsigned grid = grid_of(rows, kBwdCtas);
  if (vectors(l.op[0]) && vectors(l.op[1])) qk_norm_bwd_kernel<true><<<grid, kThreads, 0, s>>>(a);
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
