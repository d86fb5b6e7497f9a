// Per-head RMSNorm of queries and keys with their rotation, and its gradient.
//
//   y = R n,  n = x r w,  r = 1 / sqrt(mean(x^2) + eps)
//   g = R^T dy;  dw = sum g x r;  dx = r (g w - x r mean(g w x r))
//
// All in fp32, one rounding to bf16 at the end.  Memory-bound: 512 bytes a
// row forward (read and written once), 768 backward.  Eight threads hold a
// row of 128 channels as 64 pairs, thread t the pairs 8t..8t+7: pair p is
// (p, half + p) where p < half and the two plain channels (2p, 2p + 1) above,
// so a rotation never leaves its thread.
#include "conditioning.cuh"

namespace h3 {
namespace {

constexpr int kThreads = 256;
constexpr int kRowsPerCta = kThreads / 8;
constexpr int kMaxCtas = 148 * 3;  // three 256-thread CTAs per SM

struct Place {
  int b, s, h;
};

__device__ __forceinline__ Place place(uint32_t row, const QkNormOperand& o) {
  const uint32_t tok = row / (uint32_t)o.heads;
  return {(int)(tok / (uint32_t)o.tokens), (int)(tok % (uint32_t)o.tokens), (int)(row - tok * (uint32_t)o.heads)};
}

// First and second channel of pair p.
__device__ __forceinline__ int first(int p, int half) { return p < half ? p : 2 * p; }
__device__ __forceinline__ int second(int p, int half) { return p < half ? half + p : 2 * p + 1; }

__device__ __forceinline__ void load_row(const uint16_t* p, int t, int half, float* a, float* b) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    a[i] = bf2f(p[first(8 * t + i, half)]);
    b[i] = bf2f(p[second(8 * t + i, half)]);
  }
}

__device__ __forceinline__ float sum8(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 4);
  v += __shfl_xor_sync(0xffffffffu, v, 2);
  return v + __shfl_xor_sync(0xffffffffu, v, 1);
}

__device__ __forceinline__ const uint16_t* table_row(const QkNormOperand& o, const Place& at) {
  return o.table ? o.table + at.b * o.table_batch + (int64_t)at.s * o.half * 4 : nullptr;
}

__global__ void __launch_bounds__(kThreads) qk_norm_fwd_kernel(QkNormLaunch a) {
  const int t = threadIdx.x & 7;
  for (int k = 0; k < 2; ++k) {
    const QkNormOperand& o = a.op[k];
    const uint32_t rows = (uint32_t)a.batch * o.tokens * o.heads;
    for (uint32_t r0 = blockIdx.x * kRowsPerCta; r0 < rows; r0 += gridDim.x * kRowsPerCta) {
      const uint32_t row = r0 + threadIdx.x / 8;
      const bool live = row < rows;
      const Place at = place(live ? row : 0, o);
      float x[8], y[8], wx[8], wy[8];
      load_row(o.x.at(at.b, at.s, at.h), t, o.half, x, y);
      load_row(o.w, t, o.half, wx, wy);
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += x[i] * x[i] + y[i] * y[i];
      const float r = 1.0f / sqrtf(sum8(ss) / 128.f + a.eps);
      if (!live) continue;
      const uint16_t* tr = table_row(o, at);
      uint16_t* out = o.y.at(at.b, at.s, at.h);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int p = 8 * t + i;
        float u = x[i] * r * wx[i], v = y[i] * r * wy[i];
        if (tr && p < o.half) {
          const float u0 = u;
          u = bf2f(tr[4 * p]) * u0 + bf2f(tr[4 * p + 1]) * v;
          v = bf2f(tr[4 * p + 2]) * u0 + bf2f(tr[4 * p + 3]) * v;
        }
        out[first(p, o.half)] = f2bf(u);
        out[second(p, o.half)] = f2bf(v);
      }
    }
  }
}

// ws: [gridDim.x][2][128] partial sums of dw.
__global__ void __launch_bounds__(kThreads) qk_norm_bwd_kernel(QkNormLaunch a) {
  __shared__ float part[kRowsPerCta][128];
  const int t = threadIdx.x & 7;
  for (int k = 0; k < 2; ++k) {
    const QkNormOperand& o = a.op[k];
    const uint32_t rows = (uint32_t)a.batch * o.tokens * o.heads;
    float da[8] = {}, db[8] = {};
    for (uint32_t r0 = blockIdx.x * kRowsPerCta; r0 < rows; r0 += gridDim.x * kRowsPerCta) {
      const uint32_t row = r0 + threadIdx.x / 8;
      const bool live = row < rows;
      const Place at = place(live ? row : 0, o);
      float x[8], y[8], wx[8], wy[8], gx[8], gy[8];
      load_row(o.x.at(at.b, at.s, at.h), t, o.half, x, y);
      load_row(o.g.at(at.b, at.s, at.h), t, o.half, gx, gy);
      load_row(o.w, t, o.half, wx, wy);
      const uint16_t* tr = table_row(o, at);
      float ss = 0.f, c = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int p = 8 * t + i;
        if (tr && p < o.half) {
          const float g0 = gx[i];
          gx[i] = bf2f(tr[4 * p]) * g0 + bf2f(tr[4 * p + 2]) * gy[i];
          gy[i] = bf2f(tr[4 * p + 1]) * g0 + bf2f(tr[4 * p + 3]) * gy[i];
        }
        ss += x[i] * x[i] + y[i] * y[i];
        c += gx[i] * wx[i] * x[i] + gy[i] * wy[i] * y[i];
      }
      const float r = 1.0f / sqrtf(sum8(ss) / 128.f + a.eps);
      c = sum8(c) * r * r / 128.f;
      if (!live) continue;
      uint16_t* out = o.y.at(at.b, at.s, at.h);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int p = 8 * t + i;
        da[i] += gx[i] * x[i] * r;
        db[i] += gy[i] * y[i] * r;
        out[first(p, o.half)] = f2bf(r * (gx[i] * wx[i] - x[i] * c));
        out[second(p, o.half)] = f2bf(r * (gy[i] * wy[i] - y[i] * c));
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      part[threadIdx.x / 8][first(8 * t + i, o.half)] = da[i];
      part[threadIdx.x / 8][second(8 * t + i, o.half)] = db[i];
    }
    __syncthreads();
    if (threadIdx.x < 128) {
      float s = 0.f;
      for (int i = 0; i < kRowsPerCta; ++i) s += part[i][threadIdx.x];
      a.ws[((int64_t)blockIdx.x * 2 + k) * 128 + threadIdx.x] = s;
    }
  }
}

__global__ void qk_norm_dw_kernel(QkNormLaunch a, int parts) {
  float s = 0.f;
  for (int i = 0; i < parts; ++i) s += a.ws[((int64_t)i * 2 + blockIdx.x) * 128 + threadIdx.x];
  a.op[blockIdx.x].dw[threadIdx.x] = s;
}

unsigned grid_of(const QkNormLaunch& a) {
  int64_t rows = 1;
  for (const QkNormOperand& o : a.op) {
    const int64_t n = (int64_t)a.batch * o.tokens * o.heads;
    rows = n > rows ? n : rows;
  }
  const int64_t want = (rows + kRowsPerCta - 1) / kRowsPerCta;
  return (unsigned)(want < kMaxCtas ? want : kMaxCtas);
}

}  // namespace

size_t qk_norm_bwd_workspace() { return (size_t)kMaxCtas * 2 * 128 * sizeof(float); }

cudaError_t launch_qk_norm_fwd(const QkNormLaunch& a, cudaStream_t s) {
  if (!a.op[0].x.p && !a.op[1].x.p) return cudaSuccess;
  qk_norm_fwd_kernel<<<grid_of(a), kThreads, 0, s>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_qk_norm_bwd(const QkNormLaunch& a, cudaStream_t s) {
  const unsigned grid = grid_of(a);
  qk_norm_bwd_kernel<<<grid, kThreads, 0, s>>>(a);
  qk_norm_dw_kernel<<<2, 128, 0, s>>>(a, (int)grid);
  return cudaGetLastError();
}

}  // namespace h3
