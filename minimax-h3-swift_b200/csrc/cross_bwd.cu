// Gradient of cross attention: the plain kernels.  One warp per row, lane l holds channels 4l..4l+3; softmax
// statistics and sums in fp32.
#include <cmath>

#include "conditioning.cuh"

namespace h3 {
namespace {

struct F4 {
  float v[4];
};

__device__ __forceinline__ F4 load4(const uint16_t* p) {
  const uint2 u = *reinterpret_cast<const uint2*>(p + 4 * (threadIdx.x & 31));
  return {{__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
           __uint_as_float(u.y & 0xffff0000u)}};
}

__device__ __forceinline__ void store4(uint16_t* p, const F4& f, float m) {
  *reinterpret_cast<uint2*>(p + 4 * (threadIdx.x & 31)) =
      make_uint2((uint32_t)f2bf(f.v[0] * m) | ((uint32_t)f2bf(f.v[1] * m) << 16),
                 (uint32_t)f2bf(f.v[2] * m) | ((uint32_t)f2bf(f.v[3] * m) << 16));
}

__device__ __forceinline__ float dot(const F4& a, const F4& b) {
  float s = a.v[0] * b.v[0] + a.v[1] * b.v[1] + a.v[2] * b.v[2] + a.v[3] * b.v[3];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

__device__ __forceinline__ void axpy(F4& y, float a, const F4& x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) y.v[i] = fmaf(a, x.v[i], y.v[i]);
}

// this warp's row numbers
struct Walk {
  int64_t i, step;
  __device__ Walk()
      : i(((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5), step(((int64_t)gridDim.x * blockDim.x) >> 5) {}
};

__global__ void __launch_bounds__(256) cross_dq_kernel(CrossLaunch a, float* delta) {
  const CrossShape n = a.n;
  for (Walk w; w.i < (int64_t)n.batch * n.heads * n.q_len; w.i += w.step) {
    const int t = (int)(w.i % n.q_len), h = (int)(w.i / n.q_len % n.heads), b = (int)(w.i / n.q_len / n.heads);
    const int hk = h / n.group, own = kv_len_of(a.kv_lens, n.kv_len, b);
    const F4 q = load4(a.q.at(b, t, h)), g = load4(a.dout.at(b, t, h));
    const float dl = dot(g, load4(a.out.at(b, t, h))), lse = own ? a.lse[w.i] : 0.f;
    F4 dq{};
    for (int j = 0; j < own; ++j) {
      const F4 k = load4(a.k.at(b, j, hk));
      const float p = expf(dot(q, k) * a.scale - lse);
      axpy(dq, p * (dot(g, load4(a.v.at(b, j, hk))) - dl), k);
    }
    store4(a.dq.at(b, t, h), dq, a.scale);
    if ((threadIdx.x & 31) == 0) delta[w.i] = dl;
  }
}

__global__ void __launch_bounds__(256) cross_dkv_kernel(CrossLaunch a, const float* delta) {
  const CrossShape n = a.n;
  for (Walk w; w.i < (int64_t)n.batch * n.kv_heads * n.kv_len; w.i += w.step) {
    const int j = (int)(w.i % n.kv_len), hk = (int)(w.i / n.kv_len % n.kv_heads),
              b = (int)(w.i / n.kv_len / n.kv_heads);
    F4 dk{}, dv{};
    if (j < kv_len_of(a.kv_lens, n.kv_len, b)) {
      const F4 k = load4(a.k.at(b, j, hk)), v = load4(a.v.at(b, j, hk));
      for (int h = hk * n.group; h < (hk + 1) * n.group; ++h)
        for (int t = 0; t < n.q_len; ++t) {
          const int64_t r = ((int64_t)b * n.heads + h) * n.q_len + t;
          const F4 q = load4(a.q.at(b, t, h)), g = load4(a.dout.at(b, t, h));
          const float p = expf(dot(q, k) * a.scale - a.lse[r]);
          axpy(dv, p, g);
          axpy(dk, p * (dot(g, v) - delta[r]), q);
        }
    }
    store4(a.dk.at(b, j, hk), dk, a.scale);
    store4(a.dv.at(b, j, hk), dv, 1.f);
  }
}

unsigned warps_grid(int64_t rows) { return (unsigned)((rows + 7) / 8 < 148 * 8 ? (rows + 7) / 8 : 148 * 8); }

}  // namespace

size_t cross_bwd_workspace(const CrossShape& n) { return (size_t)n.batch * n.heads * n.q_len * sizeof(float); }

cudaError_t launch_cross_bwd(const CrossLaunch& a, cudaStream_t s, std::string*) {
  const int64_t rows = (int64_t)a.n.batch * a.n.heads * a.n.q_len;
  const int64_t keys = (int64_t)a.n.batch * a.n.kv_heads * a.n.kv_len;
  if (rows) cross_dq_kernel<<<warps_grid(rows), 256, 0, s>>>(a, (float*)a.ws);
  if (keys) cross_dkv_kernel<<<warps_grid(keys), 256, 0, s>>>(a, (const float*)a.ws);
  return cudaGetLastError();
}

}  // namespace h3
