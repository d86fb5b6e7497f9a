// Internal types of the conditioning calls (cross attention, shared prefix,
// q/k norm): normalised operands and the launchers of the kernel files.
#pragma once

#include "tcgen05.cuh"

namespace h3 {

// A [batch, tokens, heads, 128] operand; strides in elements, 0 on an axis of
// one element or a broadcast axis.
struct Rows {
  uint16_t* p;
  int64_t b, t, h;
  __host__ __device__ uint16_t* at(int64_t ib, int64_t it, int64_t ih) const { return p + ib * b + it * t + ih * h; }
};

struct CrossShape {
  int32_t batch, q_len, kv_len, prefix_len, heads, kv_heads, group;
};

struct CrossLaunch {
  CrossShape n;
  Rows q, out, k, v, pk, pv;  // pk, pv: batch stride 0
  Rows dout, dq, dk, dv;
  float scale;
  const int32_t* kv_lens;     // may be null
  float* lse;                 // may be null (forward)
  uint8_t* ws;
  int32_t* status;            // the context's status word of these calls (bounded waits), written only
  uint64_t wait_limit_ns;
  int32_t stall;              // test hook: barrier of each CTA that never completes (-1: none)
};

// n / d for n < 2^31, d >= 1: m = ceil(2^(31 + s) / d) with 2^s >= d.
struct Div {
  uint32_t m, s;
  __device__ uint32_t operator()(uint32_t n) const { return (uint32_t)(((uint64_t)n * m) >> (31 + s)); }
};

inline Div make_div(uint32_t d) {
  uint32_t s = 0;
  while ((1ull << s) < d) ++s;
  return {(uint32_t)(((1ull << (31 + s)) + d - 1) / d), s};
}

// Members whose lengths a kernel keeps in shared memory: with all of it taken
// by tiles, the lengths do not stay in L1, and a role that starts a unit would
// wait for L2 (1,000 cycles under load).
constexpr int kLens = 64;

// The 128-byte swizzle needs tiles on 1024-byte boundaries: so dynamic shared
// memory starts (the declaration's alignment), which this checks.
__device__ __forceinline__ bool tiles_aligned(const uint8_t* smem, int32_t* status) {
  if (!(smem_u32(smem) & 1023)) return true;
  if (threadIdx.x == 0) atomicExch(status, (int32_t)H3C_ERR_UNSUPPORTED);
  return false;
}

__device__ __forceinline__ int kv_len_of(const int32_t* kv_lens, int kv_len, int b) {
  return kv_lens ? max(0, min(kv_len, kv_lens[b])) : kv_len;
}

// (d, token, head, batch) map of an operand, boxes of 64 x box_tokens; a
// broadcast axis has one element.
inline bool make_map4(CUtensorMap* m, const Rows& r, int tokens, int heads, int batch, std::string* err,
                      int box_tokens = 128) {
  EncodeTiledFn enc = get_encode();
  if (!enc) {
    *err += "cuTensorMapEncodeTiled unavailable; ";
    return false;
  }
  cuuint64_t dims[4] = {128, (cuuint64_t)tokens, r.h ? (cuuint64_t)heads : 1, r.b ? (cuuint64_t)batch : 1};
  cuuint64_t strides[3] = {r.t ? (cuuint64_t)r.t * 2 : 256, r.h ? (cuuint64_t)r.h * 2 : 256,
                           r.b ? (cuuint64_t)r.b * 2 : 256};
  cuuint32_t box[4] = {64, (cuuint32_t)box_tokens, 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult res = enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, r.p, dims, strides, box, estr,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (res != CUDA_SUCCESS) {
    *err += "cuTensorMapEncodeTiled failed (" + std::to_string((int)res) + "); ";
    return false;
  }
  return true;
}

size_t cross_fwd_workspace(const CrossShape& n);
size_t cross_bwd_workspace(const CrossShape& n);
cudaError_t launch_cross_fwd(const CrossLaunch& a, cudaStream_t s, std::string* err);
cudaError_t launch_cross_bwd(const CrossLaunch& a, cudaStream_t s, std::string* err);

struct QkNormOperand {
  Rows x, g, y;               // rows in; gradient of the output in (backward); result out
  int32_t tokens, heads, half;
  const uint16_t* w;
  const uint16_t* table;      // null: no rotation
  int64_t table_batch;        // elements; 0: one table for the batch
  float* dw;                  // backward: fp32 [128]
};

struct QkNormLaunch {
  QkNormOperand op[2];        // queries, keys
  int32_t batch;
  float eps;
  float* ws;
};

size_t qk_norm_bwd_workspace();
cudaError_t launch_qk_norm_fwd(const QkNormLaunch& a, cudaStream_t s);
cudaError_t launch_qk_norm_bwd(const QkNormLaunch& a, cudaStream_t s);

}  // namespace h3
